"""Which pages a reordering of beams drops, with plain lists, for the tests of Kernels.paged_reorder."""


def dropped(table, parents, lens, page, n_pages):
    """Of rows [R * beams][width]: the whole pages of beams that no one goes on from which no beam has that goes on, in the
    order in which they are pushed."""
    out = []
    beams = len(parents[0])
    for r, ps in enumerate(parents):
        ps = [p if 0 <= p < beams else i for i, p in enumerate(ps)]
        rows = table[r * beams:(r + 1) * beams]
        for j in range(max(lens[r * beams:(r + 1) * beams]) // page):
            kept = {rows[p][j] for p in ps}
            for i in range(beams):
                if i in ps or j >= lens[r * beams + i] // page or rows[i][j] in kept or not 0 <= rows[i][j] < n_pages:
                    continue
                out.append(rows[i][j])
                kept.add(rows[i][j])
    return out
