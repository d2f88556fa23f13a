"""The operators of a batch whose cache is held in 8 bits and whose pages are dealt out on the GPU, and of
beam search over it, as timed cases through ``Kernels``.

A case is a dict of plain values. ``kind`` names the operator:

  append   Kernels.paged_append_fp8: bias, position rotation, keys and values into pages of e4m3 codes with
           one power of two for each 16 positions and kv head
  attend   Kernels.paged_attention_fp8: attention of the batch's tokens over such pages, with a sliding window
           and first tokens that stay visible (``window``, ``sinks``), or with a prefix whose pages all
           sequences share (``shared``)
  reserve  Kernels.paged_reserve: tokens given back and room for new ones: block tables, first rows, slot map
  beam     Kernels.beam_select: the best continuations over beams and vocabulary
  reorder  Kernels.paged_reorder: the pages of the beams that go on, last pages copied where a beam splits

Lengths of a batch spread over ``lo`` .. ``hi`` positions and ``nlo`` .. ``nhi`` new tokens per sequence
(one each: a decode step), the same ones for every seed. Rotary base 1e6 and head layouts are those of this
repository's model shapes; activations are N(0, 1), keys and values too, queries twice that; logits are
N(0, 2) with some peaks, as a language model's are.
"""
import math
import random

import torch

own = False

BF16, FP8, E8M0 = torch.bfloat16, torch.float8_e4m3fn, torch.float8_e8m0fnu
THETA = 1000000.0
BLOCK = 16                      # positions that share a scale
LEAST, MOST = -110, 119         # exponents of the scales

_kernels = None


def kernels():
    global _kernels
    if _kernels is None:
        from nanoserve_amd.ops import Kernels
        _kernels = Kernels()
    return _kernels


def _batch(name, kind, b, lo, hi, nlo=1, nhi=1, heads=28, kv=4, dim=128, page=16, window=0, sinks=0,
           shared=0):
    case = {"kind": kind, "b": b, "lo": lo, "hi": hi, "nlo": nlo, "nhi": nhi, "heads": heads,
            "kv": kv, "dim": dim, "page": page, "window": window, "sinks": sinks, "shared": shared}
    return {"name": name, **case} if name else case


def _reserve(name, b, lo, hi, nlo, nhi, page):
    case = {"kind": "reserve", "b": b, "lo": lo, "hi": hi, "nlo": nlo, "nhi": nhi, "page": page}
    return {"name": name, **case} if name else case


def _beam(name, r, beams, n, v, type, first=False):
    case = {"kind": "beam", "r": r, "beams": beams, "n": n, "v": v, "type": type, "first": first}
    return {"name": name, **case} if name else case


def _reorder(name, r, beams, lo, hi, layers, kv=4, dim=128, page=16, type="fp8"):
    case = {"kind": "reorder", "r": r, "beams": beams, "lo": lo, "hi": hi, "layers": layers, "kv": kv,
            "dim": dim, "page": page, "type": type}
    return {"name": name, **case} if name else case


def listed():
    return [
        # sixteen conversations decoding together: their tokens' keys and values, the smallest append
        _batch("append decode 16", "append", 16, 100, 8000),
        # a full prompt step of several requests, some of them later chunks of long prompts
        _batch("append prompts", "append", 6, 900, 20000, 500, 900),
        # one short conversation of the 1.5B layout: the smallest attention, where latency counts
        _batch("decode 1 at 700", "attend", 1, 700, 700, heads=12, kv=2),
        # sixteen conversations of very different lengths decoding together
        _batch("decode 16 ragged", "attend", 16, 33, 8191, page=32),
        # a few very long conversations
        _batch("decode 4 at 98k", "attend", 4, 96001, 98304, page=64),
        # the prompts of several requests, some of them behind cached tokens
        _batch("prompts ragged", "attend", 5, 2000, 8000, 301, 2000),
        # a step of 64 conversations whose drafts of up to four tokens were turned down and are made again
        _reserve("reserve drafts 64", 64, 33, 8000, 1, 4, 16),
        # the prompts of many requests let in at once
        _reserve("reserve prompts 48", 48, 500, 6000, 500, 6000, 16),
        # one request's next step with four beams, eight candidates: the smallest selection
        _beam("beam 4", 1, 4, 8, 152064, "bf16"),
        # sixteen requests with eight beams each
        _beam("beam 16 x 8", 16, 8, 16, 151936, "fp32"),
        # one request of four beams over one layer's pages
        _reorder("reorder 4", 1, 4, 333, 333, 1, type="bf16"),
        # sixteen requests with eight beams, the pages of all layers of the 7B layout
        _reorder("reorder 16 x 8", 16, 8, 100, 900, 28, page=64),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["append", "append", "decode", "decode", "prompt", "shared", "reserve", "beam",
                       "beam", "reorder"])
    if kind == "beam":
        r, beams = _log_int(rng, 1, 32), rng.choice([1, 2, 3, 4, 5, 8, 16])
        r = min(r, max(1, 128 // beams))
        return _beam(None, r, beams, rng.choice([beams, 2 * beams]), _log_int(rng, 1000, 152064),
                     rng.choice(["bf16", "fp32"]), rng.random() < 0.2)
    if kind == "reserve":
        b = _log_int(rng, 1, 1024)
        n = rng.choice([1, 4, _log_int(rng, 1, max(1, 100000 // b))])
        hi = _log_int(rng, n, max(n, min(98304, 1000000 // b)))
        return _reserve(None, b, rng.randrange(n, hi + 1), hi, rng.randrange(1, n + 1), n,
                        rng.choice([16, 32, 48, 64, 128, 256]))
    heads, kv, dim = rng.choice([(28, 4, 128), (12, 2, 128), (32, 8, 128), (16, 16, 128), (14, 2, 64),
                                 (40, 8, 128), (16, 16, 64), (16, 1, 128)])
    page = rng.choice([16, 32, 48, 64, 128, 256])
    if kind == "reorder":
        r, beams, hi = _log_int(rng, 1, 16), rng.choice([2, 3, 4, 5, 8]), _log_int(rng, 1, 1000)
        layers = _log_int(rng, 1, max(1, min(32, 200000000 // (r * (hi // page + beams) * kv * page * dim))))
        return _reorder(None, r, beams, rng.randrange(1, hi + 1), hi, layers, kv, dim, page,
                        rng.choice(["bf16", "fp8", "fp8"]))
    lay = dict(heads=heads, kv=kv, dim=dim, page=page)
    window, sinks = rng.choice([(0, 0), (0, 0), (_log_int(rng, 16, 8192), rng.choice([0, 1, 4, 64]))])
    if kind == "append":
        b = _log_int(rng, 1, 64)
        n = rng.choice([1, _log_int(rng, 1, 3000 // b)])
        hi = _log_int(rng, n + 1, 20000)
        return _batch(None, "append", b, rng.randrange(1, hi + 1), hi, rng.randrange(1, n + 1), n, **lay)
    if kind == "decode":
        b = _log_int(rng, 1, 64)
        hi = _log_int(rng, 1, min(98304, 1500000 // (b * kv)))
        return _batch(None, "attend", b, rng.randrange(1, hi + 1), hi, window=window, sinks=sinks, **lay)
    if kind == "prompt":
        b = _log_int(rng, 1, 8)
        n = _log_int(rng, 2, 4000 // b)
        hi = _log_int(rng, n, max(n, min(6000, 400000000 // (n * b * heads))))
        return _batch(None, "attend", b, rng.randrange(n, hi + 1), hi, rng.randrange(1, n + 1), n,
                      window=window, sinks=sinks, **lay)
    b = _log_int(rng, 2, 96)
    shared = _log_int(rng, 200, 16384)
    n = rng.choice([1, 1, 4])
    hi = shared + _log_int(rng, n, 900)
    return _batch(None, "attend", b, rng.randrange(shared + n, hi + 1), hi, 1, n, shared=shared,
                  window=window, sinks=sinks, **lay)


# ---------------------------------------------------------------------------------- inputs
def _gen(seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    return g


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _lengths(case):
    """(positions, new tokens) of every sequence of a batch."""
    rng = random.Random(f"{case['b']} {case['lo']} {case['hi']} {case['nlo']} {case['nhi']}")
    new = [rng.randint(case["nlo"], case["nhi"]) for _ in range(case["b"])]
    return [max(rng.randint(case["lo"], case["hi"]), n) for n in new], new


def _exponent(largest):
    """Of the scale for values up to ``largest``: the least e with largest <= 448 * 2^e, within limits."""
    m, e = torch.frexp(largest)  # 448 = 0.875 * 2^9
    return torch.where(largest > 0, e - 9 + (m > 0.875).to(e.dtype), LEAST).clamp(LEAST, MOST)


def _pool(g, pages, kv, page, dim):
    """A pool of N(0, 1) in 8 bits: codes [pages, kv, page, dim] and scales [pages, kv, page / 16]."""
    codes = torch.empty(pages, kv, page, dim, dtype=FP8, device="cuda")
    scales = torch.empty(pages, kv, page // BLOCK, dtype=torch.uint8, device="cuda")
    step = max(1, (1 << 26) // (kv * page * dim))
    for at in range(0, pages, step):
        n = min(step, pages - at)
        x = torch.randn(n, kv, page // BLOCK, BLOCK * dim, generator=g, device="cuda")
        e = _exponent(x.abs().amax(-1))
        codes[at:at + n] = torch.ldexp(x, -e[..., None]).to(FP8).view(n, kv, page, dim)
        scales[at:at + n] = (e + 127).to(torch.uint8)
    return codes, scales.view(E8M0)


def prepare(case, seed):
    g = _gen(seed)
    if case["kind"] in ("append", "attend"):
        return _prepare_batch(case, g)
    return {"reserve": _prepare_reserve, "beam": _prepare_beam, "reorder": _prepare_reorder}[case["kind"]](
        case, g)


def _prepare_batch(case, g):
    lens, new = _lengths(case)
    b, ps, kv, dim = case["b"], case["page"], case["kv"], case["dim"]
    T = sum(new)
    common = case["shared"] // ps  # whole pages of the shared prefix, one copy for the batch
    width = -(-max(lens) // ps)
    counts = [max(-(-n // ps) - common, 0) for n in lens]
    total = common + sum(counts) + 1
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.zeros(b, width, dtype=torch.int32, device="cuda")
    table[:, :common] = order[:common]
    at = common
    for i, c in enumerate(counts):
        table[i, common:common + c] = order[at:at + c]
        at += c
    k, ks = _pool(g, total, kv, ps, dim)
    v, vs = _pool(g, total, kv, ps, dim)
    state = {"case": case, "table": table, "lens": _ints(lens), "q_start": None, "most": max(lens),
             "most_new": max(new), "k_pages": k, "v_pages": v, "k_scales": ks, "v_scales": vs}
    if case["nhi"] > 1:
        state["q_start"] = torch.tensor([0] + new, device="cuda").cumsum(0).to(torch.int32)
    if case["kind"] == "append":
        width = (case["heads"] + 2 * kv) * dim
        state["qkv"] = torch.randn(T, width, generator=g, device="cuda").to(BF16)
        state["bias"] = (torch.randn(width, generator=g, device="cuda") * 0.5).to(BF16)
        state["inv_freq"] = 1.0 / THETA ** (torch.arange(0, dim, 2, device="cuda").float() / dim)
    else:
        state["q"] = (torch.randn(T, case["heads"] * dim, generator=g, device="cuda") * 2).to(BF16)
        if own:
            state["work"] = kernels().paged_attention_fp8_workspace(
                T, b, case["heads"], kv, dim, table.shape[1] * ps, ragged=case["nhi"] > 1,
                shared=common * ps)
    return state


def _prepare_reserve(case, g):
    """The batch as the step before left it: its new tokens, which this step gives back first, included."""
    lens, new = _lengths(case)
    ps, b = case["page"], case["b"]
    counts = [-(-n // ps) for n in lens]
    width = max(counts) + 1
    total = sum(counts) + 64
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    slot = torch.arange(width, device="cuda")[None] < torch.tensor(counts, device="cuda")[:, None]
    table = torch.full((b, width), -1, dtype=torch.int32, device="cuda")
    table[slot] = order[:sum(counts)]
    free = torch.full((total,), -1, dtype=torch.int32, device="cuda")
    free[:64] = order[sum(counts):]
    return {"case": case, "pages": table, "lens": _ints(lens), "new": _ints(new),
            "back": _ints([-n for n in new]), "free": free, "n_free": _ints([64]), "rows": sum(new)}


def _prepare_beam(case, g):
    rows, v = case["r"] * case["beams"], case["v"]
    x = torch.randn(rows, v, generator=g, device="cuda") * 2
    hot = torch.randint(0, v, (rows, 30), generator=g, device="cuda")
    x.scatter_add_(1, hot, torch.rand(rows, 30, generator=g, device="cuda") * 12)
    scores = -20 - 4 * torch.rand(case["r"], case["beams"], generator=g, device="cuda")
    if case["first"]:  # the step after the prompt, which all beams share: one of them counts
        scores[:, 1:] = -math.inf
    state = {"case": case, "logits": x.to(BF16) if case["type"] == "bf16" else x, "scores": scores}
    if own:
        state["work"] = kernels().beam_select_workspace(case["r"], case["beams"], v, case["n"],
                                                        state["logits"].dtype)
    return state


def _splits(case):
    """(positions of every request, parents of every request's beams): some go on twice or more, some end."""
    rng = random.Random(f"{case['r']} {case['beams']} {case['lo']} {case['hi']} {case['page']}")
    lens = [rng.randint(case["lo"], case["hi"]) for _ in range(case["r"])]
    weights = [2.0 ** -i for i in range(case["beams"])]
    parents = []
    for _ in lens:
        w = weights[:]
        rng.shuffle(w)
        parents.append(rng.choices(range(case["beams"]), [x + 0.3 for x in w], k=case["beams"]))
    return lens, parents


def _prepare_reorder(case, g):
    """Tables whose whole pages the beams of a request share, and a last page for each beam."""
    lens, parents = _splits(case)
    beams, ps, kv, dim, layers = (case[x] for x in ("beams", "page", "kv", "dim", "layers"))
    whole = [n // ps for n in lens]
    total = sum(whole) + case["r"] * beams
    order = torch.randperm(total, generator=g, device="cuda").to(torch.int32)
    table = torch.full((case["r"] * beams, max(whole) + 2), -1, dtype=torch.int32, device="cuda")
    at = 0
    for r, w in enumerate(whole):
        rows = slice(r * beams, (r + 1) * beams)
        table[rows, :w] = order[at:at + w]
        table[rows, w] = order[at + w:at + w + beams]
        at += w + beams
    state = {"case": case, "pages": table, "parents": _ints(parents),
             "lens": _ints(lens).repeat_interleave(beams)}
    for name in ("k", "v"):
        if case["type"] == "fp8":
            pool, scales = _pool(g, layers * total, kv, ps, dim)
            state[name + "_scales"] = scales.view(layers, total, kv, ps // BLOCK)
        else:
            pool = torch.randn(layers * total, kv, ps, dim, generator=g, device="cuda").to(BF16)
        state[name + "_pages"] = pool.view(layers, total, kv, ps, dim)
    return state


# ---------------------------------------------------------------------------------- one pass
def run(state):
    kind = state["case"]["kind"]
    if own:
        return {"append": _own_append, "attend": _own_attend, "reserve": _own_reserve, "beam": _own_beam,
                "reorder": _own_reorder}[kind](state)
    return {"append": _plain_append, "attend": _plain_attend, "reserve": _plain_reserve,
            "beam": _plain_beam, "reorder": _plain_reorder}[kind](state)


def _own_append(s):
    q = kernels().paged_append_fp8(s["qkv"], s["bias"], s["inv_freq"], s["table"], s["lens"], s["k_pages"],
                                   s["v_pages"], s["k_scales"], s["v_scales"], s["case"]["heads"],
                                   q_start=s["q_start"])
    return {"q": q, **{x: s[x] for x in ("k_pages", "v_pages", "k_scales", "v_scales")}}


def _own_attend(s):
    c = s["case"]
    return {"out": kernels().paged_attention_fp8(
        s["q"], s["k_pages"], s["v_pages"], s["k_scales"], s["v_scales"], s["table"], s["lens"], c["heads"],
        q_start=s["q_start"], shared=c["shared"] // c["page"] * c["page"], window=c["window"],
        sinks=c["sinks"], work=s["work"])}


def _own_reserve(s):
    k, ps = kernels(), s["case"]["page"]
    k.paged_reserve(s["back"], s["lens"], s["pages"], s["free"], s["n_free"], ps)
    q_start, slots, short = k.paged_reserve(s["new"], s["lens"], s["pages"], s["free"], s["n_free"], ps,
                                            rows=s["rows"])
    return {"q_start": q_start, "slots": slots, "short": short,
            **{x: s[x] for x in ("pages", "lens", "free", "n_free")}}


def _own_beam(s):
    scores, tokens, parents = kernels().beam_select(s["logits"], s["scores"], s["case"]["n"],
                                                    work=s["work"])
    return {"scores": scores, "tokens": tokens, "parents": parents}


def _own_reorder(s):
    pages = kernels().paged_reorder(s["parents"], s["pages"], s["lens"], s["k_pages"], s["v_pages"],
                                    s.get("k_scales"), s.get("v_scales"))
    return {"pages": pages, **{x: s[x] for x in ("k_pages", "v_pages", "k_scales", "v_scales") if x in s}}


def _positions(s):
    """(sequence, position, first new position of the sequence) of every token row."""
    seq = torch.arange(s["lens"].shape[0], device="cuda")
    if s["q_start"] is None:
        pos = s["lens"].long() - 1
        return seq, pos, pos
    T = s["qkv"].shape[0]
    start = s["q_start"].long()
    seq = torch.repeat_interleave(seq, start.diff(), output_size=T)
    first = s["lens"].long() - start.diff()
    return seq, torch.arange(T, device="cuda") - start[seq] + first[seq], first[seq]


def _plain_append(s):
    c = s["case"]
    heads, kv, dim, ps = c["heads"], c["kv"], c["dim"], c["page"]
    seq, pos, first = _positions(s)
    x = (s["qkv"].float() + s["bias"].float()).view(-1, heads + 2 * kv, dim)
    angle = (pos.double()[:, None] * s["inv_freq"].double())[:, None]
    cos, sin = angle.cos().float(), angle.sin().float()
    lo, hi = x[:, :heads + kv, :dim // 2], x[:, :heads + kv, dim // 2:]
    rot = torch.cat([lo * cos - hi * sin, hi * cos + lo * sin], -1)
    page = s["table"][seq, pos // ps].long()
    block = page * (ps // BLOCK) + pos % ps // BLOCK                  # of the pool, a token's
    held = torch.maximum(pos - pos % BLOCK, first) % BLOCK            # rows of it from before this step
    row = torch.arange(BLOCK, device="cuda")
    for new, pool, scales in ((rot[:, heads:], s["k_pages"], s["k_scales"]),
                              (x[:, heads + kv:], s["v_pages"], s["v_scales"])):
        blocks = pool.shape[0] * ps // BLOCK
        codes = pool.view(torch.uint8).view(-1, kv, ps // BLOCK, BLOCK, dim)
        exps = scales.view(torch.uint8)
        page_of, at = page[:, None], (pos % ps // BLOCK)[:, None]
        head = torch.arange(kv, device="cuda")[None]
        largest = torch.zeros(blocks, kv, device="cuda")
        largest.scatter_reduce_(0, block[:, None].expand(-1, kv), new.abs().amax(-1), "amax")
        old = exps[page_of, head, at].int() - 127
        e = _exponent(largest[block])
        e = torch.where(held[:, None] > 0, torch.maximum(e, old), e)
        before = codes[page_of, head, at]                             # [T, kv, 16, dim]
        again = torch.ldexp(before.view(FP8).float(), (old - e)[..., None, None]).to(FP8).view(torch.uint8)
        codes[page_of, head, at] = torch.where(row[:, None] < held[:, None, None, None], again, before)
        codes[page_of, head, at, (pos % BLOCK)[:, None]] = torch.ldexp(new, -e[..., None]).to(FP8).view(
            torch.uint8)
        exps[page_of, head, at] = (e + 127).to(torch.uint8)
    return {"q": rot[:, :heads].reshape(-1, heads * dim).to(BF16),
            **{x: s[x] for x in ("k_pages", "v_pages", "k_scales", "v_scales")}}


def _plain_attend(s):
    """The batch padded to its longest sequence and its most new tokens."""
    c = s["case"]
    heads, kv, dim, ps, b = c["heads"], c["kv"], c["dim"], c["page"], c["b"]
    rep, n, nn = heads // kv, s["most"], s["most_new"]
    lens = s["lens"].long()
    new = torch.ones_like(lens) if s["q_start"] is None else s["q_start"].long().diff()
    start = new.cumsum(0) - new
    ids = s["table"].long()

    def values(pool, scales):
        x = pool.view(torch.uint8)[ids].view(FP8).float().view(b, -1, kv, ps // BLOCK, BLOCK, dim)
        x *= scales.view(torch.uint8)[ids].view(E8M0).float()[..., None, None]
        return x.permute(0, 2, 1, 3, 4, 5).reshape(b, kv, -1, dim)[:, :, :n]

    tok = torch.arange(nn, device="cuda")
    rows = (start[:, None] + tok).clamp(max=s["q"].shape[0] - 1)      # those past a sequence's: not taken
    q = s["q"][rows].float().view(b, nn, kv, rep, dim).permute(0, 2, 1, 3, 4).reshape(b, kv, nn * rep, dim)
    score = q @ values(s["k_pages"], s["k_scales"]).transpose(2, 3).contiguous()
    pos = ((lens - new)[:, None] + tok).repeat_interleave(rep, 1)[:, None, :, None]
    key = torch.arange(n, device="cuda")
    hidden = key > pos
    if c["window"]:
        hidden |= (key <= pos - c["window"]) & (key >= c["sinks"])
    score.mul_(1 / math.sqrt(dim)).masked_fill_(hidden, float("-inf"))
    score = score.sub_(score.amax(-1, keepdim=True)).exp_()
    total = score.sum(-1, keepdim=True)
    out = (score @ values(s["v_pages"], s["v_scales"])) / total
    out = out.view(b, kv, nn, rep, dim).permute(0, 2, 1, 3, 4).reshape(b * nn, heads * dim)
    seq = torch.repeat_interleave(torch.arange(b, device="cuda"), new, output_size=s["q"].shape[0])
    return {"out": out[seq * nn + torch.arange(seq.shape[0], device="cuda") - start[seq]].to(BF16)}


def _plain_reserve(s):
    _plain_change(s, s["back"], 0)
    return _plain_change(s, s["new"], s["rows"])


def _plain_change(s, new, rows):
    ps, pages, free = s["case"]["page"], s["pages"], s["free"]
    old = s["lens"].clamp(min=0)
    lens = (old + new).clamp(min=0)
    had, has = ((n + ps - 1) // ps for n in (old, lens))
    j = torch.arange(pages.shape[1], device="cuda")
    out = (j >= has[:, None]) & (j < had[:, None])
    into = (j >= had[:, None]) & (j < has[:, None])
    given, taken = out.sum(), into.sum()
    top = s["n_free"].long() + given
    short = (taken - top).clamp(min=0).to(torch.int32)
    grown = new.clamp(min=0)
    start = torch.cat([grown.new_zeros(1), grown.cumsum(0).to(torch.int32)])
    bad = (short > 0) | (has > pages.shape[1]).any() | (top > free.shape[0])
    if rows:
        bad |= start[-1] > rows
    # the last page comes back first, so that what was taken together comes back as it lay
    rank = out.flatten().cumsum(0) - 1
    at = torch.where(out.flatten() & ~bad, top - 1 - rank, free.shape[0])
    free.copy_(torch.cat([free, free[:1]]).scatter(0, at, pages.flatten())[:-1])
    rank = (into.flatten().cumsum(0) - 1).view_as(into)
    pages.copy_(torch.where(into & ~bad, free[(top - 1 - rank).clamp(0, free.shape[0] - 1)], pages))
    s["n_free"].copy_(torch.where(bad, s["n_free"], (top - taken).to(torch.int32)))
    s["lens"].copy_(torch.where(bad, s["lens"], lens))
    start = torch.where(bad, 0, start)
    row = torch.arange(rows, device="cuda", dtype=torch.int32)
    seq = torch.searchsorted(start[1:], row, right=True).clamp(max=new.shape[0] - 1)
    pos = (s["lens"] - grown)[seq] + row - start[seq]
    slot = pages[seq, (pos // ps).clamp(0, pages.shape[1] - 1)].long() * ps + pos % ps
    return {"q_start": start, "slots": torch.where(row < start[-1], slot, -1),
            "short": torch.where(bad & (short == 0), -1, short).view(1), "pages": pages, "lens": s["lens"],
            "free": free, "n_free": s["n_free"]}


def _plain_beam(s):
    """In 64 bits: what decides between two beams' tokens is often far below 32 bits' step."""
    c = s["case"]
    r, beams, n, v = c["r"], c["beams"], c["n"], c["v"]
    x = s["logits"].double()
    m = x.amax(1, keepdim=True)
    x = x - (x - m).exp().sum(1, keepdim=True).log() - m
    x = (s["scores"].double().view(-1, 1) + x).view(r, beams * v)
    best, at = torch.sort(x, dim=1, descending=True, stable=True)
    at = at[:, :n].to(torch.int32)
    return {"scores": best[:, :n].float(), "tokens": at % v, "parents": at // v}


def _plain_reorder(s):
    c = s["case"]
    beams, ps = c["beams"], c["page"]
    rows = s["pages"].shape[0]
    parents = s["parents"].long()
    me = torch.arange(beams, device="cuda")
    # of a parent's children the parent itself or else the first one keeps its last page, the others get
    # the pages of the beams that ended, in order
    child = parents[:, :, None] == me                                   # [r, child, parent]
    own_way = parents == me
    keeper = torch.where(own_way.gather(1, parents), parents,
                         child.to(torch.int8).argmax(1).gather(1, parents))
    copied = keeper != me
    ended = ~child.any(1)
    rank = copied.cumsum(1) - 1
    nth = torch.sort((~ended).to(torch.int8), dim=1, stable=True).indices  # the ended ones first
    page_of = torch.where(copied, nth.gather(1, rank.clamp(min=0)), parents)
    base = torch.arange(0, rows, beams, device="cuda")[:, None]
    source, place = (base + parents).flatten(), (base + page_of).flatten()
    lens = s["lens"].long()[source]
    last = (lens // ps).clamp(max=s["pages"].shape[1] - 1)
    part = lens % ps
    j = torch.arange(s["pages"].shape[1], device="cuda")
    pages = torch.where(j < (lens // ps)[:, None], s["pages"][source], s["pages"])
    at = torch.arange(rows, device="cuda")
    to = s["pages"][place, last]
    pages[at, last] = torch.where(part > 0, to, s["pages"][at, last])
    to, frm = to.long().clamp(min=0), s["pages"][source, last].long().clamp(min=0)
    row = torch.arange(ps, device="cuda")
    fill = (row < part[:, None]) & copied.flatten()[:, None]
    for name in ("k", "v"):
        for pool, mask in ((s[name + "_pages"], fill[:, None, :, None]),
                           (s.get(name + "_scales"), fill[:, None, ::BLOCK])):
            if pool is not None:
                bits = pool.view(torch.uint8 if pool.element_size() == 1 else torch.int16)
                bits[:, to] = torch.where(mask, bits[:, frm], bits[:, to])
    return {"pages": pages, **{x: s[x] for x in ("k_pages", "v_pages", "k_scales", "v_scales") if x in s}}


# ---------------------------------------------------------------------------------- 64 bits
def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "attend": _exact_attend, "reserve": lambda s: None,
            "beam": _exact_beam, "reorder": _exact_reorder}[case["kind"]](s)


def _exact_append(s):
    """Codes before their rounding: what the pages would hold in units of the scales."""
    case = s["case"]
    heads, kv, dim, ps = case["heads"], case["kv"], case["dim"], case["page"]
    lens, new = _lengths(case)
    x = s["qkv"].double() + s["bias"].double()
    pools = {n: s[n].view(torch.uint8).view(FP8).double() for n in ("k_pages", "v_pages")}
    exps = {n: s[n].double().log2() for n in ("k_scales", "v_scales")}
    qs, row = [], 0
    for b in range(case["b"]):
        n, nn = lens[b], new[b]
        pos = torch.arange(n - nn, n, device="cuda")
        y = x[row:row + nn].view(nn, heads + 2 * kv, 2, dim // 2)
        turn = torch.polar(torch.ones((), dtype=torch.float64, device="cuda"),
                           torch.outer(pos.double(), s["inv_freq"].double()))[:, None]
        r = torch.complex(y[:, :heads + kv, 0], y[:, :heads + kv, 1]) * turn
        r = torch.stack([r.real, r.imag], 2).flatten(2)
        qs.append(r[:, :heads].flatten(1))
        row += nn
        # rows of the sequence's blocks from the first one touched on, those from before this step first
        lead = (n - nn) % BLOCK
        at = torch.arange(n - nn - lead, n, device="cuda")
        page = s["table"][b].long()[torch.div(at, ps, rounding_mode="floor")]
        heads_first = page[::BLOCK], (at[::BLOCK] % ps) // BLOCK
        for name, z in (("k", r[:, heads:]), ("v", y[:, heads + kv:].flatten(2))):
            pool, exp = pools[name + "_pages"], exps[name + "_scales"]
            old = exp[heads_first[0], :, heads_first[1]]                        # [blocks, kv]
            full = torch.zeros(old.shape[0] * BLOCK, kv, dim, dtype=torch.float64, device="cuda")
            full[lead:lead + nn] = z
            top = full.view(-1, BLOCK, kv, dim).abs().amax((1, 3))
            e = torch.ceil(torch.log2(torch.clamp(top, min=1e-300) / 448)).clamp(LEAST, MOST)
            if lead:
                e[0] = torch.maximum(e[0], old[0])
                full[:lead] = pool[page[:lead], :, at[:lead] % ps] * torch.exp2(old[0])[:, None]
            exp[heads_first[0], :, heads_first[1]] = e
            full = full / torch.exp2(e).repeat_interleave(BLOCK, 0)[..., None]
            pool[page, :, at % ps] = full[:lead + nn]
    return {"q": torch.cat(qs), **pools, **{n: torch.exp2(e) for n, e in exps.items()}}


def _exact_attend(s):
    case = s["case"]
    heads, kv, dim, ps = case["heads"], case["kv"], case["dim"], case["page"]
    lens, new = _lengths(case)
    row = 0
    out = torch.zeros(sum(new), heads, dim, dtype=torch.float64, device="cuda")
    for b in range(case["b"]):
        pos = torch.arange(lens[b], device="cuda")
        page, at = s["table"][b].long()[torch.div(pos, ps, rounding_mode="floor")], pos % ps
        qpos = torch.arange(lens[b] - new[b], lens[b], device="cuda")[:, None]
        hidden = pos > qpos
        if case["window"] > 0:
            hidden = hidden | ((pos <= qpos - case["window"]) & (pos >= case["sinks"]))
        for g in range(kv):
            k, v = (s[n + "_pages"].view(torch.uint8)[page, g, at].view(FP8).double()
                    * s[n + "_scales"].view(torch.uint8)[page, g, at // BLOCK].view(E8M0).double()[:, None]
                    for n in ("k", "v"))
            for h in range(g * heads // kv, (g + 1) * heads // kv):
                q = s["q"][row:row + new[b], h * dim:(h + 1) * dim].double()
                p = torch.softmax((q @ k.t() * dim ** -0.5).masked_fill_(hidden, -math.inf), -1)
                out[row:row + new[b], h] = p @ v
        row += new[b]
    return {"out": out.flatten(1)}


def _exact_beam(s):
    c = s["case"]
    x = s["logits"].double()
    x = x - torch.logsumexp(x, 1, keepdim=True) + s["scores"].double().reshape(-1, 1)
    best = torch.topk(x.view(c["r"], -1), c["n"], dim=1).values
    return {"scores": best, "tokens": None, "parents": None}


def _exact_reorder(s):
    case, (lens, parents) = s["case"], _splits(s["case"])
    beams, ps = case["beams"], case["page"]
    names = [n for n in ("k_pages", "v_pages", "k_scales", "v_scales") if n in s]
    for r, (n, chosen) in enumerate(zip(lens, parents)):
        ids = s["pages"][r * beams:(r + 1) * beams, n // ps].tolist()
        ended = [i for i in range(beams) if i not in chosen]
        kept = {}
        for i in sorted(range(beams), key=lambda i: chosen[i] != i):
            kept.setdefault(chosen[i], i)
        for i, p in enumerate(chosen):
            if kept[p] != i:
                to, rows = ids[ended.pop(0)], n % ps
                for name in names:
                    count = rows if name.endswith("pages") else -(-rows // BLOCK)
                    bits = s[name].view(torch.uint8 if s[name].element_size() == 1 else torch.int16)
                    bits[:, to, :, :count] = bits[:, ids[p], :, :count]
    return {"pages": None, **{n: s[n].double() for n in names}}


# ---------------------------------------------------------------------------------- work
def work(case):
    if case["kind"] == "beam":
        rows, v = case["r"] * case["beams"], case["v"]
        return {"bytes": rows * v * (2 if case["type"] == "bf16" else 4) + 4 * rows + 12 * case["r"] * case["n"],
                "flops": 3 * rows * v}
    if case["kind"] == "reorder":
        lens, parents = _splits(case)
        row = case["layers"] * case["kv"] * case["dim"] * (1 if case["type"] == "fp8" else 2)
        copied = sum((n % case["page"]) * (case["beams"] - len(set(p))) for n, p in zip(lens, parents))
        tables = sum(-(-n // case["page"]) for n in lens) * case["beams"]
        return {"bytes": 4 * row * copied + 8 * tables + 8 * case["r"] * case["beams"], "flops": 0}
    lens, new = _lengths(case)
    T = sum(new)
    if case["kind"] == "reserve":
        moved = sum(-(-n // case["page"]) - -(-(n - nn) // case["page"]) for n, nn in zip(lens, new))
        return {"bytes": 8 * T + 16 * moved + 28 * case["b"], "flops": 0}
    heads, kv, dim = case["heads"], case["kv"], case["dim"]
    if case["kind"] == "append":
        # new values are read in 16 bits; queries are written in 16, keys and values in 8
        return {"bytes": 2 * T * (2 * heads + 3 * kv) * dim + 2 * (heads + 2 * kv) * dim,
                "flops": 5 * T * (heads + 2 * kv) * dim}
    window, sinks = case["window"], case["sinks"] if case["window"] else 0
    common = case["shared"] // case["page"] * case["page"]
    pairs, rows, lowest = 0, 0, common
    for n, nn in zip(lens, new):
        pairs += sum(min(p + 1, window + min(sinks, max(p + 1 - window, 0))) if window else p + 1
                     for p in range(n - nn, n))
        low = max(n - nn + 1 - window, 0) if window else 0  # below it only the first tokens are seen
        first = min(sinks, low)
        rows += max(first - common, 0) + n - max(low, common)
        lowest = min(lowest, low)
    if common:  # the shared rows that any sequence sees, read once
        rows += min(sinks, lowest) + common - lowest
    return {"bytes": 4 * T * heads * dim + 2 * rows * kv * dim, "flops": 4 * pairs * heads * dim}
