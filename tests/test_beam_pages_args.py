"""paged_reorder with a stack of free pages: calls that the entry point and the wrapper refuse before a launch, and the list model
of the GPU tests over a long search (no GPU)."""
import random

import pytest
import torch

from beam_pages_ref import dropped
from nanoserve_amd import ops
from test_cache_ops_refusals import BF16, REORDER, _address, _cache, _z, lib, on_cpu, stub  # noqa: F401

BACK = dict(REORDER, free=_address(10), cap=64, nf=_address(11))


def _back(lib, **kw):  # noqa: F811
    a = {**BACK, **kw}
    return lib.ns_paged_reorder_back(a["par"], a["pst"], a["tab"], a["ts"], a["w"], a["lens"], a["out"], a["k"], a["v"], a["ls"],
                                     a["ps"], a["hs"], a["ks"], a["vs"], a["sl"], a["sp"], a["sh"], a["layers"], a["n"],
                                     a["page"], a["rb"], a["R"], a["beams"], a["Hk"], a["free"], a["cap"], a["nf"], None)


@on_cpu
@pytest.mark.parametrize("ok", [dict(), dict(ks=None, vs=None), dict(cap=0, free=None), dict(cap=0), dict(cap=1),
                                dict(free=_address(11) + 4), dict(nf=_address(10) + 256), dict(free=_address(3) + 12 * 8 * 4)], ids=str)
def test_takes(lib, ok):  # noqa: F811
    assert _back(lib, **ok) not in (0, -2)


@on_cpu
@pytest.mark.parametrize("bad", [
    dict(nf=None), dict(free=None), dict(cap=-1), dict(cap=1 << 31), dict(free=_address(10) + 2), dict(nf=_address(11) + 1),
    dict(nf=_address(10)), dict(nf=_address(10) + 252), dict(free=_address(11) - 252), dict(free=_address(0)),
    dict(free=_address(1) - 252), dict(free=_address(2) + 44), dict(free=_address(3) + 12 * 8 * 4 - 4), dict(nf=_address(3)),
    dict(nf=_address(2)), dict(nf=_address(1) + 4), dict(nf=_address(0)), dict(free=_address(4) + 64), dict(nf=_address(5)),
    dict(nf=_address(6) + 28), dict(free=_address(7) - 252), dict(R=0), dict(beams=65, pst=65), dict(out=_address(1))], ids=str)
def test_refusals(lib, bad):  # noqa: F811
    assert _back(lib, **bad) == -2


@pytest.mark.parametrize("bad", [
    dict(free=_z(20)), dict(n_free=_z(1)), dict(free=_z(20), n_free=_z(2)), dict(free=_z(4, 5), n_free=_z(1)),
    dict(free=_z(40)[::2], n_free=_z(1)), dict(free=_z(20, dtype=torch.int64), n_free=_z(1)),
    dict(free=_z(20), n_free=_z(1, dtype=torch.int64))], ids=str)
def test_wrapper_refuses(stub, bad):  # noqa: F811
    with pytest.raises((ValueError, TypeError)):
        stub.paged_reorder(_z(3, 4), _z(12, 5), _z(12), **_cache(), **bad)
    assert not stub.lib.calls


def test_wrapper_hands_over(stub):  # noqa: F811
    free, n_free = _z(20), _z(1)
    stub.paged_reorder(_z(3, 4), _z(12, 5), _z(12), **_cache(), free=free, n_free=n_free)
    assert list(stub.lib.calls) == ["ns_paged_reorder_back"]
    args = stub.lib.calls["ns_paged_reorder_back"]
    assert args[24:27] == (free.data_ptr(), 20, n_free.data_ptr())
    assert len(args) == len(ops.INTERNAL_SIGNATURES["ns_paged_reorder_back"]) == 28
    stub.paged_reorder(_z(0, 4), _z(0, 5), _z(0), **_cache(), free=free, n_free=n_free)
    assert len(stub.lib.calls) == 1


def test_list_model_loses_no_page():
    """8 beams on pages of 16 over 1000 steps of random parents: every page is in a row or free, where without the stack the most
    are in neither."""
    rng, beams, page, steps = random.Random(1), 8, 16, 1000
    width = steps // page + 1
    n_pages = beams * width
    free, rows, taken = list(range(n_pages)), [[-1] * width for _ in range(beams)], 0
    for n in range(steps):
        parents = [rng.randrange(beams) for _ in range(beams)]
        free += dropped(rows, [parents], [n] * beams, page, n_pages)
        w = n // page
        last = sorted(row[w] for row in rows)
        rows = [rows[p][:w] + row[w:] for p, row in zip(parents, rows)]  # (whose last pages: any order)
        if n % page == 0:
            for row in rows:
                row[w] = free.pop()
                taken += 1
        else:
            assert last == sorted(row[w] for row in rows)
        used = {x for row in rows for x in row[:w + 1]}
        assert used | set(free) == set(range(n_pages)) and len(used) + len(free) == n_pages
    assert taken > 400 and len(used) < 100
