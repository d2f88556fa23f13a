"""Calls of the 8-bit cache's, the page reservation's and beam search's operators that the entry points and wrappers
refuse before a launch, and ones that they take (no GPU)."""
import ctypes
import types

import pytest
import torch

from nanoserve_amd import Kernels, ops

BF16, I32, FP8, E8M0 = torch.bfloat16, torch.int32, torch.float8_e4m3fn, torch.float8_e8m0fnu


def _address(i):  # 0.25 GiB apart, never dereferenced: the calls that pass the checks end at the missing GPU
    return (i + 1) << 28


on_cpu = pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are no memory")


@pytest.fixture(scope="module")
def lib():
    return Kernels().lib


# ------------------------------------------------------------------ the cache in 8 bits (strides in bytes)
ATTEND = dict(q=_address(0), qs=512, k=_address(1), v=_address(2), ps=4096, hs=2048, ks=_address(7), vs=_address(8), sp=2,
              sh=1, n=8, page=16, tab=_address(3), ts=4, w=4, lens=_address(4), start=None, out=_address(5),
              work=_address(6), bytes=1 << 20, T=5, B=5, Hq=4, Hk=2, D=128, shared=0, window=0, sinks=0, scale=0.1)
APPEND = dict(qkv=_address(0), qs=1024, bias=_address(9), inv=_address(10), start=None, lens=_address(4),
              tab=_address(3), ts=4, w=4, k=_address(1), v=_address(2), ps=4096, hs=2048, ks=_address(7), vs=_address(8),
              sp=2, sh=1, n=8, page=16, out=_address(5), T=5, B=5, Hq=4, Hk=2, D=128)


def _attention(lib, **kw):
    a = {**ATTEND, **kw}
    return lib.ns_paged_attention_fp8(
        a["q"], a["qs"], a["k"], a["v"], a["ps"], a["hs"], a["ks"], a["vs"], a["sp"], a["sh"], a["n"], a["page"], a["tab"],
        a["ts"], a["w"], a["lens"], a["start"], a["out"], a["work"], a["bytes"], a["T"], a["B"], a["Hq"], a["Hk"], a["D"],
        a["shared"], a["window"], a["sinks"], a["scale"], None)


def _append(lib, **kw):
    a = {**APPEND, **kw}
    return lib.ns_paged_append_fp8(
        a["qkv"], a["qs"], a["bias"], a["inv"], a["start"], a["lens"], a["tab"], a["ts"], a["w"], a["k"], a["v"], a["ps"],
        a["hs"], a["ks"], a["vs"], a["sp"], a["sh"], a["n"], a["page"], a["out"], a["T"], a["B"], a["Hq"], a["Hk"], a["D"],
        None)


@on_cpu
@pytest.mark.parametrize("call", [_attention, _append])
@pytest.mark.parametrize("ok", [
    dict(), dict(ps=2048, hs=16384, sp=1, sh=8), dict(ps=4112), dict(sp=7, sh=3), dict(sp=1000), dict(n=1, ps=0, sp=0),
    dict(page=32, ps=8192, hs=4096, sp=4, sh=2), dict(start=_address(11)),
    # one record per page: codes and scales of both between each other
    dict(v=_address(1) + 4096, ks=_address(1) + 8192, vs=_address(1) + 8208, ps=8224, sp=8224),
    dict(v=_address(1) + 2048, ks=_address(1) + 8192, vs=_address(1) + 8194, hs=4096, ps=8208, sp=8208, sh=1)], ids=str)
def test_cache_layouts_are_taken(lib, call, ok):
    assert call(lib, **ok) not in (0, -2)


@on_cpu
@pytest.mark.parametrize("call", [_attention, _append])
@pytest.mark.parametrize("bad", [
    dict(k=None), dict(k=_address(1) + 8), dict(v=None), dict(ks=None), dict(vs=None), dict(ps=4088), dict(ps=2048),
    dict(hs=1024), dict(hs=2040), dict(sp=1), dict(sh=0), dict(sp=0), dict(sp=-2), dict(sh=-1), dict(sp=1 << 47),
    dict(page=24), dict(page=0), dict(n=0), dict(D=32), dict(D=96), dict(D=256), dict(Hk=0), dict(Hq=0), dict(T=4),
    dict(T=0), dict(B=0), dict(w=1 << 27), dict(ts=3), dict(lens=None), dict(tab=None), dict(qs=508), dict(qs=256),
    dict(out=None), dict(out=_address(5) + 8), dict(out=_address(1)), dict(out=_address(7)), dict(out=_address(8) - 16),
    dict(out=_address(3)), dict(out=_address(4))], ids=str)
def test_cache_refusals(lib, call, bad):
    assert call(lib, **bad) == -2


@on_cpu
@pytest.mark.parametrize("bad", [
    dict(Hq=5), dict(shared=-1), dict(window=-1), dict(sinks=-1), dict(scale=0.0), dict(scale=float("nan")),
    dict(w=400, ts=400, work=None), dict(w=400, ts=400, bytes=100), dict(w=400, ts=400, work=_address(7)),
    dict(w=400, ts=400, work=_address(1)), dict(q=None)], ids=str)
def test_attention_refusals(lib, bad):
    assert _attention(lib, **bad) == -2


@on_cpu
@pytest.mark.parametrize("bad", [
    dict(v=_address(1)), dict(v=_address(1) + 16), dict(vs=_address(7)), dict(vs=_address(7) + 1), dict(ks=_address(1)),
    dict(vs=_address(2) + 8 * 4096 - 1), dict(ks=_address(1) + 4096, ps=6144), dict(qkv=_address(1)), dict(qkv=_address(7)),
    dict(bias=_address(8)), dict(inv=_address(2)), dict(inv=None), dict(lens=_address(7)), dict(tab=_address(8) - 4),
    dict(out=_address(0)), dict(out=_address(9)), dict(out=_address(10) - 16), dict(bias=_address(9) + 2),
    # records in which codes and scales of the next page meet
    dict(v=_address(1) + 4096, ks=_address(1) + 8192, vs=_address(1) + 8207, ps=8208, sp=8208)], ids=str)
def test_append_refusals(lib, bad):
    assert _append(lib, **bad) == -2


# ------------------------------------------------------------------ reservation
RESERVE = dict(add=_address(0), lens=_address(1), tab=_address(2), ts=10, w=8, free=_address(3), cap=100, nf=_address(4),
               qs=_address(5), slots=_address(6), rows=64, short=_address(7), B=5, page=16)


def _reserve(lib, **kw):
    a = {**RESERVE, **kw}
    return lib.ns_paged_reserve(a["add"], a["lens"], a["tab"], a["ts"], a["w"], a["free"], a["cap"], a["nf"], a["qs"],
                                a["slots"], a["rows"], a["short"], a["B"], a["page"], None)


@on_cpu
@pytest.mark.parametrize("ok", [dict(), dict(rows=-1, slots=None), dict(rows=0, slots=None), dict(rows=1 << 20),
                                dict(cap=0, free=None), dict(B=100000, ts=8)], ids=str)
def test_reserve_takes(lib, ok):
    assert _reserve(lib, **ok) not in (0, -2)


@on_cpu
@pytest.mark.parametrize("bad", [
    dict(B=0), dict(B=1 << 24), dict(w=0), dict(page=0), dict(page=8), dict(page=24), dict(ts=7), dict(w=1 << 26, ts=1 << 26),
    dict(cap=-1), dict(cap=1 << 31), dict(rows=-2), dict(add=None), dict(lens=None), dict(tab=None), dict(free=None),
    dict(nf=None), dict(qs=None), dict(short=None), dict(slots=None), dict(slots=_address(6) + 4), dict(add=_address(0) + 2),
    dict(lens=_address(0)), dict(lens=_address(0) + 16), dict(tab=_address(3)), dict(free=_address(2) + 4 * 40),
    dict(nf=_address(3) + 396), dict(qs=_address(1) + 16), dict(slots=_address(5) + 16), dict(short=_address(6) + 8 * 63),
    dict(short=_address(4)), dict(qs=_address(0) - 20)], ids=str)
def test_reserve_refusals(lib, bad):
    assert _reserve(lib, **bad) == -2


# ------------------------------------------------------------------ selection
SELECT = dict(x=_address(0), fp32=0, rs=100, s=_address(1), os=_address(2), ot=_address(3), op=_address(4),
              work=_address(5), bytes=1 << 30, R=3, beams=4, V=100, n=8)


def _select(lib, **kw):
    a = {**SELECT, **kw}
    return lib.ns_beam_select(a["x"], a["fp32"], a["rs"], a["s"], a["os"], a["ot"], a["op"], a["work"], a["bytes"], a["R"],
                              a["beams"], a["V"], a["n"], None)


@on_cpu
@pytest.mark.parametrize("ok", [dict(), dict(fp32=1), dict(x=_address(0) + 2), dict(beams=64, n=64), dict(V=1 << 20, rs=1 << 20),
                                dict(R=16383), dict(rs=1000, os=_address(0) + 2 * 12000)], ids=str)
def test_select_takes(lib, ok):
    assert _select(lib, **ok) not in (0, -2)


@on_cpu
@pytest.mark.parametrize("bad", [
    dict(R=0), dict(beams=0), dict(beams=65), dict(n=0), dict(n=65), dict(V=0), dict(V=(1 << 20) + 1, rs=1 << 21),
    dict(R=16384), dict(rs=99), dict(x=None), dict(s=None), dict(os=None), dict(ot=None), dict(op=None), dict(work=None),
    dict(x=_address(0) + 1), dict(fp32=1, x=_address(0) + 2), dict(work=_address(5) + 8), dict(bytes=100),
    dict(ot=_address(2)), dict(op=_address(3) + 92), dict(os=_address(0)), dict(os=_address(0) + 2396), dict(ot=_address(1)),
    dict(work=_address(0)), dict(work=_address(1) - 16), dict(work=_address(4)), dict(s=_address(5))], ids=str)
def test_select_refusals(lib, bad):
    assert _select(lib, **bad) == -2


def test_select_workspace(lib):
    assert lib.ns_beam_select_workspace(3, 4, 100, 8) > 0
    for bad in ((0, 4, 100, 8), (3, 65, 100, 8), (3, 4, 0, 8), (3, 4, 100, 65), (1 << 16, 1, 100, 8)):
        assert lib.ns_beam_select_workspace(*bad) == 0


# ------------------------------------------------------------------ reordering
# 2 layers of 8 pages with 2 heads of 16 rows of 128 bytes
REORDER = dict(par=_address(0), pst=8, tab=_address(1), ts=10, w=8, lens=_address(2), out=_address(3), k=_address(4),
               v=_address(5), ls=32768, ps=4096, hs=2048, ks=_address(6), vs=_address(7), sl=16, sp=2, sh=1, layers=2, n=8,
               page=16, rb=128, R=3, beams=4, Hk=2)


def _reorder(lib, **kw):
    a = {**REORDER, **kw}
    return lib.ns_paged_reorder(a["par"], a["pst"], a["tab"], a["ts"], a["w"], a["lens"], a["out"], a["k"], a["v"], a["ls"],
                                a["ps"], a["hs"], a["ks"], a["vs"], a["sl"], a["sp"], a["sh"], a["layers"], a["n"],
                                a["page"], a["rb"], a["R"], a["beams"], a["Hk"], None)


K4 = _address(4)


@on_cpu
@pytest.mark.parametrize("ok", [
    dict(), dict(ks=None, vs=None), dict(ls=2 * 32768, v=K4 + 32768), dict(layers=1, ls=0, sl=0),
    dict(ls=4096, ps=8192, sl=2, sp=4), dict(beams=64, pst=64), dict(ls=65536, v=K4 + 32768, ks=K4 + 131072, vs=K4 + 131200),
    # one record per layer and page: K, V and their scales
    dict(v=K4 + 4096, ks=K4 + 8192, vs=K4 + 8208, ps=8224, sp=8224, ls=8 * 8224, sl=8 * 8224)], ids=str)
def test_reorder_takes(lib, ok):
    assert _reorder(lib, **ok) not in (0, -2)


@on_cpu
@pytest.mark.parametrize("bad", [
    dict(R=0), dict(beams=0), dict(beams=65, pst=65), dict(R=1 << 23), dict(w=0), dict(ts=7), dict(pst=3), dict(page=8),
    dict(page=0), dict(layers=0), dict(n=0), dict(Hk=0), dict(rb=0), dict(rb=24), dict(par=None), dict(tab=None),
    dict(lens=None), dict(out=None), dict(k=None), dict(v=None), dict(ks=None), dict(vs=None), dict(k=K4 + 8),
    dict(ps=4088), dict(ps=2048), dict(hs=1024), dict(ls=16384), dict(ls=-32768), dict(sp=1), dict(sl=8), dict(sh=0),
    dict(v=K4), dict(v=K4 + 2048), dict(v=K4 + 32768), dict(ks=K4), dict(vs=_address(6)), dict(vs=_address(6) + 31),
    dict(out=_address(1)), dict(out=_address(1) + 4), dict(out=_address(0)), dict(out=_address(2) + 44), dict(out=K4 + 16),
    dict(tab=K4 + 64), dict(lens=_address(7)), dict(par=_address(5) + 16), dict(out=_address(6) - 4),
    dict(v=K4 + 4096, ks=K4 + 8192, vs=K4 + 8207, ps=8208, sp=8208, ls=8 * 8208, sl=8 * 8208)], ids=str)
def test_reorder_refusals(lib, bad):
    assert _reorder(lib, **bad) == -2


# ------------------------------------------------------------------ the wrappers
class _Lib:
    def __init__(self):
        self.calls = {}

    def __getattr__(self, name):
        def call(*args):
            self.calls[name] = args
            return 64 if name.endswith("_workspace") else 0

        return call


@pytest.fixture
def stub(monkeypatch):
    """Kernels on CPU tensors with the library replaced."""
    def check(t, name, dtype):
        if t.dtype != dtype:
            raise TypeError(name)

    monkeypatch.setattr(ops, "_require_gpu_tensor", check)
    monkeypatch.setattr(ops, "_current_device", lambda: -1)  # what CPU tensors say
    monkeypatch.setattr(ops, "_raw_stream", lambda device: 0)
    k = Kernels.__new__(Kernels)
    k.lib = _Lib()
    return k


def _z(*shape, dtype=I32):
    return torch.zeros(*shape, dtype=torch.uint8 if dtype in (FP8, E8M0) else dtype).view(dtype)


def _cache(pages=8, heads=2, page=16, D=128, layers=None):
    lead = () if layers is None else (layers,)
    return dict(k_pages=_z(*lead, pages, heads, page, D, dtype=FP8), v_pages=_z(*lead, pages, heads, page, D, dtype=FP8),
                k_scales=_z(*lead, pages, heads, page // 16, dtype=E8M0),
                v_scales=_z(*lead, pages, heads, page // 16, dtype=E8M0))


def _attend(k, **kw):
    a = dict(q=_z(3, 512, dtype=BF16), pages=_z(3, 4), lens=_z(3), n_heads=4, **_cache())
    return k.paged_attention_fp8(**{**a, **kw})


def _add(k, **kw):
    a = dict(qkv=_z(3, 1024, dtype=BF16), bias=None, inv_freq=torch.zeros(64), pages=_z(3, 4), lens=_z(3), n_heads=4, **_cache())
    return k.paged_append_fp8(**{**a, **kw})


@pytest.mark.parametrize("call", [_attend, _add])
@pytest.mark.parametrize("bad", [
    dict(k_pages=_z(8, 2, 16, 128, dtype=BF16)), dict(v_pages=_z(9, 2, 16, 128, dtype=FP8)),
    dict(k_scales=_z(8, 2, 1, dtype=torch.uint8)), dict(k_scales=_z(8, 2, 2, dtype=E8M0)),
    dict(v_scales=_z(8, 2, 1, dtype=torch.float32)), dict(v_scales=_z(16, 2, 1, dtype=torch.uint8)[::2].view(E8M0)),
    dict(lens=_z(4)), dict(pages=_z(4, 4)), dict(pages=_z(3, 8)[:, ::2]), dict(n_heads=5), dict(q_start=_z(3)),
    dict(out=_z(3, 511, dtype=BF16)), dict(lens=_z(3, dtype=torch.int64))], ids=lambda b: next(iter(b)))
def test_cache_wrappers_refuse(stub, call, bad):
    with pytest.raises((ValueError, TypeError)):
        call(stub, **bad)
    assert not any(not n.endswith("_workspace") for n in stub.lib.calls)


@pytest.mark.parametrize("call, name, columns", [(_attend, "q", 512), (_add, "qkv", 1024)])
def test_what_the_library_refuses(stub, call, name, columns):
    """An output over the input is named, anything else has the library's code."""
    stub.lib = types.SimpleNamespace(ns_paged_append_fp8=lambda *a: -2, ns_paged_attention_fp8=lambda *a: -2,
                                     ns_paged_attention_fp8_workspace=lambda *a: 64)
    x, work = _z(3, columns, dtype=BF16), dict(work=torch.zeros(64, dtype=torch.uint8)) if call is _attend else {}
    with pytest.raises(ValueError, match="overlap"):
        call(stub, **{name: x, "out": x.view(-1)[:3 * 512].view(3, 512)}, **work)
    with pytest.raises(RuntimeError, match="-2"):
        call(stub, **{name: x, "out": _z(3, 512, dtype=BF16)}, **work)


def test_attention_workspace_must_be_contiguous(stub):
    with pytest.raises(ValueError, match="contiguous"):
        _attend(stub, work=torch.zeros(1, dtype=torch.uint8).expand(1 << 20))


def test_empty_batches(stub):
    _attend(stub, q=_z(0, 512, dtype=BF16), pages=_z(0, 4), lens=_z(0))
    _add(stub, qkv=_z(0, 1024, dtype=BF16), pages=_z(0, 4), lens=_z(0))
    a, b, c = stub.beam_select(torch.zeros(0, 10), torch.zeros(0, 4), 3)
    assert a.shape == b.shape == c.shape == (0, 3)
    assert stub.paged_reorder(_z(0, 4), _z(0, 5), _z(0), **_cache()).shape == (0, 5)
    assert not any(not n.endswith("_workspace") for n in stub.lib.calls)


def _room(k, **kw):
    a = dict(new=_z(3), lens=_z(3), pages=_z(3, 6), free=_z(20), n_free=_z(1), page_size=16, rows=10)
    return k.paged_reserve(**{**a, **kw})


@pytest.mark.parametrize("bad", [
    dict(new=_z(3, 1)), dict(new=_z(6)[::2]), dict(new=_z(0), lens=_z(0), pages=_z(0, 6)), dict(lens=_z(4)),
    dict(lens=_z(6)[::2]), dict(pages=_z(4, 6)), dict(pages=_z(3, 12)[:, ::2]), dict(free=_z(4, 5)), dict(free=_z(40)[::2]),
    dict(n_free=_z(2)), dict(rows=-1), dict(lens=_z(3, dtype=torch.int64)), dict(out=(_z(3), _z(10, dtype=torch.int64), _z(1))),
    dict(out=(_z(4), _z(9, dtype=torch.int64), _z(1))), dict(out=(_z(4), _z(10), _z(1))),
    dict(out=(_z(4), _z(10, dtype=torch.int64), _z(2))), dict(rows=None, out=(_z(4), _z(10, dtype=torch.int64), _z(1)))], ids=str)
def test_reserve_wrapper_refuses(stub, bad):
    with pytest.raises((ValueError, TypeError)):
        _room(stub, **bad)
    assert not stub.lib.calls


@pytest.mark.parametrize("bad", [dict(page_size=(1 << 32) + 16), dict(page_size=-16), dict(rows=1 << 31)], ids=str)
def test_reserve_sizes_past_32_bits(stub, bad):
    """Sizes whose low bits would pass."""
    with pytest.raises(ValueError):
        _room(stub, **bad)
    assert not stub.lib.calls


def test_select_sizes_past_32_bits(stub):
    a = dict(logits=torch.zeros(12, 50), scores=torch.zeros(3, 4), n=8)
    for bad in (dict(n=(1 << 32) + 8), dict(n=-1)):
        with pytest.raises(ValueError):
            stub.beam_select(**{**a, **bad})
    assert not stub.lib.calls
    stub.beam_select_workspace(3, 4, 50, (1 << 32) + 8, device="cpu")
    assert stub.lib.calls["ns_beam_select_workspace"] == (3, 4, 50, (1 << 31) - 1)


def test_reserve_wrapper_hands_over(stub):
    q, slots, short = _room(stub)
    assert q.shape == (4,) and slots.shape == (10,) and slots.dtype == torch.int64 and short.shape == (1,)
    assert stub.lib.calls["ns_paged_reserve"][10] == 10
    assert _room(stub, rows=None)[1] is None and stub.lib.calls["ns_paged_reserve"][9:11] == (None, -1)


@pytest.mark.parametrize("bad", [
    dict(logits=torch.zeros(11, 50)), dict(logits=torch.zeros(12, 50).t().contiguous().t()),
    dict(logits=torch.zeros(12, 50, dtype=torch.float16)), dict(scores=torch.zeros(3, 8)[:, ::2]), dict(scores=torch.zeros(12)),
    dict(scores=torch.zeros(3, 4, dtype=BF16)), dict(out=(torch.zeros(3, 8), _z(3, 8), _z(3, 7))),
    dict(out=(torch.zeros(3, 8), torch.zeros(3, 8), _z(3, 8))), dict(work=torch.zeros(128, dtype=torch.uint8)[::2])],
    ids=lambda b: next(iter(b)))
def test_select_wrapper_refuses(stub, bad):
    with pytest.raises((ValueError, TypeError)):
        stub.beam_select(**{**dict(logits=torch.zeros(12, 50), scores=torch.zeros(3, 4), n=8), **bad})
    assert "ns_beam_select" not in stub.lib.calls


@pytest.mark.parametrize("bad", [
    dict(parents=_z(12)), dict(parents=_z(3, 8)[:, ::2]), dict(parents=_z(3, 4, dtype=torch.int64)), dict(pages=_z(11, 5)),
    dict(pages=_z(12, 10)[:, ::2]), dict(lens=_z(11)), dict(v_pages=_z(8, 2, 32, 128, dtype=FP8)), dict(k_scales=None),
    dict(k_pages=_z(8, 2, 16, 128, dtype=BF16)), dict(k_scales=_z(8, 2, 2, dtype=E8M0)), dict(out=_z(12, 6)),
    dict(k_pages=_z(8, 16, 2, 128, dtype=torch.uint8).transpose(1, 2).view(FP8))], ids=lambda b: next(iter(b)))
def test_reorder_wrapper_refuses(stub, bad):
    a = dict(parents=_z(3, 4), pages=_z(12, 5), lens=_z(12), **_cache())
    with pytest.raises((ValueError, TypeError)):
        stub.paged_reorder(**{**a, **bad})
    assert not stub.lib.calls


def test_reorder_wrapper_hands_over(stub):
    """Strides in bytes, of all layers or of one; candidates' first columns as they lie."""
    c = _cache(layers=3)
    stub.paged_reorder(_z(3, 8)[:, :4], _z(12, 5), _z(12), **c)
    args = stub.lib.calls["ns_paged_reorder"]
    assert args[1] == 8 and args[9:12] == (8 * 4096, 4096, 2048) and args[14:17] == (16, 2, 1)
    assert args[17:24] == (3, 8, 16, 128, 3, 4, 2)
    pool = _z(8, 2, 16, 128, dtype=BF16)
    stub.paged_reorder(_z(3, 4), _z(12, 5), _z(12), pool, pool.clone())
    args = stub.lib.calls["ns_paged_reorder"]
    assert args[9:12] == (0, 8192, 4096) and args[12:17] == (None, None, 0, 0, 0) and args[20] == 256


def test_argument_types():
    """As many arguments as the declarations have."""
    for name, n in (("ns_paged_append_fp8", 26), ("ns_paged_attention_fp8", 30), ("ns_paged_reserve", 15),
                    ("ns_beam_select", 14), ("ns_paged_reorder", 25)):
        assert len(ops.INTERNAL_SIGNATURES[name]) == n
    assert ops.RESTYPES["ns_beam_select_workspace"] is ctypes.c_size_t


@on_cpu
def test_checks_of_layouts_are_quick(lib):
    """Records of a million pages, many layers and heads, and layouts whose check would be long, which are refused."""
    import time
    start = time.perf_counter()
    n = 1 << 20
    record = 2 * 80 * 16 * 2048 + 4096
    assert _reorder(lib, n=n, layers=80, Hk=16, ls=2 * 16 * 2048, ps=record, v=K4 + 16 * 2048, ks=K4 + record - 4096,
                    vs=K4 + record - 2048, sl=16, sp=record, sh=1, lens=1 << 61, tab=1 << 60, par=1 << 59,
                    out=1 << 58) not in (0, -2)
    assert _append(lib, n=n, ps=2048, hs=2048 * n, ks=APPEND["k"] + 2048 * n, sp=2048, sh=2048 * n + 16) == -2
    assert time.perf_counter() - start < 1.0
