"""Calls of the batch operators that the wrappers and entry points have to refuse before a launch, and what
they hand to the library for the sizes that they take (no GPU)."""
import pytest
import torch

from nanoserve_amd import Kernels, ops

P = 0x10000  # a 64 KiB-aligned non-null address: never dereferenced on these paths
BF16, I32 = torch.bfloat16, torch.int32


class _Lib:
    """Stands in for the library: keeps the arguments of every call; workspaces take 64 bytes."""

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
    monkeypatch.setattr(Kernels, "_stream", staticmethod(lambda: 0))
    k = Kernels.__new__(Kernels)
    k.lib = _Lib()
    return k


def _bf16(*shape):
    return torch.zeros(*shape, dtype=BF16)


def _ints(*shape):
    return torch.zeros(*shape, dtype=I32)


def _attend(k, **kw):
    pool = _bf16(8, 2, 16, 128)
    return k.paged_attention(_bf16(3, 512), pool, pool.clone(), _ints(3, 4), _ints(3), 4, **kw)


# a workspace whose elements are repeated or apart: the library would write `numel` bytes from its address on
@pytest.mark.parametrize("work", [torch.zeros(1, dtype=torch.uint8).expand(1 << 20),
                                  torch.zeros(1 << 21, dtype=torch.uint8)[::2]], ids=["expanded", "strided"])
@pytest.mark.parametrize("call", [
    lambda k, w: _attend(k, work=w),
    lambda k, w: k.sample(torch.zeros(2, 8), torch.zeros(2), work=w),
    lambda k, w: k.prompt_attention(_bf16(2, 256), _bf16(1, 2, 128), _bf16(1, 2, 128), 2, 0, work=w),
    lambda k, w: k.decode_attention(_bf16(256), _bf16(1, 8, 128), _bf16(1, 8, 128), _ints(1), 2, 1, 128, w),
    lambda k, w: k.decode_qkv_attention(_bf16(512), None, torch.zeros(64), _ints(1), _bf16(1, 8, 128),
                                        _bf16(1, 8, 128), 2, 1, 128, w),
    lambda k, w: k.w4_linear(_bf16(2, 128), _ints(16, 16), _bf16(16, 1), work=w)],
    ids=["paged_attention", "sample", "prompt_attention", "decode_attention", "decode_qkv_attention", "w4_linear"])
def test_workspace_must_be_contiguous(stub, call, work):
    with pytest.raises(ValueError, match="contiguous"):
        call(stub, work)
    assert not any(not n.endswith("_workspace") for n in stub.lib.calls)
    call(stub, torch.zeros(1 << 20, dtype=torch.uint8))


@pytest.mark.parametrize("n,held", [((1 << 31) + 5, (1 << 31) - 1), ((1 << 32) + 16, (1 << 31) - 1),
                                    (1 << 40, (1 << 31) - 1), (-(1 << 32), -(1 << 31)), (4096, 4096), (0, 0)])
def test_counts_past_32_bits(stub, n, held):
    """A window, first tokens or a prefix of more than 32 bits are as many as can be, not their low bits."""
    _attend(stub, window=n, sinks=n, shared=n)
    assert stub.lib.calls["ns_paged_attention"][-5:-2] == (held, held, held)
    assert stub.lib.calls["ns_paged_attention_workspace"][-1] == held


def test_negative_counts_past_32_bits_are_refused(monkeypatch):
    monkeypatch.setattr(ops, "_require_gpu_tensor", lambda *a: None)
    monkeypatch.setattr(ops, "_current_device", lambda: -1)
    monkeypatch.setattr(ops, "_raw_stream", lambda device: 0)
    work = torch.zeros(1 << 20, dtype=torch.uint8)
    for kw in (dict(window=-(1 << 32)), dict(sinks=-(1 << 33)), dict(shared=-(1 << 32))):
        with pytest.raises(RuntimeError, match="-2"):
            _attend(Kernels(), work=work, **kw)


# ------------------------------------------------------------------ entry points, with addresses that are apart
# 0.25 GiB apart, never dereferenced: the calls that pass the checks end at the missing GPU
def _address(i):
    return (i + 1) << 28


on_cpu = pytest.mark.skipif(torch.cuda.is_available(), reason="the addresses are no memory")
ATTEND = dict(q=_address(0), qs=512, k=_address(1), v=_address(2), ps=4096, hs=2048, n=8, page=16, tab=_address(3), ts=4,
              w=4, lens=_address(4), start=None, out=_address(5), work=_address(6), bytes=1 << 20, T=5, B=5, Hq=4, Hk=2,
              D=128, shared=0, window=0, sinks=0, scale=0.1)
APPEND = dict(qkv=_address(0), qs=1024, bias=_address(7), inv=_address(8), start=None, lens=_address(4),
              tab=_address(3), ts=4, w=4, k=_address(1), v=_address(2), ps=4096, hs=2048, n=8, page=16, out=_address(5),
              T=5, B=5, Hq=4, Hk=2, D=128)


@pytest.fixture(scope="module")
def lib():
    return Kernels().lib


def _attention(lib, **kw):
    a = {**ATTEND, **kw}
    return lib.ns_paged_attention(
        a["q"], a["qs"], a["k"], a["v"], a["ps"], a["hs"], a["n"], a["page"], a["tab"], a["ts"], a["w"],
        a["lens"], a["start"], a["out"], a["work"], a["bytes"], a["T"], a["B"], a["Hq"], a["Hk"], a["D"],
        a["shared"], a["window"], a["sinks"], a["scale"], None)


def _append(lib, **kw):
    a = {**APPEND, **kw}
    return lib.ns_paged_append(
        a["qkv"], a["qs"], a["bias"], a["inv"], a["start"], a["lens"], a["tab"], a["ts"], a["w"], a["k"],
        a["v"], a["ps"], a["hs"], a["n"], a["page"], a["out"], a["T"], a["B"], a["Hq"], a["Hk"], a["D"], None)


# strides in elements for 8 pages and 2 heads of 2048: pages outside, heads outside, either padded; a lone page or
# head has no stride
@on_cpu
@pytest.mark.parametrize("call", [_attention, _append])
@pytest.mark.parametrize("ok", [
    dict(), dict(ps=2048, hs=16384), dict(ps=4104), dict(ps=4608, hs=2560), dict(ps=2056, hs=16440), dict(n=1, ps=0),
    dict(n=1, ps=8), dict(n=1 << 30, ps=1 << 45)], ids=str)
def test_pool_strides_are_taken(lib, call, ok):
    assert call(lib, **ok) not in (0, -2)


@pytest.mark.parametrize("call", [_attention, _append])
@pytest.mark.parametrize("bad", [
    dict(ps=2048), dict(ps=4088), dict(ps=2048, hs=16376), dict(ps=2048, hs=4096), dict(ps=2056),
    dict(ps=2048, hs=2056), dict(ps=0), dict(hs=0), dict(ps=1 << 50), dict(hs=1 << 62)], ids=str)
def test_pages_and_heads_that_overlap_are_refused(lib, call, bad):
    if torch.cuda.is_available():
        pytest.skip("the addresses are no memory")
    assert call(lib, **bad) == -2


@on_cpu
def test_tensors_that_are_apart_are_taken(lib):
    for kw in (dict(), dict(start=_address(9)), dict(out=_address(0) + 5 * 1024), dict(out=_address(0) - 5 * 1024),
               # pools cut from one buffer: keys and values of a page beside each other, of a head beside each other,
               # of other layers, one behind the other
               dict(v=_address(1) + 2 * 4096, ps=8192), dict(v=_address(1) + 2 * 2048, ps=8192, hs=4096),
               dict(v=_address(1) + 2 * 8192, ps=5 * 4096), dict(v=_address(1) + 2 * 8 * 4096),
               dict(v=_address(1) + 2 * 16384 * 2, hs=16384, ps=2048), dict(v=_address(1) - 2 * 8 * 4096),
               # an output between two pages' rows
               dict(out=_address(1) + 2 * 4096, ps=8192, v=_address(2))):
        assert _attention(lib, **{k: w for k, w in kw.items()}) not in (0, -2), kw
        if "out" not in kw:
            assert _append(lib, **kw) not in (0, -2), kw
    assert _attention(lib, v=ATTEND["k"]) not in (0, -2)  # reads alone
    assert _append(lib, out=_address(0) + 5 * 2048) not in (0, -2)


K = ATTEND["k"]
TABLE = dict(w=400, ts=400)  # wide enough that the work may be split


@on_cpu
@pytest.mark.parametrize("bad", [
    dict(out=_address(0)), dict(out=_address(0) + 5 * 1024 - 16), dict(out=_address(0) - 5 * 1024 + 16), dict(out=K),
    dict(out=K + 2 * 8 * 4096 - 16), dict(out=K - 16), dict(out=K + 2 * 4096, ps=6144 - 1024, v=_address(2)),
    dict(out=ATTEND["v"] + 4096), dict(out=ATTEND["tab"]), dict(out=ATTEND["lens"]),
    dict(out=_address(9), start=_address(9) + 32), dict(out=ATTEND["tab"] + 2 * 400 * 4, **TABLE),
    dict(work=ATTEND["q"], **TABLE), dict(work=ATTEND["out"] + 16, **TABLE), dict(work=K, **TABLE),
    dict(work=ATTEND["v"] - 16, **TABLE), dict(work=ATTEND["lens"] - 16, **TABLE), dict(work=ATTEND["tab"] + 16, **TABLE)],
    ids=str)
def test_attention_outputs_over_inputs_are_refused(lib, bad):
    assert _attention(lib, **bad) == -2


@on_cpu
@pytest.mark.parametrize("bad", [
    dict(v=K), dict(v=K + 16), dict(v=K + 2 * 7 * 4096), dict(v=K - 16), dict(v=K + 2 * 4096 - 16, ps=8192),
    dict(v=K + 2 * 2048, ps=8192), dict(v=K + 2 * 2048, ps=8192, hs=4096 - 8), dict(out=_address(0)),
    dict(out=_address(0) + 5 * 2048 - 16), dict(out=APPEND["bias"]), dict(out=APPEND["inv"] - 16), dict(out=K),
    dict(out=APPEND["v"] + 2 * 5 * 4096), dict(out=APPEND["tab"]), dict(out=APPEND["lens"]),
    dict(out=_address(9), start=_address(9)), dict(qkv=K), dict(qkv=K - 5 * 2048 + 16), dict(bias=APPEND["v"]),
    dict(inv=K + 16), dict(lens=K + 16), dict(tab=APPEND["v"] + 4), dict(start=K + 4)], ids=str)
def test_append_outputs_over_inputs_are_refused(lib, bad):
    assert _append(lib, **bad) == -2


SAMPLE = dict(x=_address(0), fp32=0, rs=100, u=_address(1), T=_address(2), k=_address(3), p=_address(4), m=_address(5),
              out=_address(6), work=_address(7), bytes=1 << 30, B=2, V=100)


def _sample(lib, **kw):
    a = {**SAMPLE, **kw}
    return lib.ns_sample(a["x"], a["fp32"], a["rs"], a["u"], a["T"], 1.0, a["k"], 0, a["p"], 1.0, a["m"], 0.0,
                         a["out"], a["work"], a["bytes"], a["B"], a["V"], None)


@on_cpu
def test_sample_takes_what_is_apart(lib):
    for kw in (dict(), dict(T=None, k=None, p=None, m=None), dict(fp32=1), dict(out=_address(0) + 400),
               dict(out=_address(0) - 8)):
        assert _sample(lib, **kw) not in (0, -2), kw


@on_cpu
@pytest.mark.parametrize("bad", [
    dict(work=None), dict(work=SAMPLE["work"] + 8), dict(bytes=100), dict(out=SAMPLE["x"]), dict(out=SAMPLE["x"] + 396),
    dict(out=SAMPLE["x"] + 796, fp32=1), dict(out=SAMPLE["x"] + 300, rs=101, V=50), dict(work=SAMPLE["x"]),
    dict(work=SAMPLE["out"]), dict(work=SAMPLE["u"] - 16), dict(work=SAMPLE["T"] - 16), dict(work=SAMPLE["k"] - 16),
    dict(work=SAMPLE["p"]), dict(work=SAMPLE["m"] - 64)], ids=str)
def test_sample_outputs_over_inputs_are_refused(lib, bad):
    assert _sample(lib, **bad) == -2
