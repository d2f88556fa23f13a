"""Refusals of the batch operators, before any launch (no GPU): sizes, strides, alignment, metadata."""
import pytest
import torch

from nanoserve_amd import Kernels, ops

P = 0x10000  # a 64 KiB-aligned non-null address: never dereferenced on these paths
BF16, I32 = torch.bfloat16, torch.int32


@pytest.fixture(scope="module")
def lib():
    return Kernels().lib


ATTEND = dict(q=P, qs=512, k=P, v=P, ps=4096, hs=2048, n=8, page=16, tab=P, ts=4, w=4, lens=P, start=None,
              out=P, work=P, bytes=1 << 30, T=3, B=3, Hq=4, Hk=2, D=128, shared=0, window=0, sinks=0,
              scale=0.1)


@pytest.mark.parametrize("bad", [
    dict(q=None), dict(q=P + 8), dict(k=None), dict(k=P + 2), dict(v=None), dict(out=None), dict(out=P + 4),
    dict(tab=None), dict(tab=P + 2), dict(lens=None), dict(lens=P + 1), dict(start=P + 2), dict(qs=508),
    dict(qs=256), dict(ps=1024), dict(ps=4098), dict(hs=1024), dict(hs=-2048), dict(n=0), dict(page=8),
    dict(page=24), dict(page=0), dict(ts=3), dict(w=0), dict(w=1 << 27), dict(T=4), dict(T=0), dict(B=0),
    dict(Hq=5), dict(Hk=0), dict(Hq=0), dict(D=96), dict(D=256), dict(shared=-1), dict(window=-1),
    dict(sinks=-1), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("inf")), dict(scale=float("nan")),
    dict(start=P, T=1 << 29, qs=1 << 12), dict(w=400, ts=400, work=None),
    dict(w=400, ts=400, bytes=100), dict(w=400, ts=400, work=P + 8)], ids=str)
def test_paged_attention_refuses(lib, bad):
    a = {**ATTEND, **bad}
    assert lib.ns_paged_attention(
        a["q"], a["qs"], a["k"], a["v"], a["ps"], a["hs"], a["n"], a["page"], a["tab"], a["ts"], a["w"],
        a["lens"], a["start"], a["out"], a["work"], a["bytes"], a["T"], a["B"], a["Hq"], a["Hk"], a["D"],
        a["shared"], a["window"], a["sinks"], a["scale"], None) == -2


APPEND = dict(qkv=P, qs=1024, bias=P, inv=P, start=None, lens=P, tab=P, ts=4, w=4, k=P, v=P, ps=4096,
              hs=2048, n=8, page=16, out=P, T=3, B=3, Hq=4, Hk=2, D=128)


@pytest.mark.parametrize("bad", [
    dict(qkv=None), dict(qkv=P + 2), dict(qs=1016), dict(qs=1028), dict(bias=P + 2), dict(inv=None),
    dict(inv=P + 2), dict(lens=None), dict(tab=None), dict(k=None), dict(v=P + 8), dict(ps=2048, hs=2044),
    dict(hs=2040), dict(ps=1000), dict(n=-1), dict(page=17), dict(out=None), dict(out=P + 8), dict(T=2),
    dict(Hq=0), dict(Hk=-1), dict(D=72), dict(D=1024), dict(w=1 << 26), dict(ts=-4)], ids=str)
def test_paged_append_refuses(lib, bad):
    a = {**APPEND, **bad}
    assert lib.ns_paged_append(
        a["qkv"], a["qs"], a["bias"], a["inv"], a["start"], a["lens"], a["tab"], a["ts"], a["w"], a["k"],
        a["v"], a["ps"], a["hs"], a["n"], a["page"], a["out"], a["T"], a["B"], a["Hq"], a["Hk"], a["D"],
        None) == -2


def test_paged_attention_workspace_sizes(lib):
    def size(T=4, B=4, Hq=28, Hk=4, D=128, max_len=4096, ragged=0, shared=0):
        return lib.ns_paged_attention_workspace(T, B, Hq, Hk, D, max_len, ragged, shared)

    # nothing to merge: no key range of 64 rows (single tokens) or 256 (prompts) is ever split
    assert size(max_len=64) == 0 and size(max_len=256, ragged=1) == 0
    assert size() > 0 and size(shared=1) > 0 and size(max_len=64, shared=1) > 0
    # a table far wider than the batch's lengths does not grow it: the GPU's workgroups bound the parts
    assert size(max_len=1 << 29) == size(max_len=1 << 20) < 64 << 20
    assert size(D=96) == size(Hq=6) == size(T=0) == size(max_len=0) == size(shared=-1) == 0


def _pool(**kw):
    return torch.zeros(kw.get("shape", (8, 2, 16, 128)), dtype=kw.get("dtype", BF16))


def test_wrapper_refusals(monkeypatch):
    """Shapes and strides that the wrappers check (on CPU tensors; nothing is launched)."""
    k = Kernels()
    ints = dict(dtype=I32)
    with pytest.raises(ValueError):  # CPU tensors
        k.paged_attention(torch.zeros(1, 512, dtype=BF16), _pool(), _pool(), torch.zeros(1, 4, **ints),
                          torch.zeros(1, **ints), 4)

    def check(t, name, dtype):
        if t.dtype != dtype:
            raise TypeError(name)

    monkeypatch.setattr(ops, "_require_gpu_tensor", check)
    monkeypatch.setattr(ops, "_current_device", lambda: -1)  # what CPU tensors say
    monkeypatch.setattr(ops, "_raw_stream", lambda device: 0)

    def attend(q=torch.zeros(3, 512, dtype=BF16), kp=_pool(), vp=_pool(), pages=torch.zeros(3, 4, **ints),
               lens=torch.zeros(3, **ints), heads=4, **kw):
        return k.paged_attention(q, kp, vp, pages, lens, heads, **kw)

    buf = torch.zeros(4, 4096, dtype=BF16)
    for kw, err in ((dict(q=torch.zeros(3, 512)), TypeError), (dict(q=torch.zeros(512, 3, dtype=BF16).t()), ValueError),
                    (dict(heads=3), ValueError), (dict(q=torch.zeros(4, 512, dtype=BF16)), ValueError),
                    (dict(kp=_pool(dtype=torch.float16)), TypeError), (dict(vp=_pool(shape=(8, 2, 32, 128))), ValueError),
                    (dict(kp=_pool(shape=(8, 16, 2, 128)).transpose(1, 2)), ValueError),
                    (dict(pages=torch.zeros(3, 4, dtype=torch.int64)), TypeError),
                    (dict(pages=torch.zeros(2, 4, **ints)), ValueError),
                    (dict(pages=torch.zeros(4, 3, **ints).t()), ValueError),
                    (dict(lens=torch.zeros(3, 1, **ints)), ValueError),
                    (dict(lens=torch.zeros(6, **ints)[::2]), ValueError),
                    (dict(q_start=torch.zeros(3, **ints)), ValueError),
                    (dict(out=torch.zeros(3, 256, dtype=BF16)), ValueError),
                    (dict(q=buf[0, :1536].view(3, 512), out=buf[0, 512:2048].view(3, 512)), ValueError),
                    (dict(q=buf[:3, :512], out=buf[2, 500:2036].view(3, 512)), ValueError),
                    (dict(work=torch.zeros(9)), TypeError), (dict(window=-2), RuntimeError),
                    (dict(scale=0.0), RuntimeError)):
        if err is RuntimeError:
            kw["work"] = torch.zeros(1 << 20, dtype=torch.uint8)
        with pytest.raises(err):
            attend(**kw)

    def append(qkv=torch.zeros(3, 1024, dtype=BF16), bias=None, inv=torch.zeros(64), **kw):
        return k.paged_append(qkv, bias, inv, torch.zeros(3, 4, **ints), torch.zeros(3, **ints), _pool(), _pool(),
                              4, **kw)

    for kw, err in ((dict(qkv=torch.zeros(3, 1024)), TypeError), (dict(qkv=torch.zeros(3, 512, dtype=BF16)), ValueError),
                    (dict(bias=torch.zeros(512, dtype=BF16)), ValueError), (dict(inv=torch.zeros(32)), ValueError),
                    (dict(inv=torch.zeros(64).half()), TypeError), (dict(out=torch.zeros(3, 1024, dtype=BF16)), ValueError),
                    (dict(qkv=buf[:3, :1024], out=buf[2, 1000:2536].view(3, 512)), ValueError),
                    (dict(q_start=torch.zeros(5, **ints)), ValueError)):
        with pytest.raises(err):
            append(**kw)
    # tensors of another device than the current one, whose stream the launch would go to
    monkeypatch.setattr(ops, "_current_device", lambda: 0)
    for call in (attend, append):
        with pytest.raises(ValueError, match="current"):
            call()
    with pytest.raises(ValueError, match="current"):
        k.sample(torch.zeros(2, 8), torch.zeros(2))


SAMPLE = dict(x=P, fp32=0, rs=100, u=P, T=None, k=None, p=None, m=None, out=P, work=P, bytes=1 << 30, B=2, V=100)


@pytest.mark.parametrize("bad", [
    dict(x=None), dict(x=P + 1), dict(x=P + 2, fp32=1), dict(rs=99), dict(u=None), dict(u=P + 2), dict(T=P + 1),
    dict(k=P + 2), dict(p=P + 3), dict(m=P + 1), dict(out=None), dict(out=P + 2), dict(B=0), dict(V=0),
    dict(V=(1 << 20) + 1, rs=1 << 22)], ids=str)
def test_sample_refuses(lib, bad):
    a = {**SAMPLE, **bad}
    assert lib.ns_sample(a["x"], a["fp32"], a["rs"], a["u"], a["T"], 1.0, a["k"], 0, a["p"], 1.0, a["m"], 0.0,
                         a["out"], a["work"], a["bytes"], a["B"], a["V"], None) == -2


def test_sample_wrapper_refusals(monkeypatch):
    k = Kernels()
    with pytest.raises(ValueError):
        k.sample(torch.zeros(1, 8), torch.zeros(1))

    def check(t, name, dtype):
        if t.dtype != dtype:
            raise TypeError(name)

    monkeypatch.setattr(ops, "_require_gpu_tensor", check)
    monkeypatch.setattr(ops, "_current_device", lambda: -1)
    x, u = torch.zeros(2, 8), torch.zeros(2)
    for args, kw, err in (((x.half(), u), {}, TypeError), ((x.t(), torch.zeros(8)), {}, ValueError),
                          ((x[0], u), {}, ValueError), ((x, torch.zeros(3)), {}, ValueError),
                          ((x, u.double()), {}, TypeError), ((x, u), dict(temperature=-1.0), ValueError),
                          ((x, u), dict(temperature=float("nan")), ValueError), ((x, u), dict(top_k=-1), ValueError),
                          ((x, u), dict(top_p=1.5), ValueError), ((x, u), dict(top_p=-0.5), ValueError),
                          ((x, u), dict(min_p=2.0), ValueError), ((x, u), dict(top_k=torch.zeros(2)), TypeError),
                          ((x, u), dict(top_p=torch.zeros(3)), ValueError),
                          ((x, u), dict(out=torch.zeros(2, dtype=torch.int64)), TypeError),
                          ((x, u), dict(out=torch.zeros(3, dtype=I32)), ValueError)):
        with pytest.raises(err):
            k.sample(*args, **kw)
