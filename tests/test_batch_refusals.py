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
