"""ctypes bindings to libnanoserve_amd.so: the W4A16 part of the reference's ``Kernels`` class
(Uttaprexa/nanoserve python/nanoserve/ops.py:15-39, 76-97), same method names, argument
meaning, return values and exceptions.

The library is loaded with ctypes exactly as the reference loads build/libnanoserve.so; loading
needs no GPU. There is no CPU fallback: a missing library raises at construction, and tensors
that are not on the GPU raise before any native call.
"""
from __future__ import annotations

import ctypes
import os

import torch

LIB_PATH = os.path.join(os.path.dirname(os.path.abspath(__file__)), "libnanoserve_amd.so")

# Exported symbols and their ctypes signatures (include/nanoserve_w4.h,
# include/nanoserve_decode.h, include/nanoserve_probe.h); every function returns int except
# where RESTYPES says otherwise.
_VP, _I32, _I64, _F32, _SZ = (ctypes.c_void_p, ctypes.c_int, ctypes.c_longlong, ctypes.c_float,
                              ctypes.c_size_t)
SIGNATURES = {
    "ns_w4_quantize": [_VP, _VP, _VP, _I32, _I32, _I32, _VP],
    "ns_w4_linear": [_VP, _VP, _VP, _VP, _I32, _I32, _I32, _I32, _VP],
    "ns_rmsnorm": [_VP, _VP, _VP, _VP, _I32, _I32, _F32, _VP],
    "ns_rope": [_VP, _VP, _VP, _I32, _I32, _I32, _I32, _I32, _I64, _I64, _VP],
    "ns_swiglu": [_VP, _VP, _VP, _I32, _I32, _VP],
    "ns_decode_qkv": [_VP, _VP, _VP, _VP, _VP, _VP, _I32, _I32, _I32, _I32, _VP],
    "ns_decode_attention_workspace": [_I32, _I32, _I32, _I32],
    "ns_decode_attention": [_VP, _VP, _VP, _VP, _VP, _VP, _SZ, _I32, _I32, _I32, _I32, _VP],
    "ns_decode_qkv_attention": [_VP, _VP, _VP, _VP, _VP, _VP, _VP, _VP, _SZ, _I32, _I32, _I32,
                                _I32, _I32, _VP, _VP],
    "ns_decode_embed": [_VP, _VP, _VP, _I32, _I32, _VP, _I32, _VP, _VP, _VP],
    "ns_w4_gemv_decode_attn": [_VP, _VP, _VP, _I32, _I32, _VP, _VP, _VP, _I32, _I32, _I32, _VP],
}
SIGNATURES["ns_w4_gemv_decode"] = [_VP, _VP, _VP, _VP, _F32, _VP, _VP, _VP, _VP, _I32, _I32, _I32,
                                   _I32, _VP]
SIGNATURES["ns_bf16_gemv"] = [_VP, _VP, _VP, _VP, _F32, _VP, _VP, _I32, _I32, _VP]
SIGNATURES["ns_w4_repack"] = [_VP, _VP, _VP, _VP, _I32, _I32, _I32, _VP]
SIGNATURES["ns_w4_linear_packed"] = [_VP, _VP, _VP, _VP, _I32, _I32, _I32, _I32, _VP]
SIGNATURES["ns_w4_linear_packed_swiglu"] = [_VP, _VP, _VP, _VP, _I32, _I32, _I32, _I32, _VP]
SIGNATURES["ns_w4_linear_swiglu"] = [_VP, _VP, _VP, _VP, _I32, _I32, _I32, _I32, _VP]
SIGNATURES["ns_w4_linear_workspace"] = [_I32, _I32, _I32, _I32]
SIGNATURES["ns_w4_linear_ws"] = [_VP, _VP, _VP, _VP, _I32, _I32, _I32, _I32, _VP, _SZ, _VP]
SIGNATURES["ns_w4_gptq_workspace"] = [_I32]
SIGNATURES["ns_w4_gptq"] = [_VP, _VP, _VP, _VP, _VP, _SZ, _I32, _I32, _I32, _VP]
SIGNATURES["ns_decode_attention_noalloc"] = [_VP, _VP, _VP, _VP, _VP, _I32, _I32, _I32, _I32, _VP]
SIGNATURES["ns_probe_read"] = [_VP, _SZ, _VP, _I32, _I32, _I32, _VP]
SIGNATURES["ns_probe_empty"] = [_I32, _I32, _VP]
SIGNATURES["ns_probe_linear_loop"] = [_VP] * 7 + [_I32, _I32, _VP]
RESTYPES = {"ns_decode_attention_workspace": _SZ, "ns_w4_gptq_workspace": _SZ,
            "ns_w4_linear_workspace": _SZ, "ns_prompt_attention_workspace": _SZ,
            "ns_w4_linear_swiglu_rows_workspace": _SZ, "ns_paged_attention_workspace": _SZ,
            "ns_sample_workspace": _SZ, "ns_paged_attention_fp8_workspace": _SZ,
            "ns_beam_select_workspace": _SZ}
# Entry points of this package's own callers (csrc/internal_ops.h, csrc/batch_ops.h), not part of the
# public ABI.
INTERNAL_SIGNATURES = {
    "ns_prompt_qkv": [_VP] * 5 + [_I32] * 6 + [_VP],
    "ns_w4_linear_rows": [_VP] * 4 + [_I32] * 4 + [_VP],
    "ns_w4_linear_swiglu_rows_workspace": [_I32] * 4,
    "ns_w4_linear_swiglu_rows": [_VP] * 5 + [_SZ] + [_I32] * 4 + [_VP],
    "ns_prompt_attention_fits": [_I32] * 4 + [_I64],
    "ns_prompt_attention_workspace": [_I32] * 4,
    "ns_prompt_attention": [_VP, _I64, _VP, _VP, _I64, _I64, _VP, _VP, _SZ, _I32, _I32, _I32, _I32,
                            _VP],
    "ns_paged_append": [_VP, _I64] + [_VP] * 5 + [_I64, _I32, _VP, _VP, _I64, _I64, _I32, _I32, _VP]
                       + [_I32] * 5 + [_VP],
    "ns_paged_attention_workspace": [_I32] * 8,
    "ns_paged_attention": [_VP, _I64, _VP, _VP, _I64, _I64, _I32, _I32, _VP, _I64, _I32, _VP, _VP, _VP,
                           _VP, _SZ] + [_I32] * 8 + [_F32, _VP],
    "ns_paged_append_fp8": [_VP, _I64] + [_VP] * 5 + [_I64, _I32, _VP, _VP, _I64, _I64, _VP, _VP, _I64, _I64,
                                                      _I32, _I32, _VP] + [_I32] * 5 + [_VP],
    "ns_paged_attention_fp8_workspace": [_I32] * 8,
    "ns_paged_attention_fp8": [_VP, _I64, _VP, _VP, _I64, _I64, _VP, _VP, _I64, _I64, _I32, _I32, _VP, _I64, _I32,
                               _VP, _VP, _VP, _VP, _SZ] + [_I32] * 8 + [_F32, _VP],
    "ns_paged_reserve": [_VP, _VP, _VP, _I64, _I32, _VP, _I64, _VP, _VP, _VP, _I32, _VP, _I32, _I32, _VP],
    "ns_beam_select_workspace": [_I32] * 4,
    "ns_beam_select": [_VP, _I32, _I64] + [_VP] * 5 + [_SZ] + [_I32] * 4 + [_VP],
    "ns_paged_reorder": [_VP, _I64, _VP, _I64, _I32] + [_VP] * 4 + [_I64] * 3 + [_VP] * 2 + [_I64] * 3 + [_I32] * 7 + [_VP],
    "ns_paged_reorder_back": [_VP, _I64, _VP, _I64, _I32] + [_VP] * 4 + [_I64] * 3 + [_VP] * 2 + [_I64] * 3 + [_I32] * 7 +
                             [_VP, _I64, _VP, _VP],
    "ns_sample_workspace": [_I32] * 3,
    "ns_sample": [_VP, _I32, _I64, _VP, _VP, _F32, _VP, _I32, _VP, _F32, _VP, _F32, _VP, _VP, _SZ, _I32,
                  _I32, _VP],
}


if hasattr(torch._C, "_cuda_getCurrentRawStream"):
    _raw_stream = torch._C._cuda_getCurrentRawStream
else:  # pragma: no cover - older torch builds
    def _raw_stream(device):
        return torch.cuda.current_stream(device).cuda_stream


# The current device index without torch.cuda.current_device()'s initialisation check: the callers have
# GPU tensors in hand (and reading the raw stream, as probe_empty does without any, initialises the
# runtime itself).
_current_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)


def _require_gpu_tensor(t: torch.Tensor, name: str, dtype: torch.dtype) -> None:
    # (the common case first: these checks run several times per launch, 0.3 us against 0.6 each)
    if type(t) is torch.Tensor and t.is_cuda and t.dtype is dtype:
        return
    if not isinstance(t, torch.Tensor):
        raise TypeError(f"{name} must be a torch.Tensor")
    if t.device.type != "cuda":
        raise ValueError(f"{name} must be a GPU tensor (got device {t.device})")
    if t.dtype != dtype:
        raise TypeError(f"{name} must be {dtype} (got {t.dtype})")


def _rot_ptr(rot, head_dim):
    _require_gpu_tensor(rot, "rot", torch.float32)
    if not rot.is_contiguous() or rot.numel() != head_dim:
        raise ValueError("rot must be a contiguous [2, head_dim / 2] float32 tensor")
    return rot.data_ptr()


def _check_out(out: torch.Tensor, like: torch.Tensor) -> torch.Tensor:
    _require_gpu_tensor(out, "out", like.dtype)
    if out.shape != like.shape or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous tensor of shape {tuple(like.shape)}")
    return out


def _aligned_rows(x: torch.Tensor) -> torch.Tensor:
    """A contiguous tensor at a 16-byte aligned address: x, or a copy of a view that starts at
    another one."""
    return x if x.data_ptr() % 16 == 0 else x.clone()


def _overlap(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Whether two contiguous tensors share memory."""
    pa, pb = a.data_ptr(), b.data_ptr()
    return pa < pb + b.nbytes and pb < pa + a.nbytes


def _require_here(t: torch.Tensor, name: str, dtype: torch.dtype, here: int) -> None:
    """_require_gpu_tensor, and that t is on the current device ``here``, whose stream is launched on."""
    if type(t) is torch.Tensor and t.dtype is dtype and t.get_device() == here:
        return
    _require_gpu_tensor(t, name, dtype)
    if t.get_device() != here:
        raise ValueError(f"{name} is on device {t.get_device()}, the current one is {here}")


def _device_of(t: torch.Tensor, name: str, dtype: torch.dtype) -> int:
    """_require_gpu_tensor of a call's first tensor; returns the current device, which it must be on."""
    _require_gpu_tensor(t, name, dtype)
    here = _current_device()
    _require_here(t, name, dtype, here)
    return here


def _int32(n: int) -> int:
    """n held to 32 bits, for counts where more than every position means no more than that (the library's
    argument would keep the low bits alone)."""
    return max(-(1 << 31), min(n, (1 << 31) - 1))


def _strided_work():
    # elements that are apart or repeated (an expanded byte) span another range than their number says
    return ValueError("work must be contiguous")


def check_setting(name: str, t) -> None:
    """Raises unless the number t is a setting ``name`` (temperature, top_k, top_p, min_p) of Kernels.sample."""
    if not t >= 0 or (name in ("top_p", "min_p") and t > 1):
        raise ValueError(f"{name} is out of range: {t}")


def _apart(out: torch.Tensor, t: torch.Tensor, name: str) -> None:
    """Raises if the contiguous out shares memory with t, whose last dimension is contiguous."""
    a, b = out.data_ptr(), t.data_ptr()
    if out.numel() and t.numel() and a < b + 2 * ((t.shape[0] - 1) * t.stride(0) + t.shape[1]) and b < a + out.nbytes:
        raise ValueError(f"out must not overlap {name}")


class Kernels:
    """W4A16 kernels through the C ABI. ``path`` defaults to the in-tree library."""

    def __init__(self, path: str = LIB_PATH):
        path = os.path.abspath(path)
        if not os.path.exists(path):
            raise OSError(f"{path} not found: build it with `python -m nanoserve_amd.build` "
                          "(there is no CPU fallback)")
        self.lib = ctypes.CDLL(path)
        for name, args in {**SIGNATURES, **INTERNAL_SIGNATURES}.items():
            fn = getattr(self.lib, name)
            fn.argtypes = args
            fn.restype = RESTYPES.get(name, ctypes.c_int)

    # reference ops.py:32-34: the current torch stream (a hipStream_t on ROCm), read as a raw
    # handle (no Stream object per call: the eager launch path runs this for every operator)
    @staticmethod
    def _stream():
        return _raw_stream(_current_device())

    # reference ops.py:36-39
    @staticmethod
    def _check(rc: int, name: str):
        if rc != 0:
            raise RuntimeError(f"{name} failed with code {rc}")

    def w4_quantize(self, W, group=128):
        """W [N, K] bf16 -> (Wq int32 [N, K // 8], S bf16 [N, K // group]). Reference
        ops.py:76-83 (kernel: kernels/quant/w4a16.cuh:272-301)."""
        _require_gpu_tensor(W, "W", torch.bfloat16)
        N, K = W.shape
        Wq = torch.empty((N, K // 8), dtype=torch.int32, device=W.device)
        S = torch.empty((N, K // group), dtype=torch.bfloat16, device=W.device)
        W = W.contiguous()
        rc = self.lib.ns_w4_quantize(W.data_ptr(), Wq.data_ptr(), S.data_ptr(), N, K, group,
                                     self._stream())
        self._check(rc, "ns_w4_quantize")
        return Wq, S

    def w4_linear_swiglu(self, x, Wq, S, group=128, out=None):
        """x [M, K] bf16 -> [M, N // 2] bf16 = swiglu of x @ deq(Wq, S)^T whose rows are gate and
        up rows interleaved in blocks of 8 (``qwen.interleave_gate_up``): one launch, except for
        the M = 2..8 shapes whose GEMV has no SwiGLU output, which take two (not in the reference,
        whose MLP is swiglu(linear(h, "g"), linear(h, "u")), qwen.py:159)."""
        _require_gpu_tensor(x, "x", torch.bfloat16)
        _require_gpu_tensor(Wq, "Wq", torch.int32)
        _require_gpu_tensor(S, "S", torch.bfloat16)
        M, K = x.shape
        N = Wq.shape[0]
        if N % 16:
            raise ValueError("the interleaved gate/up matrix needs N % 16 == 0")
        I = N // 2
        if out is not None:
            _require_gpu_tensor(out, "out", torch.bfloat16)
            if tuple(out.shape) != (M, I) or not out.is_contiguous():
                raise ValueError(f"out must be a contiguous tensor of shape {(M, I)}")
        if M == 0:
            return out if out is not None else x.new_empty((0, I))
        # (names for the copies: an address whose copy is gone may already be another copy's)
        x, Wq, S = x.contiguous(), Wq.contiguous(), S.contiguous()
        if M > 8 and M % 128:
            x = _aligned_rows(x)
        n = int(self.lib.ns_w4_linear_swiglu_rows_workspace(M, N, K, group))
        # one launch reads x while it writes y: out may lie over x only through a tensor of its own
        # (M = 1 and multiples of 128 are the callers' to keep apart)
        y = out
        if out is None or (M > 1 and M % 128 and _overlap(out, x)):
            y = x.new_empty((M, I))
        tmp = torch.empty(n, dtype=torch.uint8, device=x.device) if n else None
        rc = self.lib.ns_w4_linear_swiglu_rows(
            x.data_ptr(), Wq.data_ptr(), S.data_ptr(), y.data_ptr(),
            None if tmp is None else tmp.data_ptr(), n, M, N, K, group, self._stream())
        self._check(rc, "ns_w4_linear_swiglu")
        return y if out is None or y is out else out.copy_(y)

    def w4_gptq(self, W, U, group=128):
        """Calibrated quantization (not in the reference, whose README.md:233-235 names it as
        the next step): W [N, K] (any float dtype) and U [K, K] fp32, the upper Cholesky factor
        of the layer's damped inverse Hessian (``nanoserve_amd.gptq.hessian_factor``) ->
        (Wq int32 [N, K // 8], S bf16 [N, K // group]) in w4_quantize's format. W is not
        modified (the kernels work on an fp32 copy; the workspace is the entry point's contract,
        they do not use it)."""
        if not isinstance(W, torch.Tensor) or not W.is_cuda:
            raise ValueError("W must be a CUDA (HIP) tensor")
        _require_gpu_tensor(U, "U", torch.float32)
        N, K = W.shape
        if tuple(U.shape) != (K, K):
            raise ValueError(f"U must be [{K}, {K}], got {tuple(U.shape)}")
        # one copy, always the kernels' own (they overwrite it)
        Wf = W.to(torch.float32, copy=True, memory_format=torch.contiguous_format)
        U = U.contiguous()
        Wq = torch.empty((N, K // 8), dtype=torch.int32, device=W.device)
        S = torch.empty((N, K // group), dtype=torch.bfloat16, device=W.device)
        nbytes = self.lib.ns_w4_gptq_workspace(N)
        work = torch.empty(max(nbytes, 16), dtype=torch.uint8, device=W.device)
        rc = self.lib.ns_w4_gptq(Wf.data_ptr(), U.data_ptr(), Wq.data_ptr(), S.data_ptr(),
                                 work.data_ptr(), work.numel(), N, K, group, self._stream())
        self._check(rc, "ns_w4_gptq")
        return Wq, S

    def w4_linear_workspace(self, M, N, K, group=128, device=None):
        """A uint8 device tensor of the workspace ``w4_linear(..., work=)`` uses for this shape
        (the K split of the M = 2..8 GEMV for K > 8192), or None when the shape needs none."""
        n = int(self.lib.ns_w4_linear_workspace(M, N, K, group))
        return torch.empty(n, dtype=torch.uint8, device=device or "cuda") if n else None

    def w4_linear(self, x, Wq, S, group=128, out=None, work=None):
        """x [M, K] bf16 -> y [M, N] bf16 = x @ deq(Wq, S)^T. Reference ops.py:85-97.

        Any M runs natively (the reference pads 3 -> 4 and 5..7 -> 8 with zero rows, and larger M
        up to a multiple of 128, which does not change any output row). ``out`` (not in the
        reference): a contiguous [M, N] bf16 tensor to write instead of a new one, for M <= 8 and
        multiples of 128 (the M the reference does not pad). ``work`` (not in the reference): a
        workspace from ``w4_linear_workspace``; with it the M = 2..8 GEMV may split long rows over
        K (ns_w4_linear_ws), without it no shape is split (ns_w4_linear)."""
        _require_gpu_tensor(x, "x", torch.bfloat16)
        _require_gpu_tensor(Wq, "Wq", torch.int32)
        _require_gpu_tensor(S, "S", torch.bfloat16)
        M, K = x.shape
        N = Wq.shape[0]
        padded = M > 8 and M % 128 != 0  # in the reference: ``out`` does not apply there
        if M == 0:
            x = x.new_zeros(1, K)
        x = x.contiguous()
        if padded:
            x = _aligned_rows(x)
        Wq = Wq.contiguous()
        S = S.contiguous()
        if out is not None:
            _require_gpu_tensor(out, "out", torch.bfloat16)
            if M == 0 or padded or tuple(out.shape) != (M, N) or not out.is_contiguous():
                raise ValueError(f"out must be a contiguous [{M}, {N}] tensor and M must need "
                                 "no padding")
            y = out
        else:
            y = x.new_empty((M or 1, N))
        if work is not None:
            _require_gpu_tensor(work, "work", torch.uint8)
            if not work.is_contiguous():
                raise _strided_work()
        if work is None or padded:
            rc = self.lib.ns_w4_linear_rows(x.data_ptr(), Wq.data_ptr(), S.data_ptr(), y.data_ptr(),
                                            max(M, 1), N, K, group, self._stream())
            self._check(rc, "ns_w4_linear")
        else:
            rc = self.lib.ns_w4_linear_ws(x.data_ptr(), Wq.data_ptr(), S.data_ptr(), y.data_ptr(),
                                          max(M, 1), N, K, group, work.data_ptr(), work.numel(),
                                          self._stream())
            self._check(rc, "ns_w4_linear_ws")
        return y if M else y[:0]

    # ------------------------------------------------------------------ decoder-step operators
    def rmsnorm(self, x, r, w, eps, out=None):
        """x [T, H] residual stream, updated in place to x + r when r is given; returns
        rmsnorm(x) * w. Reference ops.py:41-48 (kernel: kernels/fused/rmsnorm.cuh:10-52).
        ``out`` (not in the reference): a contiguous tensor like x to write the result to."""
        _require_gpu_tensor(x, "x", torch.bfloat16)
        _require_gpu_tensor(w, "w", torch.bfloat16)
        if not x.is_contiguous():
            raise ValueError("x must be contiguous (it is updated in place)")
        if r is not None:
            _require_gpu_tensor(r, "r", torch.bfloat16)
            r = r.contiguous()
        w = w.contiguous()
        y = torch.empty_like(x) if out is None else _check_out(out, x)
        rc = self.lib.ns_rmsnorm(x.data_ptr(), None if r is None else r.data_ptr(), w.data_ptr(),
                                 y.data_ptr(), x.shape[0], x.shape[1], eps, self._stream())
        self._check(rc, "ns_rmsnorm")
        return y

    def rope(self, q, k, inv_freq, n_heads, n_kv_heads, head_dim, pos0):
        """In place on q [T, Hq*D] and k [T, Hk*D] (row stride may exceed Hq*D / Hk*D).
        Reference ops.py:50-54 (kernel: kernels/fused/rope.cuh:14-46)."""
        _require_gpu_tensor(q, "q", torch.bfloat16)
        _require_gpu_tensor(k, "k", torch.bfloat16)
        _require_gpu_tensor(inv_freq, "inv_freq", torch.float32)
        for t, n in ((q, "q"), (k, "k")):
            if t.stride(-1) != 1:
                raise ValueError(f"{n} rows must be contiguous")
        inv_freq = inv_freq.contiguous()
        rc = self.lib.ns_rope(q.data_ptr(), k.data_ptr(), inv_freq.data_ptr(), q.shape[0], n_heads,
                              n_kv_heads, head_dim, pos0, q.stride(0), k.stride(0), self._stream())
        self._check(rc, "ns_rope")

    def swiglu(self, gate, up, out=None):
        """silu(gate) * up, gate and up contiguous [T, I]. Reference ops.py:56-62 (kernel:
        kernels/fused/swiglu.cuh:35-52). ``out`` (not in the reference): a contiguous tensor
        like gate to write the result to."""
        _require_gpu_tensor(gate, "gate", torch.bfloat16)
        _require_gpu_tensor(up, "up", torch.bfloat16)
        if not (gate.is_contiguous() and up.is_contiguous()):
            raise ValueError("gate and up must be contiguous")
        out = torch.empty_like(gate) if out is None else _check_out(out, gate)
        rc = self.lib.ns_swiglu(gate.data_ptr(), up.data_ptr(), out.data_ptr(), gate.shape[0],
                                gate.shape[1], self._stream())
        self._check(rc, "ns_swiglu")
        return out

    def decode_qkv(self, qkv, bias, inv_freq, pos, k_cache, v_cache, n_heads, n_kv_heads,
                   head_dim):
        """One decode token: bias add + RoPE at position pos[0] (device int32) in place on the
        fused projection output qkv [(Hq + 2Hk) * D], and the k / v heads appended to one
        layer's cache slices k_cache / v_cache [Hk, max_len, D]. The reference does these
        steps with PyTorch ops (qwen.py:119-122, 147-151)."""
        _require_gpu_tensor(qkv, "qkv", torch.bfloat16)
        _require_gpu_tensor(inv_freq, "inv_freq", torch.float32)
        _require_gpu_tensor(pos, "pos", torch.int32)
        for t, n in ((k_cache, "k_cache"), (v_cache, "v_cache")):
            _require_gpu_tensor(t, n, torch.bfloat16)
            if not t.is_contiguous():
                raise ValueError(f"{n} must be contiguous")
        if bias is not None:
            _require_gpu_tensor(bias, "bias", torch.bfloat16)
        if not qkv.is_contiguous():
            raise ValueError("qkv must be contiguous")
        rc = self.lib.ns_decode_qkv(qkv.data_ptr(), None if bias is None else bias.data_ptr(),
                                    inv_freq.data_ptr(), pos.data_ptr(), k_cache.data_ptr(),
                                    v_cache.data_ptr(), n_heads, n_kv_heads, head_dim,
                                    k_cache.shape[-2], self._stream())
        self._check(rc, "ns_decode_qkv")

    def decode_attention_workspace(self, n_heads, n_kv_heads, head_dim, max_len, device=None):
        """A uint8 device tensor of the workspace decode_attention and decode_qkv_attention
        need (per-split partial results). Launches that may overlap in time need workspaces of
        their own."""
        n = int(self.lib.ns_decode_attention_workspace(n_heads, n_kv_heads, head_dim, max_len))
        if n == 0:
            raise ValueError("unsupported attention sizes (head_dim must be 128)")
        return torch.zeros(n, dtype=torch.uint8, device=device or "cuda")

    def decode_attention(self, q, k_cache, v_cache, pos, n_heads, n_kv_heads, head_dim,
                         work, out=None):
        """Attention of one query token q [Hq * D] over cache rows 0 .. pos[0] of one layer's
        k_cache / v_cache [Hk, max_len, D]; returns out [1, Hq * D] bf16. The reference uses
        PyTorch SDPA for this (qwen.py:124-133). work: from decode_attention_workspace."""
        _require_gpu_tensor(q, "q", torch.bfloat16)
        _require_gpu_tensor(pos, "pos", torch.int32)
        _require_gpu_tensor(work, "work", torch.uint8)
        if not work.is_contiguous():
            raise _strided_work()
        if out is None:
            out = torch.empty((1, n_heads * head_dim), dtype=torch.bfloat16, device=q.device)
        rc = self.lib.ns_decode_attention(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                                          pos.data_ptr(), out.data_ptr(), work.data_ptr(),
                                          work.numel(), n_heads, n_kv_heads, head_dim,
                                          k_cache.shape[-2], self._stream())
        self._check(rc, "ns_decode_attention")
        return out

    def decode_attention_noalloc(self, q, k_cache, v_cache, pos, n_heads, n_kv_heads, head_dim,
                                 out):
        """decode_attention without a workspace, for callers that cannot allocate: the partials
        go to the library's per-GPU scratch (include/nanoserve_decode.h), so calls that overlap
        on one GPU race. ``out`` [1, Hq * D] bf16 is required (nothing is allocated here)."""
        _require_gpu_tensor(q, "q", torch.bfloat16)
        _require_gpu_tensor(pos, "pos", torch.int32)
        _require_gpu_tensor(out, "out", torch.bfloat16)
        rc = self.lib.ns_decode_attention_noalloc(q.data_ptr(), k_cache.data_ptr(),
                                                  v_cache.data_ptr(), pos.data_ptr(),
                                                  out.data_ptr(), n_heads, n_kv_heads, head_dim,
                                                  k_cache.shape[-2], self._stream())
        self._check(rc, "ns_decode_attention_noalloc")
        return out

    def decode_qkv_attention(self, qkv, bias, inv_freq, pos, k_cache, v_cache, n_heads,
                             n_kv_heads, head_dim, work, out=None, merge=True, rot=None):
        """decode_qkv followed by decode_attention in one launch, qkv left unchanged: bias +
        RoPE of the q heads, the token's k / v row appended to the cache at pos[0], attention
        over rows 0 .. pos[0]. Returns out [1, Hq * D] bf16. With ``merge=False`` the split
        partials stay in ``work`` for gemv_decode_attn (out is written only for one split).
        ``rot``: the step's rotation table from ``decode_embed`` (same outputs, fewer
        instructions per workgroup)."""
        _require_gpu_tensor(qkv, "qkv", torch.bfloat16)
        _require_gpu_tensor(inv_freq, "inv_freq", torch.float32)
        _require_gpu_tensor(pos, "pos", torch.int32)
        _require_gpu_tensor(work, "work", torch.uint8)
        if not work.is_contiguous():
            raise _strided_work()
        for t, n in ((k_cache, "k_cache"), (v_cache, "v_cache")):
            _require_gpu_tensor(t, n, torch.bfloat16)
            if not t.is_contiguous():
                raise ValueError(f"{n} must be contiguous")
        if bias is not None:
            _require_gpu_tensor(bias, "bias", torch.bfloat16)
        if not qkv.is_contiguous():
            raise ValueError("qkv must be contiguous")
        if out is None:
            out = torch.empty((1, n_heads * head_dim), dtype=torch.bfloat16, device=qkv.device)
        rc = self.lib.ns_decode_qkv_attention(
            qkv.data_ptr(), None if bias is None else bias.data_ptr(), inv_freq.data_ptr(),
            pos.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), out.data_ptr(),
            work.data_ptr(), work.numel(), n_heads, n_kv_heads, head_dim, k_cache.shape[-2],
            1 if merge else 0, None if rot is None else _rot_ptr(rot, head_dim), self._stream())
        self._check(rc, "ns_decode_qkv_attention")
        return out

    def decode_embed(self, tok, pos, embed, inv_freq, x=None, rot=None):
        """Start of a decode step (no counterpart in the reference, whose runner gathers the
        row with F.embedding, qwen.py:141): x [1, H] = embed[tok[0]] (zeros for an id outside
        the table) and rot [2, D/2] fp32 = cos, sin of pos[0] * inv_freq, the table
        decode_qkv_attention takes. Returns (x, rot)."""
        _require_gpu_tensor(tok, "tok", torch.int32)
        _require_gpu_tensor(pos, "pos", torch.int32)
        _require_gpu_tensor(embed, "embed", torch.bfloat16)
        _require_gpu_tensor(inv_freq, "inv_freq", torch.float32)
        if not embed.is_contiguous() or embed.dim() != 2:
            raise ValueError("embed must be a contiguous [vocab, H] tensor")
        vocab, H = embed.shape
        D = 2 * inv_freq.numel()
        if x is None:
            x = torch.empty((1, H), dtype=torch.bfloat16, device=embed.device)
        if rot is None:
            rot = torch.empty((2, D // 2), dtype=torch.float32, device=embed.device)
        rc = self.lib.ns_decode_embed(tok.data_ptr(), pos.data_ptr(), embed.data_ptr(), vocab, H,
                                      inv_freq.data_ptr(), D, x.data_ptr(), _rot_ptr(rot, D),
                                      self._stream())
        self._check(rc, "ns_decode_embed")
        return x, rot

    def gemv_decode_attn(self, attn_out, work, pos, max_len, n_heads, Wq, S, group=128,
                         out=None):
        """y [1, N] = a . deq(Wq, S)^T where a is the output of a preceding
        decode_qkv_attention(..., merge=False) with the same work, pos, max_len and heads: its
        split partials are merged while the activation is loaded."""
        _require_gpu_tensor(attn_out, "attn_out", torch.bfloat16)
        _require_gpu_tensor(work, "work", torch.uint8)
        if not work.is_contiguous():
            raise _strided_work()
        _require_gpu_tensor(pos, "pos", torch.int32)
        _require_gpu_tensor(Wq, "Wq", torch.int32)
        _require_gpu_tensor(S, "S", torch.bfloat16)
        N, K = Wq.shape[0], Wq.shape[1] * 8
        if out is None:
            out = torch.empty((1, N), dtype=torch.bfloat16, device=Wq.device)
        rc = self.lib.ns_w4_gemv_decode_attn(attn_out.data_ptr(), work.data_ptr(),
                                             pos.data_ptr(), max_len, n_heads, Wq.data_ptr(),
                                             S.data_ptr(), out.data_ptr(), N, K, group,
                                             self._stream())
        self._check(rc, "ns_w4_gemv_decode_attn")
        return out

    def gemv_decode(self, Wq, S, group=128, x=None, res=None, r=None, norm_w=None, eps=1e-6,
                    res_out=None, swiglu=False, out=None):
        """One-token W4 GEMV with its neighbours fused (no reference counterpart; its runner
        launches them separately, qwen.py:145-162). Activation: x [K] / [1, K], or, with res,
        rmsnorm(res + r) * norm_w (res_out receives bf16(res + r)). Output: y [1, N], or with
        ``swiglu`` (gate/up rows interleaved in blocks of 8) silu(gate) * up [1, N/2]."""
        for t, n in ((Wq, "Wq"), (S, "S")):
            _require_gpu_tensor(t, n, torch.int32 if n == "Wq" else torch.bfloat16)
            if not t.is_contiguous():
                raise ValueError(f"{n} must be contiguous")
        N, K = Wq.shape[0], Wq.shape[1] * 8
        vecs = {"x": x, "res": res, "r": r, "norm_w": norm_w, "res_out": res_out}
        for n, t in vecs.items():
            if t is not None:
                _require_gpu_tensor(t, n, torch.bfloat16)
                if t.numel() != K or not t.is_contiguous():
                    raise ValueError(f"{n} must be a contiguous tensor of {K} elements")
        n_out = N // 2 if swiglu else N
        if out is None:
            out = torch.empty((1, n_out), dtype=torch.bfloat16, device=Wq.device)
        elif out.numel() != n_out or not out.is_contiguous() or out.dtype != torch.bfloat16:
            raise ValueError(f"out must be a contiguous bf16 tensor of {n_out} elements")

        def ptr(t):
            return None if t is None else t.data_ptr()

        rc = self.lib.ns_w4_gemv_decode(ptr(x), ptr(res), ptr(r), ptr(norm_w), eps, ptr(res_out),
                                        Wq.data_ptr(), S.data_ptr(), out.data_ptr(), N, K, group,
                                        1 if swiglu else 0, self._stream())
        self._check(rc, "ns_w4_gemv_decode")
        return out

    def bf16_gemv(self, W, x=None, res=None, r=None, norm_w=None, eps=1e-6, out=None):
        """One-token bf16 product y [1, N] = a . W^T (W [N, K] bf16), the reference's lm_head
        F.linear (qwen.py:164); a is x, or with res the fused rmsnorm(res + r) * norm_w."""
        _require_gpu_tensor(W, "W", torch.bfloat16)
        if not W.is_contiguous():
            raise ValueError("W must be contiguous")
        N, K = W.shape
        for n, t in (("x", x), ("res", res), ("r", r), ("norm_w", norm_w)):
            if t is not None:
                _require_gpu_tensor(t, n, torch.bfloat16)
                if t.numel() != K or not t.is_contiguous():
                    raise ValueError(f"{n} must be a contiguous tensor of {K} elements")
        if out is None:
            out = torch.empty((1, N), dtype=torch.bfloat16, device=W.device)

        def ptr(t):
            return None if t is None else t.data_ptr()

        rc = self.lib.ns_bf16_gemv(ptr(x), ptr(res), ptr(r), ptr(norm_w), eps, W.data_ptr(),
                                   out.data_ptr(), N, K, self._stream())
        self._check(rc, "ns_bf16_gemv")
        return out

    # ------------------------------------------------------------------ prompt-pass attention
    def prompt_qkv(self, qkv, bias, inv_freq, n_heads, n_kv_heads, head_dim, pos0, k_cache=None,
                   v_cache=None):
        """T prompt tokens at positions pos0 ..: bias add + RoPE of the fused projection output
        qkv [T, (Hq + 2Hk) * D], q heads in place, k and v heads into rows pos0 .. of one layer's
        k_cache / v_cache [Hk, max_len, D], or in place without them (csrc/internal_ops.h). The
        reference does this with PyTorch ops and ns_rope (qwen.py:119-122, 147-151)."""
        _require_gpu_tensor(qkv, "qkv", torch.bfloat16)
        _require_gpu_tensor(inv_freq, "inv_freq", torch.float32)
        if qkv.dim() != 2 or not qkv.is_contiguous() or (
                qkv.shape[1] != (n_heads + 2 * n_kv_heads) * head_dim):
            raise ValueError("qkv must be a contiguous [T, (Hq + 2Hk) * D] tensor")
        if inv_freq.numel() != head_dim // 2 or not inv_freq.is_contiguous():
            raise ValueError("inv_freq must be contiguous with head_dim / 2 elements")
        if bias is not None:
            _require_gpu_tensor(bias, "bias", torch.bfloat16)
            if bias.numel() != qkv.shape[1] or not bias.is_contiguous():
                raise ValueError("bias must be contiguous with one value per column of qkv")
        for t, n in ((k_cache, "k_cache"), (v_cache, "v_cache")):
            if t is not None:
                _require_gpu_tensor(t, n, torch.bfloat16)
                if not t.is_contiguous() or t.shape[0] != n_kv_heads or t.shape[2] != head_dim:
                    raise ValueError(f"{n} must be a contiguous [Hk, max_len, D] tensor")
        if k_cache is not None and v_cache is not None and k_cache.shape != v_cache.shape:
            raise ValueError("k_cache and v_cache must have the same shape")

        def ptr(t):
            return None if t is None else t.data_ptr()

        rc = self.lib.ns_prompt_qkv(qkv.data_ptr(), ptr(bias), inv_freq.data_ptr(), ptr(k_cache),
                                    ptr(v_cache), qkv.shape[0], n_heads, n_kv_heads, head_dim,
                                    pos0, 0 if k_cache is None else k_cache.shape[1],
                                    self._stream())
        self._check(rc, "ns_prompt_qkv")

    def prompt_attention_fits(self, T, n_heads, n_kv_heads, pos0, kv_stride):
        """Whether prompt_attention takes these sizes with keys kv_stride elements apart."""
        return bool(self.lib.ns_prompt_attention_fits(T, n_heads, n_kv_heads, pos0, kv_stride))

    def prompt_attention_workspace(self, T, n_heads, n_kv_heads, pos0, device=None):
        """A uint8 device tensor of the workspace prompt_attention uses for these sizes, or None.
        Launches that may overlap in time need workspaces of their own."""
        n = int(self.lib.ns_prompt_attention_workspace(T, n_heads, n_kv_heads, pos0))
        return torch.empty(n, dtype=torch.uint8, device=device or "cuda") if n else None

    def prompt_attention(self, q, k, v, n_heads, pos0, work=None, out=None):
        """Causal grouped-query attention, head size 128: q [T, >= Hq * 128] (rows may be strided)
        at positions pos0 .. pos0 + T - 1 over k, v [Hk, >= pos0 + T, 128] (the same strides, last
        dimension contiguous: a layer's cache, or heads of the projection's rows); returns
        [T, Hq * 128] bf16. Reference: PyTorch SDPA (qwen.py:124-133)."""
        for t, n in ((q, "q"), (k, "k"), (v, "v")):
            _require_gpu_tensor(t, n, torch.bfloat16)
        T, Hk = q.shape[0], k.shape[0]
        if q.stride(1) != 1 or q.shape[1] < n_heads * 128:
            raise ValueError("q rows must be contiguous and hold n_heads * 128 values")
        if k.shape != v.shape or k.stride() != v.stride() or k.shape[2] != 128 or k.stride(2) != 1:
            raise ValueError("k and v must be alike, with contiguous rows of 128 values")
        if k.shape[1] < pos0 + T:
            raise ValueError(f"k and v must hold {pos0 + T} rows")
        if out is None:
            out = torch.empty((T, n_heads * 128), dtype=torch.bfloat16, device=q.device)
        else:
            _require_gpu_tensor(out, "out", torch.bfloat16)
            if tuple(out.shape) != (T, n_heads * 128) or not out.is_contiguous():
                raise ValueError(f"out must be a contiguous [{T}, {n_heads * 128}] tensor")
        if work is not None and not work.is_contiguous():
            raise _strided_work()
        rc = self.lib.ns_prompt_attention(
            q.data_ptr(), q.stride(0), k.data_ptr(), v.data_ptr(), k.stride(1), k.stride(0),
            out.data_ptr(), None if work is None else work.data_ptr(),
            0 if work is None else work.numel(), T, n_heads, Hk, pos0, self._stream())
        self._check(rc, "ns_prompt_attention")
        return out

    # ------------------------------------------------------------------ a batch over a paged cache
    @staticmethod
    def _batch_args(T, pages, lens, k_pages, v_pages, q_start, here, dtype=torch.bfloat16):
        """Checks of a batch's metadata and pools; returns them as the C entry points take them."""
        _require_here(pages, "pages", torch.int32, here)
        _require_here(lens, "lens", torch.int32, here)
        _require_here(k_pages, "k_pages", dtype, here)
        _require_here(v_pages, "v_pages", dtype, here)
        # (shapes and strides are read once: 0.2 us each, beside a launch of 4)
        shape, strides = k_pages.shape, k_pages.stride()
        if len(shape) != 4 or strides[3] != 1 or strides[2] != shape[3]:
            raise ValueError("k_pages must be [n_pages, Hk, page_size, D] with contiguous heads")
        if v_pages.shape != shape or v_pages.stride() != strides:
            raise ValueError("k_pages and v_pages must be alike")
        rows, steps = pages.shape, pages.stride()
        if lens.dim() != 1 or not lens.is_contiguous():
            raise ValueError("lens must be a contiguous [B] tensor")
        B = lens.numel()
        if len(rows) != 2 or rows[0] != B or steps[1] != 1:
            raise ValueError("pages must be [B, width] with contiguous rows")
        if q_start is None:
            if T != B:
                raise ValueError("without q_start every sequence has one token row")
        else:
            _require_here(q_start, "q_start", torch.int32, here)
            if q_start.dim() != 1 or q_start.shape[0] != B + 1 or not q_start.is_contiguous():
                raise ValueError("q_start must be a contiguous [B + 1] tensor")
        n_pages, Hk, page_size, D = shape
        width = rows[1]
        # (the stride of a dimension of size 1 says nothing)
        return (B, Hk, D, page_size, n_pages,
                (strides[0] if n_pages > 1 else 0, strides[1] if Hk > 1 else 0),
                (pages.data_ptr(), steps[0] if B > 1 else width, width))

    def paged_append(self, qkv, bias, inv_freq, pages, lens, k_pages, v_pages, n_heads, q_start=None,
                     out=None):
        """The new tokens of a batch of sequences: bias add and RoPE of the fused projection output
        qkv [T, (Hq + 2Hk) * D] (rows any multiple of 8 elements apart), k and v heads into the paged
        cache; returns the q heads [T, Hq * D].

        k_pages, v_pages [n_pages, Hk, page_size, D] (page_size a multiple of 16, heads contiguous,
        e.g. one layer of a larger pool), pages [B, width] int32: the pages of each sequence's
        positions 0 .. page_size - 1, page_size .. and so on. Token rows q_start[b] .. q_start[b + 1] - 1
        (int32 [B + 1], ascending; without it one row per sequence) are sequence b's, at its last
        positions: lens [B] int32 counts them. All of it is read on the device, so a captured graph
        replays at any lengths. Rows past the last sequence's are left alone, tokens whose page is
        outside the pool are not stored. Angles are position * inv_freq in float64, and a value is
        rounded once. The reference serves one sequence at a time (qwen.py:113-122)."""
        here = _device_of(qkv, "qkv", torch.bfloat16)
        _require_here(inv_freq, "inv_freq", torch.float32, here)
        if qkv.dim() != 2 or qkv.stride(1) != 1:
            raise ValueError("qkv must be [T, (Hq + 2Hk) * D] with contiguous rows")
        T, columns = qkv.shape
        B, Hk, D, page_size, n_pages, strides, table = self._batch_args(T, pages, lens, k_pages, v_pages,
                                                                        q_start, here)
        if columns != (n_heads + 2 * Hk) * D:
            raise ValueError("qkv must hold n_heads + 2 Hk heads of D values per row")
        if inv_freq.numel() != D // 2 or not inv_freq.is_contiguous():
            raise ValueError("inv_freq must be contiguous with head_dim / 2 elements")
        if bias is not None:
            _require_here(bias, "bias", torch.bfloat16, here)
            if bias.numel() != columns or not bias.is_contiguous():
                raise ValueError("bias must be contiguous with one value per column of qkv")
        if out is None:
            out = qkv.new_empty((T, n_heads * D))
        else:
            _require_here(out, "out", torch.bfloat16, here)
            if tuple(out.shape) != (T, n_heads * D) or not out.is_contiguous():
                raise ValueError(f"out must be a contiguous [{T}, {n_heads * D}] tensor")
            _apart(out, qkv, "qkv")
        if T == 0 or B == 0:
            return out
        rc = self.lib.ns_paged_append(
            qkv.data_ptr(), qkv.stride(0) if T > 1 else columns,
            None if bias is None else bias.data_ptr(), inv_freq.data_ptr(),
            None if q_start is None else q_start.data_ptr(), lens.data_ptr(), *table, k_pages.data_ptr(),
            v_pages.data_ptr(), *strides, n_pages, page_size, out.data_ptr(), T, B, n_heads, Hk, D,
            _raw_stream(here))
        self._check(rc, "ns_paged_append")
        return out

    def paged_attention_workspace(self, T, B, n_heads, n_kv_heads, head_dim, max_len, ragged=False,
                                  shared=0, device=None):
        """A uint8 device tensor of the workspace paged_attention uses for these sizes (max_len: table
        width * page_size; ragged: with q_start), or None. Launches that may overlap in time need
        workspaces of their own."""
        n = int(self.lib.ns_paged_attention_workspace(T, B, n_heads, n_kv_heads, head_dim, _int32(max_len),
                                                      int(ragged), _int32(shared)))
        return torch.empty(n, dtype=torch.uint8, device=device or "cuda") if n else None

    def paged_attention(self, q, k_pages, v_pages, pages, lens, n_heads, q_start=None, shared=0,
                        window=0, sinks=0, scale=None, work=None, out=None):
        """Causal grouped-query attention of a batch's new tokens over its paged cache, their own keys
        and values included (paged_append first; pages, lens and q_start as there): q [T, Hq * D]
        (rows any multiple of 8 elements apart), head size 64 or 128; returns [T, Hq * D] bf16.

        With ``window`` a token sees the last ``window`` positions (its own among them) and the first
        ``sinks`` ones. ``shared``: the first ``shared`` positions, as far as a sequence has them, lie in
        the same pages for every sequence (the caller's statement); their keys and values are then read
        once for the whole batch. A token that sees nothing gets zeros, one whose query or seen keys hold
        NaN gets NaN; rows past the last sequence's are left alone. ``scale`` (default 1 / sqrt(D)) must be
        positive. ``work``: from paged_attention_workspace, allocated here when it is not given. The
        reference has SDPA over one sequence's cache (qwen.py:124-133)."""
        here = _device_of(q, "q", torch.bfloat16)
        if q.dim() != 2 or q.stride(1) != 1:
            raise ValueError("q must be [T, Hq * D] with contiguous rows")
        T, columns = q.shape
        B, Hk, D, page_size, n_pages, strides, table = self._batch_args(T, pages, lens, k_pages, v_pages,
                                                                        q_start, here)
        if columns != n_heads * D:
            raise ValueError("q must hold n_heads heads of D values per row")
        if out is None:
            out = q.new_empty((T, columns))
        else:
            _require_here(out, "out", torch.bfloat16, here)
            if tuple(out.shape) != (T, columns) or not out.is_contiguous():
                raise ValueError(f"out must be a contiguous [{T}, {columns}] tensor")
            _apart(out, q, "q")
        if T == 0 or B == 0:
            return out
        if (shared | window | sinks) >> 31:  # one below 0 or past 32 bits
            shared, window, sinks = _int32(shared), _int32(window), _int32(sinks)
        if work is None:
            work = self.paged_attention_workspace(T, B, n_heads, Hk, D, table[2] * page_size,
                                                  q_start is not None, shared, device=q.device)
        else:
            _require_here(work, "work", torch.uint8, here)
            if not work.is_contiguous():
                raise _strided_work()
        rc = self.lib.ns_paged_attention(
            q.data_ptr(), q.stride(0) if T > 1 else columns, k_pages.data_ptr(), v_pages.data_ptr(),
            *strides, n_pages, page_size, *table, lens.data_ptr(),
            None if q_start is None else q_start.data_ptr(), out.data_ptr(),
            None if work is None else work.data_ptr(), 0 if work is None else work.numel(), T, B, n_heads,
            Hk, D, shared, window, sinks, D ** -0.5 if scale is None else scale, _raw_stream(here))
        self._check(rc, "ns_paged_attention")
        return out

    @staticmethod
    def _scale_args(k_scales, v_scales, n_pages, Hk, page_size, here):
        """Checks of the scales of a cache in 8 bits; returns them as the C entry points take them."""
        _require_here(k_scales, "k_scales", torch.float8_e8m0fnu, here)
        _require_here(v_scales, "v_scales", torch.float8_e8m0fnu, here)
        blocks = page_size // 16
        strides = k_scales.stride()
        if k_scales.shape != (n_pages, Hk, blocks) or (blocks > 1 and strides[2] != 1):
            raise ValueError("k_scales must be [n_pages, Hk, page_size / 16] with contiguous heads")
        if v_scales.shape != k_scales.shape or v_scales.stride() != strides:
            raise ValueError("k_scales and v_scales must be alike")
        return (k_scales.data_ptr(), v_scales.data_ptr(), strides[0] if n_pages > 1 else 0,
                strides[1] if Hk > 1 else 0)

    def paged_append_fp8(self, qkv, bias, inv_freq, pages, lens, k_pages, v_pages, k_scales, v_scales, n_heads,
                         q_start=None, out=None):
        """paged_append to a cache in 8 bits: k_pages, v_pages [n_pages, Hk, page_size, D] float8_e4m3fn (head
        size 64 or 128), k_scales, v_scales [n_pages, Hk, page_size / 16] float8_e8m0fnu, one power of two for each
        16 positions and kv head; a value is its code times its scale. Returns the q heads [T, Hq * D], bf16.

        The scale is the least with which the block's largest magnitude fits (448 of it), in 2^-110 .. 2^119; with rows of
        the block from before it rises where new ones need it and never falls, and their codes are rounded to the new
        scale (for most values exact: the exponent moves). A block of which no earlier position is the sequence's
        starts anew, whatever its scale held. NaN and infinities are stored as NaN and do not count for the scale.
        Everything else as paged_append; rows of the pages that no new token writes keep their values."""
        here = _device_of(qkv, "qkv", torch.bfloat16)
        _require_here(inv_freq, "inv_freq", torch.float32, here)
        shape, steps = qkv.shape, qkv.stride()
        if len(shape) != 2 or steps[1] != 1:
            raise ValueError("qkv must be [T, (Hq + 2Hk) * D] with contiguous rows")
        T, columns = shape
        B, Hk, D, page_size, n_pages, strides, table = self._batch_args(T, pages, lens, k_pages, v_pages,
                                                                        q_start, here, torch.float8_e4m3fn)
        scales = self._scale_args(k_scales, v_scales, n_pages, Hk, page_size, here)
        if columns != (n_heads + 2 * Hk) * D:
            raise ValueError("qkv must hold n_heads + 2 Hk heads of D values per row")
        if inv_freq.numel() != D // 2 or not inv_freq.is_contiguous():
            raise ValueError("inv_freq must be contiguous with head_dim / 2 elements")
        if bias is not None:
            _require_here(bias, "bias", torch.bfloat16, here)
            if bias.numel() != columns or not bias.is_contiguous():
                raise ValueError("bias must be contiguous with one value per column of qkv")
        if out is None:
            out = qkv.new_empty((T, n_heads * D))
        else:
            _require_here(out, "out", torch.bfloat16, here)
            if out.shape != (T, n_heads * D) or not out.is_contiguous():
                raise ValueError(f"out must be a contiguous [{T}, {n_heads * D}] tensor")
        if T == 0 or B == 0:
            return out
        rc = self.lib.ns_paged_append_fp8(
            qkv.data_ptr(), steps[0] if T > 1 else columns,
            None if bias is None else bias.data_ptr(), inv_freq.data_ptr(),
            None if q_start is None else q_start.data_ptr(), lens.data_ptr(), *table, k_pages.data_ptr(),
            v_pages.data_ptr(), *strides, *scales, n_pages, page_size, out.data_ptr(), T, B, n_heads, Hk, D,
            _raw_stream(here))
        if rc:
            _apart(out, qkv, "qkv")  # (says so; the library has refused it)
            self._check(rc, "ns_paged_append_fp8")
        return out

    def paged_attention_fp8_workspace(self, T, B, n_heads, n_kv_heads, head_dim, max_len, ragged=False,
                                      shared=0, device=None):
        """paged_attention_workspace for paged_attention_fp8."""
        n = int(self.lib.ns_paged_attention_fp8_workspace(T, B, n_heads, n_kv_heads, head_dim, _int32(max_len),
                                                          int(ragged), _int32(shared)))
        return torch.empty(n, dtype=torch.uint8, device=device or "cuda") if n else None

    def paged_attention_fp8(self, q, k_pages, v_pages, k_scales, v_scales, pages, lens, n_heads, q_start=None,
                            shared=0, window=0, sinks=0, scale=None, work=None, out=None):
        """paged_attention over a cache in 8 bits (pools and scales as paged_append_fp8 writes them): the result of
        paged_attention over a bf16 cache that holds code times scale, but for infinities in a query, which count as NaN,
        query magnitudes above 448 * 2^119, which are held to it, and those below 2^-14 of their head's largest, which are
        held to 2^-22 of it. ``work``: from paged_attention_fp8_workspace."""
        here = _device_of(q, "q", torch.bfloat16)
        shape, steps = q.shape, q.stride()
        if len(shape) != 2 or steps[1] != 1:
            raise ValueError("q must be [T, Hq * D] with contiguous rows")
        T, columns = shape
        B, Hk, D, page_size, n_pages, strides, table = self._batch_args(T, pages, lens, k_pages, v_pages,
                                                                        q_start, here, torch.float8_e4m3fn)
        scales = self._scale_args(k_scales, v_scales, n_pages, Hk, page_size, here)
        if columns != n_heads * D:
            raise ValueError("q must hold n_heads heads of D values per row")
        if out is None:
            out = q.new_empty((T, columns))
        else:
            _require_here(out, "out", torch.bfloat16, here)
            if out.shape != (T, columns) or not out.is_contiguous():
                raise ValueError(f"out must be a contiguous [{T}, {columns}] tensor")
        if T == 0 or B == 0:
            return out
        if (shared | window | sinks) >> 31:  # one below 0 or past 32 bits
            shared, window, sinks = _int32(shared), _int32(window), _int32(sinks)
        if work is None:
            work = self.paged_attention_fp8_workspace(T, B, n_heads, Hk, D, table[2] * page_size,
                                                      q_start is not None, shared, device=q.device)
        else:
            _require_here(work, "work", torch.uint8, here)
            if not work.is_contiguous():
                raise _strided_work()
        rc = self.lib.ns_paged_attention_fp8(
            q.data_ptr(), steps[0] if T > 1 else columns, k_pages.data_ptr(), v_pages.data_ptr(),
            *strides, *scales, n_pages, page_size, *table, lens.data_ptr(),
            None if q_start is None else q_start.data_ptr(), out.data_ptr(),
            None if work is None else work.data_ptr(), 0 if work is None else work.numel(), T, B, n_heads,
            Hk, D, shared, window, sinks, D ** -0.5 if scale is None else scale, _raw_stream(here))
        if rc:
            _apart(out, q, "q")
            self._check(rc, "ns_paged_attention_fp8")
        return out

    def paged_reserve(self, new, lens, pages, free, n_free, page_size, rows=None, out=None):
        """Room for a step's tokens, on the device: sequence b gets new[b] more positions (int32 [B]; below 0: gives
        back as many). lens [B] and pages [B, width] (int32, as paged_append reads them), the stack of free pages free
        [capacity] and its height n_free [1] are changed in place: pages of sequences that shrink are pushed, those that
        growing ones need are popped, in the order of the sequences. Returns (q_start [B + 1], slots, short [1]):
        the first token row of each sequence, and with ``rows`` an int64 [rows] map of every new token to page * page_size +
        its row there (an index into a pool's positions; -1 for rows behind the last sequence's). ``out``: the three of
        them (slots None without ``rows``), for a captured step.

        The call goes through as a whole or changes nothing: then q_start is 0 throughout, so that the operators that
        it is handed on to have no rows to work on (without it they take the last position for a new one), and short[0] is the number of pages that were missing, or -1 where a sequence
        would pass its table row, more tokens are new than rows, or the stack would pass its capacity; else 0. A later
        call that gives back what this one took restores the stack as it was. Pages that another sequence still
        reads (a shared prefix, beams) must not be given back. The reference keeps one sequence in one cache
        (qwen.py:103-111)."""
        here = _device_of(new, "new", torch.int32)
        _require_here(lens, "lens", torch.int32, here)
        _require_here(pages, "pages", torch.int32, here)
        _require_here(free, "free", torch.int32, here)
        _require_here(n_free, "n_free", torch.int32, here)
        shape = new.shape
        if len(shape) != 1 or not new.is_contiguous():
            raise ValueError("new must be a contiguous [B] tensor")
        B = shape[0]
        if lens.shape != shape or not lens.is_contiguous():
            raise ValueError(f"lens must be a contiguous [{B}] tensor")
        shape, strides = pages.shape, pages.stride()
        if len(shape) != 2 or shape[0] != B or strides[1] != 1:
            raise ValueError("pages must be [B, width] with contiguous rows")
        width = shape[1]
        if free.dim() != 1 or not free.is_contiguous() or n_free.numel() != 1:
            raise ValueError("free must be a contiguous [capacity] tensor and n_free hold one value")
        if rows is not None and rows >> 31:  # below 0 or past the library's 32 bits
            raise ValueError("rows must be within 0 .. 2^31 - 1")
        if (page_size | width) >> 31:
            raise ValueError("page_size and the width of pages must be within 32 bits")
        if B == 0:
            raise ValueError("the batch has no sequence")
        if out is None:
            q_start, short = new.new_empty(B + 1), new.new_empty(1)
            slots = None if rows is None else new.new_empty(rows, dtype=torch.int64)
            out = (q_start, slots, short)
        else:
            q_start, slots, short = out
            _require_here(q_start, "q_start", torch.int32, here)
            _require_here(short, "short", torch.int32, here)
            if q_start.shape != (B + 1,) or not q_start.is_contiguous() or short.numel() != 1:
                raise ValueError(f"q_start must be a contiguous [{B + 1}] tensor and short hold one value")
            if rows is not None:
                _require_here(slots, "slots", torch.int64, here)
                if slots.shape != (rows,) or not slots.is_contiguous():
                    raise ValueError(f"slots must be a contiguous [{rows}] tensor")
            elif slots is not None:
                raise ValueError("slots without rows")
        rc = self.lib.ns_paged_reserve(
            new.data_ptr(), lens.data_ptr(), pages.data_ptr(), strides[0] if B > 1 else width, width,
            free.data_ptr(), free.shape[0], n_free.data_ptr(), q_start.data_ptr(),
            None if slots is None else slots.data_ptr(), -1 if rows is None else rows, short.data_ptr(), B, page_size,
            _raw_stream(here))
        self._check(rc, "ns_paged_reserve")
        return out

    def paged_reorder(self, parents, pages, lens, k_pages, v_pages, k_scales=None, v_scales=None, out=None, free=None,
                      n_free=None):
        """The pages of beam search's sequences after a selection: beam i of request r goes on from beam parents[r, i]
        (int32 [R, beams], rows may be strided, e.g. beam_select's first columns; -1: stays). pages [R * beams, width] and
        lens [R * beams] are the batch's, request by request; the beams of a request have one length. Returns the new
        pages [R * beams, width] (contiguous, not pages itself).

        Whole pages are shared by the tables. Of the last, partly filled pages, which have to be the beams' own, one child
        keeps its parent's; for the others its rows are copied, in every layer, to the pages of beams that ended. So
        neither pages nor copies are needed beyond the beams' own, and entries behind the last position stay each
        beam's. k_pages, v_pages: bf16 [n_pages, Hk, page_size, D] or all layers' [layers, n_pages, Hk, page_size,
        D] (strides as in paged_append), or float8_e4m3fn with k_scales, v_scales as in paged_append_fp8.

        Whole pages that only ended beams had are in no row of the result. With ``free`` and ``n_free``, paged_reserve's stack, they
        are pushed on it (request by request, column by column, then by beam; it needs room for every page). Without, a
        repeated call with the same arguments gives the same, and the caller has to know which pages a request took. Pages that
        rows of another request hold too must be in all of a request's rows. The reference serves one sequence
        (qwen.py:166-177)."""
        here = _device_of(parents, "parents", torch.int32)
        _require_here(pages, "pages", torch.int32, here)
        _require_here(lens, "lens", torch.int32, here)
        fp8 = k_scales is not None
        dtype = torch.float8_e4m3fn if fp8 else torch.bfloat16
        _require_here(k_pages, "k_pages", dtype, here)
        _require_here(v_pages, "v_pages", dtype, here)
        shape, strides = parents.shape, parents.stride()
        if len(shape) != 2 or (shape[1] > 1 and strides[1] != 1):
            raise ValueError("parents must be [R, beams] with contiguous rows")
        R, beams = shape
        rows, parent_stride = R * beams, strides[0] if R > 1 else beams
        shape, strides = pages.shape, pages.stride()
        if len(shape) != 2 or shape[0] != rows or strides[1] != 1:
            raise ValueError(f"pages must be [{rows}, width] with contiguous rows")
        width = shape[1]
        table_stride = strides[0] if rows > 1 else width
        if lens.shape != (rows,) or not lens.is_contiguous():
            raise ValueError(f"lens must be a contiguous [{rows}] tensor")
        shape, strides = k_pages.shape, k_pages.stride()
        if len(shape) not in (4, 5) or strides[-1] != 1 or strides[-2] != shape[-1]:
            raise ValueError("k_pages must be [n_pages, Hk, page_size, D], or that for all layers, with contiguous heads")
        if v_pages.shape != k_pages.shape or v_pages.stride() != strides:
            raise ValueError("k_pages and v_pages must be alike")
        if len(shape) == 4:
            shape, strides = (1, *shape), (0, *strides)
        layers, n_pages, Hk, page_size, D = shape
        size = 1 if fp8 else 2
        if (width | n_pages | page_size | size * D) >> 31:
            raise ValueError("the width of pages and the sizes of a page must be within 32 bits")
        by = (size * strides[0] if layers > 1 else 0, size * strides[1] if n_pages > 1 else 0,
              size * strides[2] if Hk > 1 else 0)
        marks = (None, None, 0, 0, 0)
        if fp8:
            _require_here(k_scales, "k_scales", torch.float8_e8m0fnu, here)
            _require_here(v_scales, "v_scales", torch.float8_e8m0fnu, here)
            strides = k_scales.stride()
            if k_scales.shape != (*k_pages.shape[:-2], page_size // 16) or (page_size > 16 and strides[-1] != 1):
                raise ValueError("k_scales must be [n_pages, Hk, page_size / 16] (for all layers, as the pages) with "
                                 "contiguous heads")
            if v_scales.shape != k_scales.shape or v_scales.stride() != strides:
                raise ValueError("k_scales and v_scales must be alike")
            if len(strides) == 3:
                strides = (0, *strides)
            marks = (k_scales.data_ptr(), v_scales.data_ptr(), strides[0] if layers > 1 else 0,
                     strides[1] if n_pages > 1 else 0, strides[2] if Hk > 1 else 0)
        elif v_scales is not None:
            raise ValueError("v_scales without k_scales")
        if free is not None or n_free is not None:
            if free is None or n_free is None:
                raise ValueError("free and n_free go together")
            _require_here(free, "free", torch.int32, here)
            _require_here(n_free, "n_free", torch.int32, here)
            if free.dim() != 1 or not free.is_contiguous() or n_free.numel() != 1:
                raise ValueError("free must be a contiguous [capacity] tensor and n_free hold one value")
        if out is None:
            out = pages.new_empty((rows, width))
        else:
            _require_here(out, "out", torch.int32, here)
            if out.shape != (rows, width) or not out.is_contiguous():
                raise ValueError(f"out must be a contiguous [{rows}, {width}] tensor")
        if rows == 0:
            return out
        args = (parents.data_ptr(), parent_stride, pages.data_ptr(), table_stride, width, lens.data_ptr(), out.data_ptr(),
                k_pages.data_ptr(), v_pages.data_ptr(), *by, *marks, layers, n_pages, page_size, size * D, R, beams, Hk)
        if free is None:
            rc = self.lib.ns_paged_reorder(*args, _raw_stream(here))
            self._check(rc, "ns_paged_reorder")
        else:
            rc = self.lib.ns_paged_reorder_back(*args, free.data_ptr(), free.shape[0], n_free.data_ptr(), _raw_stream(here))
            self._check(rc, "ns_paged_reorder_back")
        return out

    # ------------------------------------------------------------------ beam search
    def beam_select_workspace(self, R, beams, vocab, n, dtype=torch.bfloat16, device=None):
        """A uint8 device tensor of the workspace beam_select uses for these sizes. Launches that may overlap in time need
        workspaces of their own."""
        size = int(self.lib.ns_beam_select_workspace(_int32(R), _int32(beams), _int32(vocab), _int32(n)))
        return torch.empty(size, dtype=torch.uint8, device=device or "cuda") if size else None

    def beam_select(self, logits, scores, n, work=None, out=None):
        """The n best continuations (at most 64) of R requests with up to 64 beams each: logits [R * beams, vocab] (bf16 or
        float32, request by request, rows may be strided, vocab at most 2^20), scores [R, beams] float32, the beams' sums of log
        probabilities so far. Returns (scores float32, tokens int32, parents int32), each [R, n]: the largest scores[r, i] +
        log softmax(logits[r, i])[v], falling, with their v and i; equal ones by beam, within a beam by falling logit, then by
        token. A beam whose score is -inf does not count (after the prompt: all but one). NaN counts as -inf and is never taken,
        +inf as the largest float32; where fewer than n are left, -inf, -1 and -1. Scores are compared in float64; the sum below
        a logarithm is good to some 2^-22, and beams whose scores lie closer than that may come in either order.
        ``work``: from beam_select_workspace, allocated here when it is not given; ``out``: the three results. The
        reference decodes one sequence greedily (qwen.py:166-177)."""
        if not isinstance(logits, torch.Tensor):
            raise TypeError("logits must be a torch.Tensor")
        fp32 = logits.dtype is torch.float32
        here = _device_of(logits, "logits", torch.float32 if fp32 else torch.bfloat16)
        _require_here(scores, "scores", torch.float32, here)
        if scores.dim() != 2 or not scores.is_contiguous():
            raise ValueError("scores must be a contiguous [R, beams] tensor")
        R, beams = scores.shape
        shape, steps = logits.shape, logits.stride()
        if len(shape) != 2 or steps[1] != 1 or shape[0] != R * beams:
            raise ValueError(f"logits must be [{R * beams}, vocab] with contiguous rows")
        V = shape[1]
        if (n | V) >> 31:  # (the library's arguments would keep the low bits alone)
            raise ValueError("n and the vocabulary must be within 32 bits")
        if out is None:
            out = (scores.new_empty((R, n)), scores.new_empty((R, n), dtype=torch.int32),
                   scores.new_empty((R, n), dtype=torch.int32))
        else:
            for t, name, dtype in zip(out, ("scores", "tokens", "parents"), (torch.float32, torch.int32, torch.int32)):
                _require_here(t, "out " + name, dtype, here)
                if t.shape != (R, n) or not t.is_contiguous():
                    raise ValueError(f"out {name} must be a contiguous [{R}, {n}] tensor")
        if R == 0:
            return out
        if work is None:
            work = self.beam_select_workspace(R, beams, V, n, logits.dtype, device=logits.device)
        else:
            _require_here(work, "work", torch.uint8, here)
            if not work.is_contiguous():
                raise _strided_work()
        rc = self.lib.ns_beam_select(logits.data_ptr(), int(fp32), steps[0] if R * beams > 1 else V,
                                     scores.data_ptr(), out[0].data_ptr(), out[1].data_ptr(), out[2].data_ptr(),
                                     None if work is None else work.data_ptr(), 0 if work is None else work.numel(), R,
                                     beams, V, n, _raw_stream(here))
        self._check(rc, "ns_beam_select")
        return tuple(out)

    # ------------------------------------------------------------------ the next token
    def sample_workspace(self, B, vocab, dtype=torch.bfloat16, device=None):
        """A uint8 device tensor of the workspace sample uses for these sizes, or None. Launches that
        may overlap in time need workspaces of their own."""
        n = int(self.lib.ns_sample_workspace(B, vocab, int(dtype == torch.float32)))
        return torch.empty(n, dtype=torch.uint8, device=device or "cuda") if n else None

    def sample(self, logits, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0, work=None, out=None):
        """One token id per row of logits [B, vocab] (bf16 or float32, rows may be strided, vocab at
        most 2^20, at most 65535 rows) from the given random numbers u [B] float32 in [0, 1): int32 [B].

        Tokens ordered by falling logit (equal ones by index): the first ``top_k`` are kept (0: all), of
        those the shortest beginning that holds ``top_p`` of their probability (at least one), of those
        the ones of at least ``min_p`` times the largest probability; the token is the first, by index,
        at which the running sum of the kept probabilities exceeds u times their sum. Temperature 0:
        the largest logit. A setting is a number or a tensor [B] (float32, top_k int32) with one for
        each row. Numbers out of range are refused; a tensor's are read on the device, where a top_k
        below 1 keeps all tokens, a temperature not above 0 is 0, a top_p from 1 on keeps all and a
        min_p above 1 is 1. NaN logits are never drawn, nor is -inf; a row without any other gives -1. The same
        arguments give the same token, eager or replayed, whatever else is in the batch. ``work``: from
        sample_workspace, allocated here when it is not given. The reference decodes greedily
        (qwen.py:166-177)."""
        if not isinstance(logits, torch.Tensor):
            raise TypeError("logits must be a torch.Tensor")
        fp32 = logits.dtype is torch.float32
        here = _device_of(logits, "logits", torch.float32 if fp32 else torch.bfloat16)
        _require_here(u, "u", torch.float32, here)
        if logits.dim() != 2 or logits.stride(1) != 1:
            raise ValueError("logits must be [B, vocab] with contiguous rows")
        B, V = logits.shape
        if tuple(u.shape) != (B,) or not u.is_contiguous():
            raise ValueError(f"u must be a contiguous [{B}] tensor")
        args = []
        for name, t, dtype in (("temperature", temperature, torch.float32), ("top_k", top_k, torch.int32),
                               ("top_p", top_p, torch.float32), ("min_p", min_p, torch.float32)):
            if isinstance(t, torch.Tensor):
                _require_here(t, name, dtype, here)
                if tuple(t.shape) != (B,) or not t.is_contiguous():
                    raise ValueError(f"{name} must be a number or a contiguous [{B}] tensor")
                args += [t.data_ptr(), 0]
            else:
                check_setting(name, t)
                args += [None, min(int(t), V) if dtype is torch.int32 else t]
        if out is None:
            out = logits.new_empty(B, dtype=torch.int32)
        else:
            _require_here(out, "out", torch.int32, here)
            if tuple(out.shape) != (B,) or not out.is_contiguous():
                raise ValueError(f"out must be a contiguous [{B}] tensor")
        if B == 0:
            return out
        if work is None:
            work = self.sample_workspace(B, V, logits.dtype, device=logits.device)
        else:
            _require_here(work, "work", torch.uint8, here)
            if not work.is_contiguous():
                raise _strided_work()
        rc = self.lib.ns_sample(logits.data_ptr(), int(fp32), logits.stride(0) if B > 1 else V, u.data_ptr(),
                                *args, out.data_ptr(), None if work is None else work.data_ptr(),
                                0 if work is None else work.numel(), B, V, _raw_stream(here))
        self._check(rc, "ns_sample")
        return out

    # ------------------------------------------------------------------ packed tile format
    def w4_repack(self, Wq, S, group=128):
        """(Wq [N, K/8] int32, S [N, K/128] bf16) -> packed tiles (Wp int32 [ceil(N/16), K/128,
        256], Sp bf16 [ceil(N/16), K/128, 16]) for w4_linear_packed (include/nanoserve_w4.h)."""
        _require_gpu_tensor(Wq, "Wq", torch.int32)
        _require_gpu_tensor(S, "S", torch.bfloat16)
        N, K = Wq.shape[0], Wq.shape[1] * 8
        NT, C = (N + 15) // 16, K // 128
        Wp = torch.empty((NT, C, 256), dtype=torch.int32, device=Wq.device)
        Sp = torch.empty((NT, C, 16), dtype=torch.bfloat16, device=Wq.device)
        Wq, S = Wq.contiguous(), S.contiguous()
        rc = self.lib.ns_w4_repack(Wq.data_ptr(), S.data_ptr(), Wp.data_ptr(), Sp.data_ptr(), N, K,
                                   group, self._stream())
        self._check(rc, "ns_w4_repack")
        return Wp, Sp

    def w4_linear_packed(self, x, Wp, Sp, N, group=128, out=None):
        """x [M, K] bf16 (M >= 2: batched decode up to 16 rows, prefill beyond) -> y [M, N]
        bf16, as w4_linear on the packed weights of w4_repack (agreeing with it to one bf16
        ulp; M > 16 with the GEMM's bf16-staged weights, as w4_linear's GEMM). M = 1 is
        rejected: the standard format (w4_linear) is the faster one there."""
        _require_gpu_tensor(x, "x", torch.bfloat16)
        _require_gpu_tensor(Wp, "Wp", torch.int32)
        _require_gpu_tensor(Sp, "Sp", torch.bfloat16)
        M, K = x.shape
        if Wp.shape[0] * 16 < N or Wp.shape[1] * 128 != K:
            raise ValueError("packed weights do not match N and x's K")
        if out is None:
            out = x.new_empty((M, N))
        x = x.contiguous()
        rc = self.lib.ns_w4_linear_packed(x.data_ptr(), Wp.data_ptr(), Sp.data_ptr(), out.data_ptr(),
                                          M, N, K, group, self._stream())
        self._check(rc, "ns_w4_linear_packed")
        return out

    def w4_linear_packed_swiglu(self, x, Wp, Sp, N, group=128, out=None):
        """x [M, K] bf16 (M > 16) -> bf16(silu(g) * u) [M, N/2] on packed weights of gate/up
        rows interleaved in blocks of 8 (qwen.interleave_gate_up, then w4_repack): the packed
        GEMM with the SwiGLU epilogue (include/nanoserve_w4.h)."""
        _require_gpu_tensor(x, "x", torch.bfloat16)
        _require_gpu_tensor(Wp, "Wp", torch.int32)
        _require_gpu_tensor(Sp, "Sp", torch.bfloat16)
        M, K = x.shape
        if Wp.shape[0] * 16 < N or Wp.shape[1] * 128 != K:
            raise ValueError("packed weights do not match N and x's K")
        if out is None:
            out = torch.empty((M, N // 2), dtype=torch.bfloat16, device=x.device)
        x = x.contiguous()
        rc = self.lib.ns_w4_linear_packed_swiglu(x.data_ptr(), Wp.data_ptr(), Sp.data_ptr(),
                                                 out.data_ptr(), M, N, K, group, self._stream())
        self._check(rc, "ns_w4_linear_packed_swiglu")
        return out

    # ------------------------------------------------------------------ measurement kernels
    def probe_read(self, buf, grid, waves, depth, sink):
        """Read-only stream over the bytes of ``buf`` (a 16-byte aligned GPU tensor) with the W4
        GEMV's access pattern (include/nanoserve_probe.h); ``sink`` a GPU int32 tensor."""
        rc = self.lib.ns_probe_read(buf.data_ptr(), buf.numel() * buf.element_size(),
                                    sink.data_ptr(), grid, waves, depth, self._stream())
        self._check(rc, "ns_probe_read")

    def probe_empty(self, grid=1, threads=64):
        """Launch an empty kernel (the per-launch floor of a graph of kernels)."""
        self._check(self.lib.ns_probe_empty(grid, threads, self._stream()), "ns_probe_empty")

    def linear_loop(self, calls, group=128):
        """Issue ns_w4_linear for each (x, Wq, S, y) of ``calls`` back to back from the C++ host
        loop of ns_probe_linear_loop (no Python between the launches), on the current stream.
        Every tensor must satisfy ns_w4_linear's own contract without padding (M <= 8 or a
        multiple of 128, contiguous, y [M, N])."""
        n = len(calls)
        ptrs, ints = ctypes.c_void_p * n, ctypes.c_int * n
        rc = self.lib.ns_probe_linear_loop(
            ptrs(*[c[0].data_ptr() for c in calls]), ptrs(*[c[1].data_ptr() for c in calls]),
            ptrs(*[c[2].data_ptr() for c in calls]), ptrs(*[c[3].data_ptr() for c in calls]),
            ints(*[c[0].shape[0] for c in calls]), ints(*[c[1].shape[0] for c in calls]),
            ints(*[c[0].shape[1] for c in calls]), group, n, self._stream())
        self._check(rc, "ns_probe_linear_loop")
