"""Tensor-level operators over the C ABI.

Each function takes torch tensors that already live on the GPU, checks layout
the way the kernels assume it, and queues the work on torch's current HIP
stream.  torch is used for device memory and streams only; all arithmetic is in
libastrai_q.so.  Together these replace the single call
``F.linear(x, weight, bias)`` of astrai/model/components/linear.py:21.
"""
from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _abi

_host = None  # the native host path once it is loaded


def _native():
    """The native host path (csrc/host.cpp).  Its functions serve the plain case -- contiguous tensors of the right
    types on the current device -- and return None for any other, which the general code below then takes."""
    global _host
    if _host is None:
        _host = _abi.host()
    return _host


_DT = {torch.float32: _abi.AQ_F32, torch.bfloat16: _abi.AQ_BF16}


_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None)
_cur_device = getattr(torch._C, "_cuda_getDevice", None)


def current_stream(device: torch.device) -> int:
    """torch's current HIP stream on ``device``, as the raw handle the C ABI takes."""
    if _raw_stream is not None:
        return _raw_stream(device.index if device.index is not None else torch.cuda.current_device())
    return torch.cuda.current_stream(device).cuda_stream


def _stream(t: torch.Tensor) -> int:
    return current_stream(t.device)


class _OnDevice:
    """``torch.cuda.device(dev)`` that costs nothing when ``dev`` already is the current device (the
    usual case; a launch goes to the current device)."""
    __slots__ = ("ctx",)

    def __init__(self, dev: torch.device):
        self.ctx = None
        if _cur_device is None or dev.index is None or _cur_device() != dev.index:
            self.ctx = torch.cuda.device(dev)

    def __enter__(self):
        if self.ctx is not None:
            self.ctx.__enter__()

    def __exit__(self, *exc):
        if self.ctx is not None:
            return self.ctx.__exit__(*exc)
        return False


def _need_gpu(*ts: Optional[torch.Tensor]) -> None:
    dev = None
    for t in ts:
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError("astrai_q operators run on the GPU only; got a CPU tensor (no CPU fallback exists)")
        if dev is None:
            dev = t.device
        elif t.device != dev:
            raise ValueError("all tensors must be on the same device")


def _dt(t: torch.Tensor, what: str) -> int:
    try:
        return _DT[t.dtype]
    except KeyError:
        raise ValueError(f"{what}: dtype {t.dtype} is not supported (float32 or bfloat16)") from None


def _rows(x: torch.Tensor, what: str) -> torch.Tensor:
    """View [..., K] as a contiguous [M, K]."""
    if x.dim() < 1:
        raise ValueError(f"{what}: needs at least one dimension")
    x2 = x.reshape(-1, x.shape[-1])
    if not x2.is_contiguous():
        x2 = x2.contiguous()
    return x2


def _check_k(K: int) -> None:
    if K <= 0 or K % 16:
        raise ValueError(f"in_dim (K) must be a positive multiple of 16, got {K}")


def quant_rowwise_i8(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Symmetric absmax int8 per row of ``x [..., K]`` -> (codes int8 [M, K], scale f32 [M])."""
    r = (_host or _native()).quant_rowwise_i8(x)
    if r is not None:
        return r
    _need_gpu(x)
    x2 = _rows(x, "quant_rowwise_i8")
    M, K = x2.shape
    _check_k(K)
    q = torch.empty((M, K), dtype=torch.int8, device=x.device)
    s = torch.empty((M,), dtype=torch.float32, device=x.device)
    if M:
        with _OnDevice(x.device):
            rc = _abi.load().aq_quant_rowwise_i8(x2.data_ptr(), _dt(x2, "x"), M, K, x2.stride(0), q.data_ptr(),
                                                 s.data_ptr(), _stream(x))
        _abi.check(rc, "aq_quant_rowwise_i8")
    return q, s


# longest rows the fused row kernels keep in registers (elements): bf16, fp32
RMSNORM_QUANT_MAX_K = {torch.bfloat16: 12288, torch.float32: 6144}
SWIGLU_QUANT_MAX_F = {torch.bfloat16: 8192, torch.float32: 4096}


def rmsnorm_quant_rowwise_i8(x: torch.Tensor, gamma: torch.Tensor, eps: float) -> Tuple[torch.Tensor, torch.Tensor]:
    """RMSNorm (gain ``gamma``, same dtype as ``x``) fused with the per-token quantisation of its
    output: ``[..., K]`` -> (codes int8 ``[M, K]``, scales float32 ``[M]``)."""
    r = (_host or _native()).rmsnorm_quant_rowwise_i8(x, gamma, eps)
    if r is not None:
        return r
    _need_gpu(x, gamma)
    x2 = _rows(x, "x")
    M, K = x2.shape
    _check_k(K)
    if gamma.dtype != x2.dtype or gamma.numel() != K:
        raise ValueError("gamma must have the activations' dtype and K elements")
    gamma = gamma.contiguous()
    q = torch.empty((M, K), dtype=torch.int8, device=x2.device)
    s = torch.empty((M,), dtype=torch.float32, device=x2.device)
    if M:
        with _OnDevice(x2.device):
            rc = _abi.load().aq_rmsnorm_quant_rowwise_i8(x2.data_ptr(), _dt(x2, "x"), gamma.data_ptr(), _dt(gamma, "gamma"),
                                                         float(eps), M, K, x2.stride(0), q.data_ptr(), s.data_ptr(),
                                                         _stream(x2))
        _abi.check(rc, "aq_rmsnorm_quant_rowwise_i8")
    return q, s


def swiglu_quant_rowwise_i8(ug: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """``ug [..., 2F] = [up | gate]`` -> codes and scales of ``up * silu(gate)`` per row
    (int8 ``[M, F]``, float32 ``[M]``), without writing the product."""
    r = (_host or _native()).swiglu_quant_rowwise_i8(ug)
    if r is not None:
        return r
    _need_gpu(ug)
    u2 = _rows(ug, "ug")
    M, F2 = u2.shape
    if F2 % 2:
        raise ValueError("the last dimension holds up and gate side by side: it must be even")
    F = F2 // 2
    _check_k(F)
    q = torch.empty((M, F), dtype=torch.int8, device=u2.device)
    s = torch.empty((M,), dtype=torch.float32, device=u2.device)
    if M:
        with _OnDevice(u2.device):
            rc = _abi.load().aq_swiglu_quant_rowwise_i8(u2.data_ptr(), _dt(u2, "ug"), M, F, u2.stride(0), q.data_ptr(),
                                                        s.data_ptr(), _stream(u2))
        _abi.check(rc, "aq_swiglu_quant_rowwise_i8")
    return q, s


# From this many input bytes on, the one-launch form of the per-tensor quantiser is the faster one (below, its
# exchange of partial maxima between workgroups costs more than the second launch: 6.9 against 4.6-5.2 us for small
# tensors, level at 16 MiB, 13.0 against 16.5 us at 32 MiB).
FP8_ONEPASS_MIN_BYTES = 16 << 20


def fp8_onepass_state(device) -> torch.Tensor:
    """The small piece of device state the one-launch per-tensor quantiser needs: zero-filled once, then reused
    for every call on that device and stream (calls that overlap in time must not share one)."""
    return torch.zeros((_abi.AQ_FP8_ONEPASS_WS_BYTES // 8,), dtype=torch.int64, device=device)


def codes_pitch(M: int, N: int, K: int, fp8: bool, residual: bool = False) -> int:
    """Bytes between the rows of the codes that a Linear ``[M, K] -> [M, N]`` reads fastest, K or the next multiple of 128."""
    return _abi.load().aq_linear_codes_pitch(int(fp8), int(residual), M, N, K)


def quant_tensor_fp8(x: torch.Tensor, state: Optional[torch.Tensor] = None,
                     onepass: Optional[bool] = None, pitch: Optional[int] = None) -> Tuple[torch.Tensor, torch.Tensor]:
    """Per-tensor OCP e4m3fn -> (codes uint8 with x's shape, scale f32 [1]).
    ``state`` (from ``fp8_onepass_state``): allows the one-launch form, which reads x from HBM once instead of
    twice -- same codes and scale; taken for tensors of ``FP8_ONEPASS_MIN_BYTES`` and more, or as ``onepass`` says.
    ``pitch`` (of a 2-D x, at least its row length and a multiple of 16): the codes' rows begin that many bytes apart."""
    if onepass is None:
        onepass = state is not None and x.numel() * x.element_size() >= FP8_ONEPASS_MIN_BYTES
    if pitch is not None and x.dim() != 2:
        raise ValueError("a pitch needs rows")
    if (state is not None or not onepass) and pitch is None:
        r = (_host or _native()).quant_tensor_fp8(x, state if onepass else None)
        if r is not None:
            return r
    _need_gpu(x)
    xc = x.contiguous()
    n = xc.numel()
    if n % 16:
        raise ValueError(f"numel must be a multiple of 16, got {n}")
    q = torch.empty(xc.shape if pitch is None else (xc.shape[0], pitch), dtype=torch.uint8, device=x.device)
    s = torch.empty((1,), dtype=torch.float32, device=x.device)
    lib, size = _abi.load(), (n,) if pitch is None else tuple(xc.shape)
    to = (q.data_ptr(),) if pitch is None else (q.data_ptr(), pitch)
    if onepass:
        if state is None:
            raise ValueError("the one-launch form needs the state tensor of fp8_onepass_state()")
        _need_gpu(state)
        if state.dtype != torch.int64 or state.numel() * 8 < _abi.AQ_FP8_ONEPASS_WS_BYTES or not state.is_contiguous() \
                or state.device != x.device:
            raise ValueError("state must come from fp8_onepass_state() for x's device")
        with _OnDevice(x.device):
            f = lib.aq_quant_tensor_fp8_onepass if pitch is None else lib.aq_quant_tensor_fp8_onepass_strided
            rc = f(xc.data_ptr(), _dt(xc, "x"), *size, *to, s.data_ptr(), state.data_ptr(), state.numel() * 8, _stream(x))
        _abi.check(rc, "aq_quant_tensor_fp8_onepass")
        return q if pitch is None else q[:, :xc.shape[1]], s
    ws = torch.empty((_abi.AQ_FP8_AMAX_WS_BYTES // 4,), dtype=torch.int32, device=x.device)  # partial maxima, stateless
    with _OnDevice(x.device):
        f = lib.aq_quant_tensor_fp8 if pitch is None else lib.aq_quant_tensor_fp8_strided
        rc = f(xc.data_ptr(), _dt(xc, "x"), *size, *to, s.data_ptr(), ws.data_ptr(), ws.numel() * 4, _stream(x))
    _abi.check(rc, "aq_quant_tensor_fp8")
    return q if pitch is None else q[:, :xc.shape[1]], s


def gemm_i8_i32(xq: torch.Tensor, wq: torch.Tensor) -> torch.Tensor:
    """acc[m, n] = sum_k xq[m, k] * wq[n, k] in exact int32."""
    _need_gpu(xq, wq)
    if xq.dtype != torch.int8 or wq.dtype != torch.int8:
        raise ValueError("gemm_i8_i32 takes int8 codes")
    if xq.dim() != 2 or wq.dim() != 2 or xq.shape[1] != wq.shape[1]:
        raise ValueError(f"shape mismatch: xq {tuple(xq.shape)} vs wq {tuple(wq.shape)}")
    xq, wq = xq.contiguous(), wq.contiguous()
    M, K = xq.shape
    N = wq.shape[0]
    _check_k(K)
    acc = torch.empty((M, N), dtype=torch.int32, device=xq.device)
    if M and N:
        with _OnDevice(xq.device):
            rc = _abi.load().aq_gemm_i8_i32(xq.data_ptr(), wq.data_ptr(), acc.data_ptr(), M, N, K, _stream(xq))
        _abi.check(rc, "aq_gemm_i8_i32")
    return acc


def _bias_args(bias: Optional[torch.Tensor], N: int):
    if bias is None:
        return None, 0
    if bias.dim() != 1 or bias.shape[0] != N:
        raise ValueError(f"bias must have shape [{N}], got {tuple(bias.shape)}")
    b = bias.contiguous()
    return b, _dt(b, "bias")


def _residual_arg(residual, M, N, out_dtype, dev):
    """A residual is added to the rounded output (``y = round(linear) + residual``, rounded again:
    the bits of a separate elementwise add); it holds M*N elements of the output's dtype."""
    if residual is None:
        return None
    if residual.dtype != out_dtype or residual.numel() != M * N or residual.device != dev:
        raise ValueError(f"residual must hold {M}x{N} {out_dtype} elements on {dev}, got {residual.dtype} "
                         f"{tuple(residual.shape)} on {residual.device}")
    if residual.dim() < 1 or residual.shape[-1] != N:
        raise ValueError(f"residual's last dimension must be {N}, got {tuple(residual.shape)}")
    return residual.contiguous()


def linear_w8a8(xq, sx, wq, sw, bias=None, out_dtype=torch.bfloat16, residual=None) -> torch.Tensor:
    """MFMA GEMM with the fused epilogue y = (acc * sx[m]) * sw[n] (+ bias[n]) (+ residual[m, n])."""
    y = (_host or _native()).linear_w8a8(xq, sx, wq, sw, bias, out_dtype, residual)
    if y is not None:
        return y
    _need_gpu(xq, sx, wq, sw, bias, residual)
    if xq.dtype != torch.int8 or wq.dtype != torch.int8:
        raise ValueError("linear_w8a8 takes int8 codes")
    if xq.dim() != 2 or wq.dim() != 2 or xq.shape[1] != wq.shape[1]:
        raise ValueError(f"shape mismatch: xq {tuple(xq.shape)} vs wq {tuple(wq.shape)}")
    M, K = xq.shape
    N = wq.shape[0]
    _check_k(K)
    if sx.dtype != torch.float32 or sw.dtype != torch.float32 or sx.numel() != M or sw.numel() != N:
        raise ValueError("sx must be float32 [M] and sw float32 [N]")
    if out_dtype not in _DT:
        raise ValueError(f"out_dtype {out_dtype} is not supported")
    xq, wq, sx, sw = xq.contiguous(), wq.contiguous(), sx.contiguous(), sw.contiguous()
    b, bdt = _bias_args(bias, N)
    r = _residual_arg(residual, M, N, out_dtype, xq.device)
    y = torch.empty((M, N), dtype=out_dtype, device=xq.device)
    if M and N:
        with _OnDevice(xq.device):
            rc = _abi.load().aq_linear_w8a8_residual(xq.data_ptr(), sx.data_ptr(), wq.data_ptr(), sw.data_ptr(),
                                                     b.data_ptr() if b is not None else None, bdt,
                                                     r.data_ptr() if r is not None else None, y.data_ptr(),
                                                     _DT[out_dtype], M, N, K, _stream(xq))
        _abi.check(rc, "aq_linear_w8a8")
    elif r is not None:
        y.copy_(r.view(M, N))
    return y


def gemv_w8a8_decode(x, wq, sw, bias=None, out_dtype=None, workspace: Optional[torch.Tensor] = None,
                     residual=None, norm=None) -> torch.Tensor:
    """Decode path for at most 16 rows of ``x [M, K]``: fused per-token quantise + int8 GEMV + epilogue.
    ``norm = (gamma [K], eps)``: RMS-normalise the rows first (the codes ``rmsnorm_quant_rowwise_i8``
    gives), in the same launch for bfloat16 rows of at most 2048 elements."""
    if workspace is None:
        gamma, eps = norm if norm is not None else (None, 0.0)
        y = (_host or _native()).gemv_w8a8_decode(x, wq, sw, bias, out_dtype, residual, gamma, eps)
        if y is not None:
            return y
    _need_gpu(x, wq, sw, bias, workspace, residual, norm[0] if norm is not None else None)
    x2 = _rows(x, "gemv_w8a8_decode")
    M, K = x2.shape
    N = wq.shape[0]
    if M > 16:
        raise ValueError(f"the decode path takes at most 16 rows, got {M}")
    if wq.dtype != torch.int8 or wq.dim() != 2 or wq.shape[1] != K:
        raise ValueError(f"wq must be int8 [N, {K}], got {wq.dtype} {tuple(wq.shape)}")
    _check_k(K)
    if sw.dtype != torch.float32 or sw.numel() != N:
        raise ValueError("sw must be float32 [N]")
    out_dtype = out_dtype or x.dtype
    if out_dtype not in _DT:
        raise ValueError(f"out_dtype {out_dtype} is not supported")
    wq, sw = wq.contiguous(), sw.contiguous()
    b, bdt = _bias_args(bias, N)
    lib = _abi.load()
    need = lib.aq_gemv_w8a8_workspace_bytes(M, K)
    if workspace is None:
        workspace = torch.empty((max(need, 16),), dtype=torch.uint8, device=x.device)
    elif workspace.numel() * workspace.element_size() < need:
        raise ValueError(f"workspace holds {workspace.numel() * workspace.element_size()} bytes, {need} needed")
    r = _residual_arg(residual, M, N, out_dtype, x.device)
    y = torch.empty((M, N), dtype=out_dtype, device=x.device)
    if norm is not None:
        gamma, eps = norm
        if gamma.dtype != x2.dtype or gamma.numel() != K:
            raise ValueError(f"the norm's gain must be {x2.dtype} [{K}], got {gamma.dtype} {tuple(gamma.shape)}")
        gamma = gamma.contiguous()
    if M and N:
        with _OnDevice(x.device):
            if norm is None:
                rc = lib.aq_gemv_w8a8_decode_residual(x2.data_ptr(), _dt(x2, "x"), wq.data_ptr(), sw.data_ptr(),
                                                      b.data_ptr() if b is not None else None, bdt,
                                                      r.data_ptr() if r is not None else None, y.data_ptr(),
                                                      _DT[out_dtype], M, N, K, workspace.data_ptr(),
                                                      workspace.numel() * workspace.element_size(), _stream(x))
            else:
                rc = lib.aq_gemv_w8a8_decode_rmsnorm(x2.data_ptr(), _dt(x2, "x"), gamma.data_ptr(), float(eps),
                                                     wq.data_ptr(), sw.data_ptr(),
                                                     b.data_ptr() if b is not None else None, bdt,
                                                     r.data_ptr() if r is not None else None, y.data_ptr(),
                                                     _DT[out_dtype], M, N, K, workspace.data_ptr(),
                                                     workspace.numel() * workspace.element_size(), _stream(x))
        _abi.check(rc, "aq_gemv_w8a8_decode")
    elif r is not None:
        y.copy_(r.view(M, N))
    return y


def gemv_swiglu_ok(x: torch.Tensor, dim_ffn: int) -> bool:
    """Whether ``gemv_w8a8_decode_swiglu`` serves these rows (bf16, at most 16 of them, K <= 2048 in whole
    512-byte steps, dim_ffn a multiple of 16)."""
    if not x.is_cuda or x.dtype not in _DT:
        return False
    rows = x.numel() // x.shape[-1] if x.shape[-1] else 0
    return bool(_abi.load().aq_gemv_w8a8_decode_swiglu_ok(_DT[x.dtype], rows, dim_ffn, x.shape[-1]))


def gemv_w8a8_decode_swiglu(x, wq, sw, bias=None, out_dtype=None, norm=None) -> torch.Tensor:
    """``up(x) * silu(gate(x))`` of an MLP at decode in ONE launch: ``wq [2F, K]`` holds the up projection's rows and
    then the gate projection's (``QuantLinear.concat([up, gate])``); returns ``h [M, F]``.  ``norm = (gamma, eps)``:
    the RMSNorm in front, folded in as in ``gemv_w8a8_decode``.  Raises ``ValueError`` for shapes
    ``gemv_swiglu_ok`` refuses."""
    _need_gpu(x, wq, sw, bias, norm[0] if norm is not None else None)
    x2 = _rows(x, "gemv_w8a8_decode_swiglu")
    M, K = x2.shape
    if wq.dtype != torch.int8 or wq.dim() != 2 or wq.shape[1] != K or wq.shape[0] % 2:
        raise ValueError(f"wq must be int8 [2F, {K}], got {wq.dtype} {tuple(wq.shape)}")
    N = wq.shape[0]
    Fh = N // 2
    _check_k(K)
    if sw.dtype != torch.float32 or sw.numel() != N:
        raise ValueError("sw must be float32 [2F]")
    out_dtype = out_dtype or x.dtype
    if out_dtype not in _DT:
        raise ValueError(f"out_dtype {out_dtype} is not supported")
    wq, sw = wq.contiguous(), sw.contiguous()
    b, bdt = _bias_args(bias, N)
    gamma, eps = (None, 0.0)
    if norm is not None:
        gamma, eps = norm
        if gamma.dtype != x2.dtype or gamma.numel() != K:
            raise ValueError(f"the norm's gain must be {x2.dtype} [{K}], got {gamma.dtype} {tuple(gamma.shape)}")
        gamma = gamma.contiguous()
    h = torch.empty((M, Fh), dtype=out_dtype, device=x.device)
    if M and Fh:
        with _OnDevice(x.device):
            rc = _abi.load().aq_gemv_w8a8_decode_swiglu(x2.data_ptr(), _dt(x2, "x"),
                                                        gamma.data_ptr() if gamma is not None else None, float(eps),
                                                        wq.data_ptr(), sw.data_ptr(),
                                                        b.data_ptr() if b is not None else None, bdt, h.data_ptr(),
                                                        _DT[out_dtype], M, Fh, K, _stream(x))
        _abi.check(rc, "aq_gemv_w8a8_decode_swiglu")
    return h


def gemv_w8a8_codes(xq, sx, wq, sw, bias=None, out_dtype=torch.bfloat16, residual=None) -> torch.Tensor:
    """The decode GEMV on activation codes the caller already holds (at most 16 rows)."""
    y = (_host or _native()).gemv_w8a8_codes(xq, sx, wq, sw, bias, out_dtype, residual)
    if y is not None:
        return y
    _need_gpu(xq, sx, wq, sw, bias, residual)
    if xq.dtype != torch.int8 or wq.dtype != torch.int8:
        raise ValueError("gemv_w8a8_codes takes int8 codes")
    if xq.dim() != 2 or wq.dim() != 2 or xq.shape[1] != wq.shape[1]:
        raise ValueError(f"shape mismatch: xq {tuple(xq.shape)} vs wq {tuple(wq.shape)}")
    M, K = xq.shape
    N = wq.shape[0]
    if M > 16:
        raise ValueError(f"the decode path takes at most 16 rows, got {M}")
    _check_k(K)
    if sx.dtype != torch.float32 or sw.dtype != torch.float32 or sx.numel() != M or sw.numel() != N:
        raise ValueError("sx must be float32 [M] and sw float32 [N]")
    if out_dtype not in _DT:
        raise ValueError(f"out_dtype {out_dtype} is not supported")
    xq, wq, sx, sw = xq.contiguous(), wq.contiguous(), sx.contiguous(), sw.contiguous()
    b, bdt = _bias_args(bias, N)
    r = _residual_arg(residual, M, N, out_dtype, xq.device)
    y = torch.empty((M, N), dtype=out_dtype, device=xq.device)
    if M and N:
        with _OnDevice(xq.device):
            rc = _abi.load().aq_gemv_w8a8_codes_residual(xq.data_ptr(), sx.data_ptr(), wq.data_ptr(), sw.data_ptr(),
                                                         b.data_ptr() if b is not None else None, bdt,
                                                         r.data_ptr() if r is not None else None, y.data_ptr(),
                                                         _DT[out_dtype], M, N, K, _stream(xq))
        _abi.check(rc, "aq_gemv_w8a8_codes")
    elif r is not None:
        y.copy_(r.view(M, N))
    return y


def _rope_args(qkv, freqs, page_table, k_cache, v_cache, n_heads, n_kv_heads, what):
    """Checks shared by the rotary / KV-write entry points; returns (qkv [B, S, W], freqs as
    float32, its batch stride in floats, page_table), contiguous."""
    _need_gpu(qkv, freqs, page_table, k_cache, v_cache)
    D = k_cache.shape[-1]
    W = (n_heads + 2 * n_kv_heads) * D
    if qkv.dtype != torch.bfloat16 or k_cache.dtype != torch.bfloat16 or v_cache.dtype != torch.bfloat16:
        raise ValueError(f"{what} takes bfloat16 activations and caches")
    if qkv.dim() not in (2, 3) or qkv.shape[-1] != W:
        raise ValueError(f"qkv must be [B, {W}] or [B, S, {W}], got {tuple(qkv.shape)}")
    if qkv.dim() == 2:
        qkv = qkv.unsqueeze(1)
    B, S = qkv.shape[0], qkv.shape[1]
    if k_cache.dim() != 4 or k_cache.shape != v_cache.shape or k_cache.shape[2] != n_kv_heads:
        raise ValueError("caches must be [n_pages, page, Hkv, D] and alike")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("caches must be contiguous")
    fr = torch.view_as_real(freqs) if freqs.is_complex() else freqs
    if fr.dtype != torch.float32 or fr.shape[0] != B or fr.numel() // max(B, 1) != S * D or fr.stride(-1) != 1:
        raise ValueError(f"freqs must be complex64 [B, (S,) {D // 2}] or float32 [B, (S,) {D // 2}, 2]")
    if B > 1 and fr.stride(0) == 0:      # one table broadcast to every sequence: no copy
        fr_stride, fr = 0, fr[0].contiguous()
    else:
        fr = fr.reshape(B, S * D).contiguous()
        fr_stride = S * D
    if fr.data_ptr() % 16:
        fr = fr.clone()
    if page_table.dtype != torch.int64 or page_table.dim() != 2 or page_table.shape[0] != B:
        raise ValueError("page_table must be int64 [B, P]")
    return qkv.contiguous(), fr, fr_stride, page_table.contiguous()


class QkNorm(NamedTuple):
    """Attention's qk-norm (``use_qk_norm``, astrai/model/components/attention.py:62-64, 86-89): the weights of the
    RMSNorm modules over the head dimension that follow the rotation of q and of k, and their epsilon."""
    q_gain: torch.Tensor
    k_gain: torch.Tensor
    eps: float


def _qk_norm_args(qk_norm, D: int, dev):
    """``(q_gain, k_gain, eps)`` checked for the kernels: bfloat16 ``[D]`` on ``dev``, 16-byte aligned."""
    if qk_norm is None:
        return None
    qg, kg, eps = qk_norm
    out = []
    for g in (qg, kg):
        if g.dtype != torch.bfloat16 or g.numel() != D or g.device != dev:
            raise ValueError(f"qk-norm gains must be bfloat16 [{D}] on {dev}, got {g.dtype} {tuple(g.shape)} on {g.device}")
        g = g.reshape(D).contiguous()
        out.append(g if g.data_ptr() % 16 == 0 else g.clone())
    if not eps >= 0.0:
        raise ValueError("qk-norm eps must not be negative")
    return out[0], out[1], float(eps)


def rope_kv_write(qkv: torch.Tensor, freqs: torch.Tensor, page_table: torch.Tensor, pos: int, k_cache: torch.Tensor,
                  v_cache: torch.Tensor, n_heads: int, n_kv_heads: int, return_k: bool = False,
                  qk_norm: Optional[QkNorm] = None):
    """New tokens of every sequence -- ``qkv [B, (Hq + 2 Hkv) * D]`` (one each, D = 64 or 128) or ``[B, S, ...]``:
    rotate q and k by ``freqs`` (complex64 ``[B, (S,) 64]`` or float32 ``[B, (S,) 64, 2]``), write k and
    v into the paged caches ``[n_pages, page, Hkv, D]`` at logical positions ``pos .. pos + S - 1``;
    returns the rotated ``q [B, (S,) Hq, D]``, and with ``return_k`` also the rotated
    ``k [B, (S,) Hkv, D]``.  With ``qk_norm`` the rotated q and k heads are RMS-normalised over D before they are
    returned and cached."""
    one = qkv.dim() == 2
    qkv, fr, fr_stride, page_table = _rope_args(qkv, freqs, page_table, k_cache, v_cache, n_heads, n_kv_heads,
                                                "rope_kv_write")
    B, S, D = qkv.shape[0], qkv.shape[1], k_cache.shape[-1]
    q = torch.empty((B, S, n_heads, D), dtype=torch.bfloat16, device=qkv.device)
    k = torch.empty((B, S, n_kv_heads, D), dtype=torch.bfloat16, device=qkv.device) if return_k else None
    norm = _qk_norm_args(qk_norm, D, qkv.device)
    if B and S:
        head = (qkv.data_ptr(), fr.data_ptr(), fr_stride, page_table.data_ptr(), page_table.shape[1], int(pos), S,
                k_cache.shape[1], k_cache.data_ptr(), v_cache.data_ptr(), k_cache.shape[0], q.data_ptr(),
                k.data_ptr() if return_k else None, B, n_heads, n_kv_heads, D)
        with _OnDevice(qkv.device):
            if norm is None:
                rc = _abi.load().aq_rope_kv_write(*head, _stream(qkv))
            else:
                rc = _abi.load().aq_rope_kv_write_qknorm(*head, norm[0].data_ptr(), norm[1].data_ptr(), norm[2],
                                                         _stream(qkv))
        _abi.check(rc, "aq_rope_kv_write" if norm is None else "aq_rope_kv_write_qknorm")
    if one:
        q, k = q.squeeze(1), (k.squeeze(1) if return_k else None)
    return (q, k) if return_k else q


def _attn_workspace(workspace, need, dev):
    if need and (workspace is None or not workspace.is_contiguous() or workspace.device != dev
                 or workspace.numel() * workspace.element_size() < need or workspace.data_ptr() % 16):
        workspace = torch.empty(need // 4, dtype=torch.float32, device=dev)
    if not need:
        return None, 0
    return workspace.data_ptr(), workspace.numel() * workspace.element_size()


class AttnPartials(NamedTuple):
    """A decode step's attention stopped before its position slices are combined: ``buf`` holds
    ``[B, n_heads, n_slices, D + 4]`` float32 (D numerators, maximum, denominator, padding)."""
    buf: torch.Tensor
    n_slices: int
    B: int
    n_heads: int
    head_dim: int


GEMV_ATTN_MAX_ROWS, GEMV_ATTN_MAX_K, GEMV_ATTN_MAX_SLICES = 8, 2048, 4
GEMV_ATTN_SLICE = 256  # positions of a slice
# Every workgroup of the projection repeats the merge of all rows, so it pays only while that is little work (rows x row
# length x slices).  A decode step with the merge in o_proj | in a launch of its own, us: 24 layers 1536 wide, 4 rows x 3
# slices (18432) 644.6 | 652.1, 5 x 3 (23040) 737.1 | 735.2, 5 x 4 (30720) 759.7 | 747.1; 8 blocks 2048 wide, 3 x 3 237.2 | 243.6,
# 4 x 3 (24576) 241.8 | 242.7, 8 x 2 (32768) 276.0 | 273.2.  Attention and o_proj alone, separate minus merged: 1 x 1536 x 3 1.3,
# 4 x 1536 x 3 0.3, 8 x 2048 x 3 -1.4.  (Level around 22000; the limit is what callers ask attn_gemv_fusable about.)
GEMV_ATTN_MAX_WORK = 32768


def attn_gemv_fusable(B: int, n_heads: int, head_dim: int, total_len: int) -> bool:
    """Whether ``gemv_w8a8_attn`` can, and should, combine this step's attention slices itself:
    within the kernel's limits, and more than one slice (a single slice has no merge launch to
    save, and the attention kernel's bf16 output is the smaller input)."""
    if not (0 < B <= GEMV_ATTN_MAX_ROWS and n_heads * head_dim <= GEMV_ATTN_MAX_K
            and GEMV_ATTN_SLICE < total_len <= GEMV_ATTN_MAX_SLICES * GEMV_ATTN_SLICE):
        return False
    slices = (total_len + GEMV_ATTN_SLICE - 1) // GEMV_ATTN_SLICE
    return B * n_heads * head_dim * slices <= GEMV_ATTN_MAX_WORK


def rope_paged_attn_decode(qkv: torch.Tensor, freqs: torch.Tensor, page_table: torch.Tensor, total_len: int,
                           k_cache: torch.Tensor, v_cache: torch.Tensor, n_heads: int, n_kv_heads: int,
                           scale: Optional[float] = None, workspace: Optional[torch.Tensor] = None,
                           partials: bool = False, seq_lens: Optional[torch.Tensor] = None,
                           qk_norm: Optional[QkNorm] = None):
    """``rope_kv_write`` at position ``total_len - 1`` and ``paged_attn_decode`` over ``total_len``
    positions as one launch (plus the small merge launch for long sequences): same caches and
    outputs, bit for bit.  Returns the attention output ``[B, Hq, D]`` -- or, with ``partials``,
    the slices' partial results (no merge launch) for ``gemv_w8a8_attn`` to combine.
    ``seq_lens`` (int64 ``[B]`` on the device): sequence b attends to its first ``seq_lens[b]`` positions only.
    ``qk_norm``: as in ``rope_kv_write``, same bits."""
    if qkv.dim() != 2:
        raise ValueError(f"one new token per sequence: qkv must be [B, W], got {tuple(qkv.shape)}")
    qkv, fr, fr_stride, page_table = _rope_args(qkv, freqs, page_table, k_cache, v_cache, n_heads, n_kv_heads,
                                                "rope_paged_attn_decode")
    B, D = qkv.shape[0], k_cache.shape[-1]
    if total_len < 1:
        raise ValueError("total_len counts the new token: at least 1")
    lib = _abi.load()
    scale = float(scale if scale is not None else D ** -0.5)
    lens_ptr = _seq_lens_ptr(seq_lens, B, qkv.device)
    norm = _qk_norm_args(qk_norm, D, qkv.device)
    tail = () if norm is None else (norm[0].data_ptr(), norm[1].data_ptr(), norm[2])
    suffix = "" if norm is None else "_qknorm"
    if partials:
        if not B:
            raise ValueError("partial results need at least one sequence")
        need = int(lib.aq_paged_attn_decode_partials_bytes(B, n_heads, int(total_len)))
        if (workspace is None or not workspace.is_contiguous() or workspace.device != qkv.device
                or workspace.dtype != torch.float32 or workspace.numel() * 4 < need or workspace.data_ptr() % 16):
            workspace = torch.empty(need // 4, dtype=torch.float32, device=qkv.device)
        entry = "aq_rope_paged_attn_decode_partials" + suffix
        with _OnDevice(qkv.device):
            rc = getattr(lib, entry)(qkv.data_ptr(), fr.data_ptr(), fr_stride, page_table.data_ptr(),
                                     page_table.shape[1], int(total_len), lens_ptr, k_cache.shape[1],
                                     k_cache.data_ptr(), v_cache.data_ptr(), k_cache.shape[0],
                                     scale, B, n_heads, n_kv_heads, D, *tail, workspace.data_ptr(),
                                     workspace.numel() * 4, _stream(qkv))
        _abi.check(rc, entry)
        return AttnPartials(workspace, int(lib.aq_paged_attn_decode_slices(int(total_len))), B, n_heads, D)
    out = torch.empty((B, n_heads, D), dtype=torch.bfloat16, device=qkv.device)
    if B:
        ws_ptr, ws_bytes = _attn_workspace(workspace, paged_attn_workspace_bytes(B, n_heads, n_kv_heads, total_len),
                                           qkv.device)
        entry = "aq_rope_paged_attn_decode" + suffix
        with _OnDevice(qkv.device):
            rc = getattr(lib, entry)(qkv.data_ptr(), fr.data_ptr(), fr_stride, page_table.data_ptr(),
                                     page_table.shape[1], int(total_len), lens_ptr, k_cache.shape[1],
                                     k_cache.data_ptr(), v_cache.data_ptr(), k_cache.shape[0], scale,
                                     out.data_ptr(), B, n_heads, n_kv_heads, D, *tail, ws_ptr, ws_bytes,
                                     _stream(qkv))
        _abi.check(rc, entry)
    return out


def gemv_w8a8_attn(parts: AttnPartials, wq, sw, bias=None, out_dtype=torch.bfloat16, residual=None) -> torch.Tensor:
    """The output projection of a decode step on attention partial results: combines the slices
    (the merge kernel's arithmetic), quantises the ``[B, n_heads * D]`` rows and multiplies, one
    launch; the bits of ``rope_paged_attn_decode`` followed by ``gemv_w8a8_decode``."""
    _need_gpu(parts.buf, wq, sw, bias, residual)
    M, K = parts.B, parts.n_heads * parts.head_dim
    N = wq.shape[0]
    if wq.dtype != torch.int8 or wq.dim() != 2 or wq.shape[1] != K:
        raise ValueError(f"wq must be int8 [N, {K}], got {wq.dtype} {tuple(wq.shape)}")
    if sw.dtype != torch.float32 or sw.numel() != N:
        raise ValueError("sw must be float32 [N]")
    if out_dtype not in _DT:
        raise ValueError(f"out_dtype {out_dtype} is not supported")
    if M > GEMV_ATTN_MAX_ROWS or K > GEMV_ATTN_MAX_K or parts.n_slices > GEMV_ATTN_MAX_SLICES:
        raise ValueError(f"gemv_w8a8_attn takes at most {GEMV_ATTN_MAX_ROWS} rows of {GEMV_ATTN_MAX_K} elements in "
                         f"{GEMV_ATTN_MAX_SLICES} slices; got {M} x {K} in {parts.n_slices}")
    if parts.buf.dtype != torch.float32 or parts.buf.numel() < M * parts.n_heads * parts.n_slices * (parts.head_dim + 4):
        raise ValueError("the partial results do not cover [B, n_heads, n_slices, D + 4] float32")
    wq, sw = wq.contiguous(), sw.contiguous()
    b, bdt = _bias_args(bias, N)
    r = _residual_arg(residual, M, N, out_dtype, wq.device)
    y = torch.empty((M, N), dtype=out_dtype, device=wq.device)
    if N:
        with _OnDevice(wq.device):
            rc = _abi.load().aq_gemv_w8a8_decode_attn(parts.buf.data_ptr(), parts.n_slices, parts.head_dim,
                                                      wq.data_ptr(), sw.data_ptr(),
                                                      b.data_ptr() if b is not None else None, bdt,
                                                      r.data_ptr() if r is not None else None, y.data_ptr(),
                                                      _DT[out_dtype], M, N, K, _stream(wq))
        _abi.check(rc, "aq_gemv_w8a8_decode_attn")
    return y


def prefill_attn_causal(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, scale: Optional[float] = None) -> torch.Tensor:
    """Causal attention of a prompt over itself: ``q [B, S, Hq, D]``, ``k`` / ``v [B, S, Hkv, D]`` (bfloat16,
    D = 64 or 128, last two dimensions contiguous, any token stride) -> ``[B, S, Hq, D]``."""
    _need_gpu(q, k, v)
    if q.dtype != torch.bfloat16 or k.dtype != torch.bfloat16 or v.dtype != torch.bfloat16:
        raise ValueError("prefill_attn_causal takes bfloat16 tensors")
    if q.dim() != 4 or k.dim() != 4 or k.shape != v.shape or q.shape[:2] != k.shape[:2] or q.shape[3] != k.shape[3]:
        raise ValueError("q must be [B, S, Hq, D] and k, v [B, S, Hkv, D]")
    B, S, Hq, D = q.shape
    Hkv = k.shape[2]

    def tokens(t, heads):
        # rows of heads*D contiguous elements, batch stride = S * token stride: otherwise copy
        if t.stride(3) == 1 and t.stride(2) == D and t.stride(0) == S * t.stride(1) and t.stride(1) % 8 == 0 \
                and t.data_ptr() % 16 == 0:
            return t, t.stride(1)
        return t.contiguous(), heads * D
    q, qs = tokens(q, Hq)
    k, ks = tokens(k, Hkv)
    v, vs = tokens(v, Hkv)
    out = torch.empty((B, S, Hq, D), dtype=torch.bfloat16, device=q.device)
    if B and S:
        with _OnDevice(q.device):
            rc = _abi.load().aq_prefill_attn_causal(q.data_ptr(), qs, k.data_ptr(), ks, v.data_ptr(), vs, out.data_ptr(),
                                                    float(scale if scale is not None else D ** -0.5), B, S, Hq, Hkv, D,
                                                    _stream(q))
        _abi.check(rc, "aq_prefill_attn_causal")
    return out


def prefill_attn_paged(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                       start: int, scale: Optional[float] = None) -> torch.Tensor:
    """Attention of ``S`` new tokens at positions ``start .. start + S`` over everything cached:
    ``q [B, S, Hq, D]`` against positions ``0 .. start + s`` of ``k_cache`` / ``v_cache
    [n_pages, page, Hkv, D]`` read through ``page_table [B, P]`` in place (the new tokens' rows
    written beforehand, ``rope_kv_write``) -> ``[B, S, Hq, D]``.  Unmapped pages are zero keys and
    values.  bfloat16, D = 64 or 128."""
    _need_gpu(q, k_cache, v_cache, page_table)
    if q.dtype != torch.bfloat16 or k_cache.dtype != torch.bfloat16 or v_cache.dtype != torch.bfloat16:
        raise ValueError("prefill_attn_paged takes bfloat16 tensors")
    if q.dim() != 4 or k_cache.dim() != 4 or k_cache.shape != v_cache.shape or q.shape[3] != k_cache.shape[3]:
        raise ValueError("q must be [B, S, Hq, D] and the caches [n_pages, page, Hkv, D]")
    if page_table.dtype != torch.int64 or page_table.dim() != 2 or page_table.shape[0] != q.shape[0]:
        raise ValueError("page_table must be int64 [B, P]")
    B, S, Hq, D = q.shape
    n_pages, page, Hkv, _ = k_cache.shape
    if start < 0 or start + S > page_table.shape[1] * page:
        raise ValueError(f"positions {start} .. {start + S} fall outside the page table")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("the caches must be contiguous")
    page_table = page_table.contiguous()
    if not (q.stride(3) == 1 and q.stride(2) == D and q.stride(0) == S * q.stride(1) and q.stride(1) % 8 == 0
            and q.data_ptr() % 16 == 0):
        q = q.contiguous()
    out = torch.empty((B, S, Hq, D), dtype=torch.bfloat16, device=q.device)
    if B and S:
        with _OnDevice(q.device):
            rc = _abi.load().aq_prefill_attn_paged(q.data_ptr(), q.stride(1), k_cache.data_ptr(), v_cache.data_ptr(),
                                                   page_table.data_ptr(), page_table.shape[1], int(start), page,
                                                   n_pages, out.data_ptr(),
                                                   float(scale if scale is not None else D ** -0.5), B, S, Hq, Hkv, D,
                                                   _stream(q))
        _abi.check(rc, "aq_prefill_attn_paged")
    return out


def paged_attn_workspace_bytes(B: int, n_heads: int, n_kv_heads: int, total_len: int) -> int:
    """Bytes of device workspace ``paged_attn_decode`` needs for this shape (0: none)."""
    return int(_abi.load().aq_paged_attn_decode_workspace_bytes(B, n_heads, n_kv_heads, int(total_len)))


def paged_attn_partials_bytes(B: int, n_heads: int, total_len: int) -> int:
    """Bytes the slices' partial results of a decode step take (also enough as its workspace)."""
    return int(_abi.load().aq_paged_attn_decode_partials_bytes(B, n_heads, int(total_len)))


def _seq_lens_ptr(seq_lens: Optional[torch.Tensor], B: int, device) -> Optional[int]:
    if seq_lens is None:
        return None
    if seq_lens.dtype != torch.int64 or seq_lens.shape != (B,) or seq_lens.device != device or not seq_lens.is_contiguous():
        raise ValueError(f"seq_lens must be a contiguous int64 [{B}] tensor on {device}")
    return seq_lens.data_ptr()


def paged_attn_decode(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                      total_len: int, scale: Optional[float] = None,
                      workspace: Optional[torch.Tensor] = None, seq_lens: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``softmax(scale * q K^T) V`` for one query token per sequence over the first ``total_len``
    positions of each sequence's pages: ``q [B, Hq, D]`` -> ``[B, Hq, D]`` (bfloat16, D = 64 or 128).
    ``workspace``: a contiguous device tensor of at least ``paged_attn_workspace_bytes`` bytes
    to reuse across calls; allocated per call when omitted or too small."""
    _need_gpu(q, k_cache, v_cache, page_table)
    if q.dtype != torch.bfloat16 or k_cache.dtype != torch.bfloat16 or v_cache.dtype != torch.bfloat16:
        raise ValueError("paged_attn_decode takes bfloat16 tensors")
    if q.dim() != 3 or k_cache.dim() != 4 or k_cache.shape != v_cache.shape or q.shape[2] != k_cache.shape[3]:
        raise ValueError("q must be [B, Hq, D] and the caches [n_pages, page, Hkv, D]")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("caches must be contiguous")
    B, Hq, D = q.shape
    Hkv = k_cache.shape[2]
    if page_table.dtype != torch.int64 or page_table.dim() != 2 or page_table.shape[0] != B:
        raise ValueError("page_table must be int64 [B, P]")
    page_table, q = page_table.contiguous(), q.contiguous()
    out = torch.empty_like(q)
    if B:
        ws_ptr, ws_bytes = _attn_workspace(workspace, paged_attn_workspace_bytes(B, Hq, Hkv, total_len), q.device)
        with _OnDevice(q.device):
            rc = _abi.load().aq_paged_attn_decode(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(),
                                                  page_table.data_ptr(), page_table.shape[1], int(total_len),
                                                  _seq_lens_ptr(seq_lens, B, q.device), k_cache.shape[1], k_cache.shape[0],
                                                  float(scale if scale is not None else D ** -0.5), out.data_ptr(),
                                                  B, Hq, Hkv, D, ws_ptr, ws_bytes, _stream(q))
        _abi.check(rc, "aq_paged_attn_decode")
    return out


def paged_attn_decode_shared(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, page_table: torch.Tensor,
                             total_len: int, shared_len: int, scale: Optional[float] = None,
                             workspace: Optional[torch.Tensor] = None, seq_lens: Optional[torch.Tensor] = None) -> torch.Tensor:
    """``paged_attn_decode`` for sequences that begin with the same pages: the entries of ``page_table`` for the first
    ``shared_len`` positions are the same in every row (the caller's promise; row 0's pages are read).  Those positions
    are read once and multiplied with all sequences' queries at once.  The results agree with ``paged_attn_decode`` within bf16
    rounding (the probabilities of all positions are rounded to bf16 on the way); ``seq_lens`` as there.  Sizes that gain nothing by it (``paged_attn_shared_positions``) run as ``paged_attn_decode``.
    ``workspace``: a contiguous device tensor to reuse across calls, of ``paged_attn_shared_workspace_bytes`` bytes; allocated per call when
    omitted or too small."""
    if workspace is None:
        y = (_host or _native()).paged_attn_decode_shared(q, k_cache, v_cache, page_table, total_len, shared_len, scale, seq_lens)
        if y is not None:
            return y
    _need_gpu(q, k_cache, v_cache, page_table)
    if q.dtype != torch.bfloat16 or k_cache.dtype != torch.bfloat16 or v_cache.dtype != torch.bfloat16:
        raise ValueError("paged_attn_decode_shared takes bfloat16 tensors")
    if q.dim() != 3 or k_cache.dim() != 4 or k_cache.shape != v_cache.shape or q.shape[2] != k_cache.shape[3]:
        raise ValueError("q must be [B, Hq, D] and the caches [n_pages, page, Hkv, D]")
    if not (k_cache.is_contiguous() and v_cache.is_contiguous()):
        raise ValueError("caches must be contiguous")
    B, Hq, D = q.shape
    n_pages, page, Hkv, _ = k_cache.shape
    if page_table.dtype != torch.int64 or page_table.dim() != 2 or page_table.shape[0] != B:
        raise ValueError("page_table must be int64 [B, P]")
    total_len, shared_len = int(total_len), int(shared_len)
    lens_ptr = _seq_lens_ptr(seq_lens, B, q.device)
    page_table, q = page_table.contiguous(), q.contiguous()
    out = torch.empty_like(q)
    if B:
        ws_ptr, ws_bytes = _attn_workspace(workspace, paged_attn_shared_workspace_bytes(B, Hq, Hkv, D, total_len, shared_len, q.device),
                                           q.device)
        with _OnDevice(q.device):
            rc = _abi.load().aq_paged_attn_decode_shared(q.data_ptr(), k_cache.data_ptr(), v_cache.data_ptr(), page_table.data_ptr(),
                                                         page_table.shape[1], total_len, shared_len, lens_ptr, page, n_pages,
                                                         float(scale if scale is not None else D ** -0.5), out.data_ptr(),
                                                         B, Hq, Hkv, D, ws_ptr, ws_bytes, _stream(q))
        _abi.check(rc, "aq_paged_attn_decode_shared")
    return out


def paged_attn_shared_positions(B: int, n_heads: int, n_kv_heads: int, head_dim: int, total_len: int, shared_len: int,
                                step: bool = False) -> int:
    """How many of the shared positions ``paged_attn_decode_shared`` reads once at these sizes; 0: nothing is gained by it, and the call is
    ``paged_attn_decode``'s.  ``step``: how many a model's step does, whose other form is ``rope_paged_attn_decode`` and which
    needs ``rope_kv_write`` in front of ``paged_attn_decode_shared``."""
    lib = _abi.load()
    rule = lib.aq_paged_attn_decode_shared_step_positions if step else lib.aq_paged_attn_decode_shared_positions
    return int(rule(B, n_heads, n_kv_heads, head_dim, int(total_len), int(shared_len)))


def paged_attn_shared_workspace_bytes(B: int, n_heads: int, n_kv_heads: int, head_dim: int, total_len: int, shared_len: int, device) -> int:
    """Bytes of device workspace ``paged_attn_decode_shared`` needs for these sizes on ``device`` (0: none)."""
    with _OnDevice(torch.device(device)):  # the positions are cut by the device's compute units
        return int(_abi.load().aq_paged_attn_decode_shared_workspace_bytes(B, n_heads, n_kv_heads, head_dim, int(total_len), int(shared_len)))


class ForkedPages(NamedTuple):
    """What ``fork_pages`` gives: the new rows ``[R, P]``, the pages' new counts ``[n_pages]``, and how many rows found no
    free page for their copy (``missing`` int32 ``[1]``; that entry of theirs is -1)."""
    page_table: torch.Tensor
    refs: torch.Tensor
    missing: torch.Tensor


class CompactedPages(NamedTuple):
    """What ``compact_pages`` gives: the renumbered table and counts, where each held page is now (``where`` int64
    ``[n_pages]``, -1: it was free), and how many are held (``live`` int32 ``[1]``: pages 0 .. live - 1)."""
    page_table: torch.Tensor
    refs: torch.Tensor
    where: torch.Tensor
    live: torch.Tensor


def _pages_args(page_table, refs, k_layers, v_layers, what):
    """Checked caches ``[layers, n_pages, page, Hkv, D]`` (or one layer's) with their table and counts ->
    (table, refs, (k, v, layers, layer_bytes, n_pages, page, row_bytes))."""
    if k_layers.dtype != v_layers.dtype or k_layers.shape != v_layers.shape or k_layers.dim() not in (4, 5):
        raise ValueError(f"{what}: the caches must be [layers, n_pages, page, Hkv, D], or one layer's, alike")
    k, v = (c.unsqueeze(0) if c.dim() == 4 else c for c in (k_layers, v_layers))
    layers, n_pages, page, heads, dim = k.shape
    if layers == 0 or k[0].numel() == 0:
        raise ValueError(f"{what}: the caches hold nothing")
    if not (k[0].is_contiguous() and v[0].is_contiguous()) or (layers > 1 and k.stride(0) != v.stride(0)):
        raise ValueError(f"{what}: a layer's pages must be contiguous, and the layers of both caches as far apart")
    if page_table.dtype != torch.int64 or page_table.dim() != 2 or page_table.shape[1] == 0:
        raise ValueError(f"{what}: page_table must be int64 [B, P]")
    if refs.dtype != torch.int32 or refs.shape != (n_pages,):
        raise ValueError(f"{what}: refs must be int32 [{n_pages}]")
    size = k.element_size()
    if heads * dim * size % 16:
        raise ValueError(f"{what}: a token's row of a layer must be a multiple of 16 bytes, got {heads * dim * size}")
    refs = refs.contiguous()
    if refs.data_ptr() % 16:
        refs = refs.clone()
    return page_table.contiguous(), refs, (k.data_ptr(), v.data_ptr(), layers, k.stride(0) * size if layers > 1 else 0,
                                                        n_pages, page, heads * dim * size)


def fork_pages(page_table: torch.Tensor, refs: torch.Tensor, parents: torch.Tensor, k_layers: torch.Tensor, v_layers: torch.Tensor,
               total_len: int, seq_lens: Optional[torch.Tensor] = None) -> ForkedPages:
    """New rows of a page table, each a fork of an old one: row i of the result goes on from row ``parents[i]`` (int64 ``[R]``;
    outside ``0 .. B - 1``: an empty row).  Whole pages are held together; the first child of a row goes on in its pages, the others
    get a free page with a copy of what is written of a page that is not full (``total_len`` positions are written, or
    ``seq_lens`` int64 ``[B]`` of them, in all layers' caches).  The first child writes on in the partly filled page whoever else holds it, as
    ``refs`` is not asked: a row that ends inside a page which another row, or another holder, still reads (a cached prompt whose last page is not
    full; with ``seq_lens``, a sequence rolled back into pages that it shares) is named twice, ``parents = [.., row, row]``, and goes on
    as its second child, which has a copy; the first is kept for those readers, or dropped in the next fork.  Old rows without a child let go of their pages: dropping beams, ending
    sequences and sampling several continuations are one call, and no call waits for the device.  ``refs`` int32
    ``[n_pages]`` counts who holds each page.  The table and the counts given are left as they are; the caches (any type, of 16-byte
    rows) are written in place, free pages only."""
    r = (_host or _native()).fork_pages(page_table, refs, parents, k_layers, v_layers, total_len, seq_lens)
    if r is not None:
        return ForkedPages(*r)
    _need_gpu(page_table, refs, parents, k_layers, v_layers)
    page_table, refs, caches = _pages_args(page_table, refs, k_layers, v_layers, "fork_pages")
    (B, P), n_pages, dev = page_table.shape, refs.numel(), refs.device
    if parents.dtype != torch.int64 or parents.dim() != 1:
        raise ValueError("parents must be int64 [R]")
    total_len = int(total_len)
    if not 0 <= total_len <= P * caches[5]:
        raise ValueError(f"{total_len} positions fall outside the page table")
    lens_ptr = _seq_lens_ptr(seq_lens, B, dev)
    parents, R = parents.contiguous(), parents.numel()
    table = torch.empty((R, P), dtype=torch.int64, device=dev)
    counts = torch.empty_like(refs)
    missing = torch.empty((1,), dtype=torch.int32, device=dev)
    lib = _abi.load()
    ws = torch.empty((lib.aq_fork_pages_workspace_bytes(n_pages, R) // 4,), dtype=torch.int32, device=dev)
    with _OnDevice(dev):
        rc = lib.aq_fork_pages(page_table.data_ptr(), B, P, refs.data_ptr(), parents.data_ptr(), R, total_len, lens_ptr, *caches,
                               table.data_ptr(), counts.data_ptr(), missing.data_ptr(), ws.data_ptr(), ws.numel() * 4, _stream(refs))
    _abi.check(rc, "aq_fork_pages")
    return ForkedPages(table, counts, missing)


def compact_pages(page_table: torch.Tensor, refs: torch.Tensor, k_layers: torch.Tensor, v_layers: torch.Tensor) -> CompactedPages:
    """Moves the pages that are held (``refs`` int32 ``[n_pages]`` above 0) to the front of all layers' caches, in place, and
    renumbers the table's entries: the last page held goes into the first free place, and so on, until pages 0 .. live - 1 are held.
    Entries that name a free page become -1.  The table and the counts given are left as they are; ``where`` tells other holders
    of pages where theirs went."""
    r = (_host or _native()).compact_pages(page_table, refs, k_layers, v_layers)
    if r is not None:
        return CompactedPages(*r)
    _need_gpu(page_table, refs, k_layers, v_layers)
    page_table, refs, caches = _pages_args(page_table, refs, k_layers, v_layers, "compact_pages")
    n_pages, dev = refs.numel(), refs.device
    table, counts = torch.empty_like(page_table), torch.empty_like(refs)
    where = torch.empty((n_pages,), dtype=torch.int64, device=dev)
    live = torch.empty((1,), dtype=torch.int32, device=dev)
    lib = _abi.load()
    ws = torch.empty((lib.aq_compact_pages_workspace_bytes(n_pages) // 4,), dtype=torch.int32, device=dev)
    with _OnDevice(dev):
        rc = lib.aq_compact_pages(page_table.data_ptr(), page_table.numel(), refs.data_ptr(), *caches, table.data_ptr(), counts.data_ptr(),
                                  where.data_ptr(), live.data_ptr(), ws.data_ptr(), ws.numel() * 4, _stream(refs))
    _abi.check(rc, "aq_compact_pages")
    return CompactedPages(table, counts, where, live)


# what the routed-expert operators take at most: experts and choices of a token, tokens, rows, values in one of them, and values of x, of h and of an
# expert's weights (codes by 31-bit offsets)
ROUTE_MAX_EXPERTS, ROUTE_MAX_CHOICES = 512, 16
EXPERTS_MAX_TOKENS, EXPERTS_MAX_ROWS, EXPERTS_MAX_WIDTH, EXPERTS_MAX_VALUES = 1 << 24, 1 << 25, 1 << 24, (1 << 31) - 17


class Routing(NamedTuple):
    """What ``route_topk`` gives for ``T`` tokens and ``k`` choices each: the weights (float32 ``[T, k]``) and the experts (int32 ``[T, k]``, -1: none),
    and the choices in the experts' order: expert e has rows ``offsets[e] .. offsets[e + 1] - 1`` (int32 ``[E + 1]``), ``rows`` (int32 ``[T, k]``) is the row of
    each choice (-1: none) and ``tokens`` (int32 ``[T k]``) the token of each row (-1 past the last one in use).  The five may share one storage."""
    weights: torch.Tensor
    experts: torch.Tensor
    rows: torch.Tensor
    tokens: torch.Tensor
    offsets: torch.Tensor


def _int32(t: torch.Tensor, shape, what: str) -> torch.Tensor:
    if t.dtype != torch.int32 or tuple(t.shape) != tuple(shape):
        raise ValueError(f"{what} must be int32 {list(shape)}, got {t.dtype} {list(t.shape)}")
    return t.contiguous()


def route_topk(logits: torch.Tensor, k: int, renormalize: bool = True) -> Routing:
    """Experts of each token from the router's logits ``[T, E]`` (float32 or bfloat16): the ``k`` largest, the largest first, equal ones the lowest
    expert first.  Weights are the softmax over the chosen logits, or over all ``E`` with ``renormalize=False``.  -inf and NaN are never
    chosen: a token with fewer than ``k`` other logits (a padded one: all -inf) has -1 and weight 0 in the places left.  The choices are sorted by
    expert on the device (by token inside an expert), so that no call waits to learn how many each got.  ``E`` at most 512, ``k`` at most 16.
    (DeepSeekMoE.forward, mlp.py:72-82, takes the top k of the probabilities rounded to the activations' type, whose ties have no order.)"""
    r = (_host or _native()).route_topk(logits, k, renormalize)
    if r is not None:
        return Routing(*r)
    _need_gpu(logits)
    if logits.dim() != 2:
        raise ValueError(f"logits must be [T, E], got {list(logits.shape)}")
    code, (T, E), k, dev = _dt(logits, "logits"), logits.shape, int(k), logits.device
    if E > 1 and logits.stride(1) != 1 or T > 1 and logits.stride(0) < E:
        logits = logits.contiguous()
    if not 0 < k <= E:
        raise ValueError(f"k must be 1 .. {E}, got {k}")
    weights = torch.empty((T, k), dtype=torch.float32, device=dev)
    experts, rows = (torch.empty((T, k), dtype=torch.int32, device=dev) for _ in range(2))
    tokens = torch.empty((T * k,), dtype=torch.int32, device=dev)
    offsets = torch.empty((E + 1,), dtype=torch.int32, device=dev)
    lib = _abi.load()
    ws = torch.empty((lib.aq_route_topk_workspace_bytes(T, E),), dtype=torch.uint8, device=dev)
    with _OnDevice(dev):
        rc = lib.aq_route_topk(logits.data_ptr(), code, T, E, logits.stride(0) if T > 1 else E, k, int(bool(renormalize)), weights.data_ptr(),
                               experts.data_ptr(), rows.data_ptr(), tokens.data_ptr(), offsets.data_ptr(), ws.data_ptr(), ws.numel(), _stream(logits))
    _abi.check(rc, "aq_route_topk")
    return Routing(weights, experts, rows, tokens, offsets)


def _grouped_args(xq, sx, wq, sw, offsets, tokens, what):
    """Checked operands of a grouped product -> (xq, sx, wq, sw, offsets, tokens, rows)."""
    _need_gpu(xq, sx, wq, sw, offsets, tokens)
    if xq.dtype != torch.int8 or xq.dim() != 2 or wq.dtype != torch.int8 or wq.dim() != 3 or wq.shape[2] != xq.shape[1]:
        raise ValueError(f"{what}: xq must be int8 [rows, K] and wq int8 [E, N, K]")
    _check_k(xq.shape[1])
    if sx.dtype != torch.float32 or sx.numel() != xq.shape[0] or sw.dtype != torch.float32 or tuple(sw.shape) != tuple(wq.shape[:2]):
        raise ValueError(f"{what}: scales must be float32, a number per row of xq and per row of each expert's weight")
    offsets = _int32(offsets, (wq.shape[0] + 1,), f"{what}: offsets")
    if tokens is not None:
        if tokens.dim() != 1:
            raise ValueError(f"{what}: tokens must be int32 [R]")
        tokens = _int32(tokens, tokens.shape, f"{what}: tokens")
    return (xq.contiguous(), sx.contiguous(), wq.contiguous(), sw.contiguous(), offsets, tokens,
            xq.shape[0] if tokens is None else tokens.numel())


def linear_w8a8_grouped(xq: torch.Tensor, sx: torch.Tensor, wq: torch.Tensor, sw: torch.Tensor, offsets: torch.Tensor,
                        tokens: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                        out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``linear_w8a8`` of several experts at once, ``wq`` int8 ``[E, N, K]``, ``sw`` ``[E, N]``, ``bias`` ``[E, N]``: rows ``offsets[e] .. offsets[e + 1] - 1``
    (int32 ``[E + 1]``, on the device; a group may be empty) of the result ``[R, N]`` are expert e's Linear on rows ``tokens[r]`` (int32 ``[R]``) of ``xq`` ``[T, K]``, or,
    without ``tokens``, on the same rows of ``xq`` ``[R, K]``: the bits of the single calls.  Rows past ``offsets[E]`` are not written.  A token
    outside ``0 .. T - 1`` counts as a row of zeros.  ``E`` at most 512, ``R`` 2^25, ``T K`` and ``N K`` below 2^31 - 16."""
    y = (_host or _native()).linear_w8a8_grouped(xq, sx, wq, sw, offsets, tokens, bias, out_dtype)
    if y is not None:
        return y
    xq, sx, wq, sw, offsets, tokens, R = _grouped_args(xq, sx, wq, sw, offsets, tokens, "linear_w8a8_grouped")
    E, N, K = wq.shape
    if out_dtype not in _DT:
        raise ValueError(f"out_dtype {out_dtype} is not supported (float32 or bfloat16)")
    bias_ptr, bias_dt = None, _abi.AQ_F32
    if bias is not None:
        _need_gpu(xq, bias)
        if tuple(bias.shape) != (E, N):
            raise ValueError(f"bias must be [{E}, {N}], got {list(bias.shape)}")
        bias = bias.contiguous()
        bias_ptr, bias_dt = bias.data_ptr(), _dt(bias, "bias")
    y = torch.empty((R, N), dtype=out_dtype, device=xq.device)
    with _OnDevice(xq.device):
        rc = _abi.load().aq_linear_w8a8_grouped(xq.data_ptr(), sx.data_ptr(), xq.shape[0], wq.data_ptr(), sw.data_ptr(), bias_ptr, bias_dt,
                                                offsets.data_ptr(), E, None if tokens is None else tokens.data_ptr(), R, y.data_ptr(),
                                                _DT[out_dtype], N, K, _stream(xq))
    _abi.check(rc, "aq_linear_w8a8_grouped")
    return y


def swiglu_w8a8_grouped(xq: torch.Tensor, sx: torch.Tensor, wq: torch.Tensor, sw: torch.Tensor, offsets: torch.Tensor,
                        tokens: Optional[torch.Tensor] = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """``h = up * silu(gate)`` of several experts at once: ``wq`` int8 ``[E, 2F, K]`` is each expert's up on top of its gate, the rest as in
    ``linear_w8a8_grouped``; up and gate are rounded to ``out_dtype`` first, as two Linears would have stored them (``gemv_w8a8_decode_swiglu``
    does the same for one MLP).  Returns ``[R, F]``; ``F`` a multiple of 16."""
    h = (_host or _native()).swiglu_w8a8_grouped(xq, sx, wq, sw, offsets, tokens, out_dtype)
    if h is not None:
        return h
    xq, sx, wq, sw, offsets, tokens, R = _grouped_args(xq, sx, wq, sw, offsets, tokens, "swiglu_w8a8_grouped")
    E, N, K = wq.shape
    if N % 32:
        raise ValueError(f"wq holds up and gate one on top of the other, of a multiple of 16 rows each: got {N} rows")
    if out_dtype not in _DT:
        raise ValueError(f"out_dtype {out_dtype} is not supported (float32 or bfloat16)")
    h = torch.empty((R, N // 2), dtype=out_dtype, device=xq.device)
    with _OnDevice(xq.device):
        rc = _abi.load().aq_swiglu_w8a8_grouped(xq.data_ptr(), sx.data_ptr(), xq.shape[0], wq.data_ptr(), sw.data_ptr(), offsets.data_ptr(), E,
                                                None if tokens is None else tokens.data_ptr(), R, h.data_ptr(), _DT[out_dtype], N // 2, K,
                                                _stream(xq))
    _abi.check(rc, "aq_swiglu_w8a8_grouped")
    return h


def combine_rows(y: torch.Tensor, rows: torch.Tensor, weights: torch.Tensor, residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The experts' outputs back in the tokens' order: ``out[t] = sum_j weights[t, j] * y[rows[t, j]]`` (``y`` ``[R, N]``, ``rows`` int32 and ``weights``
    float32 ``[T, k]``), plus ``residual[t]`` (what shared experts gave, or the residual stream), summed in fp32 in the order of j and rounded once.  Rows
    outside ``0 .. R - 1`` (-1: no expert) count for nothing.  ``k`` at most 64."""
    out = (_host or _native()).combine_rows(y, rows, weights, residual)
    if out is not None:
        return out
    _need_gpu(y, rows, weights, residual)
    if y.dim() != 2 or rows.dim() != 2:
        raise ValueError("y must be [R, N] and rows [T, k]")
    code, (R, N), (T, k) = _dt(y, "y"), y.shape, rows.shape
    rows = _int32(rows, rows.shape, "rows")
    if weights.dtype != torch.float32 or weights.shape != rows.shape:
        raise ValueError(f"weights must be float32 [{T}, {k}]")
    res = _residual_arg(residual, T, N, y.dtype, y.device)
    y, weights = y.contiguous(), weights.contiguous()
    out = torch.empty((T, N), dtype=y.dtype, device=y.device)
    with _OnDevice(y.device):
        rc = _abi.load().aq_combine_rows(y.data_ptr(), code, R, N, rows.data_ptr(), weights.data_ptr(), T, k,
                                         None if res is None else res.data_ptr(), out.data_ptr(), _stream(y))
    _abi.check(rc, "aq_combine_rows")
    return out


def experts_w8a8(x: torch.Tensor, routing: Routing, up_gate: torch.Tensor, up_gate_scale: torch.Tensor, down: torch.Tensor, down_scale: torch.Tensor,
                 residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The routed experts' MLP on ``x`` ``[T, dim]``: each token's rows through its experts' up, gate, SwiGLU and down, weighted and summed
    (``residual`` ``[T, dim]`` added).  ``up_gate`` int8 ``[E, 2F, dim]`` with scales ``[E, 2F]``, ``down`` int8 ``[E, dim, F]`` with scales ``[E, dim]``.  The bits of
    ``quant_rowwise_i8``, ``swiglu_w8a8_grouped``, ``quant_rowwise_i8``, ``linear_w8a8_grouped`` and ``combine_rows`` one after the other (what
    DeepSeekMoE.forward, mlp.py:83-91, does expert by expert), in one call that waits for nothing.  At most 64 choices a token; ``T dim``, ``T k F`` and
    ``2 F dim`` below 2^31 - 16: a longer batch is handed over in parts."""
    out = (_host or _native()).experts_w8a8(x, routing, up_gate, up_gate_scale, down, down_scale, residual)
    if out is not None:
        return out
    weights, _, rows, tokens, offsets = routing
    _need_gpu(x, weights, rows, tokens, offsets, up_gate, up_gate_scale, down, down_scale, residual)
    if x.dim() != 2:
        raise ValueError(f"x must be [T, dim], got {list(x.shape)}")
    code, (T, dim) = _dt(x, "x"), x.shape
    _check_k(dim)
    for w, what in ((up_gate, "up_gate"), (down, "down")):
        if w.dtype != torch.int8 or w.dim() != 3:
            raise ValueError(f"{what} must be int8 [E, out, in]")
    E, F = up_gate.shape[0], down.shape[2]
    if tuple(up_gate.shape) != (E, 2 * F, dim) or tuple(down.shape) != (E, dim, F) or F % 16:
        raise ValueError(f"up_gate must be [E, 2F, {dim}] and down [E, {dim}, F] with F a multiple of 16, got {list(up_gate.shape)} and {list(down.shape)}")
    for s, w, what in ((up_gate_scale, up_gate, "up_gate_scale"), (down_scale, down, "down_scale")):
        if s.dtype != torch.float32 or tuple(s.shape) != tuple(w.shape[:2]):
            raise ValueError(f"{what} must be float32 {list(w.shape[:2])}")
    if rows.dim() != 2 or rows.shape[0] != T:
        raise ValueError(f"the routing is not of {T} tokens")
    k = rows.shape[1]
    rows, tokens, offsets = _int32(rows, (T, k), "rows"), _int32(tokens, (T * k,), "tokens"), _int32(offsets, (E + 1,), "offsets")
    if weights.dtype != torch.float32 or tuple(weights.shape) != (T, k):
        raise ValueError(f"weights must be float32 [{T}, {k}]")
    res = _residual_arg(residual, T, dim, x.dtype, x.device)
    x, weights, up_gate, up_gate_scale, down, down_scale = (t.contiguous() for t in (x, weights, up_gate, up_gate_scale, down, down_scale))
    out = torch.empty_like(x)
    lib = _abi.load()
    ws = torch.empty((lib.aq_experts_w8a8_workspace_bytes(code, T, k, dim, F),), dtype=torch.uint8, device=x.device)
    with _OnDevice(x.device):
        rc = lib.aq_experts_w8a8(x.data_ptr(), code, T, dim, offsets.data_ptr(), E, tokens.data_ptr(), rows.data_ptr(), weights.data_ptr(), k,
                                 up_gate.data_ptr(), up_gate_scale.data_ptr(), down.data_ptr(), down_scale.data_ptr(), F,
                                 None if res is None else res.data_ptr(), out.data_ptr(), ws.data_ptr(), ws.numel(), _stream(x))
    _abi.check(rc, "aq_experts_w8a8")
    return out


def linear_fp8(xq, sx, wq, sw, bias=None, out_dtype=torch.bfloat16, residual=None) -> torch.Tensor:
    """FP8 e4m3fn GEMM with fp32 accumulation: y = (acc * sx[0]) * sw[0] (+ bias), cast, (+ residual)."""
    y = (_host or _native()).linear_fp8(xq, sx, wq, sw, bias, out_dtype, residual)
    if y is not None:
        return y
    _need_gpu(xq, sx, wq, sw, bias, residual)
    if xq.dtype != torch.uint8 or wq.dtype != torch.uint8:
        raise ValueError("linear_fp8 takes e4m3fn codes as uint8")
    if xq.dim() != 2 or wq.dim() != 2 or xq.shape[1] != wq.shape[1]:
        raise ValueError(f"shape mismatch: xq {tuple(xq.shape)} vs wq {tuple(wq.shape)}")
    M, K = xq.shape
    N = wq.shape[0]
    _check_k(K)
    if sx.dtype != torch.float32 or sw.dtype != torch.float32 or sx.numel() != 1 or sw.numel() != 1:
        raise ValueError("sx and sw must be float32 device scalars")
    if out_dtype not in _DT:
        raise ValueError(f"out_dtype {out_dtype} is not supported")
    wq, ld = wq.contiguous(), xq.stride(0)
    if xq.stride(1) != 1 or ld < K or ld % 16 or ld > 1 << 22 or M < 2 or xq.data_ptr() % 16:  # 2^22: the kernels' 32-bit offsets
        xq, ld = xq.contiguous(), K
    b, bdt = _bias_args(bias, N)
    r = _residual_arg(residual, M, N, out_dtype, xq.device)
    y = torch.empty((M, N), dtype=out_dtype, device=xq.device)
    if M and N:
        with _OnDevice(xq.device):
            rc = _abi.load().aq_linear_fp8_strided(xq.data_ptr(), ld, sx.data_ptr(), wq.data_ptr(), sw.data_ptr(),
                                                   b.data_ptr() if b is not None else None, bdt,
                                                   r.data_ptr() if r is not None else None, y.data_ptr(),
                                                   _DT[out_dtype], M, N, K, _stream(xq))
        _abi.check(rc, "aq_linear_fp8")
    elif r is not None:
        y.copy_(r.view(M, N))
    return y


def gemv_fp8_codes(xq, sx, wq, sw, bias=None, out_dtype=torch.bfloat16, residual=None) -> torch.Tensor:
    """The FP8 decode GEMV on codes the caller already holds (at most 16 rows; ``sx``, ``sw`` device scalars)."""
    _need_gpu(xq, sx, wq, sw, bias, residual)
    if xq.dtype != torch.uint8 or wq.dtype != torch.uint8 or xq.dim() != 2 or wq.dim() != 2 or xq.shape[1] != wq.shape[1]:
        raise ValueError(f"gemv_fp8_codes takes e4m3fn codes as uint8 [M, K] and [N, K], got {tuple(xq.shape)} / {tuple(wq.shape)}")
    M, K = xq.shape
    N = wq.shape[0]
    if M > 16:
        raise ValueError(f"the decode path takes at most 16 rows, got {M}")
    _check_k(K)
    if sx.dtype != torch.float32 or sw.dtype != torch.float32 or sx.numel() != 1 or sw.numel() != 1:
        raise ValueError("sx and sw must be float32 device scalars")
    if out_dtype not in _DT:
        raise ValueError(f"out_dtype {out_dtype} is not supported")
    xq, wq = xq.contiguous(), wq.contiguous()
    b, bdt = _bias_args(bias, N)
    r = _residual_arg(residual, M, N, out_dtype, xq.device)
    y = torch.empty((M, N), dtype=out_dtype, device=xq.device)
    if M and N:
        with _OnDevice(xq.device):
            rc = _abi.load().aq_gemv_fp8_codes_residual(xq.data_ptr(), sx.data_ptr(), wq.data_ptr(), sw.data_ptr(),
                                                        b.data_ptr() if b is not None else None, bdt,
                                                        r.data_ptr() if r is not None else None, y.data_ptr(),
                                                        _DT[out_dtype], M, N, K, _stream(xq))
        _abi.check(rc, "aq_gemv_fp8_codes")
    elif r is not None:
        y.copy_(r.view(M, N))
    return y


def gemv_fp8_decode(x, wq, sw, bias=None, out_dtype=None, workspace: Optional[torch.Tensor] = None,
                    residual=None) -> torch.Tensor:
    """FP8 decode path for at most 16 rows of ``x [M, K]``: per-tensor e4m3 cast + GEMV + epilogue, one launch for
    bfloat16 rows of at most 8192 elements (4096 for more than 8 rows)."""
    if workspace is None:
        y = (_host or _native()).gemv_fp8_decode(x, wq, sw, bias, out_dtype, residual)
        if y is not None:
            return y
    _need_gpu(x, wq, sw, bias, workspace, residual)
    x2 = _rows(x, "gemv_fp8_decode")
    M, K = x2.shape
    N = wq.shape[0]
    if M > 16:
        raise ValueError(f"the decode path takes at most 16 rows, got {M}")
    if wq.dtype != torch.uint8 or wq.dim() != 2 or wq.shape[1] != K:
        raise ValueError(f"wq must be uint8 (e4m3fn codes) [N, {K}], got {wq.dtype} {tuple(wq.shape)}")
    _check_k(K)
    if sw.dtype != torch.float32 or sw.numel() != 1:
        raise ValueError("sw must be a float32 device scalar")
    out_dtype = out_dtype or x.dtype
    if out_dtype not in _DT:
        raise ValueError(f"out_dtype {out_dtype} is not supported")
    wq = wq.contiguous()
    b, bdt = _bias_args(bias, N)
    lib = _abi.load()
    need = lib.aq_gemv_fp8_workspace_bytes(M, K)
    if workspace is None:
        workspace = torch.empty((max(need, 16),), dtype=torch.uint8, device=x.device)
    elif workspace.numel() * workspace.element_size() < need:
        raise ValueError(f"workspace holds {workspace.numel() * workspace.element_size()} bytes, {need} needed")
    r = _residual_arg(residual, M, N, out_dtype, x.device)
    y = torch.empty((M, N), dtype=out_dtype, device=x.device)
    if M and N:
        with _OnDevice(x.device):
            rc = lib.aq_gemv_fp8_decode_residual(x2.data_ptr(), _dt(x2, "x"), wq.data_ptr(), sw.data_ptr(),
                                                 b.data_ptr() if b is not None else None, bdt,
                                                 r.data_ptr() if r is not None else None, y.data_ptr(), _DT[out_dtype],
                                                 M, N, K, workspace.data_ptr(),
                                                 workspace.numel() * workspace.element_size(), _stream(x))
        _abi.check(rc, "aq_gemv_fp8_decode")
    elif r is not None:
        y.copy_(r.view(M, N))
    return y


def linear_fp8_few_rows(x, wq, sw, bias=None, residual=None) -> Optional[torch.Tensor]:
    """``linear_fp8`` of ``quant_tensor_fp8(x)`` in one launch, fp32 sums in an order of its own; None where two launches are the
    faster form of the shape (``aq_linear_few_rows_ok``) or take the type, and so decide what is wrong with it."""
    if x.dtype is not torch.bfloat16 or x.dim() != 2 or wq.dim() != 2 or wq.shape[1] != x.shape[1]:
        return None
    (M, K), N, lib = x.shape, wq.shape[0], _abi.load()
    if not lib.aq_linear_few_rows_ok(_abi.AQ_BF16, 0, 1, M, N, K):
        return None
    _need_gpu(x, wq, sw, bias, residual)
    if wq.dtype != torch.uint8 or sw.dtype != torch.float32 or sw.numel() != 1:
        raise ValueError("linear_fp8_few_rows takes e4m3fn codes as uint8 and a float32 device scalar")
    x, wq = x.contiguous(), wq.contiguous()
    b, bdt = _bias_args(bias, N)
    r = _residual_arg(residual, M, N, x.dtype, x.device)
    y = torch.empty((M, N), dtype=x.dtype, device=x.device)
    with _OnDevice(x.device):
        rc = lib.aq_linear_few_rows(x.data_ptr(), _abi.AQ_BF16, None, 0.0, wq.data_ptr(), 1, sw.data_ptr(), b.data_ptr() if b is not None else None,
                                    bdt, r.data_ptr() if r is not None else None, y.data_ptr(), _abi.AQ_BF16, M, N, K, _stream(x))
    _abi.check(rc, "aq_linear_few_rows")
    return y
