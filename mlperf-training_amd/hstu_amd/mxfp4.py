"""Microscaled 4-bit floating point (OCP MX: e2m1 values with one E8M0 scale
for 32 consecutive values of a row) on the kernels of ``csrc/hstu_mxfp4.hip``.
It stands beside the e4m3 quantizers and GEMMs (``fp8``); the reference's
microscaled format for its projections is a 6-bit one
(``ops/hip/k512_mx6_gemm.cu:1-45``).

A quantized matrix is a pair ``(codes, scales)``: uint8 [R, C / 2], two values a
byte, the even column in the low half, and uint8 [R, C / 32], E + 127 with
E = max(floor(log2 max|v|) - 2, -127) of the block.  A value is the nearest of
0, 0.5, 1, 1.5, 2, 3, 4, 6 times 2^E (ties to the even code, larger ones 6); a
block with an infinity or NaN stands for NaN (scale byte 255).

* ``quantize_mxfp4`` / ``dequantize_mxfp4``;
* ``mxfp4_mm(a, w)``: the product of two quantized matrices;
* ``mxfp4_linear(x, w)``: bf16 activations, quantized on the way.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib

_TYPES = {torch.bfloat16: _lib.HSTU_DTYPE_BF16, torch.float32: _lib.HSTU_DTYPE_FP32}
# Up to here the product's kernel quantizes its rows of x itself, one launch and the
# work and the reads of x repeated for every 16 or 32 outputs; beyond, a kernel of
# its own does it once.  Measured (us on the device, one launch / two): 5 x 5632
# (M x K) against 2048 outputs 6.9 / 7.7, 16 x 4096 against 4096 8.3 / 9.4, 8 x 8192
# against 8192 13.0 / 14.4; 16 x 8192 against 8192 16.4 / 16.1, against 2048 13.2 /
# 10.7.  A launch from Python is 8 us of the host's time more.
ROWS_QUANT = 16
VALUES_QUANT = 65536
Packed = Tuple[torch.Tensor, torch.Tensor]


def quantize_mxfp4(x: torch.Tensor) -> Packed:
    """(codes [.., C / 2], scales [.., C / 32]) of bf16 or fp32 x [.., C], C a multiple of 32."""
    if x.dtype not in _TYPES:
        raise NotImplementedError(f"x: bf16 or fp32 (got {x.dtype})")
    if x.dim() < 1 or x.shape[-1] == 0 or x.shape[-1] % 32:
        raise NotImplementedError(f"x {tuple(x.shape)}: a last dimension that is a multiple of 32")
    if not x.is_cuda:
        raise NotImplementedError("x: device tensors only")
    shape, C = x.shape, x.shape[-1]
    x2 = x if x.dim() == 2 else x.reshape(-1, C)
    R = x2.shape[0]
    s0, s1 = x2.stride()
    if s1 != 1 or (R > 1 and s0 < C):
        x2, s0 = x2.contiguous(), C
    codes = torch.empty(shape[:-1] + (C // 2,), dtype=torch.uint8, device=x.device)
    scales = torch.empty(shape[:-1] + (C // 32,), dtype=torch.uint8, device=x.device)
    if R > 0:
        _lib.launch("hstu_mxfp4_quantize", x, _TYPES[x.dtype], x2.data_ptr(), s0 if R > 1 else C, R, C,
                    codes.data_ptr(), scales.data_ptr())
    return codes, scales


def _pair(name: str, codes: torch.Tensor, scales: torch.Tensor) -> None:
    if codes.dtype != torch.uint8 or scales.dtype != torch.uint8:
        raise ValueError(f"{name}: uint8 codes and scales (got {codes.dtype}, {scales.dtype})")
    if codes.device != scales.device or not codes.is_cuda:
        raise NotImplementedError(f"{name}: codes and scales on one device")
    if (codes.dim() < 1 or codes.shape[:-1] != scales.shape[:-1] or codes.shape[-1] != 16 * scales.shape[-1]
            or codes.shape[-1] == 0):
        raise ValueError(f"{name}: codes {tuple(codes.shape)} and scales {tuple(scales.shape)}; expected [.., C / 2] "
                         "and [.., C / 32]")


def dequantize_mxfp4(codes: torch.Tensor, scales: torch.Tensor, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values [.., C] that the pair stands for, in bf16 (exact) or fp32."""
    if dtype not in _TYPES:
        raise NotImplementedError(f"dtype: bf16 or fp32 (got {dtype})")
    _pair("dequantize_mxfp4", codes, scales)
    C = 2 * codes.shape[-1]
    c2, s2 = codes.contiguous(), scales.contiguous()
    c2 = c2 if c2.data_ptr() % 4 == 0 else c2.clone()
    out = torch.empty(codes.shape[:-1] + (C,), dtype=dtype, device=codes.device)
    R = out.numel() // C
    if R > 0:
        _lib.launch("hstu_mxfp4_dequantize", codes, c2.data_ptr(), s2.data_ptr(), R, C, _TYPES[dtype], out.data_ptr(), C)
    return out


FAR = 2 ** 23  # bytes between rows from which on the product's 32-bit offsets do not reach over a tile


def _aligned(t: torch.Tensor, n: int, far: int = FAR) -> torch.Tensor:
    """A 2-D operand with unit column stride and rows at multiples of n bytes, less than ``far`` bytes apart (a
    view such as one position of every sequence is copied where they are further)."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    s0, s1 = t.stride()
    apart = s0 * t.element_size()
    if s1 == 1 and t.data_ptr() % n == 0 and (t.shape[0] <= 1 or (s0 >= t.shape[1] and apart % n == 0 and apart < far)):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % n == 0 else t.clone()


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _epilogue(bias: Optional[torch.Tensor], residual: Optional[torch.Tensor], shape, device):
    """(bias in bf16 or fp32, residual, what an entry point's name ends in): a bias is added to the fp32 sum
    with the bits it has (of fp64's, fp32's)."""
    entry = ""
    if bias is not None:
        if bias.shape != shape[-1:] or bias.device != device:
            raise ValueError(f"bias {tuple(bias.shape)} on {bias.device}; expected [{shape[-1]}] on {device}")
        if not bias.is_floating_point():
            raise NotImplementedError(f"bias: a floating type (got {bias.dtype})")
        if bias.dtype != torch.bfloat16:
            bias, entry = bias.detach().to(torch.float32), "_bias_fp32"
        bias = bias if bias.stride(0) == 1 else bias.contiguous()
        bias = bias if bias.data_ptr() % 16 == 0 else bias.clone()
    if residual is not None:
        if residual.shape != shape or residual.device != device or residual.dtype != torch.bfloat16:
            raise ValueError(f"residual {tuple(residual.shape)} {residual.dtype} on {residual.device}; expected "
                             f"{tuple(shape)} bf16 on {device}")
        residual = _aligned(residual, 16, 2 ** 63)  # 64-bit offsets
    return bias, residual, entry


def _weight(weight: Packed) -> Tuple[torch.Tensor, torch.Tensor, int, int]:
    wc, ws = weight
    _pair("weight", wc, ws)
    if wc.dim() != 2:
        raise ValueError(f"weight codes {tuple(wc.shape)}; expected [N, K / 2]")
    N, K = wc.shape[0], 2 * wc.shape[1]
    if N == 0 or N % 16 or K % 128:
        raise NotImplementedError(f"weight [{N}, {K}]: N a multiple of 16 and K of 128")
    return _aligned(wc, 16), _aligned(ws, 4), N, K


def mxfp4_mm(a: Packed, weight: Packed, bias: Optional[torch.Tensor] = None,
             residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """a @ weight^T (+ bias [N], bf16 or fp32) (+ residual [.., N], bf16) in bf16, fp32 accumulation:
    a a pair of [.., K], weight a pair of [N, K]; N a multiple of 16, K of 128.
    Forward only, as ``mxfp4_linear``."""
    _lib.forward_only("mxfp4_mm", bias, residual)
    wc, ws, N, K = _weight(weight)
    ac, as_ = a
    _pair("a", ac, as_)
    if ac.shape[-1] != K // 2 or ac.device != wc.device:
        raise ValueError(f"a codes {tuple(ac.shape)} on {ac.device} against weight [{N}, {K}] on {wc.device}")
    shape = ac.shape[:-1] + (N,)
    bias, r2, entry = _epilogue(bias, residual, shape, wc.device)
    a2, s2 = _aligned(ac, 16), _aligned(as_, 4)
    M = a2.shape[0]
    if M >= 2 ** 31 - 256:
        raise NotImplementedError("a: fewer than 2^31 rows")
    out = torch.empty(shape, dtype=torch.bfloat16, device=wc.device)
    if M > 0:
        _lib.launch("hstu_mxfp4_gemm" + entry, wc, a2.data_ptr(), _ld(a2), s2.data_ptr(), _ld(s2), wc.data_ptr(), _ld(wc),
                    ws.data_ptr(), _ld(ws), _lib.ptr(bias), _lib.ptr(r2), 0 if r2 is None else _ld(r2), out.data_ptr(),
                    N, M, N, K)
    return out


def mxfp4_linear(x: torch.Tensor, weight: Packed, bias: Optional[torch.Tensor] = None,
                 residual: Optional[torch.Tensor] = None) -> torch.Tensor:
    """quantize(x) @ weight^T (+ bias) (+ residual) in bf16, for bf16 x [.., K].
    Forward only: the result carries no gradient, and inputs that require grad are
    refused while grad mode is on."""
    _lib.forward_only("mxfp4_linear", x, bias, residual)
    if x.dtype != torch.bfloat16:
        raise NotImplementedError(f"x: bf16 (got {x.dtype})")
    wc, ws, N, K = _weight(weight)
    shape = x.shape
    if shape[-1] != K or x.device != wc.device:
        raise ValueError(f"x {tuple(shape)} on {x.device} against weight [{N}, {K}] on {wc.device}")
    M = x.numel() // K
    if M > ROWS_QUANT or M * K > VALUES_QUANT:
        return mxfp4_mm(quantize_mxfp4(x), weight, bias, residual)
    shape = shape[:-1] + (N,)
    bias, r2, entry = _epilogue(bias, residual, shape, wc.device)
    out = torch.empty(shape, dtype=torch.bfloat16, device=wc.device)
    if M > 0:
        x2 = _aligned(x, 16)
        _lib.launch("hstu_mxfp4_linear_rows" + entry, wc, x2.data_ptr(), _ld(x2), wc.data_ptr(), _ld(wc), ws.data_ptr(), _ld(ws),
                    _lib.ptr(bias), _lib.ptr(r2), 0 if r2 is None else _ld(r2), out.data_ptr(), N, M, N, K)
    return out
