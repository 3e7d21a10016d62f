"""RMS norm with the residual's addition (``csrc/hstu_rms_norm.hip``):

    h = round(x + residual)        (h = x without a residual)
    y = h / sqrt(mean(h^2) + eps) * weight

over the last dimension, for bf16 and fp32 activations and bf16 or fp32
weights of any width up to 16384.  It stands beside the weighted LayerNorm
(``triton_weighted_layer_norm_fwd``), which the reference norms with
(``ops/triton/triton_layer_norm.py:1668-1740``); the reference's HSTU layer
has no RMS norm.

* ``rms_norm``: differentiable, ``y`` or ``(y, h)``;
* ``rms_norm_fp8``: e4m3 output with the scale of each row (what
  ``fp8.fp8_gemm`` and ``gated_linear_fp8`` take as ``a_scale``) or at one given
  scale;
* ``rms_norm_fwd`` / ``rms_norm_bwd``: the two kernels.

The norm is of the rounded ``h`` that is returned, so that the gradients, for
which only that ``h`` is kept, are those of the function that was computed.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib

E4M3 = torch.float8_e4m3fn
_TYPES = {torch.bfloat16: _lib.HSTU_DTYPE_BF16, torch.float32: _lib.HSTU_DTYPE_FP32}
MAX_D = 16384


def _rows2d(t: torch.Tensor) -> torch.Tensor:
    """[rows, D] with unit column stride and disjoint rows (column slices of a wider buffer stay in place)."""
    if t.dim() == 2:
        s0, s1 = t.stride()
        if s1 == 1 and (s0 >= t.shape[1] or t.shape[0] <= 1):
            return t
        return t.contiguous()
    t = t.reshape(-1, t.shape[-1])
    return t if t.stride(1) == 1 and (t.shape[0] <= 1 or t.stride(0) >= t.shape[1]) else t.contiguous()


def _ld(t: torch.Tensor) -> int:
    """Row stride; a single row may have any."""
    n = t.shape[1]
    s = t.stride(0)
    return s if s > n else n


def _like(name: str, t: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    if t.shape != x.shape or t.dtype != x.dtype or t.device != x.device:
        raise ValueError(f"{name} {tuple(t.shape)} {t.dtype} on {t.device} must match x {tuple(x.shape)} {x.dtype} "
                         f"on {x.device}")
    return _rows2d(t)


def _check(x: torch.Tensor, weight: torch.Tensor) -> Tuple[int, torch.Tensor, int]:
    """(code of x's type, the weight with unit stride, code of its type)"""
    code, wcode = _TYPES.get(x.dtype), _TYPES.get(weight.dtype)
    if code is None:
        raise NotImplementedError(f"x: bf16 or fp32 (got {x.dtype})")
    if x.dim() < 1 or not 0 < x.shape[-1] <= MAX_D:
        raise NotImplementedError(f"x {tuple(x.shape)}: a last dimension of 1 .. {MAX_D}")
    if not x.is_cuda:
        raise NotImplementedError("x: device tensors only")
    if weight.dim() != 1 or weight.shape[0] != x.shape[-1] or weight.device != x.device:
        raise ValueError(f"weight {tuple(weight.shape)} on {weight.device} must be [{x.shape[-1]}] on {x.device}")
    if wcode is None:
        raise NotImplementedError(f"weight: bf16 or fp32 (got {weight.dtype})")
    return code, weight if weight.stride(0) == 1 else weight.contiguous(), wcode


def rms_norm_fwd(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: Optional[torch.Tensor] = None,
                 output_fp8: bool = False, scale: Optional[torch.Tensor] = None, want_rstd: bool = True
                 ) -> Tuple[torch.Tensor, torch.Tensor, Optional[torch.Tensor], Optional[torch.Tensor]]:
    """(y, h, rstd, y_scale).  ``h`` is ``x`` itself without a residual; ``rstd``
    fp32 [rows]; ``output_fp8``: y e4m3 and ``y_scale`` the fp32 scales of the
    rows, or ``scale`` (one fp32 value on the device) where it is given."""
    code, w, wcode = _check(x, weight)
    shape, device, D = x.shape, x.device, x.shape[-1]
    x2 = _rows2d(x)
    rows = x2.shape[0]
    r2 = h = None
    r_ptr = h_ptr = r_ld = 0
    if residual is not None:
        r2 = _like("residual", residual, x)
        h = torch.empty(shape, dtype=x.dtype, device=device)
        r_ptr, r_ld, h_ptr = r2.data_ptr(), _ld(r2), h.data_ptr()
    y = torch.empty(shape, dtype=E4M3 if output_fp8 else x.dtype, device=device)
    rstd = torch.empty(rows, dtype=torch.float32, device=device) if want_rstd else None
    given = y_scale = None
    if output_fp8:
        if scale is None:
            y_scale = torch.empty(rows, dtype=torch.float32, device=device)
        else:
            if scale.numel() != 1 or scale.device != device:
                raise ValueError("scale must be one value on x's device")
            given = y_scale = scale.detach().to(torch.float32).reshape(1)
    elif scale is not None:
        raise ValueError("scale goes with output_fp8")
    if rows > 0:
        _lib.launch("hstu_rms_norm_fwd", x, code, x2.data_ptr(), _ld(x2), r_ptr, r_ld, w.data_ptr(), wcode, eps, rows,
                    D, h_ptr, D, y.data_ptr(), D, _lib.HSTU_DTYPE_FP8_E4M3 if output_fp8 else code, _lib.ptr(given),
                    None if given is not None else _lib.ptr(y_scale), _lib.ptr(rstd))
    return y, x if h is None else h, rstd, y_scale


def rms_norm_bwd(dy: torch.Tensor, h: torch.Tensor, weight: torch.Tensor, rstd: torch.Tensor,
                 dh: Optional[torch.Tensor] = None, dweight_dtype: Optional[torch.dtype] = None
                 ) -> Tuple[torch.Tensor, torch.Tensor]:
    """(dx, dweight): dx is the gradient of x and of the residual; ``dh`` the
    gradient of the returned h.  dweight in ``dweight_dtype`` (the weight's)."""
    code, w, wcode = _check(h, weight)
    device, D = h.device, h.shape[-1]
    dt = w.dtype if dweight_dtype is None else dweight_dtype
    if dt not in _TYPES:
        raise NotImplementedError(f"dweight: bf16 or fp32 (got {dt})")
    h2, dy2 = _rows2d(h), _like("dy", dy, h)
    d2 = None if dh is None else _like("dh", dh, h)
    rows = h2.shape[0]
    if rstd.dtype != torch.float32 or rstd.shape != (rows,) or rstd.device != device or rstd.stride(0) != 1:
        raise ValueError(f"rstd must be contiguous fp32 [{rows}] on {device}")
    dx = torch.empty(h.shape, dtype=h.dtype, device=device)
    dw = torch.empty(D, dtype=dt, device=device)
    nbytes = _lib.fn("hstu_rms_norm_bwd_workspace_bytes")(rows, D)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
    _lib.launch("hstu_rms_norm_bwd", h, code, dy2.data_ptr(), _ld(dy2), h2.data_ptr(), _ld(h2), _lib.ptr(d2),
                0 if d2 is None else _ld(d2), w.data_ptr(), wcode, rstd.data_ptr(), rows, D, dx.data_ptr(), D,
                dw.data_ptr(), _TYPES[dt], ws.data_ptr(), nbytes)
    return dx, dw


class RMSNormFunction(torch.autograd.Function):
    """Autograd of the norm: (y, h) from (x, residual, weight).  A gradient
    that nothing asks for is None and costs nothing.  What the backward needs
    besides tensors is settled in the forward: the engine runs it on a thread of
    its own, where every Python operation costs more."""

    @staticmethod
    def forward(ctx, x, weight, eps, residual):
        ctx.set_materialize_grads(False)
        y, h, rstd, _ = rms_norm_fwd(x, weight, eps, residual)
        _lib.guard_graph(ctx, x)
        ctx.save_for_backward(h, weight, rstd)
        D = h.shape[-1]
        rows = rstd.shape[0]
        ctx.plan = (_TYPES[h.dtype], _TYPES[weight.dtype], rows, D,
                    _lib.fn("hstu_rms_norm_bwd_workspace_bytes")(rows, D), h.shape, h.dtype, h.device,
                    residual is not None)
        return (y, h) if residual is not None else y

    @staticmethod
    def backward(ctx, dy, dh=None):
        if torch.is_grad_enabled():  # only under create_graph
            raise NotImplementedError("second derivatives (create_graph=True)")
        _lib.no_tangent("the backward of rms_norm", dy, dh)
        if dy is None:  # only h was used
            return dh, None, None, dh
        h, weight, rstd = ctx.saved_tensors
        code, wcode, rows, D, nbytes, shape, dtype, device, has_residual = ctx.plan
        h2, dy2 = _rows2d(h), _rows2d(dy)
        d_ptr = d_ld = 0
        if dh is not None:
            d2 = _rows2d(dh)
            d_ptr, d_ld = d2.data_ptr(), _ld(d2)
        w = weight if weight.stride(0) == 1 else weight.contiguous()
        dx = torch.empty(shape, dtype=dtype, device=device)
        dw = torch.empty(D, dtype=weight.dtype, device=device)
        ws = torch.empty(nbytes, dtype=torch.uint8, device=device)
        _lib.launch("hstu_rms_norm_bwd", h, code, dy2.data_ptr(), _ld(dy2), h2.data_ptr(), _ld(h2), d_ptr, d_ld,
                    w.data_ptr(), wcode, rstd.data_ptr(), rows, D, dx.data_ptr(), D, dw.data_ptr(), wcode,
                    ws.data_ptr(), nbytes)
        return dx, dw, None, dx if has_residual else None


def rms_norm(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: Optional[torch.Tensor] = None):
    """``y``, or ``(y, h)`` with a residual: h = x + residual is the new residual
    stream and y its norm times ``weight``.  Differentiable in x, residual and
    weight, through y and h; not a second time, nor in forward mode."""
    _lib.no_tangent("rms_norm", x, weight, residual)
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad
                                    or (residual is not None and residual.requires_grad)):
        return RMSNormFunction.apply(x, weight, eps, residual)
    y, h, _, _ = rms_norm_fwd(x, weight, eps, residual, want_rstd=False)
    return y if residual is None else (y, h)


def rms_norm_fp8(x: torch.Tensor, weight: torch.Tensor, eps: float = 1e-6, residual: Optional[torch.Tensor] = None,
                 scale: Optional[torch.Tensor] = None):
    """``(y8, scale)`` or, with a residual, ``(y8, scale, h)``: the norm in e4m3,
    y = y8 * scale with one fp32 scale a row ([rows], max|y| / 448) or the given
    one (returned as [1]).  Forward only: nothing returned carries a gradient, and
    inputs that require grad are refused while grad mode is on."""
    _lib.forward_only("rms_norm_fp8", x, weight, residual, scale)
    y8, h, _, s = rms_norm_fwd(x, weight, eps, residual, output_fp8=True, scale=scale, want_rstd=False)
    return (y8, s) if residual is None else (y8, s, h)
