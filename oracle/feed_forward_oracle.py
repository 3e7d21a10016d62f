"""64-bit restatements of the feed-forward operators: the RMS norm with the
residual's addition, the gated projection and the microscaled 4-bit format.

Everything is computed in float64 from the formulas, on the tensors' device.
"""

from __future__ import annotations

import math
from typing import Optional, Tuple

import torch

F64 = torch.float64


# ---------------------------------------------------------------- RMS norm
def rms_norm_ref(h: torch.Tensor, weight: torch.Tensor, eps: float) -> Tuple[torch.Tensor, torch.Tensor]:
    """(y, rstd [.., 1]) of the residual stream h as it is kept."""
    h64 = h.to(F64)
    rstd = 1.0 / torch.sqrt(h64.pow(2).mean(-1, keepdim=True) + eps)
    return h64 * rstd * weight.to(F64), rstd


def rms_norm_bwd_ref(dy: torch.Tensor, h: torch.Tensor, weight: torch.Tensor, eps: float,
                     dh: Optional[torch.Tensor] = None):
    """(dx, dweight, bound_dx, bound_dw): the gradients, and for each element the
    sum of the magnitudes that meet in it, which a bound on rounding scales."""
    h64, dy64 = h.to(F64), dy.to(F64)
    rstd = 1.0 / torch.sqrt(h64.pow(2).mean(-1, keepdim=True) + eps)
    xhat, c = h64 * rstd, dy64 * weight.to(F64)
    dx = rstd * (c - xhat * (c * xhat).mean(-1, keepdim=True))
    bound = rstd * (c.abs() + xhat.abs() * (c * xhat).abs().mean(-1, keepdim=True))
    if dh is not None:
        dx = dx + dh.to(F64)
        bound = bound + dh.to(F64).abs()
    prod = (dy64 * xhat).reshape(-1, h.shape[-1])
    return dx, prod.sum(0), bound, prod.abs().sum(0)


# ---------------------------------------------------------------- gated projection
def activation_ref(name: str, g: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(a(g), a'(g)) of silu, gelu (tanh form) and sigmoid."""
    if name == "silu":
        s = torch.sigmoid(g)
        return g * s, s + g * s * (1 - s)
    if name == "sigmoid":
        s = torch.sigmoid(g)
        return s, s * (1 - s)
    k = math.sqrt(2 / math.pi)
    t = torch.tanh(k * (g + 0.044715 * g.pow(3)))
    return 0.5 * g * (1 + t), 0.5 * (1 + t) + 0.5 * g * (1 - t * t) * k * (1 + 3 * 0.044715 * g.pow(2))


def gated_ref(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, name: str) -> torch.Tensor:
    x64 = x.to(F64)
    return activation_ref(name, x64 @ w_gate.to(F64).t())[0] * (x64 @ w_up.to(F64).t())


def gated_bwd_ref(dh, x, w_gate, w_up, name):
    """(dx, dgate, dup, dg, du)"""
    x64, gate, up, dh64 = (t.to(F64) for t in (x, w_gate, w_up, dh))
    a, da = activation_ref(name, x64 @ gate.t())
    u = x64 @ up.t()
    dg, du = dh64 * u * da, dh64 * a
    return dg @ gate + du @ up, dg.t() @ x64, du.t() @ x64, dg, du


# ---------------------------------------------------------------- MXFP4
E2M1 = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)


def _pow2(e: torch.Tensor) -> torch.Tensor:
    """2^e in float64 from its bits (a device's pow and ldexp may be an ulp off)."""
    return ((e.long() + 1023) << 52).view(F64)


def mxfp4_quantize_ref(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """(values the rows stand for, float64 [R, C]; scale bytes int64 [R, C / 32]).
    E = max(floor(log2 max|x|) - 2, -127); nearest of E2M1 * 2^E, ties to the
    even code, 6 at the most; a block with an infinity or NaN is NaN (byte 255)."""
    R, C = x.shape
    b = x.to(F64).reshape(R, C // 32, 32)
    finite = torch.isfinite(b).all(-1)
    amax = torch.where(finite, b.abs().amax(-1), 1.0)
    E = (torch.frexp(amax)[1] - 3).clamp(min=-127)  # frexp: amax = m 2^e, m in [1/2, 1)
    E = torch.where(amax > 0, E, -127)
    t = (b.abs() * _pow2(-E)[..., None]).clamp(max=6.0)
    grid = torch.tensor(E2M1, dtype=F64, device=x.device)
    mid = (grid[1:] + grid[:-1]) / 2
    up = torch.bucketize(t, mid)                       # t on a midpoint goes down ...
    tie = (t == mid[up.clamp(max=6)]) & (up % 2 == 1)  # ... unless the lower code is odd
    code = up + tie.to(up.dtype)
    v = torch.copysign(grid[code], b) * _pow2(E)[..., None]
    v = torch.where(finite[..., None], v, float("nan"))
    return v.reshape(R, C), torch.where(finite, E + 127, 255).long()


def mxfp4_decode_ref(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """float64 values of packed codes [R, C / 2] (low nibble first) and scale bytes [R, C / 32]."""
    n = torch.stack((codes & 15, codes >> 4), -1).reshape(codes.shape[0], -1).long()
    grid = torch.tensor(E2M1 + tuple(-g for g in E2M1), dtype=F64, device=codes.device)
    unit = _pow2(scales.long() - 127)
    unit = torch.where(scales == 255, float("nan"), unit)
    return grid[n] * unit.repeat_interleave(32, 1)
