"""Gated feed-forward projection (``csrc/hstu_gated.hip``):

    g = x @ w_gate^T,  u = x @ w_up^T,  h = a(g) * u

with a = silu, gelu (the tanh form) or sigmoid; both products and the
activation are one kernel, and h is the only [.., F] tensor written.  Weights
are [F, D] with the contraction index contiguous, as ``fp8.bf16_gemm`` takes
them.  The UVQK projection (``hstu_compute_uqvk``) has SiLU on a column range
of one product, not the product of two.

* ``gated_linear``: differentiable, bf16, D a multiple of 256 and F of 128;
* ``gated_linear_fp8``: forward from e4m3 (``rms_norm_fp8``'s or
  ``fp8.quantize_e4m3_rows``' output), D a multiple of 128;
* ``gated_linear_fwd`` / ``gated_linear_bwd``: the two directions.

The backward takes g and u in fp32, kept by the forward or computed again
(``recompute``), and writes [dg | du], whose products with the weights and with
x are the bf16 projection GEMM and the token-axis weight gradient.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from . import _lib

ACTIVATIONS = {"silu": 0, "gelu": 1, "sigmoid": 2}
E4M3 = torch.float8_e4m3fn
Scaled = Tuple[torch.Tensor, torch.Tensor]


def _act(activation: str) -> int:
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation {activation!r} (one of {sorted(ACTIVATIONS)})")
    return ACTIVATIONS[activation]


FAR = 2 ** 24  # bytes between rows from which on the kernels' 32-bit offsets do not reach over a tile


def _rows2d(t: torch.Tensor, far: int = FAR) -> torch.Tensor:
    """[rows, width] with unit column stride and 16-byte aligned rows less than ``far`` bytes apart (a view
    such as one position of every sequence is copied where they are further)."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    s0, s1 = t.stride()
    apart = s0 * t.element_size()
    if s1 == 1 and t.data_ptr() % 16 == 0 and (t.shape[0] <= 1 or (s0 >= t.shape[1] and apart % 16 == 0 and apart < far)):
        return t
    t = t.contiguous()
    return t if t.data_ptr() % 16 == 0 else t.clone()


def _ld(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _check(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, dtype: torch.dtype, multiple: int) -> Tuple[int, int]:
    """(F, D)"""
    if x.dtype != dtype or w_gate.dtype != dtype or w_up.dtype != dtype:
        raise NotImplementedError(f"x, w_gate, w_up: {dtype} (got {x.dtype}, {w_gate.dtype}, {w_up.dtype})")
    device = x.device
    if not x.is_cuda or w_gate.device != device or w_up.device != device:
        raise NotImplementedError(f"x, w_gate, w_up: on one device (got {device}, {w_gate.device}, {w_up.device})")
    shape = w_gate.shape
    if x.dim() < 1 or len(shape) != 2 or w_up.shape != shape or shape[1] != x.shape[-1]:
        raise ValueError(f"x {tuple(x.shape)}, w_gate {tuple(shape)}, w_up {tuple(w_up.shape)}: expected "
                         "[.., D], [F, D], [F, D]")
    F, D = shape
    if D == 0 or F == 0 or D % multiple or F % 128:
        raise NotImplementedError(f"D = {D}, F = {F}: D a multiple of {multiple} and F of 128")
    if x.numel() // D >= 2 ** 31 - 256:
        raise NotImplementedError("x: fewer than 2^31 rows")
    return F, D


def gated_linear_fwd(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, activation: str = "silu",
                     keep: bool = False):
    """h [.., F] in bf16; with ``keep`` (h, gu): gu fp32 [rows, 2F] holds g and u for ``gated_linear_bwd``."""
    act = _act(activation)
    F, D = _check(x, w_gate, w_up, torch.bfloat16, 256)
    x2, g, u = _rows2d(x), _rows2d(w_gate), _rows2d(w_up)
    M = x2.shape[0]
    h = torch.empty(x.shape[:-1] + (F,), dtype=torch.bfloat16, device=x.device)
    gu = torch.empty((M, 2 * F), dtype=torch.float32, device=x.device) if keep else None
    if M > 0:
        _lib.launch("hstu_gated_fwd", x, x2.data_ptr(), _ld(x2), g.data_ptr(), _ld(g), u.data_ptr(), _ld(u), M, F, D,
                    act, h.data_ptr(), F, _lib.ptr(gu))
    return (h, gu) if keep else h


def gated_linear_bwd(dh: torch.Tensor, x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor,
                     activation: str = "silu", need_dx: bool = True, need_dw: bool = True,
                     gu: Optional[torch.Tensor] = None
                     ) -> Tuple[Optional[torch.Tensor], Optional[torch.Tensor], Optional[torch.Tensor]]:
    """(dx, dw_gate, dw_up) in bf16; None for what is not needed.  ``gu``: what
    ``gated_linear_fwd(keep=True)`` kept; without it g and u are computed again."""
    act = _act(activation)
    F, D = _check(x, w_gate, w_up, torch.bfloat16, 256)
    device = x.device
    if dh.shape != x.shape[:-1] + (F,) or dh.dtype != torch.bfloat16 or dh.device != device:
        raise ValueError(f"dh {tuple(dh.shape)} {dh.dtype}; expected {tuple(x.shape[:-1] + (F,))} bf16 on {device}")
    x2, g, u, d2 = _rows2d(x), _rows2d(w_gate), _rows2d(w_up), _rows2d(dh, 2 ** 63)  # dh: 64-bit offsets
    M = x2.shape[0]
    if gu is not None and (gu.shape != (M, 2 * F) or gu.dtype != torch.float32 or not gu.is_contiguous()
                           or gu.device != device):
        raise ValueError(f"gu {tuple(gu.shape)} {gu.dtype}; expected contiguous fp32 [{M}, {2 * F}] on {device}")
    if M == 0:
        dw = torch.zeros((2 * F, D), dtype=torch.bfloat16, device=device)
        return torch.empty_like(x) if need_dx else None, dw[:F] if need_dw else None, dw[F:] if need_dw else None
    dgu = torch.empty((M, 2 * F), dtype=torch.bfloat16, device=device)
    if gu is not None:
        _lib.launch("hstu_gated_bwd_kept", x, d2.data_ptr(), _ld(d2), gu.data_ptr(), M, F, act, dgu.data_ptr(), 2 * F)
    else:
        _lib.launch("hstu_gated_bwd", x, d2.data_ptr(), _ld(d2), x2.data_ptr(), _ld(x2), g.data_ptr(), _ld(g),
                    u.data_ptr(), _ld(u), M, F, D, act, dgu.data_ptr(), 2 * F)
    dx = dg = du = None
    bf16 = _lib.HSTU_DTYPE_BF16
    if need_dx:  # the contraction runs over both halves of dgu: the weights side by side, transposed
        wt = torch.empty((D, 2 * F), dtype=torch.bfloat16, device=device)
        dx = torch.empty(x.shape, dtype=torch.bfloat16, device=device)
        _lib.launch("hstu_gated_transpose", x, g.data_ptr(), _ld(g), u.data_ptr(), _ld(u), F, D, wt.data_ptr(), 2 * F)
        _lib.launch("hstu_bf16_gemm", x, dgu.data_ptr(), 2 * F, wt.data_ptr(), 2 * F, None, None, 0, dx.data_ptr(), D, M,
                    D, 2 * F, 0, 0)
    if need_dw:
        split = _wgrad_split(M, max(2 * F, _ld(x2)))
        if split < 0:  # rows too far apart for its offsets
            x2, split = x2.contiguous(), _wgrad_split(M, 2 * F)
        nbytes = _lib.fn("hstu_wgrad_workspace_bytes")(M, 2 * F, D, split)
        ws = torch.empty(max(nbytes, 1), dtype=torch.uint8, device=device)
        dw = torch.empty((2 * F, D), dtype=torch.bfloat16, device=device)
        _lib.launch("hstu_wgrad", x, bf16, dgu.data_ptr(), 2 * F, bf16, x2.data_ptr(), _ld(x2), M, 2 * F, D, None, None,
                    dw.data_ptr(), D, bf16, None, split, ws.data_ptr(), nbytes)
        dg, du = dw[:F], dw[F:]
    return dx, dg, du


# Keeping g and u costs 16 bytes of memory traffic a value (written and read in
# fp32), computing them again 4 D operations: equal near D = 1200 at the rates that
# these kernels reach.  Measured (us on the device a training step, computed again /
# kept): 37 429 rows x 512 -> 2048 659 / 794, 16 384 x 768 -> 3584 698 / 770, 16 384 x
# 1024 -> 4096 948 / 1013, 16 384 x 1280 -> 5120 1519 / 1493, 16 384 x 2048 -> 5632
# 2585 / 2322, 8192 x 4096 -> 10240 4347 / 3584, 512 x 2048 -> 5632 177 / 156.
RECOMPUTE_BELOW = 1280


def _wgrad_split(T: int, ld: int) -> int:
    """Token ranges for the weight gradient: the kernel's own choice (0), more where
    a range's rows would pass its 32-bit offsets; -1 where none would do."""
    most = (2 ** 31) // (2 * ld) - 256
    return -1 if most < 256 else 0 if T <= most else -(-T // most)


class GatedLinearFunction(torch.autograd.Function):
    """Autograd of the gated projection: keeps x, the weights and, with ``keep``, g and u in fp32."""

    @staticmethod
    def forward(ctx, x, w_gate, w_up, activation, keep):
        h = gated_linear_fwd(x, w_gate, w_up, activation, keep)
        h, gu = h if keep else (h, None)
        _lib.guard_graph(ctx, x)
        ctx.activation = activation
        ctx.save_for_backward(x, w_gate, w_up, gu)
        return h

    @staticmethod
    def backward(ctx, dh):
        if torch.is_grad_enabled():  # only under create_graph
            raise NotImplementedError("second derivatives (create_graph=True)")
        _lib.no_tangent("the backward of gated_linear", dh)
        x, w_gate, w_up, gu = ctx.saved_tensors
        need_x, need_g, need_u = ctx.needs_input_grad[:3]
        dx, dg, du = gated_linear_bwd(dh, x, w_gate, w_up, ctx.activation, need_x, need_g or need_u, gu)
        return dx, dg if need_g else None, du if need_u else None, None, None


def gated_linear(x: torch.Tensor, w_gate: torch.Tensor, w_up: torch.Tensor, activation: str = "silu",
                 recompute: Optional[bool] = None) -> torch.Tensor:
    """a(x @ w_gate^T) * (x @ w_up^T): x [.., D], weights [F, D], h [.., F], bf16.
    Differentiable in x and both weights.  ``recompute``: the backward computes g
    and u again (nothing but x and the weights is kept) instead of keeping them
    in fp32, 8 bytes a value of h; None: where that is the faster way (D < 1280).
    The gradients are the same bytes.  Not differentiable a second time, nor in
    forward mode."""
    _lib.no_tangent("gated_linear", x, w_gate, w_up)
    if not (torch.is_grad_enabled() and (x.requires_grad or w_gate.requires_grad or w_up.requires_grad)):
        return gated_linear_fwd(x, w_gate, w_up, activation)
    if recompute is None:
        recompute = x.shape[-1] < RECOMPUTE_BELOW
    return GatedLinearFunction.apply(x, w_gate, w_up, activation, not recompute)


def _scale(name: str, s: torch.Tensor, n: int, x: torch.Tensor) -> Tuple[torch.Tensor, int]:
    if s.device != x.device or s.numel() not in (1, n):
        raise ValueError(f"{name}: 1 or {n} values on {x.device} (got {tuple(s.shape)} on {s.device})")
    if s.dtype != torch.float32 or s.dim() != 1 or not s.is_contiguous():
        s = s.detach().to(torch.float32).reshape(-1).contiguous()
    return s, 1 if s.numel() > 1 else 0


def gated_linear_fp8(x8: torch.Tensor, x_scale: torch.Tensor, gate: Scaled, up: Scaled, activation: str = "silu"
                     ) -> torch.Tensor:
    """The forward from e4m3: x8 [.., D] with one fp32 scale or one a row, and
    ``gate``, ``up`` as pairs (e4m3 [F, D], scale: one or [F]).  h [.., F] in bf16,
    which carries no gradient; inputs that require grad are refused while grad mode is on."""
    act = _act(activation)
    (g8, gs), (u8, us) = gate, up
    _lib.forward_only("gated_linear_fp8", x8, x_scale, g8, gs, u8, us)
    F, D = _check(x8, g8, u8, E4M3, 128)
    x2, g2, u2 = _rows2d(x8), _rows2d(g8), _rows2d(u8)
    M = x2.shape[0]
    xs, xm = _scale("x_scale", x_scale, M, x8)
    gs, gm = _scale("gate scale", gs, F, x8)
    us, um = _scale("up scale", us, F, x8)
    h = torch.empty(x8.shape[:-1] + (F,), dtype=torch.bfloat16, device=x8.device)
    if M > 0:
        _lib.launch("hstu_gated_fwd_fp8", x8, x2.data_ptr(), _ld(x2), xs.data_ptr(), xm, g2.data_ptr(), _ld(g2),
                    gs.data_ptr(), gm, u2.data_ptr(), _ld(u2), us.data_ptr(), um, M, F, D, act, h.data_ptr(), F)
    return h
