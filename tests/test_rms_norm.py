"""RMS norm with the residual's addition: the kernels against the float64
formulas (``oracle/feed_forward_oracle.py``), its refusals, streams and graphs.

Tolerances.  A sum over a row is at most 32 additions in a thread, 6 across
the wave and 16 across the waves: 54 roundings of 2^-24, under 2^-18 of the
sum of the magnitudes; the reciprocal square root, the products and the mean
add fewer than 8 more.  So fp32 results are within FP32 = 2^-17 of the
magnitudes that meet in them, and a rounding to bf16 (e4m3) adds 2^-8 (2^-4) of
the value, below e4m3's normal range half of its 2^-9 step.  dweight also sums
the rows: one more rounding for each (at most) and 64 for the joins."""

import pytest
import torch

from oracle import feed_forward_oracle as orc

DEV = "cuda"
EPS = 1e-6
FP32 = 2.0 ** -17
HALF = {torch.bfloat16: 2.0 ** -8, torch.float32: 0.0}
gpu = pytest.mark.gpu


def make(rows, D, dtype, seed, scale=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(rows, D, generator=g) * scale).to(dtype)


def make_weight(D, dtype, seed=9):
    return (1.0 + 0.3 * torch.randn(D, generator=torch.Generator().manual_seed(seed))).to(dtype)


def within(got, want, tol, what):
    got, want = got.double().cpu(), want.double().cpu()
    off = (got - want).abs()
    tol = tol.double().cpu() if torch.is_tensor(tol) else tol
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} off, worst {off[bad].max():.3e}"


SHAPES = [(1, 1), (3, 7), (5, 64), (1, 512), (33, 512), (130, 513), (17, 520), (4, 1000), (9, 1024), (2, 1032),
          (6, 2048), (3, 4096), (5, 5120), (3, 8192), (2, 8200), (3, 16384), (2, 16380), (1500, 1032), (600, 8200), (2100, 256)]


@gpu
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,D", SHAPES)
def test_forward_and_backward(hip_lib, rows, D, dtype, residual):
    import hstu_amd

    wdt = torch.bfloat16 if D % 16 == 0 else torch.float32
    x, w = make(rows, D, dtype, 1).to(DEV), make_weight(D, wdt).to(DEV)
    r = make(rows, D, dtype, 2, 3.0).to(DEV) if residual else None
    dy, dh = make(rows, D, dtype, 3).to(DEV), make(rows, D, dtype, 4).to(DEV) if residual else None
    leaves = [t.requires_grad_(True) for t in (x, r, w) if t is not None]
    out = hstu_amd.rms_norm(x, w, EPS, residual=r)
    y, h = out if residual else (out, x)
    assert y.dtype == dtype and y.shape == x.shape
    if residual:
        assert torch.equal(h, (x.float() + r.float()).to(dtype))
    yr, _ = orc.rms_norm_ref(h.detach(), w.detach(), EPS)
    within(y.detach(), yr, yr.abs() * (HALF[dtype] + FP32), "y")
    grads = torch.autograd.grad([y, h] if residual else [y], leaves, [dy, dh] if residual else [dy])
    dx, dw = grads[0], grads[-1]
    dxr, dwr, bx, bw = orc.rms_norm_bwd_ref(dy, h.detach(), w.detach(), EPS, dh)
    within(dx, dxr, dxr.abs() * HALF[dtype] + bx * 2 * FP32, "dx")
    within(dw, dwr, dwr.abs() * HALF[wdt] + bw * (FP32 + (rows + 64) * 2.0 ** -24), "dweight")
    assert dw.dtype == wdt
    if residual:
        assert torch.equal(grads[1], dx)


@gpu
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,D,blocks", [(1700, 2048, 768), (1700, 4096, 768), (1600, 2050, 768), (600, 5120, 256),
                                           (520, 8192, 256), (600, 4100, 256)])
def test_blocks_of_several_rows(hip_lib, rows, D, dtype, residual, blocks):
    """Twice as many rows as the backward has blocks: the loads ahead go round more than once, and end."""
    import hstu_amd._lib as lib

    assert lib.fn("hstu_rms_norm_bwd_workspace_bytes")(rows, D) == blocks * D * 4 and rows > 2 * blocks
    test_forward_and_backward(hip_lib, rows, D, dtype, residual)


@gpu
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,D", [(1, 1), (3, 7), (33, 512), (5, 520), (4, 1000), (6, 2048), (3, 5120), (2, 16380)])
def test_e4m3_output(hip_lib, rows, D, dtype, residual):
    import hstu_amd

    x, w = make(rows, D, dtype, 5).to(DEV), make_weight(D, torch.float32).to(DEV)
    x[rows // 2] = 0  # a row of zeros has scale 1 / 448
    r = torch.zeros_like(x) if residual else None
    out = hstu_amd.rms_norm_fp8(x, w, EPS, residual=r)
    y8, s = out[0], out[1]
    if residual:
        assert torch.equal(out[2], x)
    yr, _ = orc.rms_norm_ref(x, w, EPS)
    top = yr.abs().amax(-1)
    sr = torch.where(top > 0, top, 1.0) / 448.0
    within(s, sr, sr * FP32, "scale")
    sd = s.double()[:, None]
    within(y8.float().double() * sd, yr, yr.abs() * (2.0 ** -4 + 2 * FP32) + sd * 2.0 ** -10, "y8")
    assert torch.equal(s[rows // 2], torch.tensor(1.0 / 448.0, device=DEV)) and not y8[rows // 2].float().any()
    # one given scale: saturates at 448 of it
    given = torch.tensor([float(top.max()) / 300.0], device=DEV)
    y8, s1 = hstu_amd.rms_norm_fp8(x, w, EPS, scale=given)[:2]
    if not given:  # the only row is the one of zeros: 0 / 0
        assert y8.float().isnan().all()
        return
    want = yr.clamp(-448 * given.double(), 448 * given.double())
    within(y8.float().double() * given.double(), want, want.abs() * (2.0 ** -4 + 2 * FP32) + given.double() * 2.0 ** -10,
           "y8 at a given scale")
    assert s1.shape == (1,) and torch.equal(s1, given)
    tiny = torch.tensor([float(top.max()) / 4480.0], device=DEV)
    y8, _ = hstu_amd.rms_norm_fp8(x, w, EPS, scale=tiny)
    assert float(y8.float().abs().max()) == 448.0


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_e4m3_of_the_smallest_rows(hip_lib, dtype):
    """Scales below 2^-126, whose reciprocal no fp32 value holds.  They and y are
    multiples of 2^-149: half of one more for each, 448 of them for the scale's."""
    import hstu_amd

    x = make(6, 520, dtype, 5, 3e-39).to(DEV)
    x[:, ::7] = 0
    w = make_weight(520, torch.float32).to(DEV)
    for eps in (1e-6, 1e-2):
        y8, s = hstu_amd.rms_norm_fp8(x, w, eps)
        yr, _ = orc.rms_norm_ref(x, w, eps)
        sr = yr.abs().amax(-1) / 448.0
        assert float(sr.max()) < 2.0 ** -120
        within(s, sr, sr * 2 * FP32 + 2.0 ** -149, "scale")
        sd = s.double()[:, None]
        within(y8.float().double() * sd, yr, yr.abs() * (2.0 ** -4 + 4 * FP32) + sd * 2.0 ** -10 + 450 * 2.0 ** -150, "y8")


@gpu
def test_non_finite_rows_stay_in_their_row(hip_lib):
    import hstu_amd

    x = make(6, 520, torch.bfloat16, 6).to(DEV)
    w = make_weight(520, torch.float32).to(DEV)
    clean8, clean_s = hstu_amd.rms_norm_fp8(x, w, EPS)
    clean = hstu_amd.rms_norm(x, w, EPS)
    x[1, 3], x[4, 519] = float("nan"), float("inf")
    y = hstu_amd.rms_norm(x, w, EPS)
    y8, s = hstu_amd.rms_norm_fp8(x, w, EPS)
    keep = torch.tensor([0, 2, 3, 5], device=DEV)
    assert torch.equal(y[keep], clean[keep]) and torch.equal(s[keep], clean_s[keep])
    assert torch.equal(y8[keep].float(), clean8[keep].float())
    assert y[1].isnan().all() and s[1].isnan() and y8[1].float().isnan().all()
    assert y[4, 519].isnan() and not y[4, :519].float().any()  # 1 / inf = 0, inf * 0 = NaN
    assert s[4].isnan()


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("D", [520, 513, 1032, 5120, 16384])
def test_non_finite_weights_and_scales(hip_lib, D, dtype):
    """max|y| of a row with a NaN is NaN, wherever the NaN comes from, and so are its scale and its row; an
    infinite scale takes every finite y to zero."""
    import hstu_amd

    x, w = make(5, D, dtype, 6).to(DEV), make_weight(D, torch.float32).to(DEV)
    x[3] = 0  # its y is 0, NaN where the weight is not finite
    bad = w.clone()
    bad[D // 2] = float("nan")
    y8, s = hstu_amd.rms_norm_fp8(x, bad, EPS)
    assert s.isnan().all() and y8.float().isnan().all()
    y8, s = hstu_amd.rms_norm_fp8(x, bad, EPS, scale=torch.ones(1, device=DEV))  # a given scale: the column alone
    assert y8[:, D // 2].float().isnan().all() and int(y8.float().isnan().sum()) == 5
    bad[D // 2] = float("inf")
    y8, s = hstu_amd.rms_norm_fp8(x, bad, EPS)
    live = torch.tensor([0, 1, 2, 4], device=DEV)
    assert s[live].isinf().all() and s[3].isnan() and y8[3].float().isnan().all()
    assert y8[live, D // 2].float().isnan().all() and int(y8[live].float().isnan().sum()) == 4
    assert not y8[live].float().nan_to_num(0).any()
    y8, _ = hstu_amd.rms_norm_fp8(x, w, EPS, scale=torch.full((1,), float("inf"), device=DEV))
    assert not y8.float().any()
    y8, _ = hstu_amd.rms_norm_fp8(x, w, EPS, scale=torch.full((1,), float("nan"), device=DEV))
    assert y8.float().isnan().all()


@gpu
@pytest.mark.parametrize("shape", [(0, 512), (2, 0, 512), (2, 3, 512), (512,)])
def test_leading_dimensions_and_no_rows(hip_lib, shape):
    import hstu_amd

    x = torch.randn(shape, generator=torch.Generator().manual_seed(0)).to(DEV, torch.bfloat16).requires_grad_(True)
    w = make_weight(512, torch.float32).to(DEV).requires_grad_(True)
    r = torch.zeros_like(x).requires_grad_(True)
    y, h = hstu_amd.rms_norm(x, w, EPS, residual=r)
    assert y.shape == x.shape and h.shape == x.shape
    (y.float().sum() + h.float().sum()).backward()
    assert x.grad.shape == x.shape and r.grad.shape == x.shape and w.grad.shape == w.shape
    if x.numel() == 0:
        assert not w.grad.any()
    y8, s, h = hstu_amd.rms_norm_fp8(x.detach(), w.detach(), EPS, residual=r.detach())
    assert y8.shape == x.shape and s.numel() == x.numel() // 512 and h.shape == x.shape


@gpu
@pytest.mark.parametrize("offset", [8, 3])
def test_strided_rows(hip_lib, offset):
    """Column slices of wider buffers, 16-byte aligned and not, give what contiguous copies do."""
    import hstu_amd

    x, r, dy = (make(37, 1200, torch.bfloat16, 10 + i).to(DEV)[:, offset:offset + 512] for i in range(3))
    w = make_weight(512, torch.float32).to(DEV)
    y, h, rstd, _ = hstu_amd.rms_norm_fwd(x, w, EPS, residual=r)
    y2, h2, rstd2, _ = hstu_amd.rms_norm_fwd(x.contiguous(), w, EPS, residual=r.contiguous())
    assert torch.equal(y, y2) and torch.equal(h, h2) and torch.equal(rstd, rstd2)
    dx, dw = hstu_amd.rms_norm_bwd(dy, x, w, rstd, dh=r)
    dx2, dw2 = hstu_amd.rms_norm_bwd(dy.contiguous(), x.contiguous(), w, rstd, dh=r.contiguous())
    assert torch.equal(dx, dx2) and torch.equal(dw, dw2)


@gpu
def test_gradient_against_differences(hip_lib):
    """The kernel's gradient along a direction against a difference quotient of the float64 formula."""
    import hstu_amd

    rows, D = 7, 200
    x, r = make(rows, D, torch.float32, 20).to(DEV), make(rows, D, torch.float32, 21).to(DEV)
    w = make_weight(D, torch.float32).to(DEV)
    dy, dh = make(rows, D, torch.float32, 22).to(DEV), make(rows, D, torch.float32, 23).to(DEV)
    for t in (x, r, w):
        t.requires_grad_(True)
    y, h = hstu_amd.rms_norm(x, w, EPS, residual=r)
    dx, dr, dw = torch.autograd.grad((y, h), (x, r, w), (dy, dh))

    def loss(hh, ww):
        return float((orc.rms_norm_ref(hh, ww, EPS)[0] * dy.double()).sum() + (hh * dh.double()).sum())

    vx, vw = make(rows, D, torch.float64, 24).to(DEV), make(1, D, torch.float64, 25).to(DEV)[0]
    h64, w64, e = h.detach().double(), w.detach().double(), 1e-5
    diff = (loss(h64 + e * vx, w64 + e * vw) - loss(h64 - e * vx, w64 - e * vw)) / (2 * e)
    got = float((dx.double() * vx).sum() + (dw.double() * vw).sum())
    _, _, bx, bw = orc.rms_norm_bwd_ref(dy, h.detach(), w.detach(), EPS, dh)
    # the gradients' own rounding, and the quotient's: e^2 of the third derivative and 2^-52 / e of the loss
    tol = float((bx * vx.abs()).sum() + (bw * vw.abs()).sum()) * 2 * FP32 + 1e-4
    assert abs(got - diff) <= tol
    assert torch.equal(dx, dr)


@gpu
def test_only_one_output_used(hip_lib):
    import hstu_amd

    x, r = (make(4, 512, torch.bfloat16, 30 + i).to(DEV).requires_grad_(True) for i in range(2))
    w = make_weight(512, torch.float32).to(DEV).requires_grad_(True)
    g = make(4, 512, torch.bfloat16, 32).to(DEV)
    _, h = hstu_amd.rms_norm(x, w, EPS, residual=r)
    dx, dr = torch.autograd.grad(h, (x, r), g)
    assert torch.equal(dx, g) and torch.equal(dr, g)
    y, h = hstu_amd.rms_norm(x, w, EPS, residual=r)
    dx, dr, dw = torch.autograd.grad(y, (x, r, w), g)
    dxr, dwr, bx, bw = orc.rms_norm_bwd_ref(g, h.detach(), w.detach(), EPS)
    within(dx, dxr, dxr.abs() * HALF[torch.bfloat16] + bx * 2 * FP32, "dx")
    within(dw, dwr, bw * 2 * FP32, "dweight")


@gpu
def test_same_bytes_again_and_alone(hip_lib):
    """Deterministic, and a row's result does not depend on its batch."""
    import hstu_amd

    x, dy = make(3001, 512, torch.bfloat16, 40).to(DEV), make(3001, 512, torch.bfloat16, 41).to(DEV)
    w = make_weight(512, torch.float32).to(DEV)
    y, _, rstd, _ = hstu_amd.rms_norm_fwd(x, w, EPS)
    dx, dw = hstu_amd.rms_norm_bwd(dy, x, w, rstd)
    for _ in range(3):
        dx2, dw2 = hstu_amd.rms_norm_bwd(dy, x, w, rstd)
        assert torch.equal(dx, dx2) and torch.equal(dw, dw2)
    y1, _, rstd1, _ = hstu_amd.rms_norm_fwd(x[1234:1235], w, EPS)
    assert torch.equal(y1[0], y[1234]) and torch.equal(rstd1[0], rstd[1234])


@gpu
def test_past_32_bit_offsets(hip_lib):
    import hstu_amd

    rows, D = 2 ** 22 + 5, 512  # over 2^31 values, 4 GiB
    x = torch.zeros((rows, D), dtype=torch.bfloat16, device=DEV)
    x[-9:] = make(9, D, torch.bfloat16, 50).to(DEV)
    w = make_weight(D, torch.float32).to(DEV)
    y, _, rstd, _ = hstu_amd.rms_norm_fwd(x, w, EPS)
    small, _, rstd2, _ = hstu_amd.rms_norm_fwd(x[-9:].clone(), w, EPS)
    assert torch.equal(y[-9:], small) and torch.equal(rstd[-9:], rstd2) and not y[:-9].any()
    dx, _ = hstu_amd.rms_norm_bwd(y, x, w, rstd)
    dx2, _ = hstu_amd.rms_norm_bwd(small, x[-9:].clone(), w, rstd2)
    assert torch.equal(dx[-9:], dx2)


@gpu
def test_side_stream_and_graph(hip_lib):
    import hstu_amd

    x, r = make(257, 512, torch.bfloat16, 60).to(DEV), make(257, 512, torch.bfloat16, 61).to(DEV)
    dy = make(257, 512, torch.bfloat16, 62).to(DEV)
    w = make_weight(512, torch.float32).to(DEV)

    def step():
        y, h, rstd, _ = hstu_amd.rms_norm_fwd(x, w, EPS, residual=r)
        return (y, h) + hstu_amd.rms_norm_bwd(dy, h, w, rstd, dh=dy) + hstu_amd.rms_norm_fp8(x, w, EPS)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    torch.cuda.current_stream().wait_stream(side)
    want = step()
    for a, b in zip(on_side, want):
        assert torch.equal(a.float(), b.float())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(4):
        x.copy_(make(257, 512, torch.bfloat16, 70 + k))
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, step()):
            assert torch.equal(a.float(), b.float()), k


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,D", [(1, 512), (37, 512), (5, 513), (300, 5120)])
def test_in_place(hip_lib, rows, D, dtype):
    """The C entry with h on x or on the residual, and y on x or on the residual; columns of one buffer beside each other."""
    import hstu_amd
    import hstu_amd._lib as lib

    f = lib.fn("hstu_rms_norm_fwd")
    code = lib.HSTU_DTYPE_BF16 if dtype == torch.bfloat16 else lib.HSTU_DTYPE_FP32
    x, r, w = make(rows, D, dtype, 1).to(DEV), make(rows, D, dtype, 2, 3.0).to(DEV), make_weight(D, torch.float32).to(DEV)
    y0, h0, _, _ = hstu_amd.rms_norm_fwd(x, w, EPS, residual=r)
    alone, _, _, _ = hstu_amd.rms_norm_fwd(x, w, EPS)

    def call(x, ldx, r, ldr, h, ldh, y, ldy):
        return f(code, x.data_ptr(), ldx, lib.ptr(r), ldr, w.data_ptr(), lib.HSTU_DTYPE_FP32, EPS, rows, D, lib.ptr(h), ldh,
                 y.data_ptr(), ldy, code, None, None, None, lib.stream(x))

    for on in ("h on x", "h on residual", "y on x", "y on residual"):
        a, b, new = x.clone(), r.clone(), torch.empty_like(x)
        h, y = {"h on x": (a, new), "h on residual": (b, new), "y on x": (new, a), "y on residual": (new, b)}[on]
        assert call(a, D, b, D, h, D, y, D) == 0
        assert torch.equal(h, h0) and torch.equal(y, y0), on
    a = x.clone()
    assert call(a, D, None, 0, None, 0, a, D) == 0 and torch.equal(a, alone)
    wide = torch.full((rows, 4 * D), 7.0, dtype=dtype, device=DEV)
    a, b, h, y = (wide[:, i * D:(i + 1) * D] for i in range(4))
    a.copy_(x), b.copy_(r)
    assert call(a, 4 * D, b, 4 * D, h, 4 * D, y, 4 * D) == 0
    assert torch.equal(a, x) and torch.equal(b, r) and torch.equal(h, h0) and torch.equal(y, y0)


# ---------------------------------------------------------------- refusals, without a GPU
def test_c_entry_refuses_overlaps():
    """An output that lies on rows which another row group has still to read, and an e4m3 y on anything."""
    import hstu_amd._lib as lib

    f = lib.fn("hstu_rms_norm_fwd")
    BF, F32, F8 = lib.HSTU_DTYPE_BF16, lib.HSTU_DTYPE_FP32, lib.HSTU_DTYPE_FP8_E4M3
    X, R, H, Y, D, rows = 1 << 20, 2 << 20, 3 << 20, 4 << 20, 64, 8  # stand-in addresses, never read

    def fwd(dtype=BF, x=X, ldx=D, res=R, ldr=D, h=H, ldh=D, y=Y, ldy=D, od=None, rows=rows):
        out8 = od == F8
        return f(dtype, x, ldx, res, ldr, 64, F32, 1e-6, rows, D, h, ldh, y, ldy, dtype if od is None else od, None,
                 64 if out8 else None, None, None)

    for dtype, es in ((BF, 2), (F32, 4)):
        span = rows * D * es
        for rows_ in (1, rows):
            for bad in (dict(od=F8, y=X), dict(od=F8, y=R), dict(od=F8, y=H), dict(od=F8, y=X, res=None, h=None),
                        dict(od=F8, y=X, ldy=D * es)):
                assert fwd(dtype, rows=rows_, **bad) == lib.HSTU_E_BAD_ARG, bad
        for bad in (dict(od=F8, y=X + span - 16), dict(od=F8, y=X - D * rows + 16), dict(y=X + es), dict(y=X + span - es),
                    dict(y=X - span + es), dict(h=X + es), dict(h=R - es), dict(y=R + es), dict(y=X, ldy=D + 8),
                    dict(h=X, ldh=2 * D), dict(y=H), dict(y=X, h=X), dict(y=X, res=None, h=None, ldy=2 * D),
                    dict(x=X, ldx=2 * D, y=X + es * (D - 8), ldy=2 * D), dict(x=X, ldx=2 * D, y=X + es * (D + 8), ldy=2 * D)):
            assert fwd(dtype, **bad) == lib.HSTU_E_BAD_ARG, bad


def test_refusals():
    import hstu_amd
    from hstu_amd.hstu_rms_norm import MAX_D

    w = torch.ones(8)
    with pytest.raises(NotImplementedError):
        hstu_amd.rms_norm(torch.ones(2, 8), w)  # not on a device
    with pytest.raises(NotImplementedError):
        hstu_amd.rms_norm(torch.ones(2, 8, dtype=torch.float16), w)
    with pytest.raises(NotImplementedError):
        hstu_amd.rms_norm(torch.ones(2, MAX_D + 8), torch.ones(MAX_D + 8))
    with pytest.raises(NotImplementedError):
        hstu_amd.rms_norm(torch.ones(()), w)


@gpu
def test_refusals_on_device(hip_lib):
    import hstu_amd

    x, w = torch.ones(2, 8, device=DEV), torch.ones(8, device=DEV)
    for bad in (torch.ones(1, 8, device=DEV), torch.ones(2, 8, device=DEV, dtype=torch.bfloat16), torch.ones(2, 8)):
        with pytest.raises(ValueError):
            hstu_amd.rms_norm(x, w, residual=bad)
    for bad in (torch.ones(7, device=DEV), torch.ones(8), torch.ones(1, 8, device=DEV)):
        with pytest.raises(ValueError):
            hstu_amd.rms_norm(x, bad)
    with pytest.raises(NotImplementedError):
        hstu_amd.rms_norm(x, w.half())
    with pytest.raises(ValueError):
        hstu_amd.rms_norm_fp8(x, w, scale=torch.ones(2, device=DEV))
    with pytest.raises(ValueError):
        hstu_amd.rms_norm_fwd(x, w, scale=torch.ones(1, device=DEV))
    with pytest.raises(ValueError):
        hstu_amd.rms_norm_bwd(x, x, w, torch.ones(3, device=DEV))


def test_c_entry_refusals():
    """Bad arguments are refused before any launch (no device is touched)."""
    import hstu_amd._lib as lib

    f, b, n = (lib.fn("hstu_rms_norm_" + k) for k in ("fwd", "bwd", "bwd_workspace_bytes"))
    BF, F32, F8 = lib.HSTU_DTYPE_BF16, lib.HSTU_DTYPE_FP32, lib.HSTU_DTYPE_FP8_E4M3
    P = 64  # a stand-in address, never read

    def fwd(dtype=BF, x=P, ldx=512, res=None, ldr=0, w=P, pd=F32, rows=4, D=512, h=None, ldh=0, y=P, ldy=512, od=BF,
            sin=None, sout=None):
        return f(dtype, x, ldx, res, ldr, w, pd, 1e-6, rows, D, h, ldh, y, ldy, od, sin, sout, None, None)

    assert fwd(dtype=F8) == lib.HSTU_E_BAD_ARG
    assert fwd(od=F32) == lib.HSTU_E_BAD_ARG
    assert fwd(pd=F8) == lib.HSTU_E_BAD_ARG
    assert fwd(ldx=511) == lib.HSTU_E_BAD_ARG and fwd(ldy=511) == lib.HSTU_E_BAD_ARG
    assert fwd(rows=-1) == lib.HSTU_E_BAD_ARG and fwd(D=0) == lib.HSTU_E_BAD_ARG
    assert fwd(x=None) == lib.HSTU_E_BAD_ARG and fwd(w=None) == lib.HSTU_E_BAD_ARG and fwd(y=None) == lib.HSTU_E_BAD_ARG
    assert fwd(res=P, ldr=512, h=None, ldh=512) == lib.HSTU_E_BAD_ARG
    assert fwd(res=P, ldr=512, h=P, ldh=100) == lib.HSTU_E_BAD_ARG
    assert fwd(od=F8) == lib.HSTU_E_BAD_ARG and fwd(od=F8, sin=P, sout=P) == lib.HSTU_E_BAD_ARG
    assert fwd(D=16385, ldx=40000, ldy=40000) == lib.HSTU_E_UNSUPPORTED
    assert fwd(x=65) == lib.HSTU_E_UNSUPPORTED
    assert fwd(rows=0) == 0
    assert n(-1, 512) == -1 and n(4, 0) == -1 and n(4, 16385) == -1 and n(0, 512) == 2048 and n(5000, 512) > 2048

    def bwd(rows=4, D=512, dy=P, ld=512, dw=P, dwt=F32, ws=P, nb=1 << 30, rstd=P, dtype=BF):
        return b(dtype, dy, ld, P, 512, None, 0, P, F32, rstd, rows, D, P, 512, dw, dwt, ws, nb, None)

    assert bwd(dtype=F8) == lib.HSTU_E_BAD_ARG and bwd(dwt=F8) == lib.HSTU_E_BAD_ARG
    assert bwd(ld=100) == lib.HSTU_E_BAD_ARG and bwd(dw=None) == lib.HSTU_E_BAD_ARG
    assert bwd(dy=None) == lib.HSTU_E_BAD_ARG and bwd(rstd=None) == lib.HSTU_E_BAD_ARG
    assert bwd(nb=100) == lib.HSTU_E_BAD_ARG and bwd(ws=None) == lib.HSTU_E_BAD_ARG
    assert bwd(rstd=66) == lib.HSTU_E_UNSUPPORTED
