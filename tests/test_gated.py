"""Gated feed-forward projection: the kernels against the float64 formulas
(``oracle/feed_forward_oracle.py``), gradients, refusals, streams and graphs.

Tolerances.  A sum of n products in the matrix cores is n additions, each off by
at most 2^-23 of the sum of the magnitudes S (a unit: they need not round to
nearest); scales and the activation add fewer than 16 such units, its argument's
2^-24 |z| among them (|z| <= 88 where it matters: 2^-17 of a(g) u).  |a'| < 1.13 and
|a''| < 1.  The one rounding of h, dg and du is 2^-8 of the value.  dx and dW sum dg
and du as they are rounded: 2^-8 of the magnitudes that meet, the sum's own
units and their own rounding.  Rounding errors are independent and spread over
their range, so the 2-norm of two of them is under sqrt(2 / 3) 2^-8 of the result's
where the terms are independent too: NORM = 2^-8."""

import pytest
import torch

from oracle import feed_forward_oracle as orc

DEV = "cuda"
ACTS = ["silu", "gelu", "sigmoid"]
ULP, HALF, NORM, ARG = 2.0 ** -23, 2.0 ** -8, 2.0 ** -8, 2.0 ** -17
gpu = pytest.mark.gpu


def rnd(shape, seed, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(torch.bfloat16)


def weights(F, D, seed=0):
    return rnd((F, D), 100 + seed, 1.5 * D ** -0.5).to(DEV), rnd((F, D), 200 + seed, D ** -0.5).to(DEV)


def within(got, want, tol, what):
    off = (got.double() - want).abs()
    bad = ~(off <= tol)
    assert not bad.any(), f"{what}: {int(bad.sum())} of {bad.numel()} off, worst {off[bad].max():.3e}"


def h_bound(x, wg, wu, name):
    """(h, what h may be off)."""
    x, wg, wu = x.double(), wg.double(), wu.double()
    g, u = x @ wg.t(), x @ wu.t()
    sg, su = x.abs() @ wg.abs().t(), x.abs() @ wu.abs().t()
    a, _ = orc.activation_ref(name, g)
    h = a * u
    n = (x.shape[-1] + 16) * ULP
    return h, h.abs() * (HALF + ARG) + n * (1.13 * sg * u.abs() + a.abs() * su + 1.13 * n * sg * su)


SHAPES = [(1, 256, 128), (3, 256, 128), (16, 512, 256), (17, 512, 384), (33, 256, 640), (64, 512, 128), (65, 768, 128),
          (127, 512, 256), (129, 512, 256), (300, 1024, 384), (9, 256, 5632), (1027, 512, 2048), (2050, 256, 512),
          (4100, 512, 640), (2100, 256, 1024), (1700, 768, 1152)]


@gpu
@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("M,D,F", SHAPES)
def test_forward(hip_lib, M, D, F, name):
    import hstu_amd

    x = rnd((M, D), 1).to(DEV)
    wg, wu = weights(F, D)
    h = hstu_amd.gated_linear(x, wg, wu, name)
    assert h.shape == (M, F) and h.dtype == torch.bfloat16
    want, tol = h_bound(x, wg, wu, name)
    within(h, want, tol, "h")


@gpu
@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("M,D,F", SHAPES)
def test_backward(hip_lib, M, D, F, name):
    import hstu_amd

    x, dh = rnd((M, D), 1).to(DEV).requires_grad_(True), rnd((M, F), 2, 0.5).to(DEV)
    wg, wu = (w.requires_grad_(True) for w in weights(F, D))
    h = hstu_amd.gated_linear(x, wg, wu, name)
    dx, dgate, dup = torch.autograd.grad(h, (x, wg, wu), dh)
    xd, gd, ud = x.detach(), wg.detach(), wu.detach()
    rx, rg, ru, dg, du = orc.gated_bwd_ref(dh, xd, gd, ud, name)
    xa, ga, ua, da = xd.double().abs(), gd.double().abs(), ud.double().abs(), dh.double().abs()
    sg, su = xa @ ga.t(), xa @ ua.t()
    n = (D + 16) * ULP
    u = (xd.double() @ ud.double().t()).abs()
    # dg and du as they are rounded: their own rounding, and the sums' that they come from
    og = dg.abs() * (HALF + ARG) + n * da * (1.13 * su + u * sg + n * su * sg) + da * u * ARG
    ou = du.abs() * (HALF + ARG) + n * da * 1.13 * sg
    top_g, top_u = dg.abs() + og, du.abs() + ou
    within(dx, rx, rx.abs() * HALF + og @ ga + ou @ ua + 2 * F * ULP * (top_g @ ga + top_u @ ua), "dx")
    within(dgate, rg, rg.abs() * HALF + og.t() @ xa + (M + 64) * ULP * (top_g.t() @ xa), "dgate")
    within(dup, ru, ru.abs() * HALF + ou.t() @ xa + (M + 64) * ULP * (top_u.t() @ xa), "dup")
    if M * F >= 4096:  # enough terms for the norm to be near its mean
        for got, want in ((dx, rx), (dgate, rg), (dup, ru)):
            assert float((got.double() - want).norm() / want.norm()) <= NORM


@gpu
@pytest.mark.parametrize("modes", [(0, 0), (1, 1), (1, 0), (0, 1)])
@pytest.mark.parametrize("M,D,F", [(1, 128, 128), (5, 384, 128), (17, 512, 256), (65, 256, 384), (129, 1024, 128),
                                   (300, 640, 256), (1027, 512, 1024), (9, 128, 5632), (4100, 256, 512), (2100, 384, 1024),
                                   (1700, 640, 1152)])
def test_e4m3(hip_lib, M, D, F, modes):
    import hstu_amd

    def e4m3(v, by_row):
        a = v.float().abs()
        s = (a.amax(-1, keepdim=True) if by_row else a.max().reshape(1, 1)) / 448
        return (v.float() / s).clamp(-448, 448).to(torch.float8_e4m3fn), s.reshape(-1)

    wg, wu = weights(F, D)
    (x8, xs), (g8, gs), (u8, us) = (e4m3(t, m) for t, m in ((rnd((M, D), 3).to(DEV), modes[0]), (wg, modes[1]), (wu, modes[1])))
    h = hstu_amd.gated_linear_fp8(x8, xs, (g8, gs), (u8, us))
    x = x8.double() * xs.double().reshape(-1, 1)
    want, tol = h_bound(x, g8.double() * gs.double().reshape(-1, 1), u8.double() * us.double().reshape(-1, 1), "silu")
    within(h, want, tol, "h")


@gpu
@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("M,D,F", [(1, 256, 128), (40, 512, 384), (130, 1024, 256), (1030, 256, 640)])
def test_kept_and_computed_again_give_the_same_bytes(hip_lib, M, D, F, name):
    import hstu_amd

    x, dh = rnd((M, D), 31).to(DEV).requires_grad_(True), rnd((M, F), 32).to(DEV)
    wg, wu = (w.requires_grad_(True) for w in weights(F, D, 3))
    both = []
    for recompute in (True, False, None):
        h = hstu_amd.gated_linear(x, wg, wu, name, recompute=recompute)
        both.append((h.detach(),) + torch.autograd.grad(h, (x, wg, wu), dh))
    for other in both[1:]:
        assert all(torch.equal(a, b) for a, b in zip(both[0], other))
    h, gu = hstu_amd.gated_linear_fwd(x, wg, wu, name, keep=True)
    assert torch.equal(h, both[0][0]) and gu.shape == (M, 2 * F) and gu.dtype == torch.float32
    n = (D + 16) * ULP
    for part, w in ((gu[:, :F], wg), (gu[:, F:], wu)):
        want = x.detach().double() @ w.detach().double().t()
        within(part, want, n * (x.detach().double().abs() @ w.detach().double().abs().t()), "kept")
    with torch.no_grad():
        assert torch.equal(hstu_amd.gated_linear(x, wg, wu, name), h)


@gpu
def test_large_arguments(hip_lib):
    """Gates far out on both sides: silu, gelu and sigmoid saturate without NaN, values and derivatives."""
    import hstu_amd

    x = torch.zeros((2, 256), dtype=torch.bfloat16, device=DEV)
    x[0, 0], x[1, 0] = 1.0, -1.0
    wg, wu = torch.zeros((128, 256), dtype=torch.bfloat16, device=DEV), torch.zeros((128, 256), dtype=torch.bfloat16, device=DEV)
    wg[:, 0] = torch.tensor([0.0, 1, 10, 60, 87, 89, 100, 1e4] * 16, device=DEV)
    wu[:, 0] = 1.0
    for name in ACTS:
        want, tol = h_bound(x, wg, wu, name)
        within(hstu_amd.gated_linear(x, wg, wu, name), want, tol + 2.0 ** -100, name)
        dh = torch.ones((2, 128), dtype=torch.bfloat16, device=DEV)
        for got in hstu_amd.gated_linear_bwd(dh, x, wg, wu, name):
            assert torch.isfinite(got.float()).all(), name


@gpu
@pytest.mark.parametrize("M", [26, 200, 1100])
@pytest.mark.parametrize("name", ACTS)
def test_every_size_of_the_gate(hip_lib, name, M):
    """g = v and u = 1 exactly: a(v) and a'(v) from 0 to bf16's largest.  Far on the
    negative side they are products with an s below 2^-126, at most 88 of it; a'
    changes sign, so what its argument is off counts by itself."""
    import hstu_amd

    v = torch.tensor([0, 1e-30, 1e-3, 0.3, 1, 1.28, 5, 30, 60, 86, 1e3, 1e20, 3e38], dtype=torch.bfloat16)
    v = torch.cat((v, -v)).repeat(-(-M // 26))[:M]
    F = 1024
    x = torch.zeros((M, 256), dtype=torch.bfloat16)
    x[:, 0], x[:, 1] = v, 1
    wg, wu, dh = torch.zeros((F, 256)), torch.zeros((F, 256)), torch.zeros((M, F))
    wg[5, 0] = wu[5, 1] = 1
    dh[:, 5] = 1
    x, wg, wu, dh = (t.to(torch.bfloat16).to(DEV) for t in (x, wg, wu, dh))
    h = hstu_amd.gated_linear(x, wg, wu, name)
    kept, gu = hstu_amd.gated_linear_fwd(x, wg, wu, name, keep=True)
    assert torch.equal(kept, h)
    a, da = orc.activation_ref(name, v.to(DEV).double())
    within(h[:, 5], a, a.abs() * (HALF + ARG) + 2.0 ** -110, "h")
    for keep in (None, gu):
        dx = hstu_amd.gated_linear_bwd(dh, x, wg, wu, name, gu=keep)[0]
        within(dx[:, 1], a, a.abs() * (HALF + ARG) + 2.0 ** -110, "du")
        within(dx[:, 0], da, da.abs() * HALF + 2 * ARG, "dg")


@gpu
def test_gradient_against_differences(hip_lib):
    """The kernels' gradient along a direction against a difference quotient of the float64 formula."""
    import hstu_amd

    M, D, F = 37, 256, 128
    x, dh = rnd((M, D), 5).to(DEV), rnd((M, F), 6).to(DEV)
    wg, wu = weights(F, D, 1)
    for name in ACTS:
        grads = hstu_amd.gated_linear_bwd(dh, x, wg, wu, name)
        base = [t.double() for t in (x, wg, wu)]
        vs = [torch.randn(t.shape, generator=torch.Generator().manual_seed(7 + i), dtype=torch.float64).to(DEV)
              for i, t in enumerate(base)]

        def loss(e):
            return float((orc.gated_ref(*(b + e * v for b, v in zip(base, vs)), name) * dh.double()).sum())

        e = 1e-5
        diff = (loss(e) - loss(-e)) / (2 * e)
        got = float(sum((g.double() * v).sum() for g, v in zip(grads, vs)))
        # each gradient is off by 2^-8 of its 2-norm at most, along v by that times a unit normal number:
        # four of its deviations, over the three gradients
        tol = 4 * HALF * float(sum(g.double().norm() ** 2 for g in grads)) ** 0.5 + 1e-4
        assert abs(got - diff) <= tol, name


@gpu
def test_strided_and_leading_dimensions(hip_lib):
    import hstu_amd

    wide, wgu = rnd((40, 1024), 8).to(DEV), rnd((256, 512), 9, 0.05).to(DEV)
    x, wg, wu = wide[:, 512:768], wgu[:, :256], wgu[:, 256:]  # columns of wider buffers
    want = hstu_amd.gated_linear(x.contiguous(), wg.contiguous(), wu.contiguous())
    assert torch.equal(hstu_amd.gated_linear(x, wg, wu), want)
    assert torch.equal(hstu_amd.gated_linear(wide[:, 3:259], wg, wu),
                       hstu_amd.gated_linear(wide[:, 3:259].contiguous(), wg, wu))
    x3 = x.contiguous().view(5, 8, 256).requires_grad_(True)
    h = hstu_amd.gated_linear(x3, wg, wu)
    assert h.shape == (5, 8, 256) and torch.equal(h.reshape(40, 256), want)
    (dx,) = torch.autograd.grad(h.float().sum(), (x3,))  # an expanded gradient
    assert dx.shape == x3.shape
    ones = torch.ones((40, 256), dtype=torch.bfloat16, device=DEV)
    assert torch.equal(dx.reshape(40, 256), hstu_amd.gated_linear_bwd(ones, x, wg, wu)[0])
    # both weights of one [2F, D] parameter: their gradients meet in it
    both = rnd((256, 256), 10, 0.1).to(DEV).requires_grad_(True)
    out = hstu_amd.gated_linear(x, both[:128], both[128:])
    (db,) = torch.autograd.grad(out, (both,), ones[:, :128])
    _, dg, du = hstu_amd.gated_linear_bwd(ones[:, :128], x, both[:128].detach(), both[128:].detach())
    assert torch.equal(db, torch.cat((dg, du)))
    # one weight on both sides: its gradient is the sum
    same = both[:128].detach().clone().requires_grad_(True)
    (ds,) = torch.autograd.grad(hstu_amd.gated_linear(x, same, same), (same,), ones[:, :128])
    _, dg, du = hstu_amd.gated_linear_bwd(ones[:, :128], x, same.detach(), same.detach())
    assert torch.equal(ds, dg + du)


@gpu
def test_no_rows_and_partial_gradients(hip_lib):
    import hstu_amd

    wg, wu = (w.requires_grad_(True) for w in weights(128, 256))
    x = torch.zeros((0, 256), dtype=torch.bfloat16, device=DEV, requires_grad=True)
    h = hstu_amd.gated_linear(x, wg, wu)
    assert h.shape == (0, 128)
    dx, dg, du = torch.autograd.grad(h, (x, wg, wu), torch.zeros_like(h))
    assert dx.shape == x.shape and not dg.any() and not du.any()
    x = rnd((20, 256), 11).to(DEV)
    dh = rnd((20, 128), 12).to(DEV)
    full = hstu_amd.gated_linear_bwd(dh, x, wg, wu)
    (dg,) = torch.autograd.grad(hstu_amd.gated_linear(x, wg, wu.detach()), (wg,), dh)
    assert torch.equal(dg, full[1])
    xr = x.clone().requires_grad_(True)
    (dx,) = torch.autograd.grad(hstu_amd.gated_linear(xr, wg.detach(), wu.detach()), (xr,), dh)
    assert torch.equal(dx, full[0])


@gpu
def test_rows_past_the_last_are_left(hip_lib):
    """The C entry writes M rows and F columns of a larger buffer, nothing else."""
    import hstu_amd._lib as lib

    D, F = 256, 640
    wg, wu = weights(F, D)
    for M in (1, 17, 130, 4100):  # every form
        x = rnd((M, D), 13).to(DEV)
        out = torch.full((M + 140, F + 8), 7.0, dtype=torch.bfloat16, device=DEV)
        st = lib.fn("hstu_gated_fwd")(x.data_ptr(), D, wg.data_ptr(), D, wu.data_ptr(), D, M, F, D, 0, out.data_ptr(),
                                      F + 8, None, lib.stream(x))
        assert st == 0
        assert (out[M:] == 7).all() and (out[:, F:] == 7).all()
        assert not (out[:M, :F] == 7).all()


@gpu
def test_side_stream_graph_and_same_bytes(hip_lib):
    import hstu_amd

    x, dh = rnd((333, 512), 14).to(DEV), rnd((333, 256), 15).to(DEV)
    wg, wu = weights(256, 512)

    def step():
        from hstu_amd.fp8 import quantize_e4m3_rows

        (a8, s), (g8, gs), (u8, us) = (quantize_e4m3_rows(t) for t in (x, wg, wu))
        return ((hstu_amd.gated_linear(x, wg, wu),) + hstu_amd.gated_linear_bwd(dh, x, wg, wu)
                + (hstu_amd.gated_linear_fp8(a8, s, (g8, gs), (u8, us)),))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    torch.cuda.current_stream().wait_stream(side)
    want = step()
    assert all(torch.equal(a, b) for a, b in zip(on_side, want))
    assert all(torch.equal(a, b) for a, b in zip(step(), want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(4):
        x.copy_(rnd((333, 512), 20 + k))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, step())), k


# ---------------------------------------------------------------- each form by name
def form(M, F, k_bytes):
    """The form that a call of M rows takes (the dispatch of csrc/hstu_gated.hip), so that a case below fails when
    a changed threshold takes it to another one."""
    if M <= 32 if F <= 4096 else F > 8192 and M <= 16:
        return "rows"
    return "middle" if -(-M // 64) * (F // 32) <= 768 or k_bytes < 256 else "tile"


@gpu
@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("M,D,F", [(2100, 256, 1024), (1700, 1280, 1152)])
def test_tile_form_keeps_g_and_u(hip_lib, M, D, F, name):
    assert form(M, F, 2 * D) == "tile"
    test_kept_and_computed_again_give_the_same_bytes(hip_lib, M, D, F, name)


@gpu
@pytest.mark.parametrize("name", ACTS)
def test_tile_form_at_every_size_of_the_gate(hip_lib, name):
    assert form(2100, 1024, 512) == "tile"
    test_every_size_of_the_gate(hip_lib, name, 2100)


@gpu
@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("M,D,F,which", [(5, 256, 8320, "rows"), (16, 256, 10240, "rows"), (17, 256, 8320, "middle"),
                                         (1900, 2304, 640, "middle"), (1700, 1280, 1152, "tile")])
def test_wide_blocks(hip_lib, M, D, F, which, name):
    """The row form of many columns, and wide x, whose dx has more than eight column tiles (their grouped order)."""
    assert form(M, F, 2 * D) == which
    test_forward(hip_lib, M, D, F, name)
    test_backward(hip_lib, M, D, F, name)


def e4m3_bound(x, wg, wu, name):
    """(h, what h may be off) of e4m3 operands as the values they stand for.  Beyond h_bound's units: the matrix
    cores take eight consecutive products together and cut each toward zero at 2^-13 of the largest's power of
    two, so a sum is off by up to 8 * 2^-13 of the largest magnitudes' product in each eight."""
    h, tol = h_bound(x, wg, wu, name)
    top = [t.abs().unflatten(1, (-1, 8)).amax(-1) for t in (x, wg, wu)]
    n = (x.shape[-1] + 16) * ULP
    g, u = x @ wg.t(), x @ wu.t()
    cut_g, cut_u = 2.0 ** -10 * (top[0] @ top[1].t()), 2.0 ** -10 * (top[0] @ top[2].t())
    su = u.abs() + n * (x.abs() @ wu.abs().t()) + cut_u
    return h, tol + 1.13 * cut_g * su + (orc.activation_ref(name, g)[0].abs() + 1.13 * n * (x.abs() @ wg.abs().t())) * cut_u


@gpu
def test_e4m3_sums_of_eight(hip_lib):
    """What the bound above says of the instruction, at its edge: 2^16 - 2^16 + v with v beside the first, u alone in
    sigmoid's saturation.  v is kept from 2^3 on, in steps of it; beside neither it is exact."""
    import hstu_amd

    one, F = torch.ones(1, device=DEV), 128

    def u_of(k, v):
        x, wg, wu = torch.zeros((1, 128), device=DEV), torch.zeros((F, 128), device=DEV), torch.zeros((F, 128), device=DEV)
        x[0, 0] = x[0, 64] = 256
        wu[:, 0], wu[:, 64], x[0, k], wu[:, k], x[0, 100], wg[:, 100] = 256, -256, 1, v, 8, 8
        x8, g8, u8 = (t.to(torch.float8_e4m3fn) for t in (x, wg, wu))
        return float(hstu_amd.gated_linear_fp8(x8, one, (g8, one), (u8, one), "sigmoid")[0, 0])

    for v in (1.0, 7.0, 8.0, 15.0, 28.0, -15.0):
        for k in (1, 65):
            assert abs(u_of(k, v) - v) < 8, (k, v)  # 2^16 2^-13
        assert u_of(30, v) == v


@gpu
@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("modes", [(0, 0, 1), (0, 1, 0), (1, 0, 1), (1, 1, 0), (1, 1, 1), (0, 0, 0)])
@pytest.mark.parametrize("M,D,F,which", [(5, 384, 256, "rows"), (20, 128, 640, "rows"), (9, 256, 8320, "rows"),
                                         (65, 256, 384, "middle"), (4100, 128, 512, "middle"), (2100, 384, 1024, "tile")])
def test_e4m3_activations_and_scales(hip_lib, M, D, F, which, modes, name):
    """Scales of x, gate and up by row or one, each by itself."""
    import hstu_amd

    def e4m3(v, by_row):
        a = v.float().abs()
        s = (a.amax(-1, keepdim=True) if by_row else a.max().reshape(1, 1)) / 448
        return (v.float() / s).clamp(-448, 448).to(torch.float8_e4m3fn), s.reshape(-1)

    assert form(M, F, D) == which
    x, wg, wu = rnd((M, D), 3).to(DEV), *weights(F, D)
    (x8, xs), (g8, gs), (u8, us) = (e4m3(t, m) for t, m in zip((x, wg, wu), modes))
    h = hstu_amd.gated_linear_fp8(x8, xs, (g8, gs), (u8, us), name)
    x, wg, wu = (q.double() * s.double().reshape(-1, 1) for q, s in ((x8, xs), (g8, gs), (u8, us)))
    want, tol = e4m3_bound(x, wg, wu, name)
    within(h, want, tol, "h")
    assert float((h.double() - want).norm() / want.norm()) <= NORM  # random operands: their cuts are independent


@gpu
@pytest.mark.parametrize("name", ACTS)
@pytest.mark.parametrize("M,which", [(26, "rows"), (200, "middle"), (2100, "tile")])
def test_e4m3_at_every_size_of_the_gate(hip_lib, name, M, which):
    """g = +-v and u = v, exactly, by the row's scale: a(g) u from 0 to 1e36, an s below 2^-126 as 0."""
    import hstu_amd

    v = torch.tensor([0, 1e-30, 1e-3, 0.3, 1, 1.28, 5, 30, 60, 86, 100, 1e3, 1e18]).bfloat16().float()
    v = torch.cat((v, v)).repeat(-(-M // 26))[:M].to(DEV)
    sign = torch.cat((torch.ones(13), -torch.ones(13))).repeat(-(-M // 26))[:M].to(DEV)
    F = 1024
    assert form(M, F, 256) == which
    x, wg, wu = torch.zeros((M, 256), device=DEV), torch.zeros((F, 256), device=DEV), torch.zeros((F, 256), device=DEV)
    x[:, 0], x[:, 1], wg[5, 0], wu[5, 1] = sign, 1, 1, 1
    x8, g8, u8 = (t.to(torch.float8_e4m3fn) for t in (x, wg, wu))
    one = torch.ones(1, device=DEV)
    h = hstu_amd.gated_linear_fp8(x8, v, (g8, one), (u8, one), name)
    want = orc.activation_ref(name, (sign * v).double())[0] * v.double()
    within(h[:, 5], want, want.abs() * (HALF + ARG) + 2.0 ** -100, "h")
    assert not h[:, :5].any()


# ---------------------------------------------------------------- refusals
def test_refusals():
    import hstu_amd

    bf = torch.bfloat16
    x, w = torch.zeros(2, 256, dtype=bf), torch.zeros(128, 256, dtype=bf)
    with pytest.raises(NotImplementedError):
        hstu_amd.gated_linear(x, w, w)  # not on a device
    with pytest.raises(ValueError):
        hstu_amd.gated_linear(x, w, w, "relu")
    with pytest.raises(NotImplementedError):
        hstu_amd.gated_linear(x.float(), w, w)


@gpu
def test_refusals_on_device(hip_lib):
    import hstu_amd

    bf = torch.bfloat16

    def z(*shape, dtype=bf):
        return torch.zeros(shape, dtype=dtype, device=DEV)

    for args in ((z(2, 256), z(128, 512), z(128, 512)), (z(2, 256), z(128, 256), z(256, 256))):
        with pytest.raises(ValueError):
            hstu_amd.gated_linear(*args)
    for args in ((z(2, 128), z(128, 128), z(128, 128)), (z(2, 256), z(64, 256), z(64, 256)),
                 (z(2, 256), z(128, 256), torch.zeros(128, 256, dtype=bf)),
                 (z(2, 256), z(128, 256, dtype=torch.float32), z(128, 256))):
        with pytest.raises(NotImplementedError):
            hstu_amd.gated_linear(*args)
    with pytest.raises(ValueError):
        hstu_amd.gated_linear_bwd(z(2, 256), z(2, 256), z(128, 256), z(128, 256))
    x8, w8 = z(2, 256).to(torch.float8_e4m3fn), z(128, 256).to(torch.float8_e4m3fn)
    s = z(1, dtype=torch.float32)
    with pytest.raises(ValueError):
        hstu_amd.gated_linear_fp8(x8, z(3, dtype=torch.float32), (w8, s), (w8, s))
    with pytest.raises(ValueError):
        hstu_amd.gated_linear_fp8(x8, s, (w8, z(2, dtype=torch.float32)), (w8, s))
    with pytest.raises(NotImplementedError):
        hstu_amd.gated_linear_fp8(x8, s, (w8.to(bf), s), (w8, s))


def test_c_entry_refusals():
    """Bad arguments are refused before any launch (no device is touched)."""
    import hstu_amd._lib as lib

    P = 64  # a stand-in address, never read
    fwd, bwd, f8 = (lib.fn("hstu_gated_" + n) for n in ("fwd", "bwd", "fwd_fp8"))

    def f(x=P, ldx=256, g=P, ldg=256, u=P, ldu=256, M=4, F=128, D=256, act=0, h=P, ldh=128, keep=None):
        return fwd(x, ldx, g, ldg, u, ldu, M, F, D, act, h, ldh, keep, None)

    for bad in (dict(M=-1), dict(F=0), dict(D=0), dict(act=3), dict(act=-1), dict(ldx=255), dict(ldg=8), dict(ldu=8),
                dict(ldh=127), dict(x=None), dict(g=None), dict(u=None), dict(h=None)):
        assert f(**bad) == lib.HSTU_E_BAD_ARG, bad
    for bad in (dict(F=64), dict(D=128), dict(x=72), dict(ldx=260), dict(h=72), dict(ldh=132), dict(keep=72)):
        assert f(**bad) == lib.HSTU_E_UNSUPPORTED, bad
    assert f(M=0) == 0

    def b(dh=P, lddh=128, M=4, out=P, ldo=256):
        return bwd(dh, lddh, P, 256, P, 256, P, 256, M, 128, 256, 0, out, ldo, None)

    for bad in (dict(dh=None), dict(lddh=100), dict(ldo=255), dict(out=None), dict(M=-1)):
        assert b(**bad) == lib.HSTU_E_BAD_ARG, bad
    for bad in (dict(dh=66), dict(lddh=132), dict(ldo=260)):
        assert b(**bad) == lib.HSTU_E_UNSUPPORTED, bad

    def e(xs=P, gs=P, us=P, D=128, M=4):
        return f8(P, 128, xs, 1, P, 128, gs, 1, P, 128, us, 1, M, 128, D, 0, P, 128, None)

    for bad in (dict(xs=None), dict(gs=None), dict(us=None), dict(D=256)):
        assert e(**bad) == lib.HSTU_E_BAD_ARG, bad
    assert e(D=64) == lib.HSTU_E_UNSUPPORTED and e(xs=65) == lib.HSTU_E_UNSUPPORTED
    kept, tr = lib.fn("hstu_gated_bwd_kept"), lib.fn("hstu_gated_transpose")

    def k(dh=P, lddh=128, keep=P, rows=4, F=128, act=0, out=P, ldo=256):
        return kept(dh, lddh, keep, rows, F, act, out, ldo, None)

    for bad in (dict(dh=None), dict(keep=None), dict(out=None), dict(rows=-1), dict(F=0), dict(act=3), dict(lddh=100),
                dict(ldo=255)):
        assert k(**bad) == lib.HSTU_E_BAD_ARG, bad
    for bad in (dict(F=100), dict(dh=72), dict(keep=72), dict(out=72), dict(lddh=132), dict(ldo=260)):
        assert k(**bad) == lib.HSTU_E_UNSUPPORTED, bad
    assert k(rows=0) == 0

    def t(g=P, ldg=256, u=P, ldu=256, F=128, D=256, out=P, ldo=256):
        return tr(g, ldg, u, ldu, F, D, out, ldo, None)

    for bad in (dict(g=None), dict(u=None), dict(out=None), dict(ldg=255), dict(ldu=100), dict(ldo=200), dict(F=0), dict(D=0)):
        assert t(**bad) == lib.HSTU_E_BAD_ARG, bad
    for bad in (dict(F=96), dict(D=200), dict(g=72), dict(out=72), dict(ldg=260), dict(ldo=260)):
        assert t(**bad) == lib.HSTU_E_UNSUPPORTED, bad
