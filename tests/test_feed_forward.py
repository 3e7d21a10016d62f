"""The feed-forward operators run together, as a sublayer uses them: norm, gated
projection, 4-bit product and the residual stream between them, in training and
in serving, eagerly and captured.

Every stage is held against the float64 formulas at the inputs that it got, so
that no rounding of an earlier stage counts.  Tolerances: an output rounded once
to bf16 is off by at most 2^-8 of its value, and so is the 2-norm of the
difference (NORM); gradients of a product carry two independent roundings, under
sqrt(2 / 3) 2^-8 in the 2-norm, and the sums' own error in fp32 is under 2^-14 of
it at these sizes: NORM + 2^-14.  e4m3 is off by 2^-4 of the value, or half of a
2^-9 step below its normal range."""

import pytest
import torch

from oracle import feed_forward_oracle as orc

DEV = "cuda"
EPS = 1e-6
NORM = 2.0 ** -8 + 2.0 ** -14
gpu = pytest.mark.gpu


def rnd(shape, seed, std=1.0):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(torch.bfloat16).to(DEV)


def norm_weight(D, seed):
    return (1.0 + 0.3 * torch.randn(D, generator=torch.Generator().manual_seed(seed))).to(torch.bfloat16).to(DEV)


def close(got, want, what):
    err, size = float((got.double() - want).norm()), float(want.norm())
    assert err <= NORM * size, f"{what}: {err / size:.3e}"


@gpu
@pytest.mark.parametrize("name", ["silu", "gelu"])
@pytest.mark.parametrize("M,D,F", [(40, 256, 384), (700, 512, 1024), (130, 1280, 640), (2100, 256, 512)])
def test_training_sublayers(hip_lib, M, D, F, name):
    """Two sublayers on one residual stream, the second's norm adding the first's output."""
    import hstu_amd

    x, r = rnd((M, D), 1).requires_grad_(True), rnd((M, D), 2, 2.0).requires_grad_(True)
    layers = [[t.requires_grad_(True) for t in (norm_weight(D, 3 + i), rnd((F, D), 10 + i, 1.5 * D ** -0.5),
                                                rnd((F, D), 20 + i, D ** -0.5), rnd((D, F), 30 + i, F ** -0.5))]
              for i in range(2)]
    cur, stream, kept = x, r, []
    for w, wg, wu, wd in layers:
        y, h = hstu_amd.rms_norm(cur, w, EPS, residual=stream)
        a = hstu_amd.gated_linear(y, wg, wu, name)
        out = torch.nn.functional.linear(a, wd)
        for t in (y, h, a, out):
            t.retain_grad()
        kept.append((cur, stream, y, h, a, out))
        cur, stream = out, h
    (cur.float() * rnd((M, D), 40).float() + stream.float() * rnd((M, D), 41).float()).sum().backward()
    for (w, wg, wu, wd), (i, s, y, h, a, out) in zip(layers, kept):
        with torch.no_grad():
            assert torch.equal(h, (i.float() + s.float()).bfloat16())
            close(y, orc.rms_norm_ref(h, w, EPS)[0], "y")
            close(a, orc.gated_ref(y, wg, wu, name), "a")
            dx, dg, du = orc.gated_bwd_ref(a.grad, y, wg, wu, name)[:3]
            for got, want, what in ((y.grad, dx, "dy"), (wg.grad, dg, "dgate"), (wu.grad, du, "dup")):
                close(got, want, what)
            # h's gradient has two sources in the first layer: what the later norm
            # sends back arrives in h.grad with the direct one
            dx, dw, _, _ = orc.rms_norm_bwd_ref(y.grad, h, w, EPS, h.grad)
            for got, want, what in ((i.grad, dx, "dx"), (w.grad, dw, "dweight")):
                close(got, want, what)
    assert torch.equal(x.grad, r.grad) and x.grad.data_ptr() != r.grad.data_ptr()


@gpu
@pytest.mark.parametrize("M,D,F", [(1, 512, 1024), (5, 2048, 5632), (33, 256, 640), (300, 512, 1024), (2100, 256, 512)])
def test_serving_sublayer(hip_lib, M, D, F):
    """e4m3 norm -> e4m3 gated projection -> 4-bit product on the residual, then the next norm into the e4m3 GEMM."""
    import hstu_amd
    from hstu_amd.fp8 import fp8_gemm, quantize_e4m3_rows

    x, r, w, w2 = rnd((M, D), 1), rnd((M, D), 2, 2.0), norm_weight(D, 3), norm_weight(D, 4)
    pairs = [(q, s.reshape(-1)) for q, s in (quantize_e4m3_rows(rnd((n, D), 10 + i, D ** -0.5))
                                             for i, n in enumerate((F, F, 128)))]
    (g8, gs), (u8, us), (n8, ns) = pairs
    gd, ud, nd = (q.double() * s.double()[:, None] for q, s in pairs)
    down = hstu_amd.quantize_mxfp4(rnd((D, F), 20, F ** -0.5))
    y8, s, h = hstu_amd.rms_norm_fp8(x, w, EPS, residual=r)
    a = hstu_amd.gated_linear_fp8(y8, s, (g8, gs), (u8, us))
    out = hstu_amd.mxfp4_linear(a, down, residual=h)
    z8, zs = hstu_amd.rms_norm_fp8(out, w2, EPS)
    last = fp8_gemm(z8, zs, (n8, ns))

    for q, sc, src, wt in ((y8, s, h, w), (z8, zs, out, w2)):
        want, sd = orc.rms_norm_ref(src, wt, EPS)[0], sc.double()[:, None]
        off = (q.double() * sd - want).abs()
        assert (off <= want.abs() * (2.0 ** -4 + 2.0 ** -16) + sd * 2.0 ** -10).all()
    close(a, orc.gated_ref(y8.double() * s.double()[:, None], gd, ud, "silu"), "a")
    av = orc.mxfp4_decode_ref(*hstu_amd.quantize_mxfp4(a))
    close(out, av @ orc.mxfp4_decode_ref(*down).t() + h.double(), "out")
    close(last, z8.double() * zs.double()[:, None] @ nd.t(), "last")


@gpu
@pytest.mark.parametrize("M", [1, 40])
def test_serving_sublayer_captured(hip_lib, M):
    import hstu_amd
    from hstu_amd.fp8 import quantize_e4m3_rows

    D, F = 512, 1024
    x, r, w = rnd((M, D), 1), rnd((M, D), 2), norm_weight(D, 3)
    gate, up = ((q, s.reshape(-1)) for q, s in (quantize_e4m3_rows(rnd((F, D), 10 + i, D ** -0.5)) for i in range(2)))
    down = hstu_amd.quantize_mxfp4(rnd((D, F), 20, F ** -0.5))

    def step():
        cur, stream = x, r
        for _ in range(3):
            y8, s, stream = hstu_amd.rms_norm_fp8(cur, w, EPS, residual=stream)
            cur = hstu_amd.mxfp4_linear(hstu_amd.gated_linear_fp8(y8, s, gate, up), down)
        return cur, stream

    step()
    graphs = []
    for _ in range(2):  # two graphs replayed in turn share nothing
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            graphs.append((g, step()))
    for k in range(4):
        x.copy_(rnd((M, D), 50 + k))
        for g, _ in graphs:
            g.replay()
        want = step()
        torch.cuda.synchronize()
        for _, got in graphs:
            assert all(torch.equal(p, q) for p, q in zip(got, want)), k


@gpu
@pytest.mark.parametrize("D", [512, 1280])
def test_training_captured(hip_lib, D):
    """Forward and backward through autograd in one graph; the leaves' other graphs are gone, or the capture is refused."""
    import hstu_amd

    M, F = 300, 384
    x, r = rnd((M, D), 1).requires_grad_(True), rnd((M, D), 2).requires_grad_(True)
    w, wg, wu = norm_weight(D, 3), rnd((F, D), 10, D ** -0.5), rnd((F, D), 11, D ** -0.5)
    leaves = (x, r) + tuple(t.requires_grad_(True) for t in (w, wg, wu))
    da, dh = rnd((M, F), 12), rnd((M, D), 13)

    def forward():
        y, h = hstu_amd.rms_norm(x, w, EPS, residual=r)
        return hstu_amd.gated_linear(y, wg, wu), h

    def step():
        a, h = forward()
        return (a.detach(), h.detach()) + torch.autograd.grad((a, h), leaves, (da, dh))

    alive = forward()  # an eager graph on the default stream
    with pytest.raises(hstu_amd.HstuKernelError):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            forward()
    with pytest.raises(hstu_amd.HstuKernelError):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            hstu_amd.gated_linear(da.new_zeros(M, D), wg, wu)
    del alive
    step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(4):
        with torch.no_grad():
            x.copy_(rnd((M, D), 50 + k))
        graph.replay()
        torch.cuda.synchronize()
        want = step()
        assert all(torch.equal(p, q) for p, q in zip(captured, want)), k


@gpu
def test_no_second_derivative(hip_lib):
    import hstu_amd

    x, w = rnd((4, 256), 1).requires_grad_(True), norm_weight(256, 2)
    wg, wu = rnd((128, 256), 3, 0.1), rnd((128, 256), 4, 0.1)
    for y in (hstu_amd.rms_norm(x, w), hstu_amd.gated_linear(x, wg, wu)):
        with pytest.raises(NotImplementedError):
            torch.autograd.grad(y.float().sum(), x, create_graph=True)


def test_no_forward_mode(monkeypatch):
    """A dual tensor does not require grad, and its tangent is refused, not dropped; other tensors in a dual
    level are served.  Checked without a device: nothing is launched."""
    import torch.autograd.forward_ad as fwd
    from hstu_amd import hstu_gated, hstu_rms_norm

    served = []
    monkeypatch.setattr(hstu_rms_norm, "rms_norm_fwd", lambda x, *a, **k: served.append(x) or (x, x, x, x))
    monkeypatch.setattr(hstu_gated, "gated_linear_fwd", lambda x, *a, **k: served.append(x) or x)
    x, w, wg = torch.ones(4, 256), torch.ones(256), torch.ones(128, 256)
    with fwd.dual_level():
        def dual(t):
            return fwd.make_dual(t, torch.ones_like(t))

        with torch.no_grad():  # forward mode goes on without grad mode
            for args in ((dual(x), w), (x, dual(w)), (x, w, 1e-6, dual(x))):
                with pytest.raises(NotImplementedError):
                    hstu_rms_norm.rms_norm(*args)
        for args in ((dual(x), wg, wg), (x, dual(wg), wg), (x, wg, dual(wg))):
            with pytest.raises(NotImplementedError):
                hstu_gated.gated_linear(*args)
        assert not served
        hstu_rms_norm.rms_norm(x, w)
        hstu_gated.gated_linear(x, wg, wg)
        assert len(served) == 2
    for t in (x, w, wg):
        t.requires_grad_(True)
    with fwd.dual_level():  # reverse mode over dual inputs, too
        with pytest.raises(NotImplementedError):
            hstu_rms_norm.rms_norm(dual(x), w)
        with pytest.raises(NotImplementedError):
            hstu_gated.gated_linear(x, wg, dual(wg))


@gpu
def test_no_forward_mode_through_the_backward(hip_lib):
    """Reverse mode with a dual gradient."""
    import hstu_amd
    import torch.autograd.forward_ad as fwd

    x, w = rnd((4, 256), 1).requires_grad_(True), norm_weight(256, 2)
    wg, wu = rnd((128, 256), 3, 0.1), rnd((128, 256), 4, 0.1)
    for y in (hstu_amd.rms_norm(x, w), hstu_amd.gated_linear(x, wg, wu)):
        g = torch.ones_like(y)
        with fwd.dual_level():
            with pytest.raises(NotImplementedError):
                torch.autograd.grad(y, x, fwd.make_dual(g, g))


def forward_only_calls(dev):
    """Each forward-only entry point with the names of its inputs that could carry a derivative."""
    import hstu_amd

    def z(*shape, dtype=torch.bfloat16):
        return torch.zeros(shape, dtype=dtype, device=dev)

    f8, f32, u8 = torch.float8_e4m3fn, torch.float32, torch.uint8
    packed = (z(16, 64, dtype=u8), z(16, 4, dtype=u8))
    return (
        (dict(x=z(2, 128), w=z(128), r=z(2, 128), s=z(1, dtype=f32)),
         lambda x, w, r, s: hstu_amd.rms_norm_fp8(x, w, EPS, residual=r, scale=s)),
        (dict(x=z(2, 128).to(f8), xs=z(2, dtype=f32), gs=z(128, dtype=f32), us=z(1, dtype=f32)),
         lambda x, xs, gs, us: hstu_amd.gated_linear_fp8(x, xs, (z(128, 128).to(f8), gs), (z(128, 128).to(f8), us))),
        (dict(x=z(2, 128), b=z(16), r=z(2, 16)), lambda x, b, r: hstu_amd.mxfp4_linear(x, packed, bias=b, residual=r)),
        (dict(b=z(16), r=z(16, 16)), lambda b, r: hstu_amd.mxfp4_mm(packed, packed, bias=b, residual=r)),
    )


def test_forward_only_refuses_derivatives():
    """An input that requires grad would be cut off from the result without a word.  Refused before any look at
    the device, so this runs without one."""
    import torch.autograd.forward_ad as fwd

    for inputs, call in forward_only_calls("cpu"):
        for name, t in inputs.items():
            with pytest.raises(NotImplementedError, match="forward only"):
                call(**{**inputs, name: t.clone().requires_grad_(True)})
            if t.dtype == torch.float8_e4m3fn:
                continue
            with fwd.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
                call(**{**inputs, name: fwd.make_dual(t, torch.ones_like(t))})


@gpu
def test_forward_only_without_grad_mode(hip_lib):
    for inputs, call in forward_only_calls(DEV):
        leaves = {name: t.clone().requires_grad_(True) for name, t in inputs.items()}
        with torch.no_grad():
            out = call(**leaves)
        for t in out if isinstance(out, tuple) else (out,):
            assert not t.requires_grad
        call(**inputs)  # nor anything refused where nothing requires grad


@pytest.mark.parametrize("name,limit,es", [("hstu_gated", 2 ** 24, 2), ("mxfp4", 2 ** 23, 2), ("mxfp4", 2 ** 23, 1)])
def test_rows_far_apart_are_copied(name, limit, es):
    """Views whose rows are too far apart for the kernels' 32-bit offsets, as the last position of every
    sequence: copied; the farthest that the kernels take stay in place.  The memory is never touched whole."""
    import importlib

    mod = importlib.import_module("hstu_amd." + name)
    fit = mod._rows2d if name == "hstu_gated" else lambda t: mod._aligned(t, 16)
    dtype = torch.bfloat16 if es == 2 else torch.uint8
    for apart, copied in ((limit - 16, False), (limit, True), (4 * limit, True)):
        base = torch.empty(3 * apart // es + 64, dtype=dtype)
        view = base.as_strided((3, 32), (apart // es, 1))
        view.copy_(torch.arange(96).reshape(3, 32))
        got = fit(view)
        assert torch.equal(got, view) and (got.data_ptr() != view.data_ptr()) == copied
        assert mod._ld(got) * es < limit
        one = view[1:2]  # a single row has no distance
        assert fit(one).data_ptr() == one.data_ptr() and mod._ld(fit(one)) == 32


@gpu
def test_last_position_of_every_sequence(hip_lib):
    """hidden[:, -1] of long sequences: rows of activations, of dh and of the residual 16 MiB apart and more."""
    import hstu_amd
    from hstu_amd.fp8 import quantize_e4m3_rows

    for seqs, D in ((8, 512), (40, 256)):
        F = 256
        hidden = torch.zeros((seqs, 2 ** 24 // D, D), dtype=torch.bfloat16, device=DEV)  # 32 MiB a sequence
        x = hidden[:, -1]
        x.copy_(rnd((seqs, D), 1))
        wg, wu, w = rnd((F, D), 2, D ** -0.5), rnd((F, D), 3, D ** -0.5), norm_weight(D, 4)
        pair = hstu_amd.quantize_mxfp4(rnd((D, D), 5, D ** -0.5))
        (g8, gs), (u8, us) = quantize_e4m3_rows(wg), quantize_e4m3_rows(wu)
        x8 = x.to(torch.float8_e4m3fn)
        far8 = torch.zeros((seqs, 2 ** 24), dtype=torch.float8_e4m3fn, device=DEV)[:, :D]
        far8.copy_(x8)
        s = torch.ones(seqs, device=DEV)

        def all_of(x, x8):
            leaf = x.detach().requires_grad_(True)
            h = hstu_amd.gated_linear(leaf, wg, wu)
            dh = x[:, :F]
            return ((h.detach(),) + hstu_amd.gated_linear_bwd(dh, x, wg, wu) + torch.autograd.grad(h, leaf, dh)
                    + (hstu_amd.gated_linear_fp8(x8, s, (g8, gs.reshape(-1)), (u8, us.reshape(-1))),
                       hstu_amd.mxfp4_linear(x, pair), hstu_amd.mxfp4_linear(x.contiguous(), pair, residual=x),
                       hstu_amd.rms_norm(x, w)))

        for got, want in zip(all_of(x, far8), all_of(x.contiguous(), x8)):
            assert torch.equal(got, want)


@pytest.mark.parametrize("use", [lambda t: t, lambda t: t[:4], lambda t: t.t().t(), lambda t: t.float().bfloat16()[1:5]])
def test_capture_guard_sees_leaves_through_views(monkeypatch, use):
    """A leaf that an eager graph on the default stream holds is refused in a capture also where both use a part
    of it, its transpose or a cast (gate and up of one parameter).  Without a device: the streams are stand-ins."""
    from hstu_amd import HstuKernelError, _lib, hstu_gated, hstu_rms_norm

    stream, capturing = [0], [False]
    monkeypatch.setattr(_lib, "_raw", (lambda: 0, lambda index: stream[0], None, lambda: capturing[0]))
    monkeypatch.setattr(hstu_gated, "gated_linear_fwd", lambda x, *a, **k: x.new_ones(2, 128))
    monkeypatch.setattr(hstu_rms_norm, "rms_norm_fwd", lambda x, *a, **k: (torch.ones_like(x), x, x.new_ones(len(x)), None))
    monkeypatch.setattr(_lib, "fn", lambda name: lambda *a: 4)
    leaf = torch.ones(8, 8, dtype=torch.bfloat16, requires_grad=True)
    other = torch.ones(8, 8, dtype=torch.bfloat16)

    for call in (lambda t: hstu_gated.gated_linear(other, use(t), use(t), recompute=True), lambda t: hstu_rms_norm.rms_norm(use(t), other)):
        def capture():
            stream[0], capturing[0] = 7, True
            try:
                return call(leaf)
            finally:
                stream[0], capturing[0] = 0, False

        alive = call(leaf)
        with pytest.raises(HstuKernelError):
            capture()
        del alive
        capture()  # let go of: served
