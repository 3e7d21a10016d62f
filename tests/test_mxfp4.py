"""Microscaled 4-bit format: quantisation bit for bit, the product within the
sum's rounding, against ``oracle/feed_forward_oracle.py``.

Tolerance of the product: a code times a code is exact, the scales are powers
of two; a sum of K products is K additions, each off by at most 2^-23 of the sum of
the magnitudes (a unit: the matrix cores need not round to nearest), 16 more for
the joins, bias and residual; the output's rounding is 2^-8 of the value."""

import pytest
import torch

from oracle import feed_forward_oracle as orc

DEV = "cuda"
ULP, HALF = 2.0 ** -23, 2.0 ** -8
gpu = pytest.mark.gpu


def rnd(shape, seed, std=1.0, dtype=torch.bfloat16):
    return (torch.randn(shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype)


def pack_ref(x):
    """The oracle's pair of uint8 tensors."""
    v, e = orc.mxfp4_quantize_ref(x)
    unit = orc._pow2(e - 127).repeat_interleave(32, 1)
    t = (v / unit).abs()
    code = torch.zeros_like(t, dtype=torch.int64)
    for i, m in enumerate(orc.E2M1):
        code[t == m] = i
    code = code + 8 * torch.signbit(v)
    pair = code.reshape(x.shape[0], -1, 2)
    return (pair[..., 0] + 16 * pair[..., 1]).to(torch.uint8), e.to(torch.uint8)


def same_values(got, want):
    got, want = got.double(), want.double()
    return torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0), want.nan_to_num(0))


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 64), (7, 96), (33, 512), (5, 5632), (1000, 160), (2, 32768)])
def test_quantize(hip_lib, rows, cols, dtype):
    import hstu_amd

    x = (rnd((rows, cols), 1, 1.0, torch.float32) * torch.exp2(rnd((rows, 1), 2, 20.0, torch.float32).clamp(-60, 60))).to(dtype)
    want, e = orc.mxfp4_quantize_ref(x.to(DEV))
    codes, scales = hstu_amd.quantize_mxfp4(x.to(DEV))
    assert codes.shape == (rows, cols // 2) and scales.shape == (rows, cols // 32)
    assert torch.equal(scales.long(), e)
    assert torch.equal(orc.mxfp4_decode_ref(codes, scales), want)
    for out in (torch.bfloat16, torch.float32):
        v = hstu_amd.dequantize_mxfp4(codes, scales, out)
        assert v.dtype == out and torch.equal(v.double(), want)


@gpu
def test_quantize_every_code_and_tie(hip_lib):
    """Every bf16 magnitude of a block's range, both signs, next to a 4 that fixes the scale at 1."""
    import hstu_amd

    v = torch.arange(0, 0x4100, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)  # 0 .. 8
    v = torch.cat((v, -v)).to(DEV)
    v = v[v.abs() < 8]
    pad = (-v.numel()) % 31
    v = torch.cat((v, v.new_zeros(pad))).reshape(-1, 31)
    x = torch.cat((torch.full((v.shape[0], 1), 4.0, dtype=v.dtype, device=DEV), v), 1)
    codes, scales = hstu_amd.quantize_mxfp4(x)
    want, e = orc.mxfp4_quantize_ref(x)
    assert torch.equal(scales.long(), e) and torch.equal(orc.mxfp4_decode_ref(codes, scales), want)
    assert int(e.min()) == int(e.max()) == 127


@gpu
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
def test_quantize_special_blocks(hip_lib, dtype):
    import hstu_amd

    info = torch.finfo(dtype)
    tiny = info.smallest_normal
    x = torch.zeros((12, 64), dtype=dtype)
    x[1, 5] = info.max
    x[2] = -info.max
    x[3, :32] = tiny * torch.linspace(0, 1, 32).to(dtype)  # subnormals
    x[4, 3] = tiny * 1.5
    x[5, 7] = float("inf")
    x[6, 40] = float("-inf")
    x[7, 0] = float("nan")
    x[8, 1], x[8, 33] = 1.0, -0.0
    x[9] = 6.0
    x[10] = 7.75  # rounds to 8, which is not a code: 6
    x[11, ::2] = -1.25
    x = x.to(DEV)
    codes, scales = hstu_amd.quantize_mxfp4(x)
    want, e = orc.mxfp4_quantize_ref(x)
    assert torch.equal(scales.long(), e)
    assert int(scales[0, 0]) == 0 and scales[5].tolist() == [255, 0] and scales[6].tolist() == [0, 255]
    assert same_values(orc.mxfp4_decode_ref(codes, scales), want)
    for out in (torch.bfloat16, torch.float32):
        assert same_values(hstu_amd.dequantize_mxfp4(codes, scales, out), want)


@gpu
def test_quantize_strides_and_shapes(hip_lib):
    import hstu_amd

    wide = rnd((40, 400), 3).to(DEV)
    for part in (wide[:, 8:264], wide[:, 3:259], wide[::2, :256], wide.t()[:64, :32]):
        a, b = hstu_amd.quantize_mxfp4(part), hstu_amd.quantize_mxfp4(part.contiguous())
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    c, s = hstu_amd.quantize_mxfp4(wide[:, :384].reshape(4, 10, 384))
    assert c.shape == (4, 10, 192) and s.shape == (4, 10, 12)
    assert hstu_amd.dequantize_mxfp4(c, s).shape == (4, 10, 384)
    c, s = hstu_amd.quantize_mxfp4(wide[:0, :64])
    assert c.shape == (0, 32) and hstu_amd.dequantize_mxfp4(c, s).shape == (0, 64)


@gpu
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("bias", [False, True])
@pytest.mark.parametrize("M,N,K", [(1, 16, 128), (3, 48, 256), (16, 64, 384), (17, 80, 128), (33, 272, 640),
                                   (64, 128, 512), (65, 256, 256), (130, 272, 1152), (257, 512, 1024), (300, 1040, 384),
                                   (1027, 528, 2048), (2050, 768, 256), (515, 2064, 896),
                                   (2600, 2576, 128), (2600, 2576, 256), (2600, 2576, 384), (2600, 2576, 512),
                                   (2600, 2576, 640), (2600, 2576, 768), (2600, 2576, 1024), (2600, 2576, 1152)])
def test_product(hip_lib, M, N, K, bias, residual):
    import hstu_amd

    x, w = rnd((M, K), 4, 2.0).to(DEV), rnd((N, K), 5, K ** -0.5, torch.float32).to(DEV)
    w[: N // 2] *= 2.0 ** -9  # weights of very different scales
    b = rnd((N,), 6).to(DEV) if bias else None
    r = rnd((M, N), 7).to(DEV) if residual else None
    a, wq = hstu_amd.quantize_mxfp4(x), hstu_amd.quantize_mxfp4(w)
    got = hstu_amd.mxfp4_mm(a, wq, bias=b, residual=r)
    av, wv = orc.mxfp4_decode_ref(*a), orc.mxfp4_decode_ref(*wq)
    want = av @ wv.t()
    mag = av.abs() @ wv.abs().t()
    for t in (b, r):
        if t is not None:
            want, mag = want + t.double(), mag + t.double().abs()
    off = (got.double() - want).abs()
    tol = want.abs() * HALF + (K + 16) * ULP * mag
    assert got.shape == (M, N) and (off <= tol).all(), float((off / tol).max())
    lin = hstu_amd.mxfp4_linear(x, wq, bias=b, residual=r)
    off = (lin.double() - want).abs()
    assert (off <= tol).all(), float((off / tol).max())


@gpu
@pytest.mark.parametrize("bias,residual", [(False, False), (True, True)])
@pytest.mark.parametrize("N", [8192, 8208])
@pytest.mark.parametrize("M,K", [(1, 128), (7, 384), (16, 1024), (16, 4096), (3, 8192)])
def test_few_rows_of_many_outputs(hip_lib, M, N, K, bias, residual):
    """Two column blocks a workgroup where x is quantised on the way, the last one of 16 columns or of 32."""
    from hstu_amd import mxfp4

    assert M <= mxfp4.ROWS_QUANT and M * K <= mxfp4.VALUES_QUANT
    test_product(hip_lib, M, N, K, bias, residual)


@gpu
def test_product_special_values(hip_lib):
    """NaN blocks make their rows (columns) NaN and no others; zero blocks and far scales are exact."""
    import hstu_amd

    for M in (4, 40, 300, 20000):  # every form
        K, N = 256, 272
        x, w = rnd((M, K), 8).to(DEV), rnd((N, K), 9).to(DEV)
        x[1, 64:96] = 0
        x[2] = 0
        clean = hstu_amd.mxfp4_linear(x, hstu_amd.quantize_mxfp4(w))
        assert not clean[2].any()
        x[0, 200], w[5, 3] = float("nan"), float("inf")
        got = hstu_amd.mxfp4_linear(x, hstu_amd.quantize_mxfp4(w))
        assert got[0].isnan().all() and got[:, 5].isnan().all()
        keep = torch.ones((M, N), dtype=torch.bool, device=DEV)
        keep[0], keep[:, 5] = False, False
        assert torch.equal(got[keep], clean[keep])
        # one block each at the two ends of the scales: 2^100 against 2^-100
        x, w = torch.zeros((M, K), dtype=torch.bfloat16, device=DEV), torch.zeros((N, K), dtype=torch.bfloat16, device=DEV)
        x[:, 32:64], w[:, 32:64] = 2.0 ** 100, 2.0 ** -100
        assert (hstu_amd.mxfp4_linear(x, hstu_amd.quantize_mxfp4(w)) == 32.0).all()


@gpu
def test_each_scale_and_block_has_its_place(hip_lib):
    """One value in each block in turn, every block with a scale of its own."""
    import hstu_amd

    for M, N, K in ((5, 32, 512), (40, 48, 512), (260, 272, 1024), (6300, 1040, 1024)):
        blocks = K // 32
        x = torch.zeros((M, K), device=DEV)
        w = torch.zeros((N, K), device=DEV)
        g = torch.Generator().manual_seed(3)
        for t in (x, w):
            at = torch.randint(0, 32, (t.shape[0], blocks), generator=g).to(DEV)
            e = torch.randint(-6, 7, (t.shape[0], blocks), generator=g).to(DEV)
            t.view(t.shape[0], blocks, 32).scatter_(2, at[..., None], torch.exp2(e.float())[..., None])
        got = hstu_amd.mxfp4_linear(x.bfloat16(), hstu_amd.quantize_mxfp4(w))
        want = x.double() @ w.double().t()
        assert ((got.double() - want).abs() <= want * HALF).all()


@gpu
def test_rows_past_the_last_are_left_and_strides(hip_lib):
    import hstu_amd
    import hstu_amd._lib as lib

    N, K = 272, 256
    for M in (1, 17, 130, 20000):  # every form
        a, w = hstu_amd.quantize_mxfp4(rnd((M, K), 10).to(DEV)), hstu_amd.quantize_mxfp4(rnd((N, K), 11).to(DEV))
        want = hstu_amd.mxfp4_mm(a, w)
        out = torch.full((M + 260, N + 8), 7.0, dtype=torch.bfloat16, device=DEV)
        st = lib.fn("hstu_mxfp4_gemm")(a[0].data_ptr(), K // 2, a[1].data_ptr(), K // 32, w[0].data_ptr(), K // 2,
                                       w[1].data_ptr(), K // 32, None, None, 0, out.data_ptr(), N + 8, M, N, K,
                                       lib.stream(out))
        assert st == 0 and (out[M:] == 7).all() and (out[:, N:] == 7).all()
        assert torch.equal(out[:M, :N], want)
        # codes and scales as slices of wider buffers
        wide = [torch.full((t.shape[0], t.shape[1] + 64), 255, dtype=torch.uint8, device=DEV) for t in a + w]
        for t, s in zip(wide, a + w):
            t[:, 16:16 + s.shape[1]] = s
        ac, as_, wc, ws = (t[:, 16:16 + s.shape[1]] for t, s in zip(wide, a + w))
        assert torch.equal(hstu_amd.mxfp4_mm((ac, as_), (wc, ws)), want)
        r = torch.zeros((M, N + 24), dtype=torch.bfloat16, device=DEV)[:, 8:8 + N]
        assert torch.equal(hstu_amd.mxfp4_mm(a, w, residual=r), want)


@gpu
def test_side_stream_graph_and_same_bytes(hip_lib):
    import hstu_amd

    x, x2 = rnd((37, 512), 12).to(DEV), rnd((600, 512), 13).to(DEV)
    w = hstu_amd.quantize_mxfp4(rnd((528, 512), 14).to(DEV))

    def step():
        q = hstu_amd.quantize_mxfp4(x2)
        return (hstu_amd.mxfp4_linear(x, w), hstu_amd.mxfp4_mm(q, w), hstu_amd.dequantize_mxfp4(*q), q[0], q[1])

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        on_side = step()
    torch.cuda.current_stream().wait_stream(side)
    want = step()
    assert all(torch.equal(a, b) for a, b in zip(on_side, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for k in range(4):
        x.copy_(rnd((37, 512), 20 + k))
        x2.copy_(rnd((600, 512), 30 + k))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, step())), k


@gpu
def test_past_32_bit_offsets(hip_lib):
    import hstu_amd

    rows, cols = 2 ** 22 + 3, 512  # over 2^31 values
    x = torch.zeros((rows, cols), dtype=torch.bfloat16, device=DEV)
    x[-5:] = rnd((5, cols), 15).to(DEV)
    codes, scales = hstu_amd.quantize_mxfp4(x)
    c, s = hstu_amd.quantize_mxfp4(x[-5:].clone())
    assert torch.equal(codes[-5:], c) and torch.equal(scales[-5:], s) and not codes[:-5].any()
    v = hstu_amd.dequantize_mxfp4(codes, scales)
    assert torch.equal(v[-5:], hstu_amd.dequantize_mxfp4(c, s)) and not v[:-5].any()
    del x, v
    w = hstu_amd.quantize_mxfp4(rnd((528, cols), 16).to(DEV))  # an output of over 2^31 values
    out = hstu_amd.mxfp4_mm((codes, scales), w)
    assert torch.equal(out[-5:], hstu_amd.mxfp4_mm((codes[-1029:], scales[-1029:]), w)[-5:])
    assert not out[:-5].any()


@gpu
@pytest.mark.parametrize("residual", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.float64])
@pytest.mark.parametrize("M,N,K", [(5, 48, 384), (16, 8208, 128), (24, 272, 256), (300, 272, 640), (2600, 2576, 384)])
def test_bias_keeps_its_bits(hip_lib, M, N, K, dtype, residual):
    """A bias is not rounded to bf16 on the way to the fp32 sum.  Every code is 0, so the sum is exact: the bias
    (fp32 at the most: 2^-24), plus the residual (one rounding, 2^-24 of the magnitudes), rounded to bf16 once.
    Biases next to the middle of two bf16 values, which their own rounding would move to the other one."""
    import hstu_amd

    b = rnd((N,), 6, 1.0, torch.float32)
    b = (b.bfloat16().float() * (1 + 2.0 ** -8 + 2.0 ** -10 * torch.rand(N, generator=torch.Generator().manual_seed(3)))).to(dtype).to(DEV)
    r = rnd((M, N), 7, 2.0 ** -8).to(DEV) if residual else None
    x, w = torch.zeros((M, K), dtype=torch.bfloat16, device=DEV), hstu_amd.quantize_mxfp4(torch.zeros((N, K), device=DEV))
    want, mag = b.double().expand(M, N), b.double().abs().expand(M, N)
    if residual:
        want, mag = want + r.double(), mag + r.double().abs()
    tol = want.abs() * HALF + mag * 2.0 ** -23
    got = [hstu_amd.mxfp4_linear(x, w, bias=b, residual=r), hstu_amd.mxfp4_mm(hstu_amd.quantize_mxfp4(x), w, bias=b, residual=r)]
    for out in got:
        off = (out.double() - want).abs()
        assert (off <= tol).all(), float((off / tol).max())
        # half a step of bf16 at this value, not of the largest mantissa's: nearest, but for the ties of fp32
        near = b.float().expand(M, N) + (r.float() if residual else 0)
        assert torch.equal(out, near.bfloat16())
    odd = torch.zeros(N + 1, dtype=dtype, device=DEV)[1:].copy_(b)  # not 16-byte aligned; every second of a longer one
    for same in (odd, torch.stack((b, b), 1)[:, 0]):
        assert torch.equal(hstu_amd.mxfp4_linear(x, w, bias=same, residual=r), got[0])
    with pytest.raises(NotImplementedError):
        hstu_amd.mxfp4_linear(x, w, bias=torch.zeros(N, dtype=torch.int32, device=DEV))


def test_bias_type_goes_to_the_entry_point():
    """No bias is cast to bf16 (no device is touched)."""
    from hstu_amd import mxfp4

    for dtype, kept, entry in ((torch.bfloat16, torch.bfloat16, ""), (torch.float32, torch.float32, "_bias_fp32"),
                               (torch.float16, torch.float32, "_bias_fp32")):
        b = rnd((48,), 6, 1.0, dtype)
        got = mxfp4._epilogue(b, None, (2, 48), b.device)
        assert got[0].dtype == kept and torch.equal(got[0], b.to(kept)) and got[2] == entry


def test_tile_epilogue_orders_its_lanes():
    """The tile form's outputs pass between the lanes of a wave through LDS, the residual before them: each
    exchange has a wave-level order between the lanes' writes and the others' reads, in the source, since a
    compiler that leaves the order alone hides a missing one."""
    from pathlib import Path

    src = (Path(__file__).parents[1] / "mlperf-training_amd" / "csrc" / "hstu_mxfp4.hip").read_text()
    body = src[src.index("void __launch_bounds__(kMxThreads, 2) mx_tile_kernel"):]
    body = body[body.index("auto line_at"):body.index("hipError_t set_mx_lds")]
    resid_in = body.index("*(u32x4*)(smem + line_at(")          # rows in, lane = row and chunk of a line
    meet = body.index("smem + out_at(nb, run)")                 # the accumulators' lanes
    lines_out = body.rindex("*(const u32x4*)(smem + line_at(")  # whole lines again
    assert resid_in < meet < lines_out
    assert "wave_lds_order();" in body[resid_in:meet] and "wave_lds_order();" in body[meet:lines_out]


# ---------------------------------------------------------------- refusals
def test_oracle_packs_and_unpacks():
    x = rnd((5, 96), 1, 3.0)
    v, e = orc.mxfp4_quantize_ref(x)
    codes, scales = pack_ref(x)
    assert torch.equal(orc.mxfp4_decode_ref(codes, scales), v)
    assert float((v - x.double()).abs().max()) <= float(x.abs().max()) / 4


def test_refusals():
    import hstu_amd

    with pytest.raises(NotImplementedError):
        hstu_amd.quantize_mxfp4(torch.zeros(2, 32))  # not on a device
    with pytest.raises(NotImplementedError):
        hstu_amd.quantize_mxfp4(torch.zeros(2, 33))
    with pytest.raises(NotImplementedError):
        hstu_amd.quantize_mxfp4(torch.zeros(2, 32, dtype=torch.float16))
    with pytest.raises(NotImplementedError):
        hstu_amd.mxfp4_linear(torch.zeros(2, 128), (torch.zeros(16, 64), torch.zeros(16, 4)))
    u = torch.uint8
    with pytest.raises(NotImplementedError):
        hstu_amd.dequantize_mxfp4(torch.zeros(2, 16, dtype=u), torch.zeros(2, 1, dtype=u))


@gpu
def test_refusals_on_device(hip_lib):
    import hstu_amd

    def u(*shape):
        return torch.zeros(shape, dtype=torch.uint8, device=DEV)

    good = (u(16, 64), u(16, 4))
    a = (u(3, 64), u(3, 4))
    for bad in ((u(16, 64), u(16, 5)), (u(16, 64), u(15, 4)), (u(16, 64).float(), u(16, 4))):
        with pytest.raises(ValueError):
            hstu_amd.dequantize_mxfp4(*bad)
        with pytest.raises(ValueError):
            hstu_amd.mxfp4_mm(a, bad)
        with pytest.raises(ValueError):
            hstu_amd.mxfp4_mm(bad, good)
    with pytest.raises(ValueError):
        hstu_amd.mxfp4_mm((u(3, 128), u(3, 8)), good)
    for bad in ((u(8, 64), u(8, 4)), (u(16, 48), u(16, 3))):
        with pytest.raises(NotImplementedError):
            hstu_amd.mxfp4_mm((u(3, bad[0].shape[1]), u(3, bad[1].shape[1])), bad)
    with pytest.raises(ValueError):
        hstu_amd.mxfp4_mm(a, good, bias=torch.zeros(15, device=DEV))
    with pytest.raises(ValueError):
        hstu_amd.mxfp4_mm(a, good, residual=torch.zeros(3, 16, device=DEV))
    with pytest.raises(NotImplementedError):
        hstu_amd.dequantize_mxfp4(*good, dtype=torch.float16)


def test_c_entry_refusals():
    """Bad arguments are refused before any launch (no device is touched)."""
    import hstu_amd._lib as lib

    P = 64  # a stand-in address, never read
    q, d, g = (lib.fn("hstu_mxfp4_" + n) for n in ("quantize", "dequantize", "gemm"))
    BF = lib.HSTU_DTYPE_BF16
    assert q(9, P, 64, 2, 64, P, P, None) == lib.HSTU_E_BAD_ARG
    assert q(BF, P, 63, 2, 64, P, P, None) == lib.HSTU_E_BAD_ARG
    assert q(BF, None, 64, 2, 64, P, P, None) == lib.HSTU_E_BAD_ARG
    assert q(BF, P, 64, -1, 64, P, P, None) == lib.HSTU_E_BAD_ARG
    assert q(BF, P, 64, 2, 48, P, P, None) == lib.HSTU_E_UNSUPPORTED
    assert q(BF, 65, 64, 2, 64, P, P, None) == lib.HSTU_E_UNSUPPORTED
    assert q(BF, P, 64, 0, 64, P, P, None) == 0
    assert d(P, P, 2, 64, 9, P, 64, None) == lib.HSTU_E_BAD_ARG
    assert d(P, P, 2, 64, BF, P, 63, None) == lib.HSTU_E_BAD_ARG
    assert d(P, None, 2, 64, BF, P, 64, None) == lib.HSTU_E_BAD_ARG
    assert d(P, P, 2, 64, BF, 72, 64, None) == lib.HSTU_E_UNSUPPORTED
    assert d(P, P, 0, 64, BF, P, 64, None) == 0

    def gemm(A=P, lda=64, sa=P, ldsa=4, W=P, ldw=64, sw=P, ldsw=4, bias=None, res=None, ldr=0, C=P, ldc=16, M=2, N=16, K=128):
        return g(A, lda, sa, ldsa, W, ldw, sw, ldsw, bias, res, ldr, C, ldc, M, N, K, None)

    for bad in (dict(M=-1), dict(N=0), dict(K=0), dict(lda=63), dict(ldw=48), dict(ldsa=3), dict(ldsw=3), dict(ldc=15),
                dict(res=P, ldr=8), dict(A=None), dict(W=None), dict(sa=None), dict(sw=None), dict(C=None)):
        assert gemm(**bad) == lib.HSTU_E_BAD_ARG, bad
    for bad in (dict(N=8), dict(N=24, ldc=24), dict(K=96), dict(A=72), dict(lda=72), dict(sa=66), dict(ldsw=6), dict(C=72),
                dict(ldc=20), dict(bias=66), dict(res=66, ldr=16)):
        assert gemm(**bad) == lib.HSTU_E_UNSUPPORTED, bad
    assert gemm(M=0) == 0
    rows = lib.fn("hstu_mxfp4_linear_rows")

    def linear(x=P, ldx=128, W=P, ldw=64, sw=P, ldsw=4, res=None, ldr=0, C=P, ldc=16, M=2, N=16, K=128):
        return rows(x, ldx, W, ldw, sw, ldsw, None, res, ldr, C, ldc, M, N, K, None)

    for bad in (dict(M=-1), dict(ldx=127), dict(x=None), dict(W=None), dict(sw=None), dict(C=None), dict(ldc=8),
                dict(res=P, ldr=8)):
        assert linear(**bad) == lib.HSTU_E_BAD_ARG, bad
    for bad in (dict(x=72), dict(ldx=132), dict(K=96), dict(N=24, ldc=24)):
        assert linear(**bad) == lib.HSTU_E_UNSUPPORTED, bad
    assert linear(M=0) == 0
