"""MXFP4 quantization, dequantization and products on the GPU against plain
64-bit restatements (kc_mxfp4).

Quantization and dequantization are exact by definition: bit for bit.
Products of two E2M1 values are multiples of 1/4 up to 36, so with equal scales
and K <= 14336 every partial sum is a multiple of 1/4 below 2^19 (2^21 steps) and
exact in fp32 in any order: bit for bit.  In general each of the K additions into an
fp32 accumulator is off by at most 2^-23 of the sum of the magnitudes (the
matrix core truncates), so an fp32 output is within K * 2^-23 * sum |product|
of the exact one and a bf16 output a rounding (2^-8 of its size) more.
"""
import numpy as np
import pytest

import kc_mxfp4 as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(gpu):
    import kernel_craft_torch_ops
    return kernel_craft_torch_ops


def _t(gpu, a):
    return gpu.from_numpy(np.ascontiguousarray(a)).cuda()


def _bf16(gpu, a):
    return gpu.from_numpy(np.ascontiguousarray(a, dtype=np.float32)).cuda().bfloat16()


def _f64(t):
    return t.double().cpu().numpy()


def _shift(gpu, t, by):
    """A copy of t whose memory starts `by` elements into an allocation."""
    buf = gpu.empty(t.numel() + by, dtype=t.dtype, device="cuda")
    out = buf[by:].view(t.shape)
    out.copy_(t)
    return out


def _check_quantized(ops, x):
    codes, scales = ops.mxfp4_quantize(x)
    ec, es = ref.quantize(_f64(x))
    np.testing.assert_array_equal(scales.cpu().numpy(), es)
    np.testing.assert_array_equal(codes.cpu().numpy(), ec)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("rows,cols", [(1, 32), (3, 64), (7, 96), (1, 4096), (129, 544), (2003, 5120)])
def test_quantize_rows(gpu, ops, rows, cols, dtype):
    rng = np.random.default_rng(rows * 7 + cols)
    x = rng.standard_normal((rows, cols)) * np.exp2(rng.integers(-20, 20, (rows, 1)))
    x[rng.random((rows, cols)) < 0.1] = 0.0
    _check_quantized(ops, gpu.from_numpy(x).cuda().to(getattr(gpu, dtype)))


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_quantize_unaligned_input(gpu, ops, dtype):
    x = _shift(gpu, gpu.randn(5, 96, device="cuda").to(getattr(gpu, dtype)), 1)
    _check_quantized(ops, x)


def test_quantize_every_bf16_value_at_every_scale(gpu, ops):
    """Every finite bf16 value under block maxima of every binade at and
    above its own: each block holds the maximum and 31 values."""
    bits = np.arange(0x8000, dtype=np.uint16)
    bits = bits[bits < 0x7F80]
    for up in (0, 1, 2, 3, 4, 8):
        top = np.minimum(bits.astype(np.int64) // 128 + up, 254) * 128 + 127   # the binade's largest value
        blk = np.empty((len(bits), 32), dtype=np.uint16)
        blk[:, 0] = top
        blk[:, 1::2] = bits[:, None]
        blk[:, 2::2] = bits[:, None] | 0x8000
        x = gpu.from_numpy(blk.view(np.int16)).cuda().view(gpu.bfloat16)
        _check_quantized(ops, x)
        _check_quantized(ops, x.float())


def test_quantize_fp32_around_every_midpoint(gpu, ops):
    """fp32 values at, one step under and one step over every rounding
    boundary, at every scale byte 0 .. 252."""
    e = np.arange(-127, 126)
    mids = np.concatenate([ref.MID, ref.GRID, [5.999, 7.9]])
    x = np.ldexp(mids[None, :], e[:, None])
    vals = np.concatenate([x, x, x], 1).astype(np.float32)
    n = mids.size
    vals[:, n:2 * n] = np.nextafter(vals[:, n:2 * n], np.float32(0))
    vals[:, 2 * n:] = np.nextafter(vals[:, 2 * n:], np.float32(np.inf))
    blk = np.zeros((len(e), 2, 32), dtype=np.float32)
    blk[:, :, 0] = np.ldexp(np.float32(7.5), e)[:, None]    # sets the scale to 2^e
    flat = vals.reshape(len(e), -1)[:, :62]
    flat = np.minimum(flat, blk[:, 0, :1])
    blk[:, 0, 1:] = flat[:, :31]
    blk[:, 1, 1:flat.shape[1] - 30] = -flat[:, 31:]
    _check_quantized(ops, gpu.from_numpy(blk.reshape(len(e), 64)).cuda())


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_quantize_special_blocks(gpu, ops, dtype):
    """Zeros, negative zeros, subnormals, the largest values, NaN and
    infinities (each alone in its block)."""
    dt = getattr(gpu, dtype)
    x = gpu.randn(10, 64, device="cuda").to(dt)
    x[0] = 0.0
    x[1] = -0.0
    x[2] = 0.0
    x[2, 5] = gpu.finfo(dt).smallest_normal / 4
    x[3, 40] = float("nan")
    x[4, 3] = float("inf")
    x[5, 63] = -float("inf")
    x[6, 7] = gpu.finfo(dt).max
    x[7] *= 1e-38
    x[8] = gpu.finfo(dt).smallest_normal
    _check_quantized(ops, x)
    codes, scales = ops.mxfp4_quantize(x)
    back = ops.mxfp4_dequantize(codes, scales, out_dtype=dt)
    assert bool(gpu.isnan(back[3, 32:]).all()) and not bool(gpu.isnan(back[3, :32]).any())
    assert bool(gpu.isnan(back[4, :32]).all()) and bool(gpu.isnan(back[5, 32:]).all())


@pytest.mark.parametrize("out", ["bfloat16", "float32"])
@pytest.mark.parametrize("off", [0, 1])
def test_dequantize_every_code_at_every_scale(gpu, ops, out, off):
    codes = np.tile(np.concatenate([np.arange(16), np.arange(16)[::-1]]).astype(np.uint8), (256, 1))
    packed = codes[:, 0::2] | (codes[:, 1::2] << 4)
    scales = np.arange(256, dtype=np.uint8)[:, None]
    dt = getattr(gpu, out)
    if off:
        from kernel_craft_torch_ops import _get_lib
        from kc_abi import check, ptr, stream
        buf = gpu.empty(256 * 32 + 1, dtype=dt, device="cuda")
        got = buf[1:].view(256, 32)
        fn = _get_lib().kc_dequantize_mxfp4_bf16 if out == "bfloat16" else _get_lib().kc_dequantize_mxfp4_f32
        c, s = _t(gpu, packed), _t(gpu, scales)
        check("dequantize", fn(ptr(c), ptr(s), ptr(got), 256, 32, stream()))
    else:
        got = ops.mxfp4_dequantize(_t(gpu, packed), _t(gpu, scales), out_dtype=dt)
    want = gpu.from_numpy(ref.values(packed, scales)).to(dt)   # one rounding, where a value leaves the range
    np.testing.assert_array_equal(got.float().cpu().numpy(), want.float().numpy())


def _mx(rng, rows, cols, lo=120, hi=134):
    return (rng.integers(0, 256, (rows, cols // 2), dtype=np.uint8),
            rng.integers(lo, hi, (rows, cols // 32), dtype=np.uint8))


W4A4_SHAPES = [(1, 1, 32), (1, 16, 64), (2, 33, 96), (5, 100, 160), (16, 16, 128), (17, 31, 288), (33, 257, 512),
               (64, 300, 1024), (65, 129, 1056), (100, 513, 4096), (128, 256, 2048), (255, 260, 544),
               (256, 256, 256), (257, 511, 768), (300, 1000, 1312), (513, 1025, 320), (1, 4096, 4096),
               (8, 6144, 4096), (32, 1100, 14336), (700, 264, 96), (20, 8200, 288), (33, 9001, 1024), (64, 12300, 544),
              (50, 28672, 256), (5, 13000, 2080), (130, 4100, 1600), (1100, 3000, 1056), (2100, 2100, 2112), (64, 8192, 992),
              # several groups of steps, K a multiple of 128 and not, on every larger tile
              (500, 6144, 2176), (700, 5000, 2208), (300, 4096, 2176), (300, 4096, 2080), (300, 4096, 4224),
              (300, 4096, 4128), (300, 28672, 2112), (400, 2100, 2176),
              # several spans a wave and a tail with one to four tiles of tokens, one and two of rows
              (9, 3000, 5152), (9, 12500, 5152), (25, 3000, 5152), (25, 5000, 5152), (40, 3000, 5152),
              (40, 6100, 5152), (60, 3000, 5152)]


@pytest.mark.parametrize("out", ["bfloat16", "float32"])
@pytest.mark.parametrize("M,N,K", W4A4_SHAPES)
def test_w4a4_layout_is_exact(gpu, ops, M, N, K, out):
    """Equal scales: every sum is exact, in any order."""
    rng = np.random.default_rng(M + 3 * N + 7 * K)
    (qx, _), (qw, _) = _mx(rng, M, K), _mx(rng, N, K)
    sx, sw = np.full((M, K // 32), 127, np.uint8), np.full((N, K // 32), 126, np.uint8)
    y = ops.mxfp4_gemm_w4a4(_t(gpu, qx), _t(gpu, sx), _t(gpu, qw), _t(gpu, sw), out_dtype=getattr(gpu, out))
    want = gpu.from_numpy(ref.values(qx, sx) @ ref.values(qw, sw).T)
    assert gpu.equal(y.cpu(), want.to(y.dtype))


@pytest.mark.parametrize("M,N,K", W4A4_SHAPES)
def test_w4a4_scales(gpu, ops, M, N, K):
    """A scale of its own for every block."""
    rng = np.random.default_rng(M + 5 * N + K)
    (qx, sx), (qw, sw) = _mx(rng, M, K), _mx(rng, N, K)
    x, w = ref.values(qx, sx), ref.values(qw, sw)
    args = [_t(gpu, a) for a in (qx, sx, qw, sw)]
    exact, size = x @ w.T, np.abs(x) @ np.abs(w).T
    y = ops.mxfp4_gemm_w4a4(*args, out_dtype=gpu.float32)
    assert (np.abs(_f64(y) - exact) <= K * 2.0 ** -23 * size).all()
    y = ops.mxfp4_gemm_w4a4(*args)
    assert (np.abs(_f64(y) - exact) <= K * 2.0 ** -23 * size + 2.0 ** -8 * np.abs(exact)).all()


@pytest.mark.parametrize("M,N,K", [(5, 300, 2176), (100, 513, 2176), (300, 4096, 2176), (500, 6144, 2176), (40, 9000, 4224)])
def test_products_with_scales_at_odd_addresses(gpu, ops, M, N, K):
    """Codes must be aligned, scale bytes need not be.  W4A4 sums in one order
    wherever they lie; bf16 activations may take another kernel."""
    rng = np.random.default_rng(M + N + K)
    (qx, sx), (qw, sw) = _mx(rng, M, K), _mx(rng, N, K)
    x, w = _bf16(gpu, rng.standard_normal((M, K))), ref.values(qw, sw)
    exact, size = _f64(x) @ w.T, np.abs(_f64(x)) @ np.abs(w).T
    qx, sx, qw, sw = [_t(gpu, a) for a in (qx, sx, qw, sw)]
    y = ops.mxfp4_gemm_w4a4(qx, sx, qw, sw)
    for by in (1, 2, 3):
        assert gpu.equal(ops.mxfp4_gemm_w4a4(qx, _shift(gpu, sx, by), qw, _shift(gpu, sw, by)), y)
        a16 = ops.mxfp4_gemm_bf16(qw, _shift(gpu, sw, by), x)
        assert (np.abs(_f64(a16) - exact) <= K * 2.0 ** -23 * size + 2.0 ** -8 * np.abs(exact)).all()


@pytest.mark.parametrize("M", [1, 40, 300])
def test_w4a4_one_block_at_a_time(gpu, ops, M):
    """A matrix whose only block with values walks over K: a scale of the
    wrong block (or row) shows."""
    N, K = 300, 1056
    rng = np.random.default_rng(M)
    qx, _ = _mx(rng, M, K)
    qw, _ = _mx(rng, N, K)
    sx = rng.integers(100, 150, (M, K // 32), dtype=np.uint8)
    sw = rng.integers(100, 150, (N, K // 32), dtype=np.uint8)
    for b in range(K // 32):
        one = np.zeros_like(qx)
        one[:, 16 * b:16 * b + 16] = qx[:, 16 * b:16 * b + 16]
        y = ops.mxfp4_gemm_w4a4(_t(gpu, one), _t(gpu, sx), _t(gpu, qw), _t(gpu, sw), out_dtype=gpu.float32)
        want = ref.values(one, sx) @ ref.values(qw, sw).T     # one block: exact in fp32
        np.testing.assert_array_equal(y.cpu().numpy(), want.astype(np.float32))


@pytest.mark.parametrize("M", [2, 48, 260])
def test_w4a4_nan_scale_stays_in_its_row_and_column(gpu, ops, M):
    N, K = 270, 416
    rng = np.random.default_rng(M)
    (qx, sx), (qw, sw) = _mx(rng, M, K), _mx(rng, N, K)
    sx[M - 1, K // 32 - 1] = 255
    sw[3, 0] = 255
    y = ops.mxfp4_gemm_w4a4(*(_t(gpu, a) for a in (qx, sx, qw, sw)), out_dtype=gpu.float32).cpu().numpy()
    want = np.zeros((M, N), bool)
    want[M - 1] = True
    want[:, 3] = True
    np.testing.assert_array_equal(np.isnan(y), want)


A16_SHAPES = [(1, 1, 32), (1, 17, 64), (3, 40, 96), (1, 4096, 4096), (7, 1000, 1056), (13, 2048, 4096),
              (16, 16, 128), (17, 515, 544), (31, 96, 2048), (33, 129, 320), (48, 600, 1024), (64, 1100, 14336),
              (65, 300, 800), (128, 260, 4096), (130, 33, 288), (1, 28672, 512), (1, 77, 2048), (1, 1000, 2080),
              (1, 130, 16384), (1, 50, 16416), (1, 301, 10240), (40, 4097, 320), (20, 9000, 288), (60, 17000, 256),
              (33, 28672, 256), (200, 8200, 96), (128, 6144, 384), (500, 4100, 640),
              (64, 20003, 256), (300, 1000, 1152), (32, 28672, 128),
              # several spans of 1024 a wave and a tail, in every tile shape
              (5, 300, 9248), (5, 4200, 9248), (13, 9000, 5152), (9, 17000, 5152), (20, 9000, 5152),
              (20, 17000, 5152), (48, 17000, 5152),
              # the tiles in LDS: even and odd steps, a half step at the end
              (100, 4500, 2176), (100, 4500, 2304), (45, 16500, 2176), (60, 16500, 2304), (60, 16500, 2176),
              (100, 22000, 2176), (120, 16500, 1024)]


@pytest.mark.parametrize("M,N,K", A16_SHAPES)
def test_a16_layout_is_exact(gpu, ops, M, N, K):
    """Integer activations up to 8 and equal scales: every partial sum is a
    multiple of 1/2 below 2^20."""
    rng = np.random.default_rng(M + 3 * N + 7 * K)
    qw, _ = _mx(rng, N, K)
    sw = np.full((N, K // 32), 127, np.uint8)
    x = rng.integers(-8, 9, (M, K)).astype(np.float64)
    y = ops.mxfp4_gemm_bf16(_t(gpu, qw), _t(gpu, sw), _bf16(gpu, x))
    want = gpu.from_numpy(x @ ref.values(qw, sw).T)
    assert gpu.equal(y.cpu(), want.bfloat16())


@pytest.mark.parametrize("M,N,K", A16_SHAPES)
def test_a16_scales(gpu, ops, M, N, K):
    rng = np.random.default_rng(M + 5 * N + K)
    qw, sw = _mx(rng, N, K)
    x = _bf16(gpu, rng.standard_normal((M, K)))
    w, xd = ref.values(qw, sw), _f64(x)
    exact, size = xd @ w.T, np.abs(xd) @ np.abs(w).T
    y = ops.mxfp4_gemm_bf16(_t(gpu, qw), _t(gpu, sw), x)
    assert (np.abs(_f64(y) - exact) <= K * 2.0 ** -23 * size + 2.0 ** -8 * np.abs(exact)).all()


@pytest.mark.parametrize("M", [1, 20])
def test_a16_one_block_at_a_time(gpu, ops, M):
    N, K = 130, 1056
    rng = np.random.default_rng(M)
    qw, _ = _mx(rng, N, K)
    sw = rng.integers(60, 190, (N, K // 32), dtype=np.uint8)
    for b in range(K // 32):
        x = np.zeros((M, K))
        x[:, 32 * b:32 * b + 32] = rng.integers(-8, 9, (M, 32))
        y = ops.mxfp4_gemm_bf16(_t(gpu, qw), _t(gpu, sw), _bf16(gpu, x))
        want = gpu.from_numpy(x @ ref.values(qw, sw).T).bfloat16()
        assert gpu.equal(y.cpu(), want)


def test_a16_nan_and_infinity(gpu, ops):
    """A NaN scale marks its column, a NaN or infinite activation its row."""
    M, N, K = 5, 70, 288
    rng = np.random.default_rng(0)
    qw, sw = _mx(rng, N, K)
    qw &= 0x77
    qw |= 0x11   # positive weights: an infinity stays one
    sw[9, 8] = 255
    x = rng.standard_normal((M, K))
    x[2, 100] = np.nan
    x[4, 287] = np.inf
    y = ops.mxfp4_gemm_bf16(_t(gpu, qw), _t(gpu, sw), _bf16(gpu, x)).float().cpu().numpy()
    assert np.isnan(y[:, 9]).all() and np.isnan(y[2]).all()
    rest = np.delete(y, 9, 1)
    assert np.isposinf(rest[4]).all() and np.isfinite(np.delete(rest, [2, 4], 0)).all()


@pytest.mark.parametrize("M", [0, 4])
@pytest.mark.parametrize("N", [0, 40])
@pytest.mark.parametrize("K", [0, 64])
def test_empty_shapes(gpu, ops, M, N, K):
    z = lambda *s: gpu.zeros(*s, dtype=gpu.uint8, device="cuda")  # noqa: E731
    for dt in (gpu.bfloat16, gpu.float32):
        y = ops.mxfp4_gemm_w4a4(z(M, K // 2), z(M, K // 32), z(N, K // 2), z(N, K // 32), out_dtype=dt)
        assert y.shape == (M, N) and (not y.numel() or float(y.abs().max()) == 0)
        q, s = ops.mxfp4_quantize(gpu.zeros(M, K, dtype=dt, device="cuda"))
        assert ops.mxfp4_dequantize(q, s, out_dtype=dt).shape == (M, K)
    y = ops.mxfp4_gemm_bf16(z(N, K // 2), z(N, K // 32), gpu.zeros(M, K, dtype=gpu.bfloat16, device="cuda"))
    assert y.shape == (M, N) and (not y.numel() or float(y.abs().max()) == 0)


def test_strided_views_are_taken_as_values(gpu, ops):
    x = gpu.randn(64, 300, device="cuda").bfloat16().t()[::3]      # [100, 64], neither stride 1
    q, s = ops.mxfp4_quantize(x)
    qc, sc = ops.mxfp4_quantize(x.contiguous())
    assert gpu.equal(q, qc) and gpu.equal(s, sc)
    w, ws = ops.mxfp4_quantize(gpu.randn(96, 64, device="cuda"))
    assert gpu.equal(ops.mxfp4_gemm_bf16(w[::2], ws[::2], x), ops.mxfp4_gemm_bf16(w[::2].contiguous(),
                                                                                 ws[::2].contiguous(), x.contiguous()))


@pytest.mark.parametrize("M", [3, 700])
def test_other_stream_and_graph_replays(gpu, ops, M):
    """A linear layer (quantize, product) on a side stream and captured, each
    replay on new activations; eager work runs between the replays."""
    torch = gpu
    w, ws = ops.mxfp4_quantize(torch.randn(500, 1024, device="cuda") * 0.02)
    x = torch.randn(M, 1024, device="cuda").bfloat16()

    def layer(a):
        return ops.mxfp4_gemm_w4a4(*ops.mxfp4_quantize(a), w, ws), ops.mxfp4_gemm_bf16(w, ws, a)

    want = layer(x)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = layer(x)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = layer(x)
    for i in range(4):
        x.copy_(torch.randn(M, 1024, device="cuda").bfloat16())
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(out, layer(x)))


# The products with bf16 activations over the whole range of scales: Y = X W^T, W as
# mxfp4_dequantize gives it in bf16, whichever kernel the number of tokens leads to.
# M 1: the GEMV (K from 2048), or the matrix cores (K 96); 5 and 40 tokens in registers, 100 in LDS tiles.
A16_KERNELS = [(1, 2080), (1, 96), (5, 2176), (40, 2080), (100, 2176)]


def _one_block_rows(rng, N, K, byte, low=0):
    """N rows with codes in one block each, of any scale in `byte`; all others zero.  `low`: the smallest code."""
    qw, sw = np.zeros((N, K // 32, 16), np.uint8), np.full((N, K // 32), 127, np.uint8)
    at, rows = rng.integers(0, K // 32, N), np.arange(N)
    codes = rng.integers(low, 8, (N, 32), dtype=np.uint8) | (rng.integers(0, 2, (N, 32), dtype=np.uint8) << 3)
    qw[rows, at] = codes[:, 0::2] | (codes[:, 1::2] << 4)
    sw[rows, at] = byte
    return qw.reshape(N, K // 2), sw


@pytest.mark.parametrize("M,K", A16_KERNELS)
@pytest.mark.parametrize("first,last,x_exponent", [(0, 127, 60), (128, 252, -60), (64, 110, 120), (150, 252, -120)])
def test_a16_every_scale(gpu, ops, M, K, first, last, x_exponent):
    """One block a row: with activations n 2^e, |n| <= 8, its 32 terms are multiples of one
    power of two, at most 32 * 48 * 2 of them, and exact in fp32 in any order.  Activations
    of 2^123 on scales far below 1, and of 2^-120 on large ones, among them: the terms
    are in fp32's range only with their scale."""
    rng = np.random.default_rng(M + first)
    N = 16500 if M == 100 else 520
    byte = np.resize(np.arange(first, last + 1), N)
    qw, sw = _one_block_rows(rng, N, K, byte)
    x = np.ldexp(rng.integers(-8, 9, (M, K)).astype(np.float64), x_exponent)
    y = ops.mxfp4_gemm_bf16(_t(gpu, qw), _t(gpu, sw), _bf16(gpu, x))
    want = gpu.from_numpy(x @ ref.values(qw, sw).T).float().bfloat16()    # exact in fp32
    assert gpu.equal(y.cpu(), want)


@pytest.mark.parametrize("M,K", A16_KERNELS)
def test_a16_subnormal_activations(gpu, ops, M, K):
    """bf16's subnormal activations on large scales."""
    rng = np.random.default_rng(M)
    N = 16500 if M == 100 else 300
    qw, sw = _one_block_rows(rng, N, K, np.resize(np.arange(180, 250), N))
    x = np.ldexp(rng.integers(-8, 9, (M, K)).astype(np.float64), -133)
    y = ops.mxfp4_gemm_bf16(_t(gpu, qw), _t(gpu, sw), _bf16(gpu, x))
    want = gpu.from_numpy(x @ ref.values(qw, sw).T).float().bfloat16()
    assert gpu.equal(y.cpu(), want)


@pytest.mark.parametrize("M,K", A16_KERNELS)
def test_a16_weights_past_the_range_are_bf16_infinities(gpu, ops, M, K):
    """Scale bytes 253 and 254 with codes whose value leaves bf16's range."""
    rng = np.random.default_rng(M)
    N = 16500 if M == 100 else 64
    qw, sw = _one_block_rows(rng, N, K, np.resize([253, 254], N), low=6)
    qw &= 0x77  # positive
    x = np.full((M, K), 2.0 ** -20)
    w = ops.mxfp4_dequantize(_t(gpu, qw), _t(gpu, sw))
    assert bool(gpu.isinf(w).any(1).all())
    y = ops.mxfp4_gemm_bf16(_t(gpu, qw), _t(gpu, sw), _bf16(gpu, x))
    assert bool((y == float("inf")).all())


@pytest.mark.parametrize("M,K", A16_KERNELS)
def test_a16_nan_scale_marks_its_column(gpu, ops, M, K):
    rng = np.random.default_rng(M)
    N = 16500 if M == 100 else 70
    qw, sw = _mx(rng, N, K)
    sw[9, K // 32 - 1], sw[69, 0] = 255, 255
    y = ops.mxfp4_gemm_bf16(_t(gpu, qw), _t(gpu, sw), _bf16(gpu, rng.standard_normal((M, K))))
    want = np.zeros(N, bool)
    want[[9, 69]] = True
    assert (gpu.isnan(y).cpu().numpy() == want).all()


@pytest.mark.parametrize("M,K", A16_KERNELS + [(20, 96), (64, 2176), (300, 2176), (300, 2080)])
def test_quantized_nan_blocks_reach_every_product(gpu, ops, M, K):
    """A weight block with a NaN or an infinity, as the quantizer stores it (codes 0, byte 255):
    its column is NaN in both products, nothing else is; and so for a token's block."""
    g = gpu.Generator("cuda").manual_seed(M)
    N = 16500 if M == 100 else 300
    w = gpu.randn(N, K, generator=g, device="cuda")
    w[7, K - 1] = float("nan")
    w[N - 1, 3] = float("inf")
    qw, sw = ops.mxfp4_quantize(w)
    assert int(sw[7, -1]) == 255 and not qw[7, -16:].any()
    x = gpu.randn(M, K, generator=g, device="cuda").bfloat16()
    cols = gpu.zeros(N, dtype=gpu.bool, device="cuda")
    cols[[7, N - 1]] = True
    assert gpu.equal(gpu.isnan(ops.mxfp4_gemm_bf16(qw, sw, x)), cols[None].expand(M, N))
    for out in (gpu.bfloat16, gpu.float32):
        assert gpu.equal(gpu.isnan(ops.mxfp4_gemm_w4a4(*ops.mxfp4_quantize(x), qw, sw, out_dtype=out)), cols[None].expand(M, N))
    x[M // 2, K // 2] = float("nan")
    rows = gpu.zeros(M, dtype=gpu.bool, device="cuda")
    rows[M // 2] = True
    want = rows[:, None] | cols
    assert gpu.equal(gpu.isnan(ops.mxfp4_gemm_bf16(qw, sw, x)), want)
    assert gpu.equal(gpu.isnan(ops.mxfp4_gemm_w4a4(*ops.mxfp4_quantize(x), qw, sw)), want)
