"""The residual sum with its norms, on the GPU, against 64 bits (the tolerances
stand in kc_serving.residual; a bf16 output is rounded by 2^-8 of its value
more), and its types and routes against each other bit for bit."""
import numpy as np
import pytest

import kc_serving as ref

pytestmark = pytest.mark.gpu

TYPES = [("bfloat16", "bfloat16"), ("bfloat16", "float32"), ("float32", "float32")]
SHAPES = [(1, 4096), (1, 1), (3, 8), (5, 33), (2, 2048), (4, 2056), (7, 4104), (2, 5120), (3, 8192), (2, 8200), (1, 14336),
          (2, 32768), (1, 32761), (2, 16384), (2, 16385), (3, 8193), (5, 7), (4, 15), (3, 1023), (2, 1031), (300, 512),
          (2100, 1024), (2, 777), (0, 64), (4, 0)]
FORMS = [(False, None), (True, None), (False, "channel"), (True, "channel"), (False, "value"), (True, "value")]


@pytest.fixture(scope="module")
def ops(gpu):
    import kernel_craft_torch_ops
    return kernel_craft_torch_ops


def _np(t):
    return t.double().cpu().numpy()


def _inputs(torch, T, D, ydt, hdt, post, gate, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    rand = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
    y, h = rand(T, D).to(ydt), rand(T, D)
    h[:, ::97] *= 20
    gamma, pg = ((1 + 0.3 * rand(D)).to(ydt) for _ in range(2))
    gt = {None: None, "channel": rand(D).to(ydt), "value": rand(T, D).to(ydt)}[gate]
    return y, h.to(hdt), gamma, pg if post else None, gt


def _half(torch, dtype, want):
    return 2.0 ** -8 * np.abs(want) if dtype == torch.bfloat16 else 0.0


@pytest.mark.parametrize("ydt,hdt", TYPES)
@pytest.mark.parametrize("T,D", SHAPES)
def test_against_64_bits(gpu, ops, T, D, ydt, hdt):
    ydt, hdt = getattr(gpu, ydt), getattr(gpu, hdt)
    for i, (post, gate) in enumerate(FORMS):
        args = _inputs(gpu, T, D, ydt, hdt, post, gate, seed=D + i)
        alpha = (1.0, 0.22, -1.5)[i % 3]
        h, n = ops.residual_rmsnorm(*args, alpha, eps=1e-5)
        assert h.dtype == hdt and n.dtype == ydt and h.shape == n.shape == (T, D)
        if T == 0 or D == 0:
            continue
        x, want, off, off_n = ref.residual(*(None if a is None else _np(a) for a in args), alpha, 1e-5)
        assert (np.abs(_np(h) - x) <= off + _half(gpu, hdt, x) * (1 + 1e-3)).all()
        assert (np.abs(_np(n) - want) <= off_n + _half(gpu, ydt, want) * (1 + 1e-3)).all()


@pytest.mark.parametrize("ydt,hdt", TYPES)
@pytest.mark.parametrize("T,D", SHAPES)
def test_fp8(gpu, ops, T, D, ydt, hdt):
    """The quantized form: the same h', and the bits of the row quantizer on the
    n that the same values give in fp32."""
    ydt, hdt = getattr(gpu, ydt), getattr(gpu, hdt)
    for i, (post, gate) in enumerate(FORMS):
        args = _inputs(gpu, T, D, ydt, hdt, post, gate, seed=D + i)
        h, codes, scales = ops.residual_rmsnorm_fp8_quantize(*args, 0.22)
        h1, n1 = ops.residual_rmsnorm(*args, 0.22)
        wide = [None if a is None else a.float() for a in args]
        h32, n32 = ops.residual_rmsnorm(*wide, 0.22)
        assert gpu.equal(h, h1) and gpu.equal(h, h32.to(hdt)) and gpu.equal(n1, n32.to(ydt))
        q, s = ops.fp8_quantize_rows(n32)
        assert codes.dtype == gpu.int8 and gpu.equal(codes, q) and gpu.equal(scales, s)


@pytest.mark.parametrize("ydt,hdt", TYPES)
def test_views(gpu, ops, ydt, hdt):
    """Rows at any stride and alignment: the bits of contiguous ones."""
    ydt, hdt = getattr(gpu, ydt), getattr(gpu, hdt)
    for D in (512, 515):
        y, h, gamma, post, gate = _inputs(gpu, 6, D, ydt, hdt, True, "value")
        want = ops.residual_rmsnorm(y, h, gamma, post, gate, 0.5)
        for lead, tail in ((0, 8), (8, 0), (1, 2), (0, 1)):
            def wide(t):
                w = gpu.full((t.shape[0], lead + D + tail), float("nan"), dtype=t.dtype, device="cuda")
                w[:, lead:lead + D] = t
                return w[:, lead:lead + D]
            for a in ((wide(y), h, gate), (y, wide(h), gate), (y, h, wide(gate)), (wide(y), wide(h), wide(gate)),
                      (y.t().contiguous().t(), h, gate)):
                got = ops.residual_rmsnorm(a[0], a[1], gamma, post, a[2], 0.5)
                assert all(gpu.equal(g, w) for g, w in zip(got, want))
        # a row for all tokens
        got = ops.residual_rmsnorm(y[:1].expand(6, D), h, gamma, post, gate[:1].expand(6, D), 0.5)
        want = ops.residual_rmsnorm(y[:1].repeat(6, 1), h, gamma, post, gate[0], 0.5)
        assert all(gpu.equal(g, w) for g, w in zip(got, want))


@pytest.mark.parametrize("ydt,hdt", TYPES)
@pytest.mark.parametrize("D", [7, 8, 520, 523, 4104])
def test_gammas_and_gates_at_any_address(gpu, ops, D, ydt, hdt):
    """Rows of weights that begin between 16 bytes, in both forms: the bits of
    aligned ones."""
    ydt, hdt = getattr(gpu, ydt), getattr(gpu, hdt)
    y, h, gamma, post, gate = _inputs(gpu, 5, D, ydt, hdt, True, "channel")
    def moved(t):
        return gpu.cat([t[:1], t])[1:]
    for f in (ops.residual_rmsnorm, ops.residual_rmsnorm_fp8_quantize):
        want = f(y, h, gamma, post, gate, 0.7)
        for a in ((moved(gamma), post, gate), (gamma, moved(post), gate), (gamma, post, moved(gate))):
            assert all(gpu.equal(g, w) for g, w in zip(f(y, h, *a, 0.7), want))


@pytest.mark.parametrize("D", [3, 13, 64, 515])
def test_nothing_behind_the_rows(gpu, ops, D):
    """Outputs at odd addresses between other bytes: those stay."""
    import ctypes
    import kc_abi
    L, T = kc_abi.lib(), 3
    y, h, gamma, post, gate = _inputs(gpu, T, D, gpu.bfloat16, gpu.bfloat16, True, "value")
    want = ops.residual_rmsnorm_fp8_quantize(y, h, gamma, post, gate, 0.5)
    h_out = gpu.full((T * D + 9,), 7.0, device="cuda").bfloat16()
    codes = gpu.full((T * D + 9,), 99, dtype=gpu.int8, device="cuda")
    scales = gpu.full((T + 2,), 7.0, device="cuda")
    a = ops.Residual(y.data_ptr(), h.data_ptr(), gate.data_ptr(), post.data_ptr(), gamma.data_ptr(), D, D, D, T, D, 0.5,
                     1e-6)
    assert L.kc_residual_rmsnorm_quantize_fp8_bf16(ctypes.byref(a), kc_abi.ptr(h_out[1:]), kc_abi.ptr(codes[1:]),
                                                   kc_abi.ptr(scales[1:]), kc_abi.stream()) == 0
    for got, w, was in zip((h_out, codes, scales), want, (7, 99, 7)):
        n = w.numel()
        assert gpu.equal(got[1:1 + n], w.flatten())
        assert bool((got[:1] == was).all()) and bool((got[1 + n:] == was).all())


def test_two_streams_at_once(gpu, ops):
    args = [_inputs(gpu, 700, 515 + i, gpu.bfloat16, gpu.float32, True, "value") for i in range(2)]
    want = [ops.residual_rmsnorm(*a) for a in args]
    streams = [gpu.cuda.Stream() for _ in args]
    gpu.cuda.synchronize()
    got = []
    for _ in range(5):
        for s, a in zip(streams, args):
            with gpu.cuda.stream(s):
                got.append(ops.residual_rmsnorm(*a))
    gpu.cuda.synchronize()
    assert all(gpu.equal(g, w) for i, o in enumerate(got) for g, w in zip(o, want[i % 2]))


def test_extreme_rows(gpu, ops):
    """Zeros (only eps under the roots), large and tiny rows, a NaN, an
    infinity: each stays in its row; NaN quantizes to +448 as elsewhere."""
    y, h, gamma, post, _ = _inputs(gpu, 6, 300, gpu.float32, gpu.float32, True, None)
    y, h = y.clone(), h.clone()
    y[0] = 0
    h[0] = 0
    h[1] *= 2.0 ** 50
    y[2] *= 2.0 ** -70
    h[2] *= 2.0 ** -70
    y[3, 7] = float("nan")
    h[4, 9] = float("inf")
    hn, n = ops.residual_rmsnorm(y, h, gamma, post)
    x, want, off, off_n = ref.residual(_np(y[[0, 1, 2, 5]]), _np(h[[0, 1, 2, 5]]), _np(gamma), _np(post), None, 1.0, 1e-6)
    assert (np.abs(_np(hn[[0, 1, 2, 5]]) - x) <= off).all() and (np.abs(_np(n[[0, 1, 2, 5]]) - want) <= off_n).all()
    assert bool(gpu.isnan(n[3]).all()) and bool(gpu.isnan(n[4, 9])) and bool(gpu.isinf(hn[4, 9]))
    _, codes, scales = ops.residual_rmsnorm_fp8_quantize(y, h, gamma, post)
    q, s = ops.fp8_quantize_rows(n)
    assert gpu.equal(codes, q) and gpu.equal(scales, s) and float(scales[0]) == 1


def test_streams_and_graph(gpu, ops):
    """On a stream of its own, and replayed from a graph on new values."""
    args = _inputs(gpu, 50, 4096, gpu.bfloat16, gpu.bfloat16, True, "channel")
    new = [_inputs(gpu, 50, 4096, gpu.bfloat16, gpu.bfloat16, True, "channel", seed=s) for s in (1, 2, 3)]
    side = gpu.cuda.Stream()
    side.wait_stream(gpu.cuda.current_stream())
    with gpu.cuda.stream(side):
        ops.residual_rmsnorm_fp8_quantize(*args, 0.3)
    gpu.cuda.current_stream().wait_stream(side)
    graph = gpu.cuda.CUDAGraph()
    with gpu.cuda.graph(graph):
        out = ops.residual_rmsnorm_fp8_quantize(*args, 0.3)
    for n in new:
        for a, b in zip(args, n):
            a.copy_(b)
        graph.replay()
        gpu.cuda.synchronize()
        assert all(gpu.equal(a, b) for a, b in zip(out, ops.residual_rmsnorm_fp8_quantize(*n, 0.3)))
