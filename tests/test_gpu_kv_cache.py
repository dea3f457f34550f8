"""Head norms with rotation, and the quantized paged cache that keys and values
are written to and read back from, on the GPU.

Norm and rotation against 64 bits: in fp32 the sum of D squares, the square
root, the division and five more roundings leave each of an output's two terms
within (D / 2 + 8) * 2^-24 of its size, and a bf16 output a rounding (2^-8 of
its size) more.  The fused forms, the kernels' own routes and the cache rows
are compared bit for bit: with the two calls, and with the quantizers on the
same rows.
"""
import numpy as np
import pytest

import kc_mxfp4 as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(gpu):
    import kernel_craft_torch_ops
    return kernel_craft_torch_ops


def _np(t):
    return t.double().cpu().numpy()


def _tables(torch, rows, half, seed=0):
    a = torch.from_numpy(np.random.default_rng(seed).uniform(-7, 7, (rows, half)))
    return a.cos().float().cuda(), a.sin().float().cuda()


def _heads(torch, T, Hq, Hkv, D, dtype, seed=0, extra=0):
    """q, k, v as views of one projection's rows (`extra` more elements a row), and gammas."""
    g = torch.Generator("cuda").manual_seed(seed)
    width = (Hq + 2 * Hkv) * D
    rows = torch.randn(T, width + extra, generator=g, device="cuda").to(dtype)
    qkv = rows[:, :width].unflatten(1, (Hq + 2 * Hkv, D))
    gam = [(1 + 0.3 * torch.randn(D, generator=g, device="cuda")).to(dtype) for _ in range(2)]
    return qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:], gam[0], gam[1]


def _pool(torch, pages, page, H, D, fmt, fill=None):
    if fmt == "fp8":
        k = [torch.zeros(pages, page, H, D, dtype=torch.int8, device="cuda"),
             torch.zeros(pages, page, H, dtype=torch.float32, device="cuda")]
    else:
        k = [torch.zeros(pages, page, H, D // 2, dtype=torch.uint8, device="cuda"),
             torch.zeros(pages, page, H, D // 32, dtype=torch.uint8, device="cuda")]
    pool = k + [t.clone() for t in k]
    if fill is not None:
        for t in pool:
            t.fill_(fill)
    return pool


SHAPES = [  # T, q heads, kv heads, D, R, interleaved
    (1, 32, 8, 128, 128, False), (1, 1, 1, 64, 64, False), (5, 8, 2, 128, 64, False), (3, 4, 4, 128, 128, True),
    (7, 28, 4, 128, 128, False), (2, 5, 1, 96, 96, False), (9, 3, 1, 80, 80, False), (4, 6, 2, 80, 32, True),
    (6, 2, 2, 256, 128, False), (2, 4, 1, 512, 512, False), (3, 2, 1, 16, 16, False), (3, 2, 1, 48, 16, True),
    (3, 3, 1, 40, 40, False), (2, 2, 1, 33, 20, True), (2, 1, 1, 1, 0, False), (2, 2, 1, 576, 64, False),
    (3, 2, 1, 1024, 1024, False), (2, 2, 2, 100, 50, True), (300, 7, 1, 64, 64, False), (2100, 4, 1, 128, 128, False),
    (4, 3, 1, 80, 40, False), (4, 3, 1, 56, 24, True), (11, 0, 2, 64, 64, False), (11, 2, 0, 64, 64, True), (5, 40, 8, 128, 0, False),
]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("T,Hq,Hkv,D,R,inter", SHAPES)
def test_norm_rope(gpu, ops, T, Hq, Hkv, D, R, inter, dtype):
    dt = getattr(gpu, dtype)
    q, k, _, qg, kg = _heads(gpu, T, Hq, Hkv, D, dt, seed=D + T)
    cos, sin = _tables(gpu, 50, R // 2)
    pos = gpu.from_numpy(np.random.default_rng(T).integers(0, 50, T).astype(np.int32)).cuda()
    out = ops.qk_norm_rope(q, k, qg, kg, cos, sin, pos, eps=1e-5, interleaved=inter)
    for x, g, y in ((q, qg, out[0]), (k, kg, out[1])):
        assert y.is_contiguous() and y.dtype == dt and y.shape == x.shape
        want, size = ref.norm_rope(_np(x), _np(g), cos.cpu().numpy(), sin.cpu().numpy(), pos.cpu().numpy(), 1e-5, inter)
        tol = (D / 2 + 8) * 2.0 ** -24 * size
        if dtype == "bfloat16":
            tol = tol + 2.0 ** -8 * np.abs(want)
        assert (np.abs(_np(y) - want) <= tol).all()


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("extra", [0, 1, 8])
def test_norm_rope_routes_agree(gpu, ops, dtype, extra):
    """Any row stride, and the row as its own tensor: the same bits."""
    dt = getattr(gpu, dtype)
    for D, R, inter in ((128, 128, False), (96, 32, True), (80, 48, False)):
        q, k, _, qg, kg = _heads(gpu, 6, 5, 2, D, dt, extra=extra)
        cos, sin = _tables(gpu, 9, R // 2)
        pos = gpu.arange(6, device="cuda", dtype=gpu.int32)
        a = ops.qk_norm_rope(q, k, qg, kg, cos, sin, pos, interleaved=inter)
        b = ops.qk_norm_rope(q.contiguous(), k.contiguous(), qg, kg, cos, sin, pos, interleaved=inter)
        # heads that do not follow one another are copied
        c = ops.qk_norm_rope(q.transpose(0, 1).contiguous().transpose(0, 1), k, qg, kg, cos, sin, pos, interleaved=inter)
        assert all(gpu.equal(x, y) and gpu.equal(x, z) for x, y, z in zip(a, b, c))


@pytest.mark.parametrize("D", [64, 33])
def test_positions_outside_the_tables(gpu, ops, D):
    """Padding (negative) gives zeros, a position past the tables NaN; neither
    reaches the cache; the others are as without them."""
    R = 32
    q, k, v, qg, kg = _heads(gpu, 5, 3, 2, D, gpu.bfloat16)
    cos, sin = _tables(gpu, 10, R // 2)
    pos = gpu.tensor([3, -1, 10, 9, -2147483648], dtype=gpu.int32, device="cuda")
    yq, yk = ops.qk_norm_rope(q, k, qg, kg, cos, sin, pos)
    for y in (yq, yk):
        assert float(y[[1, 4]].abs().max()) == 0 and bool(gpu.isnan(y[2]).all()) and bool(gpu.isfinite(y[[0, 3]]).all())
    pool = _pool(gpu, 2, 4, 2, D, "fp8", fill=5)
    slots = gpu.arange(5, device="cuda")
    y = ops.qk_norm_rope_cache(q, k, v, qg, kg, cos, sin, pos, slots, *pool)
    assert gpu.equal(gpu.nan_to_num(y, 7.0), gpu.nan_to_num(yq, 7.0))
    for t in pool:
        flat = t.flatten(0, 1)
        assert bool((flat[[1, 2, 4, 5, 6, 7]] == 5).all()) and not bool((flat[[0, 3]] == 5).all())


def test_empty_tables(gpu, ops):
    """No table rows: every position is outside."""
    q, k, _, qg, kg = _heads(gpu, 2, 1, 1, 64, gpu.float32)
    e = gpu.zeros(0, 32, device="cuda")
    y, _ = ops.qk_norm_rope(q, k, qg, kg, e, e, gpu.tensor([0, -1], dtype=gpu.int32, device="cuda"))
    assert bool(gpu.isnan(y[0]).all()) and float(y[1].abs().max()) == 0


def test_norm_of_extreme_heads(gpu, ops):
    """Zeros (only eps under the root), large and tiny values, a NaN: each
    stays in its head."""
    q, k, _, qg, kg = _heads(gpu, 4, 2, 1, 128, gpu.bfloat16)
    q = q.clone()
    q[0, 0] = 0
    q[1, 0] *= 2.0 ** 60
    q[2, 0] *= 2.0 ** -60
    q[3, 0, 77] = float("nan")
    cos, sin = _tables(gpu, 4, 64)
    pos = gpu.arange(4, device="cuda", dtype=gpu.int32)
    y, _ = ops.qk_norm_rope(q, k, qg, kg, cos, sin, pos)
    want, size = ref.norm_rope(_np(q), _np(qg), cos.cpu().numpy(), sin.cpu().numpy(), np.arange(4), 1e-6, False)
    got = _np(y)
    assert np.isnan(got[3, 0]).all() and np.isfinite(got[3, 1]).all() and (got[0, 0] == 0).all()
    for t, h in ((0, 1), (1, 0), (1, 1), (2, 0), (3, 1)):
        assert (np.abs(got[t, h] - want[t, h]) <= 72 * 2.0 ** -24 * size[t, h] + 2.0 ** -8 * np.abs(want[t, h])).all()


def _rows_expected(torch, ops, x, fmt):
    """Codes and scales of rows x [T, H, D] by the row quantizers."""
    T, H, D = x.shape
    if fmt == "fp8":
        c, s = ops.fp8_quantize_rows(x.reshape(T * H, D))
        return c.view(T, H, D), s.view(T, H)
    c, s = ops.mxfp4_quantize(x.reshape(T * H, D))
    return c.view(T, H, D // 2), s.view(T, H, D // 32)


WRITES = [(1, 8, 128, 16, "fp8"), (1, 8, 128, 16, "mxfp4"), (37, 2, 64, 1, "fp8"), (37, 2, 64, 7, "mxfp4"),
          (20, 3, 96, 16, "fp8"), (20, 3, 96, 16, "mxfp4"), (9, 1, 80, 32, "fp8"), (12, 2, 33, 5, "fp8"),
          (5, 1, 256, 64, "mxfp4"), (4, 2, 1024, 4, "fp8"), (4, 2, 1024, 4, "mxfp4"), (3000, 4, 128, 48, "fp8"),
          (3000, 4, 128, 48, "mxfp4"), (3, 1, 32, 2, "mxfp4"), (6, 2, 576, 8, "mxfp4"), (2, 5, 1, 3, "fp8")]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("T,H,D,page,fmt", WRITES)
def test_write_then_read(gpu, ops, T, H, D, page, fmt, dtype):
    """Rows in a shuffled order of slots, some tokens padding: the row
    quantizers' bits, everything else of the pool as it was; read back in the
    order of the slots."""
    dt = getattr(gpu, dtype)
    rng = np.random.default_rng(T * 31 + D)
    pages = -(-T // page) + 2
    _, k, v, _, _ = _heads(gpu, T, 1, H, D, dt, seed=T)
    order = rng.permutation(pages * page)[:T]
    slots = order.astype(np.int64)
    slots[rng.random(T) < 0.2] = -1
    if T > 4:
        slots[1], slots[3] = pages * page, -(2 ** 40)     # outside the pool
    pool = _pool(gpu, pages, page, H, D, fmt, fill=3)
    before = [t.clone() for t in pool]
    ops.kv_cache_write(k, v, gpu.from_numpy(slots).cuda(), *pool)
    live = (slots >= 0) & (slots < pages * page)
    at, tok = gpu.from_numpy(slots[live]).cuda(), gpu.from_numpy(np.flatnonzero(live)).cuda()
    for i, x in ((0, k), (2, v)):
        c, s = _rows_expected(gpu, ops, x.contiguous(), fmt)
        before[i].flatten(0, 1)[at] = c[tok]
        before[i + 1].flatten(0, 1)[at] = s[tok]
    assert all(gpu.equal(a, b) for a, b in zip(pool, before))
    # the whole pool as one sequence, its pages in another order
    table = gpu.from_numpy(rng.permutation(pages).astype(np.int32)[None]).cuda()
    cu = gpu.tensor([0, pages * page], dtype=gpu.int32, device="cuda")
    got = ops.kv_cache_read(*pool, table, cu, pages * page, out_dtype=dt)
    for i, y in ((0, got[0]), (2, got[1])):
        c, s = pool[i][table[0].long()].flatten(0, 1), pool[i + 1][table[0].long()].flatten(0, 1)
        if fmt == "fp8":
            want = (c.view(gpu.float8_e4m3fn).float() * s[..., None]).to(dt)
        else:
            want = gpu.from_numpy(ref.values(c.cpu().numpy(), s.cpu().numpy())).to(dt).cuda()
        assert gpu.equal(y, want)


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("T,Hq,Hkv,D,R,inter", [(1, 32, 8, 128, 128, False), (5, 7, 1, 64, 64, True),
                                                (9, 4, 2, 96, 32, False), (9, 4, 2, 96, 64, False),
                                                (6, 2, 2, 32, 32, False), (40, 16, 4, 256, 128, False),
                                                (9, 4, 2, 80, 40, False), (5, 4, 2, 224, 40, True),
                                                (3, 2, 1, 576, 64, False), (2300, 4, 2, 128, 128, False),
                                                (4, 0, 3, 64, 64, False)])
def test_fused_equals_the_two_calls(gpu, ops, T, Hq, Hkv, D, R, inter, dtype, fmt):
    if fmt == "mxfp4" and D % 32:
        pytest.skip("MXFP4 rows are whole blocks")
    dt = getattr(gpu, dtype)
    q, k, v, qg, kg = _heads(gpu, T, Hq, Hkv, D, dt, seed=T + D)
    cos, sin = _tables(gpu, 64, R // 2)
    rng = np.random.default_rng(T)
    pos = gpu.from_numpy(rng.integers(0, 64, T).astype(np.int32)).cuda()
    page, pages = 16, -(-T // 16) + 1
    slots = gpu.from_numpy(rng.permutation(pages * page)[:T].astype(np.int64)).cuda()
    one, two = _pool(gpu, pages, page, Hkv, D, fmt, 1), _pool(gpu, pages, page, Hkv, D, fmt, 1)
    yq = ops.qk_norm_rope_cache(q, k, v, qg, kg, cos, sin, pos, slots, *one, interleaved=inter)
    wq, wk = ops.qk_norm_rope(q, k, qg, kg, cos, sin, pos, interleaved=inter)
    ops.kv_cache_write(wk, v, slots, *two)
    assert gpu.equal(yq, wq)
    assert all(gpu.equal(a, b) for a, b in zip(one, two))


@pytest.mark.parametrize("dtype,fmt,inter", [("bfloat16", "fp8", False), ("bfloat16", "mxfp4", True),
                                             ("float32", "fp8", True), ("float32", "mxfp4", False)])
def test_long_batches_equal_their_parts(gpu, ops, dtype, fmt, inter):
    """More than 64 MB of heads are read past the cache: the same bits as the batch in
    parts, in which they are not."""
    T, Hq, Hkv, D, parts = (9601 if dtype == "bfloat16" else 4801), 8, 20, 128, 4
    q, k, v, gq, gk = _heads(gpu, T, Hq, Hkv, D, getattr(gpu, dtype))
    cos, sin = _tables(gpu, 1000, D // 2)
    pos = (gpu.arange(T, device="cuda") % 1003 - 1).int()
    slots = gpu.randperm(T + 7, device="cuda")[:T] - 3
    args = lambda a, b: (q[a:b], k[a:b], gq, gk, cos, sin, pos[a:b])
    cuts = [T * i // parts for i in range(parts + 1)]
    pieces = [ops.qk_norm_rope(*args(a, b), interleaved=inter) for a, b in zip(cuts, cuts[1:])]
    got = ops.qk_norm_rope(*args(0, T), interleaved=inter)
    for whole, part in zip(got, zip(*pieces)):
        assert gpu.equal(whole.view(gpu.uint8), gpu.cat(part).view(gpu.uint8))
    caches = []
    for step in ("whole", "parts", "whole", "parts"):
        cache = _pool(gpu, T // 16 + 1, 16, Hkv, D, fmt)
        ends = [0, T] if step == "whole" else cuts
        for a, b in zip(ends, ends[1:]):
            if len(caches) < 2:
                ops.qk_norm_rope_cache(q[a:b], k[a:b], v[a:b], gq, gk, cos, sin, pos[a:b], slots[a:b], *cache,
                                       interleaved=inter)
            else:
                ops.kv_cache_write(k[a:b], v[a:b], slots[a:b], *cache)
        caches.append(cache)
    for one, other in (caches[:2], caches[2:]):
        for a, b in zip(one, other):
            assert gpu.equal(a.view(gpu.uint8), b.view(gpu.uint8))


@pytest.mark.parametrize("fmt,D", [("fp8", 64), ("fp8", 33), ("mxfp4", 64)])
def test_read_of_a_ragged_batch(gpu, ops, fmt, D):
    """Empty sequences, a page that ends inside the batch, missing pages, pages
    outside the pool, rows behind the last sequence."""
    from kc_abi import check, ptr, stream
    H, page, pages = 2, 4, 9
    g = gpu.Generator("cuda").manual_seed(1)
    k = gpu.randn(pages * page, H, D, generator=g, device="cuda")
    v = gpu.randn(pages * page, H, D, generator=g, device="cuda")
    pool = _pool(gpu, pages, page, H, D, fmt)
    ops.kv_cache_write(k, v, gpu.arange(pages * page, device="cuda"), *pool)
    lengths = [0, 5, 0, 0, 9, 1, 4, 0]
    cu = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int32)
    table = np.array([[-1, -1], [7, 2], [0, 0], [-1, 5], [1, -1], [9, 0], [8, 3], [-5, -5]], dtype=np.int32)
    total = int(cu[-1]) + 6
    slots = ref.slots_of([[p if p < pages else -1 for p in row] for row in table], cu, page, total)
    lib = ops._get_lib()
    outs = [gpu.full((total, H, D), 42.0, device="cuda") for _ in range(2)]
    cache, _, _ = ops._kv_cache("test", *pool)
    import ctypes
    tb, cd = gpu.from_numpy(table).cuda(), gpu.from_numpy(cu).cuda()
    check("read", lib.kc_kv_cache_read_f32(ctypes.byref(cache), ptr(tb), 2, ptr(cd), len(lengths), total,
                                           ptr(outs[0]), ptr(outs[1]), stream()))
    whole = ops.kv_cache_read(*pool, gpu.arange(pages, device="cuda", dtype=gpu.int32)[None],
                              gpu.tensor([0, pages * page], dtype=gpu.int32, device="cuda"), pages * page,
                              out_dtype=gpu.float32)
    for got, src in zip(outs, whole):
        for t in range(total):
            if slots[t] == -2:
                assert bool((got[t] == 42.0).all())
            elif slots[t] == -1:
                assert bool(gpu.isnan(got[t]).all())
            else:
                assert gpu.equal(got[t], src[slots[t]])
    # the operator's own outputs hold the same rows
    n = int(cu[-1])
    again = ops.kv_cache_read(*pool, tb, cd, n, out_dtype=gpu.float32)
    for got, y in zip(outs, again):
        assert gpu.equal(gpu.nan_to_num(got[:n], 9.0), gpu.nan_to_num(y, 9.0))
    # fewer tokens asked for than the batch holds
    part = ops.kv_cache_read(*pool, tb, cd, 7, out_dtype=gpu.float32)
    assert all(gpu.equal(gpu.nan_to_num(a[:7], 9.0), gpu.nan_to_num(b, 9.0)) for a, b in zip(again, part))


def test_read_with_descending_starts_stays_in_bounds(gpu, ops):
    """Starts that do not ascend are the caller's mistake: rows come from
    the pool, are NaN, or are left, and nothing outside is touched."""
    pool = _pool(gpu, 3, 4, 1, 64, "fp8", fill=1)
    cu = gpu.tensor([0, 9, 4, 8], dtype=gpu.int32, device="cuda")
    table = gpu.tensor([[0], [1], [2]], dtype=gpu.int32, device="cuda")
    k, v = ops.kv_cache_read(*pool, table, cu, 8)
    assert k.shape == (8, 1, 64) and gpu.equal(gpu.isnan(k), gpu.isnan(v))


@pytest.mark.parametrize("D", [128, 72])
def test_special_values_in_the_cache(gpu, ops, D):
    """NaN, infinities, zero and huge rows: as the row quantizers treat them."""
    k = gpu.randn(8, 2, D, device="cuda").bfloat16()
    k[0, 0, 3] = float("nan")
    k[1, 0, 5] = float("inf")
    k[2, 0] = 0
    k[3, 1] *= 2.0 ** 120
    k[4, 1] *= 2.0 ** -125
    k[5, 0] = float("nan")
    v = k.flip(0).contiguous()
    for fmt in ("fp8", "mxfp4"):
        if fmt == "mxfp4" and D % 32:
            continue
        pool = _pool(gpu, 2, 4, 2, D, fmt)
        ops.kv_cache_write(k, v, gpu.arange(8, device="cuda"), *pool)
        for i, x in ((0, k), (2, v)):
            c, s = _rows_expected(gpu, ops, x, fmt)
            assert gpu.equal(pool[i].flatten(0, 1), c)
            assert gpu.equal(gpu.nan_to_num(pool[i + 1].flatten(0, 1).float(), 1.0),
                             gpu.nan_to_num(s.float(), 1.0))


def test_zero_tokens(gpu, ops):
    q, k, v, qg, kg = _heads(gpu, 0, 4, 2, 64, gpu.bfloat16)
    cos, sin = _tables(gpu, 4, 32)
    none32, none64 = gpu.zeros(0, dtype=gpu.int32, device="cuda"), gpu.zeros(0, dtype=gpu.int64, device="cuda")
    pool = _pool(gpu, 1, 4, 2, 64, "fp8")
    a, b = ops.qk_norm_rope(q, k, qg, kg, cos, sin, none32)
    assert a.shape == (0, 4, 64) and b.shape == (0, 2, 64)
    assert ops.qk_norm_rope_cache(q, k, v, qg, kg, cos, sin, none32, none64, *pool).shape == (0, 4, 64)
    ops.kv_cache_write(k, v, none64, *pool)
    k, v = ops.kv_cache_read(*pool, gpu.zeros(0, 3, dtype=gpu.int32, device="cuda"),
                             gpu.zeros(1, dtype=gpu.int32, device="cuda"), 0)
    assert k.shape == v.shape == (0, 2, 64)
    k, v = ops.kv_cache_read(*pool, gpu.zeros(2, 0, dtype=gpu.int32, device="cuda"),
                             gpu.tensor([0, 0, 3], dtype=gpu.int32, device="cuda"), 3)
    assert bool(gpu.isnan(k).all()) and bool(gpu.isnan(v).all())


def test_slots_past_32_bits(gpu, ops):
    """A pool of more than 2^32 bytes of keys: rows at its far end."""
    page, H, D = 256, 8, 128
    pages = (1 << 32) // (page * H * D) + 3
    pool = _pool(gpu, pages, page, H, D, "fp8")
    T = 5
    _, k, v, _, _ = _heads(gpu, T, 1, H, D, gpu.bfloat16)
    slots = pages * page - 1 - gpu.arange(T, device="cuda") * 300
    ops.kv_cache_write(k, v, slots, *pool)
    for i, x in ((0, k), (2, v)):
        c, s = _rows_expected(gpu, ops, x.contiguous(), "fp8")
        assert gpu.equal(pool[i].flatten(0, 1)[slots], c) and gpu.equal(pool[i + 1].flatten(0, 1)[slots], s)
    table = gpu.arange(pages - 3, pages, device="cuda", dtype=gpu.int32)[None]
    got = ops.kv_cache_read(*pool, table, gpu.tensor([0, 3 * page], dtype=gpu.int32, device="cuda"), 3 * page)
    want = (pool[0][-3:].view(gpu.float8_e4m3fn).float() * pool[1][-3:][..., None]).bfloat16().flatten(0, 1)
    assert gpu.equal(got[0], want) and float(want.abs().max()) > 0


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
def test_decoder_layer_front(gpu, ops, fmt):
    """The operators together, as a decoder layer runs them: RMSNorm, 4-bit
    quantization, QKV product, heads into the cache and the context back; a
    prompt, then single tokens, the last ones replayed from a graph."""
    torch = gpu
    hidden, Hq, Hkv, D, page = 512, 8, 2, 64, 16
    g = torch.Generator("cuda").manual_seed(3)
    wq = ops.mxfp4_quantize(torch.randn((Hq + 2 * Hkv) * D, hidden, generator=g, device="cuda") * 0.05)
    norm, qg, kg = (1 + 0.1 * torch.randn(n, generator=g, device="cuda").bfloat16() for n in (hidden, D, D))
    cos, sin = _tables(torch, 64, D // 2)
    pool = _pool(torch, 8, page, Hkv, D, fmt)
    table = torch.tensor([[5, 1, 6, 0]], dtype=torch.int32, device="cuda")
    h_all = torch.randn(60, hidden, generator=g, device="cuda").bfloat16()

    def step(h, pos, slots, cu, total):
        x, sx = ops.mxfp4_quantize(ops.rmsnorm(h, norm))
        qkv = ops.mxfp4_gemm_w4a4(x, sx, *wq).unflatten(1, (Hq + 2 * Hkv, D))
        q = ops.qk_norm_rope_cache(qkv[:, :Hq], qkv[:, Hq:Hq + Hkv], qkv[:, Hq + Hkv:], qg, kg, cos, sin, pos, slots,
                                   *pool)
        return q, ops.kv_cache_read(*pool, table, cu, total)

    def at(lo, hi):
        pos = torch.arange(lo, hi, device="cuda", dtype=torch.int32)
        slots = table[0].long()[pos.long() // page] * page + pos % page
        return pos, slots, torch.tensor([0, hi], dtype=torch.int32, device="cuda"), hi

    # plain form of the whole, in 64 bits but for the stored roundings
    def plain(h):
        hf = h.double()
        y = (hf / (hf.square().mean(-1, keepdim=True) + 1e-6).sqrt() * norm.double()).bfloat16()
        x = torch.from_numpy(ref.values(*ref.quantize(_np(y)))).cuda()
        w = torch.from_numpy(ref.values(*(a.cpu().numpy() for a in wq))).cuda()
        qkv = (x @ w.t()).bfloat16().unflatten(1, (Hq + 2 * Hkv, D))
        pos = np.arange(len(h))
        rot = [torch.from_numpy(ref.norm_rope(_np(a), _np(gm), cos.cpu().numpy(), sin.cpu().numpy(), pos, 1e-6, False)[0])
               for a, gm in ((qkv[:, :Hq], qg), (qkv[:, Hq:Hq + Hkv], kg))]
        return rot[0], rot[1], qkv[:, Hq + Hkv:].double().cpu()

    got_q, kv = step(h_all[:50], *at(0, 50))
    rows = [got_q]
    for t in range(50, 55):
        q, kv = step(h_all[t:t + 1], *at(t, t + 1))
        rows.append(q)
    h = h_all[55:56].clone()
    pos, slots, cu, _ = at(55, 56)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(h, pos, slots, cu, 60)
    for t in range(55, 60):
        h.copy_(h_all[t:t + 1])
        p, s, c, _ = at(t, t + 1)
        pos.copy_(p), slots.copy_(s), cu.copy_(c)
        graph.replay()
        torch.cuda.synchronize()
        rows.append(out[0].clone())
        assert torch.equal(out[0], step(h, pos, slots, cu, 60)[0])
    kv = out[1]
    wq_, wk, wv = plain(h_all)
    # A flipped rounding (bf16 of the norm, then a 4-bit code: a relative 2^-8 of
    # values, half a step of 4-bit ones) moves single products; the whole
    # stays within the formats' half steps of its size.
    half_step = {"fp8": 2.0 ** -4, "mxfp4": 2.0 ** -2}[fmt]
    rel = lambda a, b: float((a.double().cpu() - b).norm() / b.norm())  # noqa: E731
    assert rel(torch.cat(rows), wq_) <= 2.0 ** -6
    assert rel(kv[0], wk) <= half_step + 2.0 ** -6 and rel(kv[1], wv) <= half_step + 2.0 ** -6


@pytest.mark.parametrize("Hq,Hkv", [(32, 8), (16, 16)])
@pytest.mark.parametrize("inter", [False, True])
@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
def test_long_bf16_batches_of_whole_head_groups_equal_their_parts(gpu, ops, fmt, inter, Hq, Hkv):
    """More than 64 MB of heads (read past the cache) whose groups of 8, a wave's, are of one
    tensor: the same bits as the batch in parts, in which they are not read past it.
    32 + 8 heads pass 64 MB with their norm, 16 + 16 also when keys and values are written alone."""
    T, D, parts = 8211, 128, 5
    q, k, v, gq, gk = _heads(gpu, T, Hq, Hkv, D, gpu.bfloat16, seed=Hq)
    cos, sin = _tables(gpu, 1000, D // 2)
    pos = (gpu.arange(T, device="cuda") % 1003 - 1).int()
    slots = gpu.randperm(T + 7, device="cuda")[:T] - 3
    cuts = [T * i // parts for i in range(parts + 1)]
    assert T * (Hq + Hkv) * D * 2 > 64 << 20 and (Hkv == 8 or T * 2 * Hkv * D * 2 > 64 << 20)

    def over(ends, call):
        return [call(slice(a, b)) for a, b in zip(ends, ends[1:])]

    def norm(s):
        return ops.qk_norm_rope(q[s], k[s], gq, gk, cos, sin, pos[s], interleaved=inter)

    whole, pieces = norm(slice(0, T)), over(cuts, norm)
    for i in range(2):
        assert gpu.equal(whole[i].view(gpu.uint8), gpu.cat([p[i] for p in pieces]).view(gpu.uint8))
    caches = [_pool(gpu, T // 16 + 1, 16, Hkv, D, fmt) for _ in range(5)]

    def fused(cache):
        return lambda s: ops.qk_norm_rope_cache(q[s], k[s], v[s], gq, gk, cos, sin, pos[s], slots[s], *cache,
                                                interleaved=inter)

    y = over([0, T], fused(caches[0])) + [gpu.cat(over(cuts, fused(caches[1])))]
    assert all(gpu.equal(t.view(gpu.uint8), whole[0].view(gpu.uint8)) for t in y)
    over([0, T], lambda s: ops.kv_cache_write(k[s], v[s], slots[s], *caches[2]))
    over(cuts, lambda s: ops.kv_cache_write(k[s], v[s], slots[s], *caches[3]))
    # the fused write's keys are the normed ones, where a position is in the table
    kept = gpu.where((pos >= 0) & (pos < 1000), slots, -1)
    ops.kv_cache_write(whole[1], v, kept, *caches[4])
    for one, other in ((0, 1), (2, 3), (0, 4)):
        for a, b in zip(caches[one], caches[other]):
            assert gpu.equal(a.view(gpu.uint8), b.view(gpu.uint8))


@pytest.mark.parametrize("fmt,D", [("fp8", 64), ("fp8", 33), ("mxfp4", 64)])
@pytest.mark.parametrize("starts", [[0, 9, 4, 8], [3, 1, 6, 8], [0, -5, 4, 7], [2, 2 ** 30, -2 ** 31, 2 ** 31 - 1], [8, 8, 0, 0]])
def test_read_with_descending_starts_keeps_to_pool_and_outputs(gpu, ops, starts, fmt, D):
    """Starts that do not ascend are the caller's mistake: each row is a row of the pool,
    keys' and values' the same one, or all NaN, or left as it was; nothing is
    written outside the outputs.  Every slot holds values of its own."""
    import ctypes
    from kc_abi import check, ptr, stream
    H, page, pages, total, guard = 2, 4, 3, 8, 5
    g = gpu.Generator("cuda").manual_seed(2)
    pool = _pool(gpu, pages, page, H, D, fmt)
    rows = [gpu.randn(pages * page, H, D, generator=g, device="cuda") for _ in range(2)]
    ops.kv_cache_write(*rows, gpu.arange(pages * page, device="cuda"), *pool)
    every = ops.kv_cache_read(*pool, gpu.arange(pages, device="cuda", dtype=gpu.int32)[None],
                              gpu.tensor([0, pages * page], dtype=gpu.int32, device="cuda"), pages * page,
                              out_dtype=gpu.float32)
    cu = gpu.tensor(starts, dtype=gpu.int32, device="cuda")
    table = gpu.tensor([[0, 2], [1, -1], [2, 7]], dtype=gpu.int32, device="cuda")
    outs = [gpu.full((total + 2 * guard, H, D), 42.0, device="cuda") for _ in range(2)]
    cache, _, _ = ops._kv_cache("test", *pool)
    check("read", ops._get_lib().kc_kv_cache_read_f32(ctypes.byref(cache), ptr(table), 2, ptr(cu), 3, total,
                                                      ptr(outs[0][guard:]), ptr(outs[1][guard:]), stream()))
    for y in outs:
        assert bool((y[:guard] == 42.0).all()) and bool((y[guard + total:] == 42.0).all())
    for t in range(guard, guard + total):
        def kind(y, src):
            if bool((y == 42.0).all()):
                return "left"
            if bool(gpu.isnan(y).all()):
                return "NaN"
            same = (src == y).flatten(1).all(1).nonzero().flatten().tolist()
            assert len(same) == 1, "not a row of the pool"
            return same[0]
        assert kind(outs[0][t], every[0]) == kind(outs[1][t], every[1])


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
def test_read_leaves_rows_before_the_first_sequence(gpu, ops, fmt):
    """Sequences that start behind the outputs' first rows: those rows are left as they were."""
    import ctypes
    from kc_abi import check, ptr, stream
    pool = _pool(gpu, 2, 4, 1, 64, fmt)
    ops.kv_cache_write(gpu.randn(8, 1, 64, device="cuda"), gpu.randn(8, 1, 64, device="cuda"),
                       gpu.arange(8, device="cuda"), *pool)
    cu = gpu.tensor([3, 5, 9], dtype=gpu.int32, device="cuda")
    table = gpu.tensor([[0], [1]], dtype=gpu.int32, device="cuda")
    outs = [gpu.full((11, 1, 64), 42.0, device="cuda") for _ in range(2)]
    cache, _, _ = ops._kv_cache("test", *pool)
    check("read", ops._get_lib().kc_kv_cache_read_f32(ctypes.byref(cache), ptr(table), 1, ptr(cu), 2, 11, ptr(outs[0]),
                                                      ptr(outs[1]), stream()))
    want = ops.kv_cache_read(*pool, table, cu - 3, 6, out_dtype=gpu.float32)
    for y, w in zip(outs, want):
        assert bool((y[[0, 1, 2, 9, 10]] == 42.0).all()) and gpu.equal(y[3:9], w)


@pytest.mark.parametrize("fused", [False, True])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("D", [128, 80, 33])
def test_fp8_scales_are_the_rounded_quotient(gpu, ops, D, dtype, fused):
    """Rows whose largest magnitude is 7 n: x / scale then meets midpoints of E4M3 exactly, so a
    scale that is off by one step of fp32 (a multiplication with a rounded 1 / 448)
    shows in the codes.  Scales and codes against 64 bits, bit for bit."""
    T, H, dt = 300, 2, getattr(gpu, dtype)
    rng = np.random.default_rng(D)
    x = rng.integers(-120, 121, (T, H, D)).astype(np.float64)
    top = 7.0 * rng.integers(1, 18, (T, H))
    x = np.clip(x, -top[..., None], top[..., None])
    x[..., 0] = top
    x = np.ldexp(x, rng.integers(-30, 30, (T, H, 1)))
    v = gpu.from_numpy(x).cuda().to(dt)
    assert np.array_equal(_np(v), x)
    pool = _pool(gpu, T, 1, H, D, "fp8")
    slots = gpu.arange(T, device="cuda")
    if fused:
        one = gpu.ones(D, device="cuda").to(dt)
        none = gpu.zeros(1, 0, device="cuda")
        ops.qk_norm_rope_cache(v, v, v, one, one, none, none, gpu.zeros(T, device="cuda", dtype=gpu.int32), slots, *pool)
    else:
        ops.kv_cache_write(v, v, slots, *pool)
    scale = (np.abs(x).max(-1) / 448.0).astype(np.float32)
    a = x / scale.astype(np.float64)[..., None]
    ulp = np.exp2(np.maximum(np.floor(np.log2(np.maximum(np.abs(a), 2.0 ** -30))), -6) - 3)
    want = np.rint(a / ulp) * ulp
    for i in (2,) if fused else (0, 2):
        np.testing.assert_array_equal(pool[i + 1][:, 0].cpu().numpy(), scale)
        np.testing.assert_array_equal(pool[i][:, 0].view(gpu.float8_e4m3fn).double().cpu().numpy(), want)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_more_rows_than_one_launch_holds(gpu, ops, dtype):
    """Over 2^26 heads in one call (of 2 values: one wave each): the rows around every place
    where a further launch can start, and the last ones, as by themselves."""
    dt, T, D, Hkv = getattr(gpu, dtype), (1 << 25) + 77, 2, 1
    g = gpu.Generator("cuda").manual_seed(5)
    q, k, v = (gpu.randn(T, Hkv, D, generator=g, device="cuda").to(dt) for _ in range(3))
    qg, kg = ((1 + 0.3 * gpu.randn(D, generator=g, device="cuda")).to(dt) for _ in range(2))
    cos, sin = _tables(gpu, 50, 1)
    pos = (gpu.arange(T, device="cuda") % 50).int()
    slots = T - 1 - gpu.arange(T, device="cuda")
    most = (1 << 24) - 1
    at = sorted({a for n in (2, 3) for a in range(0, T, 4 * most // n)} | {T})
    near = [slice(max(0, a - 40), min(T, a + 40)) for a in at]
    whole = ops.qk_norm_rope(q, k, qg, kg, cos, sin, pos)
    pools = [_pool(gpu, T, 1, Hkv, D, "fp8", 1) for _ in range(2)]
    y = ops.qk_norm_rope_cache(q, k, v, qg, kg, cos, sin, pos, slots, *pools[0])
    ops.kv_cache_write(whole[1], v, slots, *pools[1])
    assert gpu.equal(y, whole[0]) and all(gpu.equal(a, b) for a, b in zip(*pools))
    for s in near:
        part = ops.qk_norm_rope(q[s], k[s], qg, kg, cos, sin, pos[s])
        assert all(gpu.equal(a[s], b) for a, b in zip(whole, part))
        for i, x in ((0, whole[1]), (2, v)):
            c, scale = _rows_expected(gpu, ops, x[s], "fp8")
            assert gpu.equal(pools[0][i].flatten(0, 1)[slots[s]], c)
            assert gpu.equal(pools[0][i + 1].flatten(0, 1)[slots[s]], scale)


ACROSS = [(32, 16), (32, 8), (64, 16), (64, 40), (96, 96), (96, 32), (96, 48), (128, 32), (128, 96), (128, 24), (160, 80),
          (192, 96), (224, 224), (256, 96), (512, 160), (576, 48), (1024, 96)]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("Hq,Hkv,T", [(8, 8, 5), (7, 3, 9), (0, 1, 1), (4, 2, 700)])
@pytest.mark.parametrize("D,R", ACROSS)
def test_mxfp4_blocks_across_half_rotations(gpu, ops, D, R, Hq, Hkv, T, dtype):
    """Half-split heads whose half rotation is no whole number of blocks of 32: the fused
    call's cache is that of the two calls, with zeros, a NaN and an infinity among the values."""
    dt = getattr(gpu, dtype)
    q, k, v, qg, kg = _heads(gpu, T, Hq, Hkv, D, dt, seed=D + R)
    v[0, 0, D - 1] = float("inf")
    v[-1, -1, :8] = float("nan")
    k[-1, 0, D // 2] = float("nan")
    v[T // 2, 0] = 0
    cos, sin = _tables(gpu, 64, R // 2)
    pos = (gpu.arange(T, device="cuda") % 64).int()
    pages = T // 16 + 2
    slots = gpu.randperm(pages * 16, device="cuda")[:T]
    one, two = (_pool(gpu, pages, 16, Hkv, D, "mxfp4", 1) for _ in range(2))
    yq = ops.qk_norm_rope_cache(q, k, v, qg, kg, cos, sin, pos, slots, *one)
    wq, wk = ops.qk_norm_rope(q, k, qg, kg, cos, sin, pos)
    ops.kv_cache_write(wk, v, slots, *two)
    assert gpu.equal(yq, wq)
    assert all(gpu.equal(a, b) for a, b in zip(one, two))


@pytest.mark.parametrize("D,R", [(96, 96), (128, 32)])
def test_mxfp4_fused_write_is_no_slower_than_two_calls(gpu, ops, D, R):
    """Half a rotation that is no whole number of blocks keeps the kernel that a whole one has
    (one wave a head was 4 to 5 times the two calls' time; the bound is 1.5)."""
    torch, T, Hq, Hkv = gpu, 8000, 32, 8
    q, k, v, qg, kg = _heads(torch, T, Hq, Hkv, D, torch.bfloat16)
    cos, sin = _tables(torch, 100, R // 2)
    pos, slots = (torch.arange(T, device="cuda") % 100).int(), torch.randperm(T, device="cuda")
    pool = _pool(torch, T // 16, 16, Hkv, D, "mxfp4")

    def fused():
        ops.qk_norm_rope_cache(q, k, v, qg, kg, cos, sin, pos, slots, *pool)

    def two():
        ops.kv_cache_write(ops.qk_norm_rope(q, k, qg, kg, cos, sin, pos)[1], v, slots, *pool)

    def least(f):
        f()
        times = []
        for _ in range(5):
            a, b = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            a.record()
            for _ in range(10):
                f()
            b.record()
            torch.cuda.synchronize()
            times.append(a.elapsed_time(b))
        return min(times)

    assert least(fused) <= 1.5 * least(two)


@pytest.mark.parametrize("fmt,D", [("fp8", 128), ("fp8", 33), ("mxfp4", 128), ("mxfp4", 96)])
def test_a_pool_without_pages(gpu, ops, fmt, D):
    """No page: every slot is outside, every position reads as NaN."""
    q, k, v, qg, kg = _heads(gpu, 5, 4, 2, D, gpu.bfloat16)
    cos, sin = _tables(gpu, 5, D // 2)
    pos, slots = gpu.arange(5, device="cuda").int(), gpu.arange(5, device="cuda")
    pool = _pool(gpu, 0, 16, 2, D, fmt)
    ops.kv_cache_write(k, v, slots, *pool)
    y = ops.qk_norm_rope_cache(q, k, v, qg, kg, cos, sin, pos, slots, *pool)
    assert gpu.equal(y, ops.qk_norm_rope(q, k, qg, kg, cos, sin, pos)[0])
    got = ops.kv_cache_read(*pool, gpu.zeros(1, 1, dtype=gpu.int32, device="cuda"),
                            gpu.tensor([0, 5], dtype=gpu.int32, device="cuda"), 5)
    assert all(bool(gpu.isnan(t).all()) for t in got)


def test_calls_on_two_streams_at_once(gpu, ops):
    """The operators keep nothing between calls: two batches on two streams, many times, give
    what they give alone."""
    torch = gpu
    w, ws = ops.mxfp4_quantize(torch.randn(768, 512, device="cuda") * 0.05)
    cos, sin = _tables(torch, 300, 32)
    gam = torch.ones(64, device="cuda").bfloat16()

    def layer(x, pool):
        qkv = ops.mxfp4_gemm_w4a4(*ops.mxfp4_quantize(x), w, ws).unflatten(1, (12, 64))
        T = x.shape[0]
        pos = torch.arange(T, device="cuda", dtype=torch.int32)
        q = ops.qk_norm_rope_cache(qkv[:, :8], qkv[:, 8:10], qkv[:, 10:], gam, gam, cos, sin, pos, pos.long(), *pool)
        return (q, *ops.kv_cache_read(*pool, torch.arange(20, device="cuda", dtype=torch.int32)[None],
                                      torch.tensor([0, T], dtype=torch.int32, device="cuda"), T),
                ops.mxfp4_gemm_bf16(w, ws, x))

    xs = [torch.randn(T, 512, device="cuda").bfloat16() for T in (1, 300)]
    pools = [_pool(torch, 20, 16, 2, 64, fmt) for fmt in ("fp8", "mxfp4")]
    want = [layer(x, p) for x, p in zip(xs, pools)]
    streams = [torch.cuda.Stream() for _ in xs]
    got = [[], []]
    torch.cuda.synchronize()
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(layer(xs[i], pools[i]))
    torch.cuda.synchronize()
    for i in range(2):
        for out in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(out, want[i]))
