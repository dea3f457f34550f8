"""Attention of each sequence's newest token over the quantized cache, on the
GPU, against 64 bits on the values that the cache holds (the tolerance stands
in kc_serving.attention_tolerance).  The pool's other rows, and everything
behind a sequence's end, are NaN throughout."""
import ctypes

import numpy as np
import pytest

import kc_serving as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(gpu):
    import kernel_craft_torch_ops
    return kernel_craft_torch_ops


def nan_pool(torch, pages, page, H, D, fmt):
    if fmt == "fp8":
        return [t for _ in range(2) for t in (
            torch.full((pages, page, H, D), 127, dtype=torch.int8, device="cuda"),
            torch.full((pages, page, H), float("nan"), device="cuda"))]
    return [t for _ in range(2) for t in (
        torch.full((pages, page, H, D // 2), 17, dtype=torch.uint8, device="cuda"),
        torch.full((pages, page, H, D // 32), 255, dtype=torch.uint8, device="cuda"))]


def fill(torch, ops, lens, H, D, page, fmt, seed=0, spare=3, wide=2, window=0):
    """A cache that holds the visible positions of sequences of `lens`, pages
    shuffled; entries of the table behind a sequence's end, and those that the
    window hides, lead nowhere.  Returns (pool, table)."""
    rng = np.random.default_rng(seed)
    need = [-(-n // page) for n in lens]
    width = max(need + [1]) + wide
    order = rng.permutation(sum(need) + spare).astype(np.int32)
    table = rng.choice(np.array([-1, 2 ** 31 - 1, len(order), -2 ** 31], np.int32), (len(lens), width))
    slots, at = [], 0
    for b, n in enumerate(lens):
        table[b, :need[b]] = order[at:at + need[b]]
        at += need[b]
        first = max(0, n - window) if window else 0
        pos = np.arange(first, n)
        slots.append(table[b, pos // page].astype(np.int64) * page + pos % page)
        table[b, :first // page] = -1
    slots = np.concatenate(slots)
    g = torch.Generator("cuda").manual_seed(seed)
    k, v = (torch.randn(len(slots), H, D, generator=g, device="cuda") *
            (0.2 + 2 * torch.rand(len(slots), H, 1, generator=g, device="cuda")) for _ in range(2))
    pool = nan_pool(torch, len(order), page, H, D, fmt)
    ops.kv_cache_write(k, v, torch.from_numpy(slots).cuda(), *pool)
    return pool, torch.from_numpy(table).cuda()


def queries(torch, B, Hq, D, dtype, seed=0, size=1.0):
    g = torch.Generator("cuda").manual_seed(seed + 1)
    return (size * torch.randn(B, Hq, D, generator=g, device="cuda")).to(dtype)


def check(torch, ops, q, pool, table, lens, fmt, window=0, scale=None):
    B, Hq, D = q.shape
    page = pool[0].shape[1]
    d_lens = torch.tensor(lens, dtype=torch.int32, device="cuda")
    got = ops.kv_cache_attention(q, *pool, table, d_lens, scale=scale, window=window)
    assert got.dtype == q.dtype and got.shape == q.shape and got.is_contiguous()
    k, v = ref.rows_of(pool, fmt)
    want, mean, size = ref.attention(q.double().cpu().numpy(), k, v, table.cpu().numpy(), lens, page,
                                     D ** -0.5 if scale is None else scale, window)
    tol = ref.attention_tolerance(mean, size, want, D, max([1] + list(lens)), q.dtype == torch.bfloat16)
    y = got.double().cpu().numpy()
    bad = np.isnan(want)
    assert np.array_equal(np.isnan(y), bad)
    assert (np.abs(y - want)[~bad] <= tol[~bad]).all(), np.nanmax(np.abs(y - want) / np.maximum(tol, 1e-30))
    return got


LENS = [0, 1, 2, 31, 32, 33, 64, 65, 100, 0, 500, 127, 128, 129]
SHAPES = [  # q heads, kv heads, D, page, format
    (32, 8, 128, 16, "fp8"), (32, 8, 128, 16, "mxfp4"), (8, 8, 64, 1, "fp8"), (8, 8, 64, 48, "mxfp4"),
    (7, 1, 128, 32, "fp8"), (14, 2, 96, 7, "mxfp4"), (16, 1, 128, 64, "fp8"), (40, 2, 128, 64, "mxfp4"),
    (5, 1, 80, 16, "fp8"), (28, 4, 96, 5, "fp8"), (12, 3, 256, 16, "fp8"), (4, 1, 256, 33, "mxfp4"),
    (6, 3, 33, 16, "fp8"), (2, 2, 1, 3, "fp8"), (4, 2, 32, 16, "mxfp4"), (3, 1, 192, 16, "fp8"), (6, 1, 192, 8, "mxfp4"),
    (2, 1, 576, 16, "fp8"), (2, 1, 1024, 16, "mxfp4"), (9, 9, 16, 4, "fp8"), (66, 11, 64, 16, "fp8"), (10, 5, 112, 16, "fp8"),
    (4, 2, 48, 16, "fp8"), (4, 1, 144, 3, "fp8"), (8, 2, 160, 16, "fp8"), (8, 2, 160, 16, "mxfp4"), (2, 1, 176, 16, "fp8"),
    (2, 1, 208, 16, "fp8"), (2, 1, 224, 64, "fp8"), (5, 1, 224, 16, "mxfp4"), (3, 1, 240, 16, "fp8"),
    (72, 72, 64, 16, "fp8"), (64, 1, 128, 16, "fp8"), (1, 1, 1000, 16, "fp8"), (3, 1, 257, 16, "fp8"), (2, 1, 999, 5, "fp8"),
    (6, 2, 300, 16, "fp8"), (5, 1, 512, 16, "fp8"), (8, 2, 320, 16, "mxfp4"), (4, 4, 72, 16, "fp8"), (7, 1, 65, 16, "fp8"),
]


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("Hq,H,D,page,fmt", SHAPES)
def test_against_64_bits(gpu, ops, Hq, H, D, page, fmt, dtype):
    pool, table = fill(gpu, ops, LENS, H, D, page, fmt, seed=Hq + D)
    q = queries(gpu, len(LENS), Hq, D, getattr(gpu, dtype))
    check(gpu, ops, q, pool, table, LENS, fmt)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("window", [1, 2, 31, 32, 33, 100, 499, 500, 501, 2 ** 40])
def test_window(gpu, ops, window, dtype):
    for Hq, H, D, page, fmt in ((8, 2, 128, 16, "fp8"), (8, 2, 64, 7, "mxfp4"), (2, 1, 40, 16, "fp8")):
        pool, table = fill(gpu, ops, LENS, H, D, page, fmt, seed=window % 1000, window=window)
        check(gpu, ops, queries(gpu, len(LENS), Hq, D, getattr(gpu, dtype)), pool, table, LENS, fmt, window)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("lens", [[20000], [3, 9000, 0, 17], [33], [7], [64] * 40, [300] * 130, [0, 0, 0], [1] * 700,
                                  [4000, 1] * 9])
def test_long_and_many(gpu, ops, lens, dtype):
    """One sequence over all the stretches, and more sequences than stretches."""
    for Hq, H, D, page, fmt in ((8, 2, 128, 64, "fp8"), (4, 1, 128, 32, "mxfp4"), (3, 3, 24, 16, "fp8")):
        pool, table = fill(gpu, ops, lens, H, D, page, fmt, seed=len(lens))
        check(gpu, ops, queries(gpu, len(lens), Hq, D, getattr(gpu, dtype)), pool, table, lens, fmt)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_few_pages(gpu, ops, dtype):
    """Tables so short that no sequence is split: one launch."""
    for wide, page, lens in ((0, 16, [16, 3, 0, 1, 32]), (0, 1, [5, 1, 0]), (0, 64, [64, 63, 0, 33] * 20)):
        for Hq, H, D, fmt in ((32, 8, 128, "fp8"), (4, 2, 64, "mxfp4"), (3, 1, 20, "fp8")):
            pool, table = fill(gpu, ops, lens, H, D, page, fmt, wide=wide)
            check(gpu, ops, queries(gpu, len(lens), Hq, D, getattr(gpu, dtype)), pool, table, lens, fmt)


def test_lengths_that_the_table_does_not_have(gpu, ops):
    """Past the table: NaN; below zero: no position."""
    for D, page, wide in ((128, 16, 0), (128, 16, 30), (33, 16, 0)):
        pool, table = fill(gpu, ops, [40, 20, 16], 2, D, page, "fp8", wide=wide)
        room = table.shape[1] * page
        table = table.where((table >= 0) & (table < len(pool[0])), table.new_zeros(()))
        for window in (0, 3):
            check(gpu, ops, queries(gpu, 3, 4, D, gpu.bfloat16), pool, table, [room + 1, -3, 16], "fp8", window)
            check(gpu, ops, queries(gpu, 3, 4, D, gpu.float32), pool, table, [40, 2 ** 31 - 1, -2 ** 31], "fp8", window)


@pytest.mark.parametrize("D", [128, 33])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_missing_pages(gpu, ops, D, dtype):
    """A visible position without a page: NaN for its sequence alone."""
    lens = [100, 100, 100, 700, 5]
    pool, table = fill(gpu, ops, lens, 2, D, 16, "fp8", window=90)
    q = queries(gpu, 5, 8, D, getattr(gpu, dtype))
    table[1, 6] = -1
    table[3, 40] = len(pool[0])
    y = check(gpu, ops, q, pool, table, lens, "fp8", window=90)
    assert gpu.isnan(y).flatten(1).all(1).tolist() == [False, True, False, True, False]
    assert bool(gpu.isnan(ops.kv_cache_attention(q, *pool, table, gpu.tensor(lens, dtype=gpu.int32, device="cuda"))[0]).all())


def test_no_pool(gpu, ops):
    pool = nan_pool(gpu, 0, 16, 2, 64, "fp8")
    i32 = dict(dtype=gpu.int32, device="cuda")
    y = ops.kv_cache_attention(queries(gpu, 2, 4, 64, gpu.bfloat16), *pool, gpu.zeros(2, 3, **i32),
                               gpu.tensor([0, 4], **i32))
    assert float(y[0].abs().max()) == 0 and bool(gpu.isnan(y[1]).all())
    y = ops.kv_cache_attention(queries(gpu, 2, 4, 64, gpu.float32), *pool, gpu.zeros(2, 0, **i32), gpu.tensor([0, 4], **i32))
    assert float(y[0].abs().max()) == 0 and bool(gpu.isnan(y[1]).all())
    for B, Hq in ((0, 4), (2, 0)):
        assert ops.kv_cache_attention(queries(gpu, B, Hq, 64, gpu.bfloat16), *pool, gpu.zeros(B, 3, **i32),
                                      gpu.zeros(B, **i32)).shape == (B, Hq, 64)


@pytest.mark.parametrize("D,fmt", [(128, "fp8"), (128, "mxfp4"), (33, "fp8")])
def test_large_and_equal_scores(gpu, ops, D, fmt):
    """Scores of thousands, all alike, or far apart in one sequence: no overflow,
    and one position may take all the weight."""
    lens = [300, 1, 64, 2000]
    pool, table = fill(gpu, ops, lens, 2, D, 16, fmt)
    for dtype in (gpu.bfloat16, gpu.float32):
        for size, scale in ((100.0, None), (0.0, None), (1.0, 0.0), (1.0, 50.0), (1.0, -3.0), (30.0, 1e-6)):
            check(gpu, ops, queries(gpu, 4, 8, D, dtype, size=size), pool, table, lens, fmt, scale=scale)


@pytest.mark.parametrize("D", [128, 288])
def test_the_largest_queries(gpu, ops, D):
    """fp32 queries that bf16 would round to infinity: one value a head, against
    keys of a quarter there, so that every product and sum stays in fp32."""
    lens = [90, 3, 300]
    pool, table = fill(gpu, ops, lens, 2, D, 16, "mxfp4")
    k = gpu.ones(90, 2, D, device="cuda")
    at = gpu.arange(90, device="cuda")
    slots = table[0, at // 16].long() * 16 + at % 16
    q = gpu.zeros(3, 8, D, device="cuda")
    for h in range(8):
        k[:, h // 4, 3 * h] = 0.25 * (1 - 2 * (at % (h + 2) == 0).float())
        q[0, h, 3 * h] = 3.402e38 * (-1.0) ** h
    ops.kv_cache_write(k, gpu.randn(90, 2, D, device="cuda"), slots, *pool)
    check(gpu, ops, q, pool, table, lens, "mxfp4", scale=2.0 ** -126)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("D", [128, 16, 33, 288])
def test_the_range_of_fp8_scores(gpu, ops, D, dtype):
    """Queries and keys whose products with each other stay in fp32, but not those
    with the keys' codes (up to 448) or the scales' with the scale of the call."""
    lens = [90, 3, 300]
    pool, table = fill(gpu, ops, lens, 2, D, 16, "fp8")
    at = gpu.arange(90, device="cuda")
    slots = table[0, at // 16].long() * 16 + at % 16
    v = gpu.randn(90, 2, D, device="cuda")
    # one value a head, of nearly fp32's largest, against keys of a quarter there
    k = gpu.ones(90, 2, D, device="cuda")
    q = gpu.zeros(3, 8, D, device="cuda")
    for h in range(8):
        k[:, h // 4, 2 * h] = 0.25 * (1 - 2 * (at % (h + 2) == 0).float())
        q[0, h, 2 * h] = 3.3e38 * (-1.0) ** h
    ops.kv_cache_write(k, v, slots, *pool)
    check(gpu, ops, q.to(getattr(gpu, dtype)), pool, table, lens, "fp8", scale=2.0 ** -126)
    # large against small, both ways
    for size in (3e35, 1e-30):
        ops.kv_cache_write(gpu.randn(90, 2, D, device="cuda") / size, v, slots, *pool)
        q = queries(gpu, 3, 8, D, getattr(gpu, dtype))
        q[0] = (size * queries(gpu, 1, 8, D, gpu.float32)[0]).to(q.dtype)
        check(gpu, ops, q, pool, table, lens, "fp8")


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("D", [128, 33])
def test_any_finite_scale_of_a_key(gpu, ops, D, dtype):
    """Zero, negative, denormal and far apart, in one tile."""
    lens = [70, 40]
    pool, table = fill(gpu, ops, lens, 2, D, 16, "fp8")
    at = gpu.arange(70, device="cuda")
    kinds = gpu.tensor([0.0, -0.01, 2.0 ** -140, 2.0 ** -149, 0.02, 2.0 ** -101, -(2.0 ** -130)], device="cuda")
    pool[1][table[0, at // 16].long(), at % 16] = kinds[at % 7, None].expand(70, 2).contiguous()
    check(gpu, ops, queries(gpu, 2, 8, D, getattr(gpu, dtype)), pool, table, lens, "fp8")

@pytest.mark.parametrize("D,fmt", [(128, "fp8"), (64, "mxfp4"), (33, "fp8")])
def test_nan_and_infinite_queries(gpu, ops, D, fmt):
    """A query head's NaN or infinity, and a key's or value's NaN, stay where they are."""
    lens = [200, 200, 70]
    pool, table = fill(gpu, ops, lens, 2, D, 16, fmt)
    for dtype in (gpu.bfloat16, gpu.float32):
        q = queries(gpu, 3, 8, D, dtype)
        plain = check(gpu, ops, q, pool, table, lens, fmt)
        q[0, 1, 5] = float("nan")
        q[1, 6, 0] = float("inf")
        y = ops.kv_cache_attention(q, *pool, table, gpu.tensor(lens, dtype=gpu.int32, device="cuda"))
        bad = gpu.zeros(3, 8, dtype=gpu.bool, device="cuda")
        bad[0, 1] = bad[1, 6] = True
        assert bool(gpu.isnan(y[bad]).all()) and gpu.equal(y[~bad], plain[~bad])
    one = [t.clone() for t in pool]
    page = int(table[1, 3])
    one[3][page, 2, 1] = float("nan") if fmt == "fp8" else 255  # the scale of one value row, of the second head
    q = queries(gpu, 3, 8, D, gpu.bfloat16)
    y = ops.kv_cache_attention(q, *one, table, gpu.tensor(lens, dtype=gpu.int32, device="cuda"))
    assert bool(gpu.isnan(y[1, 4:]).all()) and not bool(gpu.isnan(y[1, :4]).any()) and not bool(gpu.isnan(y[[0, 2]]).any())


def test_views_and_alignment(gpu, ops):
    """Queries as views of a fused projection, a cache that does not begin at 16
    bytes, a table that is a view: the same values."""
    lens = [50, 333, 0, 64]
    for D, fmt in ((128, "fp8"), (128, "mxfp4"), (64, "fp8")):
        pool, table = fill(gpu, ops, lens, 2, D, 16, fmt)
        d_lens = gpu.tensor(lens, dtype=gpu.int32, device="cuda")
        rows = gpu.randn(4, 12 * D + 8, device="cuda").bfloat16()
        for lead in (0, 8, 1):
            q = rows[:, lead:lead + 8 * D].unflatten(1, (8, D))
            want = ops.kv_cache_attention(q.contiguous(), *pool, table, d_lens)
            assert gpu.equal(ops.kv_cache_attention(q, *pool, table, d_lens), want)
            wide = gpu.cat([table, table], 1)[:, :table.shape[1]]
            assert gpu.equal(ops.kv_cache_attention(q, *pool, wide, d_lens), want)
        for off in (1, 4, 8):
            def moved(t):
                raw = gpu.zeros(t.numel() * t.element_size() + 16, dtype=gpu.uint8, device="cuda")
                at = off if t.element_size() == 1 else 4 * (off % 4)
                m = raw[at:at + t.numel() * t.element_size()].view(t.dtype).view(t.shape)
                return m.copy_(t)
            check(gpu, ops, queries(gpu, 4, 8, D, gpu.bfloat16), [moved(t) for t in pool], table, lens, fmt)


def test_offsets_past_32_bits(gpu, ops):
    """Pages whose codes lie beyond 4 GiB."""
    H, D, page, pages = 8, 128, 64, 70000
    lens = [200, 90]
    for dtype in (gpu.bfloat16, gpu.float32):
        pool, table = fill(gpu, ops, lens, H, D, page, "fp8", wide=0)
        far = [gpu.zeros((pages,) + t.shape[1:], dtype=t.dtype, device="cuda") for t in pool]
        for t, s in zip(far, pool):
            t[pages - len(s):] = s
        q = queries(gpu, 2, 32, D, dtype)
        d_lens = gpu.tensor(lens, dtype=gpu.int32, device="cuda")
        real = (table >= 0) & (table < len(pool[0]))
        moved = gpu.where(real, table + (pages - len(pool[0])), -1)
        assert gpu.equal(ops.kv_cache_attention(q, *far, moved, d_lens), ops.kv_cache_attention(q, *pool, table, d_lens))


def test_results_repeat(gpu, ops):
    """The same bits every time, and on two streams at once."""
    lens = [3000, 1, 700, 0, 64] * 8
    pool, table = fill(gpu, ops, lens, 8, 128, 16, "fp8")
    q = queries(gpu, len(lens), 32, 128, gpu.bfloat16)
    d_lens = gpu.tensor(lens, dtype=gpu.int32, device="cuda")
    want = ops.kv_cache_attention(q, *pool, table, d_lens)
    streams = [gpu.cuda.Stream() for _ in range(2)]
    gpu.cuda.synchronize()
    got = []
    for _ in range(10):
        for s in streams:
            with gpu.cuda.stream(s):
                got.append(ops.kv_cache_attention(q, *pool, table, d_lens))
    gpu.cuda.synchronize()
    assert all(gpu.equal(y, want) for y in got)


def test_pages_in_several_places(gpu, ops):
    """Sequences that share the pages of a prefix, and a page twice in one: the
    values of a cache that holds copies."""
    lens = [100, 90, 64, 3]
    for D, fmt in ((128, "fp8"), (64, "mxfp4"), (33, "fp8")):
        pool, table = fill(gpu, ops, lens, 2, D, 16, fmt)
        table[1, :5] = table[0, :5]
        table[2, 2] = table[2, 0]
        table[3, 0] = table[0, 1]
        for dtype in (gpu.bfloat16, gpu.float32):
            check(gpu, ops, queries(gpu, 4, 8, D, dtype), pool, table, lens, fmt)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_windows_of_a_large_batch(gpu, ops, dtype):
    """More sequences than a wave has lanes, some empty, some within the window."""
    lens = [(37 * i * i) % 301 * (i % 7 != 3) for i in range(150)] + [2500, 0]
    for Hq, H, D, page, fmt in ((16, 4, 128, 16, "fp8"), (8, 1, 64, 48, "mxfp4"), (3, 1, 20, 16, "fp8")):
        pool, table = fill(gpu, ops, lens, H, D, page, fmt, window=129)
        check(gpu, ops, queries(gpu, len(lens), Hq, D, getattr(gpu, dtype)), pool, table, lens, fmt, 129)


def test_two_graphs_replayed_in_turn(gpu, ops):
    """Captured once each, replayed while lengths and queries change in place,
    with eager calls between."""
    lens = [500, 20, 0, 64, 1200]
    pool, table = fill(gpu, ops, lens, 2, 128, 16, "mxfp4")
    d_lens = gpu.tensor(lens, dtype=gpu.int32, device="cuda")
    qs = [queries(gpu, 5, 8, 128, gpu.bfloat16, seed=s) for s in (0, 5)]
    side = gpu.cuda.Stream()
    side.wait_stream(gpu.cuda.current_stream())
    with gpu.cuda.stream(side):
        ops.kv_cache_attention(qs[0], *pool, table, d_lens)
    gpu.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for q in qs:
        g = gpu.cuda.CUDAGraph()
        with gpu.cuda.graph(g):
            outs.append(ops.kv_cache_attention(q, *pool, table, d_lens))
        graphs.append(g)
    for i in range(5):
        d_lens.copy_(gpu.tensor([max(0, n - 7 * i) for n in lens], dtype=gpu.int32))
        for q in qs:
            q.normal_()
        want = [ops.kv_cache_attention(q, *pool, table, d_lens) for q in qs]
        for g in graphs:
            g.replay()
        gpu.cuda.synchronize()
        assert all(gpu.equal(a, b) for a, b in zip(outs, want))


def test_rows_do_not_depend_on_their_neighbours_output(gpu, ops):
    """Nothing is written behind the output, and a workspace's content does not matter."""
    import kc_abi
    lens = [300, 0, 5]
    pool, table = fill(gpu, ops, lens, 2, 64, 16, "fp8")
    q = queries(gpu, 3, 6, 64, gpu.float32)
    d_lens = gpu.tensor(lens, dtype=gpu.int32, device="cuda")
    want = ops.kv_cache_attention(q, *pool, table, d_lens)
    cache = ops.KvCache(*(t.data_ptr() for t in pool), len(pool[0]), 16, 2, 64, 0)
    L = kc_abi.lib()
    need = L.kc_kv_cache_attention_workspace(ctypes.byref(cache), table.shape[1], 3, 6)
    for byte in (0, 255, 127):
        work = gpu.full((need + 64,), byte, dtype=gpu.uint8, device="cuda")
        out = gpu.full((4, 6, 64), 9.0, device="cuda")
        st = L.kc_kv_cache_attention_f32(kc_abi.ptr(q), q.stride(0), 6, ctypes.byref(cache), kc_abi.ptr(table),
                                         table.shape[1], kc_abi.ptr(d_lens), 3, 64 ** -0.5, 0, kc_abi.ptr(work), need,
                                         kc_abi.ptr(out), kc_abi.stream())
        assert st == 0 and gpu.equal(out[:3], want) and bool((out[3] == 9).all())
        assert bool((work[need:] == byte).all())
    assert L.kc_kv_cache_attention_f32(kc_abi.ptr(q), q.stride(0), 6, ctypes.byref(cache), kc_abi.ptr(table),
                                       table.shape[1], kc_abi.ptr(d_lens), 3, 64 ** -0.5, 0, kc_abi.ptr(work), need - 1,
                                       kc_abi.ptr(out), kc_abi.stream()) == 1
    assert L.kc_get_last_error() == 1


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
def test_serving_steps(gpu, ops, fmt):
    """Steps as a server runs them: pages for the new tokens, their heads normed,
    rotated and written to the cache, attention over it, the residual sum and
    norm, sequences that end and come anew; against 64 bits on the cache as it
    is, and the cache against kv_cache_read."""
    B, Hq, H, D, page, width = 6, 8, 2, 64, 16, 12
    i32 = dict(dtype=gpu.int32, device="cuda")
    pages = 40
    gpu.manual_seed(9)
    pool = nan_pool(gpu, pages, page, H, D, fmt)
    lens, table = gpu.zeros(B, **i32), gpu.full((B, width), -1, **i32)
    free, count = gpu.randperm(pages, device="cuda").to(gpu.int32), gpu.full((1,), pages, **i32)
    angle = gpu.rand(width * page, D // 2, device="cuda") * 6
    gam = [(1 + 0.2 * gpu.randn(D, device="cuda")).bfloat16() for _ in range(2)]
    rng = np.random.default_rng(4)
    w = gpu.randn(Hq * D, Hq * D, device="cuda").bfloat16() * (Hq * D) ** -0.5
    wq, ws = ops.fp8_quantize_rows(w)
    gamma = (1 + 0.2 * gpu.randn(Hq * D, device="cuda")).bfloat16()
    for step in range(8):
        new = rng.integers(1, 40, B) if step % 4 == 0 else np.ones(B, int)
        total = int(new.sum())
        old = lens.tolist()
        lens, count, cu_new, cu, positions, slots = ops.kv_cache_extend(
            lens, gpu.tensor(new, **i32), table, free, count, page, total)
        served = [a != b for a, b in zip(old, lens.tolist())]
        qkv = gpu.randn(total, (Hq + 2 * H) * D, device="cuda").bfloat16()
        q, k, v = (t.unflatten(1, (-1, D)) for t in qkv.split([Hq * D, H * D, H * D], 1))
        q = ops.qk_norm_rope_cache(q, k, v, *gam, angle.cos(), angle.sin(), positions, slots, *pool)
        last = q[cu_new[1:].long() - 1]
        y = check(gpu, ops, last, pool, table, lens.tolist(), fmt)
        keys, values = ops.kv_cache_read(*pool, table, cu, int(cu[-1]), out_dtype=gpu.float32)
        assert bool(gpu.isfinite(keys).all()) and bool(gpu.isfinite(values).all())
        x = gpu.randn(B, Hq * D, device="cuda").bfloat16()
        x, codes, scales = ops.residual_rmsnorm_fp8_quantize(y.flatten(1), x, gamma, alpha=0.5)
        out = ops.fp8_gemm_w8a8(codes, scales, wq, ws)
        assert bool(gpu.isfinite(out).all())
        assert any(served)
        done = gpu.tensor(rng.random(B) < 0.3, device="cuda")
        lens, count = ops.kv_cache_release(done, lens, table, free, count, page)
        held = sum(-(-n // page) for n in lens.tolist())
        assert int(count) == pages - held and len(free[:pages - held].unique()) == pages - held


def workspace(ops, pool, table, B, Hq):
    """Bytes that attention over this cache needs; 0 where no sequence is split."""
    import kc_abi
    pages, page, H = pool[0].shape[:3]
    fp8 = pool[1].dim() == 3
    D = pool[0].shape[3] * (1 if fp8 else 2)
    cache = ops.KvCache(*(t.data_ptr() for t in pool), pages, page, H, D, 0 if fp8 else 1)
    return kc_abi.lib().kc_kv_cache_attention_workspace(ctypes.byref(cache), table.shape[1], B, Hq), cache


def split(ops, pool, table, B, Hq):
    need, _ = workspace(ops, pool, table, B, Hq)
    assert need > 0
    return need


def wide_for(page, positions=2000):
    return -(-positions // page)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("Hq,H,D,page,fmt", SHAPES)
def test_split_against_64_bits(gpu, ops, Hq, H, D, page, fmt, dtype):
    """Tables so wide that every sequence is cut into stretches and joined: ends
    of sequences inside a stretch, whole ones, empty ones between them."""
    lens = LENS + [700, 3]
    pool, table = fill(gpu, ops, lens, H, D, page, fmt, seed=Hq + D, wide=wide_for(page))
    split(ops, pool, table, len(lens), Hq)
    check(gpu, ops, queries(gpu, len(lens), Hq, D, getattr(gpu, dtype)), pool, table, lens, fmt)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("window", [1300, 1313, 1999])
def test_split_windows(gpu, ops, window, dtype):
    import kc_abi
    lens = [3000, window - 1, window, window + 1, 0, 5, 2500]
    for Hq, H, D, page, fmt in ((8, 2, 128, 16, "fp8"), (8, 2, 64, 7, "mxfp4"), (3, 1, 40, 16, "fp8")):
        pool, table = fill(gpu, ops, lens, H, D, page, fmt, seed=window, window=window)
        q = queries(gpu, len(lens), Hq, D, getattr(gpu, dtype))
        d_lens = gpu.tensor(lens, dtype=gpu.int32, device="cuda")
        assert any("join_kernel" in n for n in kc_abi.kernels_of(
            lambda: ops.kv_cache_attention(q, *pool, table, d_lens, window=window)))
        check(gpu, ops, q, pool, table, lens, fmt, window)


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_split_lengths_that_the_table_does_not_have(gpu, ops, dtype):
    for D in (128, 80, 33):
        pool, table = fill(gpu, ops, [40, 20, 16, 900], 2, D, 16, "fp8", wide=wide_for(16))
        split(ops, pool, table, 4, 4)
        room = table.shape[1] * 16
        table = table.where((table >= 0) & (table < len(pool[0])), table.new_zeros(()))
        q = queries(gpu, 4, 4, D, getattr(gpu, dtype))
        check(gpu, ops, q, pool, table, [room + 1, -3, 16, 900], "fp8")
        check(gpu, ops, q, pool, table, [40, 2 ** 31 - 1, -2 ** 31, 900], "fp8")
        check(gpu, ops, q, pool, table, [40, 7, 2 ** 31 - 1, 900], "fp8", window=1500)


@pytest.mark.parametrize("fmt,D", [("fp8", 128), ("mxfp4", 64), ("fp8", 208), ("fp8", 33)])
@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
def test_split_missing_pages(gpu, ops, D, fmt, dtype):
    """NaN through the join, for the sequence whose page is missing alone."""
    lens = [100, 100, 100, 700, 5, 300]
    pool, table = fill(gpu, ops, lens, 2, D, 16, fmt, wide=wide_for(16))
    split(ops, pool, table, 6, 8)
    table[1, 6] = -1
    table[3, 40] = len(pool[0])
    y = check(gpu, ops, queries(gpu, 6, 8, D, getattr(gpu, dtype)), pool, table, lens, fmt)
    assert gpu.isnan(y).flatten(1).all(1).tolist() == [False, True, False, True, False, False]


@pytest.mark.parametrize("D,fmt", [(128, "fp8"), (64, "mxfp4"), (160, "fp8"), (33, "fp8")])
def test_split_nan_and_infinite_queries(gpu, ops, D, fmt):
    lens = [200, 200, 70]
    pool, table = fill(gpu, ops, lens, 2, D, 16, fmt, wide=wide_for(16))
    split(ops, pool, table, 3, 8)
    d_lens = gpu.tensor(lens, dtype=gpu.int32, device="cuda")
    for dtype in (gpu.bfloat16, gpu.float32):
        q = queries(gpu, 3, 8, D, dtype)
        plain = check(gpu, ops, q, pool, table, lens, fmt)
        q[0, 1, 5] = float("nan")
        q[1, 6, 0] = float("inf")
        y = ops.kv_cache_attention(q, *pool, table, d_lens)
        bad = gpu.zeros(3, 8, dtype=gpu.bool, device="cuda")
        bad[0, 1] = bad[1, 6] = True
        assert bool(gpu.isnan(y[bad]).all()) and gpu.equal(y[~bad], plain[~bad])
    one = [t.clone() for t in pool]
    one[3][int(table[1, 3]), 2, 1] = float("nan") if fmt == "fp8" else 255  # one value row's scale, of the second head
    y = ops.kv_cache_attention(queries(gpu, 3, 8, D, gpu.bfloat16), *one, table, d_lens)
    assert bool(gpu.isnan(y[1, 4:]).all()) and not bool(gpu.isnan(y[1, :4]).any()) and not bool(gpu.isnan(y[[0, 2]]).any())


def test_split_large_and_equal_scores(gpu, ops):
    lens = [300, 1, 64, 2000]
    for D, fmt in ((128, "fp8"), (128, "mxfp4"), (33, "fp8")):
        pool, table = fill(gpu, ops, lens, 2, D, 16, fmt, wide=wide_for(16))
        split(ops, pool, table, 4, 8)
        for dtype in (gpu.bfloat16, gpu.float32):
            for size, scale in ((100.0, None), (0.0, None), (1.0, 0.0), (1.0, 50.0), (1.0, -3.0)):
                check(gpu, ops, queries(gpu, 4, 8, D, dtype, size=size), pool, table, lens, fmt, scale=scale)


def test_split_views(gpu, ops):
    """Queries that are views, a cache that begins at 16 bytes and no more: the
    same values from the same kernel."""
    lens = [50, 333, 0, 64, 900]
    for D, fmt in ((128, "fp8"), (128, "mxfp4"), (64, "fp8")):
        pool, table = fill(gpu, ops, lens, 2, D, 16, fmt, wide=wide_for(16))
        split(ops, pool, table, 5, 8)
        d_lens = gpu.tensor(lens, dtype=gpu.int32, device="cuda")
        rows = gpu.randn(5, 12 * D + 8, device="cuda").bfloat16()
        for lead in (0, 8, 1):
            q = rows[:, lead:lead + 8 * D].unflatten(1, (8, D))
            want = ops.kv_cache_attention(q.contiguous(), *pool, table, d_lens)
            assert gpu.equal(ops.kv_cache_attention(q, *pool, table, d_lens), want)

            def moved(t):
                raw = gpu.zeros(t.numel() * t.element_size() + 16, dtype=gpu.uint8, device="cuda")
                return raw[16:].view(t.dtype).view(t.shape).copy_(t)
            assert gpu.equal(ops.kv_cache_attention(q, *[moved(t) for t in pool], table, d_lens), want)


def test_split_offsets_past_32_bits(gpu, ops):
    """Pages whose codes lie beyond 4 GiB."""
    H, D, page, pages = 8, 128, 64, 70000
    lens = [2000, 90]
    for dtype in (gpu.bfloat16, gpu.float32):
        pool, table = fill(gpu, ops, lens, H, D, page, "fp8")
        split(ops, pool, table, 2, 32)
        far = [gpu.zeros((pages,) + t.shape[1:], dtype=t.dtype, device="cuda") for t in pool]
        for t, s in zip(far, pool):
            t[pages - len(s):] = s
        q = queries(gpu, 2, 32, D, dtype)
        d_lens = gpu.tensor(lens, dtype=gpu.int32, device="cuda")
        real = (table >= 0) & (table < len(pool[0]))
        moved = gpu.where(real, table + (pages - len(pool[0])), -1)
        assert gpu.equal(ops.kv_cache_attention(q, *far, moved, d_lens), ops.kv_cache_attention(q, *pool, table, d_lens))


@pytest.mark.parametrize("dtype", ["bfloat16", "float32"])
@pytest.mark.parametrize("B", [65, 600, 1100])
def test_split_more_sequences_than_threads(gpu, ops, B, dtype):
    """A thread counts the tiles of several sequences, some of them empty."""
    lens = [(37 * i) % 90 * (i % 5 != 2) for i in range(B)]
    lens[B // 2] = 4000
    lens[-1] = 0
    for Hq, H, D, page, fmt in ((8, 2, 64, 16, "fp8"), (2, 1, 128, 32, "mxfp4"), (2, 1, 20, 16, "fp8")):
        pool, table = fill(gpu, ops, lens, H, D, page, fmt, seed=B)
        split(ops, pool, table, B, Hq)
        check(gpu, ops, queries(gpu, B, Hq, D, getattr(gpu, dtype)), pool, table, lens, fmt)


@pytest.mark.parametrize("D", [64, 33])
def test_any_content_of_the_workspace(gpu, ops, D):
    """What the workspace holds does not matter, NaN included; nothing is written
    behind it or the output; one byte less is refused."""
    import kc_abi
    lens = [4000, 1, 0, 700]
    pool, table = fill(gpu, ops, lens, 2, D, 16, "fp8")
    d_lens = gpu.tensor(lens, dtype=gpu.int32, device="cuda")
    need, cache = workspace(ops, pool, table, 4, 6)
    assert need > 64
    L = kc_abi.lib()
    for fn, dtype in ((L.kc_kv_cache_attention_f32, gpu.float32), (L.kc_kv_cache_attention_bf16, gpu.bfloat16)):
        q = queries(gpu, 4, 6, D, dtype)
        want = check(gpu, ops, q, pool, table, lens, "fp8")

        def call(work, bytes_, out):
            return fn(kc_abi.ptr(q), q.stride(0), 6, ctypes.byref(cache), kc_abi.ptr(table), table.shape[1],
                      kc_abi.ptr(d_lens), 4, D ** -0.5, 0, kc_abi.ptr(work), bytes_, kc_abi.ptr(out), kc_abi.stream())
        for byte in (0, 255, 127, 129):
            work = gpu.full((need + 256,), byte, dtype=gpu.uint8, device="cuda")
            out = gpu.full((5, 6, D), 9.0, dtype=dtype, device="cuda")
            assert call(work, need, out) == 0
            assert gpu.equal(out[:4], want) and bool((out[4] == 9).all()) and bool((work[need:] == byte).all())
        assert call(work, need - 1, out) == 1 and L.kc_get_last_error() == 1


@pytest.mark.parametrize("fmt,D", [("fp8", 128), ("mxfp4", 128), ("fp8", 33)])
def test_split_graphs_replayed_in_turn(gpu, ops, fmt, D):
    """Two captured calls, replayed while lengths that move every stretch's bounds,
    and queries, change in place, with eager calls between."""
    most = [4000, 20, 0, 64, 1200]
    pool, table = fill(gpu, ops, most, 2, D, 16, fmt)
    split(ops, pool, table, 5, 8)
    d_lens = gpu.tensor(most, dtype=gpu.int32, device="cuda")
    qs = [queries(gpu, 5, 8, D, dtype, seed=5) for dtype in (gpu.bfloat16, gpu.float32)]
    side = gpu.cuda.Stream()
    side.wait_stream(gpu.cuda.current_stream())
    with gpu.cuda.stream(side):
        for q in qs:
            ops.kv_cache_attention(q, *pool, table, d_lens)
    gpu.cuda.current_stream().wait_stream(side)
    graphs, outs = [], []
    for q in qs:
        g = gpu.cuda.CUDAGraph()
        with gpu.cuda.graph(g):
            outs.append(ops.kv_cache_attention(q, *pool, table, d_lens))
        graphs.append(g)
    for lens in (most, [3999, 0, 0, 64, 1199], [17, 20, 0, 0, 1200], [0] * 5, [4000, 1, 0, 33, 3], [2048, 20, 0, 1, 0]):
        d_lens.copy_(gpu.tensor(lens, dtype=gpu.int32))
        for q in qs:
            q.normal_()
        want = [check(gpu, ops, q, pool, table, lens, fmt) for q in qs]
        for _ in range(2):
            for g in graphs:
                g.replay()
        gpu.cuda.synchronize()
        assert all(gpu.equal(a, b) for a, b in zip(outs, want))


@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
def test_long_results_repeat(gpu, ops, fmt):
    """The same bits behind other calls, which leave other parts in the same memory."""
    lens = [0, 5000, 18000, 40000]
    pool, table = fill(gpu, ops, lens, 2, 128, 64, fmt, wide=0)
    split(ops, pool, table, 4, 8)
    d_lens = gpu.tensor(lens, dtype=gpu.int32, device="cuda")
    q, other = (queries(gpu, 4, 8, 128, gpu.bfloat16, seed=s) for s in (1, 2))
    want = check(gpu, ops, q, pool, table, lens, fmt)
    got = []
    for _ in range(20):
        ops.kv_cache_attention(other, *pool, table, d_lens)
        got.append(ops.kv_cache_attention(q, *pool, table, d_lens))
    assert all(gpu.equal(y, want) for y in got)
