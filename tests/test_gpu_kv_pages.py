"""Pages of the cache given to the requests of a step and taken back, on the
GPU, against the same rules request after request: whole numbers, equal."""
import numpy as np
import pytest

import kc_serving as ref

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops(gpu):
    import kernel_craft_torch_ops
    return kernel_craft_torch_ops


def _dev(torch, a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def _state(rng, lens, page, width, free, spare=4):
    """A table with the pages of `lens` (entries behind them left over from
    others), and a stack of `free` pages in a capacity of all."""
    need = [min(-(-max(int(n), 0) // page), width) for n in lens]
    order = rng.permutation(sum(need) + free + spare).astype(np.int32)
    table = rng.integers(0, 1000, (len(lens), width)).astype(np.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = order[at:at + n]
        at += n
    stack = np.full(len(order), -7, np.int32)
    stack[:free] = order[at:at + free]
    return table, stack


def _extend(torch, ops, lens, new, table, stack, count, page, rows):
    want = ref.extend(lens, new, table, stack, count, page, rows)
    args = [_dev(torch, np.asarray(a, np.int32)) for a in (lens, new, table, stack, [count])]
    before = [a.clone() for a in args]
    for _ in range(2):  # again on the same inputs: the same
        got = (*ops.kv_cache_extend(*args, page, rows), args[2])
        for name, g, w in zip(("lens", "count", "cu_new", "cu_seqlens", "positions", "slots", "table"), got, want):
            assert g.dtype == (torch.int64 if name == "slots" else torch.int32)
            assert np.array_equal(g.cpu().numpy(), w), name
    assert all(torch.equal(a, b) for i, (a, b) in enumerate(zip(args, before)) if i != 2)
    return got


EXTENDS = [  # requests, longest, new, page, width to spare, share of the pages that there are, rows to spare
    (1, 0, 1, 16, 0, 1.0, 0), (1, 16, 1, 16, 0, 1.0, 0), (1, 700, 1, 16, 3, 0.0, 0), (64, 500, 1, 16, 2, 1.0, 0),
    (64, 500, 1, 16, 2, 0.5, 0), (9, 100, 60, 7, 1, 1.0, 5), (9, 100, 60, 7, 1, 0.6, 0), (33, 40, 90, 1, 0, 0.7, 3),
    (256, 300, 1, 16, 1, 0.8, 0), (257, 30, 4, 16, 1, 1.0, 2), (1000, 300, 1, 32, 1, 0.9, 0), (1024, 60, 3, 16, 1, 1.0, 1), (1025, 60, 3, 16, 1, 0.5, 0),
    (3000, 50, 2, 8, 1, 0.8, 700), (5, 9000, 3000, 64, 2, 1.0, 0), (2, 1, 5000, 3, 0, 1.0, 0),
]


@pytest.mark.parametrize("B,ctx,new,page,wide,share,spare", EXTENDS)
def test_extend(gpu, ops, B, ctx, new, page, wide, share, spare):
    rng = np.random.default_rng(B * 7 + ctx)
    lens = rng.integers(0, ctx + 1, B)
    fresh = np.ones(B, int) if new == 1 else rng.integers(0, new + 1, B)
    need = sum(-(-(a + b) // page) - -(-a // page) for a, b in zip(lens, fresh))
    width = -(-int((lens + fresh).max()) // page) + wide
    free = int(need * share)
    table, stack = _state(rng, lens, page, width, free)
    got = _extend(gpu, ops, lens, fresh, table, stack, free, page, int(fresh.sum()) + spare)
    # the pages in use are the table's and no two rows share a slot
    slots = got[5][got[5] >= 0]
    assert len(slots.unique()) == len(slots)


def test_extend_limits(gpu, ops):
    """Requests that pass the table or the rows are left out, those that lack no
    page are served behind one that finds none; lengths below zero count as
    none, and sums past 31 bits stay there."""
    rng = np.random.default_rng(5)
    lens = np.array([30, 31, 32, -5, 15, 2 ** 31 - 1, 2 ** 31 - 1, 3, 64, 65])
    fresh = np.array([2, 1, 1, 4, 30, 1, 2 ** 31 - 1, -3, 1, 0])
    table, stack = _state(rng, np.clip(lens, 0, 64), 16, 4, 3)
    for rows in (0, 40, 2 ** 16):
        for count in (3, 1, 0, -2, 10 ** 6):
            _extend(gpu, ops, lens, fresh, table, stack, count, 16, rows)


def test_extend_of_nothing(gpu, ops):
    z = np.zeros
    for B, width, rows in ((0, 4, 0), (0, 0, 5), (3, 0, 4), (3, 2, 0)):
        _extend(gpu, ops, z(B), z(B), z((B, width)), z(6), 2, 16, rows)
    _extend(gpu, ops, [0, 0], [1, 0], z((2, 2)), z(0), 0, 16, 1)


def test_extend_keeps_pages_that_were_marked_missing(gpu, ops):
    """A page that is held but missing (-1) gives no slot."""
    table = np.array([[-1, 3, 0], [4, -1, 0]])
    got = _extend(gpu, ops, [5, 20], [3, 3], table, np.array([9, 8, 7]), 3, 16, 6)
    assert got[4].tolist() == [5, 6, 7, 20, 21, 22] and got[5].tolist() == [-1] * 6


RELEASES = [(256, 70, 16), (257, 70, 16), (1, 0, 16), (1, 100, 16), (64, 500, 16), (64, 33, 1), (1000, 300, 32), (1025, 90, 7), (3000, 40, 8), (3, 40000, 2)]


@pytest.mark.parametrize("B,ctx,page", RELEASES)
@pytest.mark.parametrize("dtype", ["bool", "uint8"])
def test_release(gpu, ops, B, ctx, page, dtype):
    rng = np.random.default_rng(B + ctx)
    lens = rng.integers(0, ctx + 1, B).astype(np.int32)
    lens[0] = ctx
    finished = rng.random(B) < 0.5
    finished[0] = True
    table, stack = _state(rng, lens, page, -(-ctx // page) + 1, 5)
    for count in (5, 0, len(stack) - 3, len(stack)):  # the last two: more than there is room for
        want = ref.release(finished, lens, table, stack, count, page)
        st = _dev(gpu, stack)
        got = ops.kv_cache_release(_dev(gpu, finished).to(getattr(gpu, dtype)), _dev(gpu, lens), _dev(gpu, table), st,
                                   _dev(gpu, np.array([count], np.int32)), page)
        for g, w in zip((*got, st), want):
            assert np.array_equal(g.cpu().numpy(), w)


def test_release_of_nothing(gpu, ops):
    i32 = dict(dtype=gpu.int32, device="cuda")
    for B, width, cap in ((0, 3, 4), (2, 0, 4), (2, 3, 0)):
        got = ops.kv_cache_release(gpu.ones(B, dtype=gpu.bool, device="cuda"), gpu.full((B,), -3, **i32),
                                   gpu.zeros(B, width, **i32), gpu.zeros(cap, **i32), gpu.zeros(1, **i32), 16)
        assert got[0].tolist() == [0] * B and got[1].tolist() == [0]


def test_views_and_streams(gpu, ops):
    """Inputs that are read may be views, on any stream."""
    rng = np.random.default_rng(3)
    lens, fresh = rng.integers(0, 90, 20), rng.integers(0, 5, 20)
    table, stack = _state(rng, lens, 16, 8, 30)
    rows = int(fresh.sum())
    want = ref.extend(lens, fresh, table, stack, 30, 16, rows)
    pair = _dev(gpu, np.stack([lens, fresh], 1).astype(np.int32))
    t, st = _dev(gpu, table), _dev(gpu, stack.repeat(2))[::2]
    gpu.cuda.synchronize()
    with gpu.cuda.stream(gpu.cuda.Stream()):
        got = ops.kv_cache_extend(pair[:, 0], pair[:, 1], t, st, gpu.full((1,), 30, dtype=gpu.int32, device="cuda"), 16,
                                  rows)
        got = [g.cpu().numpy() for g in (*got, t)]
    assert all(np.array_equal(g, w) for g, w in zip(got, want))


def test_two_pools_on_two_streams(gpu, ops):
    """Steps over tables of their own, at once: each as alone."""
    rng = np.random.default_rng(8)
    jobs = []
    for B in (300, 40):
        lens, fresh = rng.integers(0, 90, B), rng.integers(0, 5, B)
        table, stack = _state(rng, lens, 16, 8, B)
        rows = int(fresh.sum())
        want = ref.extend(lens, fresh, table, stack, B, 16, rows)
        jobs.append(([_dev(gpu, np.asarray(a, np.int32)) for a in (lens, fresh, table, stack, [B])], rows, want))
    streams = [gpu.cuda.Stream() for _ in jobs]
    gpu.cuda.synchronize()
    got = []
    for _ in range(6):
        for s, (args, rows, want) in zip(streams, jobs):
            with gpu.cuda.stream(s):
                got.append(((*ops.kv_cache_extend(*args, 16, rows), args[2]), want))
    gpu.cuda.synchronize()
    assert all(np.array_equal(g.cpu().numpy(), w) for gs, ws in got for g, w in zip(gs, ws))


def test_many_steps_in_a_graph(gpu, ops):
    """A step that extends, releases and feeds its results back, captured once
    and replayed, against the rules on the host; other eager work between."""
    rng = np.random.default_rng(11)
    B, page, width = 37, 4, 30
    lens = rng.integers(0, 30, B).astype(np.int32)
    table, stack = _state(rng, lens, page, width, 200)
    count = 200
    dev = [_dev(gpu, np.asarray(a, np.int32)) for a in (lens, np.ones(B), table, stack, [count])]
    done = gpu.zeros(B, dtype=gpu.bool, device="cuda")
    d_lens, d_new, d_table, d_stack, d_count = dev

    def step():
        out = ops.kv_cache_extend(d_lens, d_new, d_table, d_stack, d_count, page, 2 * B)
        d_lens.copy_(out[0])
        d_count.copy_(out[1])
        back = ops.kv_cache_release(done, d_lens, d_table, d_stack, d_count, page)
        d_lens.copy_(back[0])
        d_count.copy_(back[1])
        return out

    saved = [t.clone() for t in dev]
    side = gpu.cuda.Stream()
    side.wait_stream(gpu.cuda.current_stream())
    with gpu.cuda.stream(side):
        step()
    gpu.cuda.current_stream().wait_stream(side)
    graph = gpu.cuda.CUDAGraph()
    with gpu.cuda.graph(graph):
        out = step()
    for t, s in zip(dev, saved):
        t.copy_(s)
    for i in range(12):
        finished, fresh = rng.random(B) < 0.15, rng.integers(0, 3, B).astype(np.int32)
        done.copy_(_dev(gpu, finished))
        d_new.copy_(_dev(gpu, fresh))
        gpu.randn(1000, device="cuda").sum().item()
        graph.replay()
        gpu.cuda.synchronize()
        *want, table = ref.extend(lens, fresh, table, stack, count, page, 2 * B)
        assert all(np.array_equal(g.cpu().numpy(), w) for g, w in zip(out[2:], want[2:])), i
        lens, count, stack = ref.release(finished, want[0], table, stack, want[1][0], page)
        count = int(count[0])
        assert np.array_equal(d_lens.cpu().numpy(), lens) and int(d_count) == count
        assert np.array_equal(d_stack.cpu().numpy()[:count], stack[:count])
        # no page twice
        held = [table[b, :-(-int(n) // page)] for b, n in enumerate(lens)]
        pages = np.concatenate(held + [stack[:count]])
        assert len(np.unique(pages)) == len(pages) == sum(map(len, held)) + count
