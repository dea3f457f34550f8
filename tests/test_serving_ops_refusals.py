"""What the page, attention and residual operators refuse before they launch
anything: the operators by ValueError, the C entries by their status.  No GPU is
touched (the pointers are never followed)."""
import ctypes

import pytest
import torch

import kc_abi
import kernel_craft_torch_ops as ops

BF, F32, I32 = torch.bfloat16, torch.float32, torch.int32


def z(*shape, dtype=I32):
    return torch.zeros(*shape, dtype=dtype)


def _pool(H=2, D=64, fmt="fp8"):
    if fmt == "fp8":
        return [z(4, 8, H, D, dtype=torch.int8), z(4, 8, H, dtype=F32)] * 2
    return [z(4, 8, H, D // 2, dtype=torch.uint8), z(4, 8, H, D // 32, dtype=torch.uint8)] * 2


def _attend(q=None, pool=None, table=None, lens=None, **kw):
    return ops.kv_cache_attention(z(3, 4, 64, dtype=BF) if q is None else q, *(pool or _pool()),
                                  z(3, 5) if table is None else table, z(3) if lens is None else lens, **kw)


def _extend(lens=None, new=None, table=None, free=None, count=None, page=16, total=3):
    return ops.kv_cache_extend(z(3) if lens is None else lens, z(3) if new is None else new,
                               z(3, 5) if table is None else table, z(9) if free is None else free,
                               z(1) if count is None else count, page, total)


def _release(done=None, lens=None, table=None, free=None, count=None, page=16):
    return ops.kv_cache_release(z(3, dtype=torch.bool) if done is None else done, z(3) if lens is None else lens,
                                z(3, 5) if table is None else table, z(9) if free is None else free,
                                z(1) if count is None else count, page)


def _residual(y=None, h=None, gamma=None, **kw):
    a = (z(3, 64, dtype=BF) if y is None else y, z(3, 64, dtype=BF) if h is None else h,
         z(64, dtype=BF) if gamma is None else gamma)
    with pytest.raises(ValueError) as one:
        ops.residual_rmsnorm(*a, **kw)
    with pytest.raises(ValueError) as two:
        ops.residual_rmsnorm_fp8_quantize(*a, **kw)
    assert str(one.value).split(":")[1] == str(two.value).split(":")[1]
    raise one.value


@pytest.mark.parametrize("call,match", [
    (lambda: _attend(q=z(3, 4, 64, dtype=torch.float16)), "dtype"),
    (lambda: _attend(q=z(3, 256, dtype=BF)), "tokens, heads"),
    (lambda: _attend(q=z(3, 4, 32, dtype=BF)), "tokens, heads"),
    (lambda: _attend(q=z(3, 5, 64, dtype=BF)), "multiple"),
    (lambda: _attend(q=z(2, 4, 64, dtype=BF)), "block_table"),
    (lambda: _attend(table=z(3, 5, dtype=torch.int64)), "dtype"),
    (lambda: _attend(table=z(15)), "block_table"),
    (lambda: _attend(lens=z(3, dtype=torch.int64)), "dtype"),
    (lambda: _attend(lens=z(4)), "seq_lens"),
    (lambda: _attend(window=-1), "window"),
    (lambda: _attend(pool=_pool()[:2] + _pool(fmt="mxfp4")[2:]), "dtype"),
    (lambda: _attend(pool=[_pool()[0].transpose(0, 1)] + _pool()[1:]), "contiguous"),
    (lambda: _attend(), "GPU only"),
    (lambda: _attend(pool=_pool(fmt="mxfp4")), "GPU only"),
    (lambda: _extend(lens=z(3, dtype=torch.int64)), "dtype"),
    (lambda: _extend(lens=z(2)), "block_table"),
    (lambda: _extend(new=z(2)), "new_lens"),
    (lambda: _extend(new=z(3, dtype=torch.int64)), "dtype"),
    (lambda: _extend(table=z(15)), "block_table"),
    (lambda: _extend(table=z(5, 3).t()), "contiguous"),
    (lambda: _extend(free=z(3, 3)), "free_pages"),
    (lambda: _extend(free=z(9, dtype=torch.int64)), "dtype"),
    (lambda: _extend(count=z(2)), "free_count"),
    (lambda: _extend(count=z(1, dtype=torch.int64)), "dtype"),
    (lambda: _extend(page=0), "page_size"),
    (lambda: _extend(page=2 ** 32 + 16), "page_size"),
    (lambda: _release(page=2 ** 31), "page_size"),
    (lambda: _extend(total=-1), "total_new"),
    (lambda: _extend(total=2 ** 31), "total_new"),
    (lambda: _extend(), "GPU only"),
    (lambda: _release(done=z(3)), "dtype"),
    (lambda: _release(done=z(2, dtype=torch.bool)), "finished"),
    (lambda: _release(free=z(18)[::2]), "contiguous"),
    (lambda: _release(lens=z(4)), "block_table"),
    (lambda: _release(page=-1), "page_size"),
    (lambda: _release(), "GPU only"),
    (lambda: _residual(y=z(3, 64, dtype=torch.float16)), "dtype"),
    (lambda: _residual(h=z(3, 64, dtype=torch.float16)), "dtype"),
    (lambda: _residual(y=z(3, 64, dtype=F32), gamma=z(64, dtype=F32)), "dtype"),
    (lambda: _residual(h=z(2, 64, dtype=BF)), "rows, cols"),
    (lambda: _residual(y=z(64, dtype=BF), h=z(64, dtype=BF)), "rows, cols"),
    (lambda: _residual(gamma=z(64, dtype=F32)), "dtype"),
    (lambda: _residual(gamma=z(63, dtype=BF)), "gamma"),
    (lambda: _residual(post_gamma=z(1, 64, dtype=BF)), "gamma"),
    (lambda: _residual(post_gamma=z(64, dtype=F32)), "dtype"),
    (lambda: _residual(gate=z(64, dtype=F32)), "dtype"),
    (lambda: _residual(gate=z(3, 1, dtype=BF)), "gate"),
    (lambda: _residual(gate=z(2, 64, dtype=BF)), "gate"),
    (lambda: _residual(), "GPU only"),
])
def test_operators_refuse(call, match):
    with pytest.raises(ValueError, match=match):
        call()


@pytest.mark.parametrize("heads", [0, 4])
@pytest.mark.parametrize("fmt", ["fp8", "mxfp4"])
def test_a_cache_without_heads(fmt, heads):
    with pytest.raises(ValueError, match="multiple"):
        _attend(q=z(3, heads, 64, dtype=BF), pool=_pool(H=0, fmt=fmt))


P = ctypes.c_void_p(0x1000)
ODD = ctypes.c_void_p(0x1008)


def _cache(**kw):
    a = dict(k_codes=0x1000, k_scales=0x1000, v_codes=0x1000, v_scales=0x1000, num_pages=4, page_size=16, kv_heads=2,
             head_dim=64, format=0)
    a.update(kw)
    return ctypes.byref(ops.KvCache(**a))


def _call(L, cache=None, q=P, heads=8, table=P, pages=20, lens=P, seqs=3, window=0, work=P, size=1 << 40, out=P):
    return L.kc_kv_cache_attention_bf16(q, 512, heads, cache or _cache(), table, pages, lens, seqs, 1.0, window, work,
                                        size, out, None)


def _pages(**kw):
    a = dict(block_table=0x1000, free_pages=0x1000, free_count=0x1000, max_pages=5, num_pages=9, page_size=16, seqs=3)
    a.update(kw)
    return ctypes.byref(ops.KvPages(**a))


def _res(**kw):
    a = dict(y=0x1000, h=0x1000, gate=None, post_gamma=None, gamma=0x1000, y_stride=64, h_stride=64, gate_stride=0,
             rows=3, cols=64, alpha=1.0, eps=1e-6)
    a.update(kw)
    return ctypes.byref(ops.Residual(**a))


@pytest.mark.parametrize("call,why", [
    (lambda L: _call(L, heads=7), "multiple"),
    (lambda L: _call(L, heads=-2), "negative"),
    (lambda L: _call(L, pages=-1), "negative"),
    (lambda L: _call(L, seqs=-1), "negative"),
    (lambda L: _call(L, window=-1), "window"),
    (lambda L: _call(L, seqs=1 << 22), "too large"),
    (lambda L: _call(L, heads=1 << 16), "too large"),
    (lambda L: _call(L, pages=1 << 31), "too large"),
    (lambda L: _call(L, pages=1 << 27, seqs=17), "too large"),
    (lambda L: _call(L, pages=(1 << 31) - 1, seqs=17), "too large"),
    (lambda L: _call(L, cache=_cache(num_pages=1 << 28)), "slots"),
    (lambda L: _call(L, cache=_cache(head_dim=1025)), "1024"),
    (lambda L: _call(L, cache=_cache(head_dim=48, format=1)), "multiple of 32"),
    (lambda L: _call(L, cache=_cache(format=2)), "format"),
    (lambda L: _call(L, cache=_cache(v_scales=None)), "null"),
    (lambda L: _call(L, q=None), "null"),
    (lambda L: _call(L, table=None), "null"),
    (lambda L: _call(L, lens=None), "null"),
    (lambda L: _call(L, out=None), "null"),
    (lambda L: _call(L, pages=200, size=100), "workspace"),
    (lambda L: _call(L, pages=200, work=None), "workspace"),
    (lambda L: _call(L, pages=200, work=ODD), "workspace"),
    (lambda L: L.kc_kv_cache_attention_f32(P, 512, 8, None, P, 20, P, 3, 1.0, 0, P, 1 << 40, P, None), "null"),
    (lambda L: L.kc_kv_cache_extend(None, P, P, 3, P, P, P, P, P, P, None), "null"),
    (lambda L: L.kc_kv_cache_extend(_pages(page_size=0), P, P, 3, P, P, P, P, P, P, None), "shape"),
    (lambda L: L.kc_kv_cache_extend(_pages(seqs=-1), P, P, 3, P, P, P, P, P, P, None), "shape"),
    (lambda L: L.kc_kv_cache_extend(_pages(max_pages=-1), P, P, 3, P, P, P, P, P, P, None), "shape"),
    (lambda L: L.kc_kv_cache_extend(_pages(num_pages=1 << 31), P, P, 3, P, P, P, P, P, P, None), "too large"),
    (lambda L: L.kc_kv_cache_extend(_pages(seqs=(1 << 20) + 1), P, P, 3, P, P, P, P, P, P, None), "too large"),
    (lambda L: L.kc_kv_cache_extend(_pages(), P, P, -1, P, P, P, P, P, P, None), "total_new"),
    (lambda L: L.kc_kv_cache_extend(_pages(), P, P, 1 << 31, P, P, P, P, P, P, None), "total_new"),
    (lambda L: L.kc_kv_cache_extend(_pages(block_table=None), P, P, 3, P, P, P, P, P, P, None), "null"),
    (lambda L: L.kc_kv_cache_extend(_pages(free_pages=None), P, P, 3, P, P, P, P, P, P, None), "null"),
    (lambda L: L.kc_kv_cache_extend(_pages(free_count=None), P, P, 3, P, P, P, P, P, P, None), "null"),
    *[(lambda L, i=i: L.kc_kv_cache_extend(_pages(), *[None if i == j else P for j in range(2)], 3,
                                           *[None if i == j else P for j in range(2, 8)], None), "null") for i in range(8)],
    *[(lambda L, i=i: L.kc_kv_cache_release(_pages(), *[None if i == j else P for j in range(4)], None), "null")
      for i in range(4)],
    (lambda L: L.kc_kv_cache_release(_pages(page_size=-4), P, P, P, P, None), "shape"),
    (lambda L: L.kc_residual_rmsnorm_bf16(None, P, P, None), "null"),
    (lambda L: L.kc_residual_rmsnorm_bf16(_res(y=None), P, P, None), "null"),
    (lambda L: L.kc_residual_rmsnorm_f32(_res(h=None), P, P, None), "null"),
    (lambda L: L.kc_residual_rmsnorm_bf16_f32(_res(gamma=None), P, P, None), "null"),
    (lambda L: L.kc_residual_rmsnorm_bf16(_res(), None, P, None), "null"),
    (lambda L: L.kc_residual_rmsnorm_bf16(_res(), P, None, None), "null"),
    (lambda L: L.kc_residual_rmsnorm_quantize_fp8_bf16(_res(), P, P, None, None), "null"),
    (lambda L: L.kc_residual_rmsnorm_quantize_fp8_f32(_res(rows=-1), P, P, P, None), "negative"),
    (lambda L: L.kc_residual_rmsnorm_quantize_fp8_bf16_f32(_res(cols=-1), P, P, P, None), "negative"),
    (lambda L: L.kc_residual_rmsnorm_bf16(_res(cols=32769), P, P, None), "32768"),
])
def test_entries_refuse(call, why):
    L = kc_abi.lib()
    L.kc_get_last_error()
    assert call(L) == 1
    assert why in L.kc_last_error_string().decode()
    assert L.kc_get_last_error() == 1


def test_empty_calls_are_noops():
    L = kc_abi.lib()
    assert _call(L, seqs=0, q=None, lens=None, out=None, table=None, work=None, size=0) == 0
    assert _call(L, heads=0) == 0
    assert L.kc_residual_rmsnorm_bf16(_res(rows=0, y=None), None, None, None) == 0
    assert L.kc_residual_rmsnorm_quantize_fp8_f32(_res(cols=0, y=None), None, None, None, None) == 0
    assert L.kc_get_last_error() == 0


def test_workspace_of_refused_calls():
    L = kc_abi.lib()
    assert L.kc_kv_cache_attention_workspace(_cache(), 20, 3, 7) == -1 and L.kc_get_last_error() == 1
    assert L.kc_kv_cache_attention_workspace(_cache(), 20, 0, 8) == 0
    assert L.kc_kv_cache_attention_workspace(_cache(), 20, 3, 8) == 0  # short tables are not split
    assert L.kc_kv_cache_attention_workspace(_cache(), 200, 3, 8) > 0
