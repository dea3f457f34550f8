"""What the MXFP4, head-norm and cache operators refuse before they launch
anything: the operators by ValueError, the C entries by their status.  No GPU is
touched (the pointers are never followed)."""
import ctypes

import pytest
import torch

import kc_abi
import kc_mxfp4 as ref
import kernel_craft_torch_ops as ops

U8, BF = torch.uint8, torch.bfloat16


def z(*shape, dtype=U8):
    return torch.zeros(*shape, dtype=dtype)


def _heads(T=3, H=2, D=64, dtype=BF):
    return z(T, H, D, dtype=dtype)


def _rope(q=None, k=None, qg=None, kg=None, cos=None, sin=None, pos=None):
    return (q if q is not None else _heads(H=4), k if k is not None else _heads(),
            qg if qg is not None else z(64, dtype=BF), kg if kg is not None else z(64, dtype=BF),
            cos if cos is not None else z(9, 32, dtype=torch.float32),
            sin if sin is not None else z(9, 32, dtype=torch.float32),
            pos if pos is not None else z(3, dtype=torch.int32))


def _pool(H=2, D=64, fmt="fp8"):
    if fmt == "fp8":
        return [z(4, 8, H, D, dtype=torch.int8), z(4, 8, H, dtype=torch.float32)] * 2
    return [z(4, 8, H, D // 2), z(4, 8, H, D // 32)] * 2


SLOTS = z(3, dtype=torch.int64)


@pytest.mark.parametrize("call,match", [
    (lambda: ops.mxfp4_quantize(z(4, 64, dtype=torch.float16)), "dtype"),
    (lambda: ops.mxfp4_quantize(z(4, 48, dtype=BF)), "multiple of 32"),
    (lambda: ops.mxfp4_quantize(z(64, dtype=BF)), "rows, K"),
    (lambda: ops.mxfp4_quantize(z(4, 64, dtype=BF)), "GPU only"),
    (lambda: ops.mxfp4_dequantize(z(4, 32), z(4, 1)), "K / 32"),
    (lambda: ops.mxfp4_dequantize(z(4, 32), z(3, 2)), "K / 32"),
    (lambda: ops.mxfp4_dequantize(z(4, 32), z(4, 2), out_dtype=torch.float16), "out_dtype"),
    (lambda: ops.mxfp4_dequantize(z(4, 32, dtype=torch.int8), z(4, 2)), "dtype"),
    (lambda: ops.mxfp4_dequantize(z(4, 32), z(4, 2)), "GPU only"),
    (lambda: ops.mxfp4_gemm_w4a4(z(4, 32), z(4, 2), z(4, 48), z(4, 3)), "K=64"),
    (lambda: ops.mxfp4_gemm_w4a4(z(4, 32), z(4, 2), z(4, 32), z(4, 1)), "K / 32"),
    (lambda: ops.mxfp4_gemm_w4a4(z(4, 32), z(4, 2), z(4, 32), z(4, 2), out_dtype=torch.float16), "out_dtype"),
    (lambda: ops.mxfp4_gemm_w4a4(z(4, 32), z(4, 2), z(4, 32), z(4, 2)), "GPU only"),
    (lambda: ops.mxfp4_gemm_bf16(z(4, 32), z(4, 2), z(2, 32, dtype=BF)), "M, 64"),
    (lambda: ops.mxfp4_gemm_bf16(z(4, 32), z(4, 2), z(2, 64, dtype=torch.float32)), "dtype"),
    (lambda: ops.mxfp4_gemm_bf16(z(4, 32), z(4, 2), z(2, 64, dtype=BF)), "GPU only"),
    (lambda: ops.qk_norm_rope(*_rope(q=z(3, 4, 64, dtype=torch.float16))), "dtype"),
    (lambda: ops.qk_norm_rope(*_rope(q=z(3, 256, dtype=BF))), "tokens, heads"),
    (lambda: ops.qk_norm_rope(*_rope(k=_heads(dtype=torch.float32))), "dtype"),
    (lambda: ops.qk_norm_rope(*_rope(k=_heads(T=2))), "tokens, heads"),
    (lambda: ops.qk_norm_rope(*_rope(k=_heads(D=32))), "tokens, heads"),
    (lambda: ops.qk_norm_rope(*_rope(qg=z(32, dtype=BF))), "gamma"),
    (lambda: ops.qk_norm_rope(*_rope(kg=z(64, dtype=torch.float32))), "dtype"),
    (lambda: ops.qk_norm_rope(*_rope(cos=z(9, 16, dtype=torch.float32))), "rotary_dim"),
    (lambda: ops.qk_norm_rope(*_rope(cos=z(9, 33, dtype=torch.float32), sin=z(9, 33, dtype=torch.float32))),
     "rotary_dim"),
    (lambda: ops.qk_norm_rope(*_rope(pos=z(3, dtype=torch.int64))), "dtype"),
    (lambda: ops.qk_norm_rope(*_rope(pos=z(2, dtype=torch.int32))), "positions"),
    (lambda: ops.qk_norm_rope(*_rope()), "GPU only"),
    (lambda: ops.kv_cache_write(_heads(), _heads(), z(2, dtype=torch.int64), *_pool()), "slots"),
    (lambda: ops.kv_cache_write(_heads(), _heads(), z(3, dtype=torch.int32), *_pool()), "dtype"),
    (lambda: ops.kv_cache_write(_heads(), _heads(H=1), SLOTS, *_pool()), "tokens, heads"),
    (lambda: ops.kv_cache_write(_heads(), _heads(dtype=torch.float32), SLOTS, *_pool()), "dtype"),
    (lambda: ops.kv_cache_write(_heads(D=32), _heads(D=32), SLOTS, *_pool()), "tokens, heads"),
    (lambda: ops.kv_cache_write(_heads(), _heads(), SLOTS, *_pool()[:3], z(4, 8, 1, dtype=torch.float32)), "scales"),
    (lambda: ops.kv_cache_write(_heads(), _heads(), SLOTS, *_pool()[:2], *_pool(fmt="mxfp4")[2:]), "dtype"),
    (lambda: ops.kv_cache_write(_heads(D=48), _heads(D=48), SLOTS, *[z(4, 8, 2, 24), z(4, 8, 2, 1)] * 2), "scales"),
    (lambda: ops.kv_cache_write(_heads(), _heads(), SLOTS, _pool()[0].transpose(0, 1), *_pool()[1:]), "contiguous"),
    (lambda: ops.kv_cache_write(_heads(), _heads(), SLOTS, *_pool()), "GPU only"),
    (lambda: ops.qk_norm_rope_cache(*_rope()[:2], _heads(), *_rope()[2:], SLOTS, *_pool(D=32)), "head_dim"),
    (lambda: ops.qk_norm_rope_cache(*_rope()[:2], _heads(H=1), *_rope()[2:], SLOTS, *_pool()), "tokens, heads"),
    (lambda: ops.qk_norm_rope_cache(*_rope()[:2], _heads(), *_rope()[2:], SLOTS[:2], *_pool()), "slots"),
    (lambda: ops.qk_norm_rope_cache(*_rope()[:2], _heads(), *_rope()[2:], SLOTS, *_pool()), "GPU only"),
    (lambda: ops.kv_cache_read(*_pool(), z(2, 3, dtype=torch.int32), z(2, dtype=torch.int32), 4), "cu_seqlens"),
    (lambda: ops.kv_cache_read(*_pool(), z(2, 3, dtype=torch.int64), z(3, dtype=torch.int32), 4), "dtype"),
    (lambda: ops.kv_cache_read(*_pool(), z(2, 3, dtype=torch.int32), z(3, dtype=torch.int32), -1), "negative"),
    (lambda: ops.kv_cache_read(*_pool(), z(2, 3, dtype=torch.int32), z(3, dtype=torch.int32), 4,
                               out_dtype=torch.float16), "out_dtype"),
    (lambda: ops.kv_cache_read(*_pool(), z(2, 3, dtype=torch.int32), z(3, dtype=torch.int32), 4), "GPU only"),
])
def test_operators_refuse(call, match):
    with pytest.raises(ValueError, match=match):
        call()


P = ctypes.c_void_p(0x1000)
ODD = ctypes.c_void_p(0x1008)


def _cache(**kw):
    a = dict(k_codes=0x1000, k_scales=0x1000, v_codes=0x1000, v_scales=0x1000, num_pages=4, page_size=16, kv_heads=2,
             head_dim=64, format=0)
    a.update(kw)
    return ctypes.byref(ops.KvCache(**a))


def _rp(**kw):
    a = dict(cos_table=0x1000, sin_table=0x1000, positions=0x1000, table_rows=8, rotary_dim=64, interleaved=0)
    a.update(kw)
    return ctypes.byref(ops.Rope(**a))


@pytest.mark.parametrize("call,why", [
    (lambda L: L.kc_quantize_mxfp4_bf16(P, P, P, 4, 48, None), "multiple of 32"),
    (lambda L: L.kc_quantize_mxfp4_f32(P, P, P, -1, 64, None), "negative"),
    (lambda L: L.kc_quantize_mxfp4_f32(P, None, P, 1, 64, None), "null"),
    (lambda L: L.kc_quantize_mxfp4_f32(P, P, P, 1 << 60, 64, None), "too large"),
    (lambda L: L.kc_quantize_mxfp4_bf16(P, ctypes.c_void_p(0x1002), P, 1, 64, None), "aligned"),
    (lambda L: L.kc_dequantize_mxfp4_bf16(P, P, None, 1, 64, None), "null"),
    (lambda L: L.kc_dequantize_mxfp4_f32(P, P, P, 1, 33, None), "multiple of 32"),
    (lambda L: L.kc_gemm_mxfp4_w4a4_bf16(P, P, P, P, P, 4, 4, 48, None), "multiple of 32"),
    (lambda L: L.kc_gemm_mxfp4_w4a4_f32(P, P, P, P, None, 4, 4, 64, None), "null"),
    (lambda L: L.kc_gemm_mxfp4_w4a4_f32(P, None, P, P, P, 4, 4, 64, None), "null"),
    (lambda L: L.kc_gemm_mxfp4_w4a4_bf16(ODD, P, P, P, P, 4, 4, 64, None), "aligned"),
    (lambda L: L.kc_gemm_mxfp4_w4a4_bf16(P, P, P, P, P, -4, 4, 64, None), "negative"),
    (lambda L: L.kc_gemm_mxfp4_w4a4_bf16(P, P, P, P, P, 1 << 40, 1 << 40, 64, None), "too large"),
    (lambda L: L.kc_gemm_mxfp4_bf16(P, P, P, P, 4, 4, 16, None), "multiple of 32"),
    (lambda L: L.kc_gemm_mxfp4_bf16(P, P, ODD, P, 4, 4, 64, None), "aligned"),
    (lambda L: L.kc_gemm_mxfp4_bf16(P, P, P, None, 4, 4, 64, None), "null"),
    (lambda L: L.kc_gemm_mxfp4_bf16(P, P, P, P, 1 << 21, 4, 64, None), "too large"),
    (lambda L: L.kc_gemm_mxfp4_bf16(P, P, P, P, 4, 4, 1 << 25, None), "too large"),
    (lambda L: L.kc_gemm_mxfp4_w4a4_f32(P, P, P, P, P, 4, 1 << 29, 64, None), "too large"),
    (lambda L: L.kc_qk_norm_rope_bf16(P, 256, P, 256, P, P, None, 1e-6, 3, 2, 2, 64, P, P, None), "null rope"),
    (lambda L: L.kc_qk_norm_rope_bf16(P, 256, P, 256, P, P, _rp(rotary_dim=66), 1e-6, 3, 2, 2, 64, P, P, None),
     "rotary_dim"),
    (lambda L: L.kc_qk_norm_rope_bf16(P, 256, P, 256, P, P, _rp(rotary_dim=3), 1e-6, 3, 2, 2, 64, P, P, None),
     "rotary_dim"),
    (lambda L: L.kc_qk_norm_rope_bf16(P, 256, P, 256, P, P, _rp(positions=None), 1e-6, 3, 2, 2, 64, P, P, None),
     "null"),
    (lambda L: L.kc_qk_norm_rope_f32(P, 256, None, 256, P, P, _rp(), 1e-6, 3, 2, 2, 64, P, P, None), "null"),
    (lambda L: L.kc_qk_norm_rope_f32(P, 256, P, 256, P, P, _rp(), 1e-6, 3, 2, 2, 1025, P, P, None), "head_dim"),
    (lambda L: L.kc_qk_norm_rope_f32(P, 256, P, 256, P, P, _rp(), 1e-6, -3, 2, 2, 64, P, P, None), "negative"),
    (lambda L: L.kc_kv_cache_write_bf16(P, 128, P, 128, P, 3, None, None), "null cache"),
    (lambda L: L.kc_kv_cache_write_bf16(P, 128, P, 128, P, 3, _cache(format=7), None), "format"),
    (lambda L: L.kc_kv_cache_write_bf16(P, 128, P, 128, P, 3, _cache(head_dim=48, format=1), None), "multiple of 32"),
    (lambda L: L.kc_kv_cache_write_bf16(P, 128, P, 128, P, 3, _cache(head_dim=2048), None), "head_dim"),
    (lambda L: L.kc_kv_cache_write_bf16(P, 128, P, 128, P, 3, _cache(page_size=0), None), "shape"),
    (lambda L: L.kc_kv_cache_write_bf16(P, 128, P, 128, None, 3, _cache(), None), "null"),
    (lambda L: L.kc_kv_cache_write_f32(P, 128, P, 128, P, -1, _cache(), None), "negative"),
    (lambda L: L.kc_kv_cache_write_f32(P, 128, P, 128, P, 3, _cache(k_codes=None), None), "null cache pointer"),
    (lambda L: L.kc_qk_norm_rope_cache_bf16(P, 256, P, 128, None, 128, P, P, _rp(), 1e-6, 3, 2, P, _cache(), P, None),
     "null"),
    (lambda L: L.kc_qk_norm_rope_cache_f32(P, 256, P, 128, P, 128, P, P, _rp(rotary_dim=128), 1e-6, 3, 2, P, _cache(),
                                           P, None), "rotary_dim"),
    (lambda L: L.kc_kv_cache_read_bf16(_cache(), P, -1, P, 2, 9, P, P, None), "negative"),
    (lambda L: L.kc_kv_cache_read_bf16(_cache(), None, 2, P, 2, 9, P, P, None), "null"),
    (lambda L: L.kc_kv_cache_read_f32(_cache(), P, 2, P, 2, 9, P, None, None), "null"),
])
def test_entries_refuse(call, why):
    L = kc_abi.lib()
    L.kc_get_last_error()
    assert call(L) == 1
    assert why in L.kc_last_error_string().decode()
    assert L.kc_get_last_error() == 1


def test_nothing_to_do_succeeds():
    """Empty calls return before any GPU call."""
    L = kc_abi.lib()
    L.kc_get_last_error()
    assert L.kc_quantize_mxfp4_bf16(None, None, None, 0, 64, None) == 0
    assert L.kc_quantize_mxfp4_f32(None, None, None, 5, 0, None) == 0
    assert L.kc_gemm_mxfp4_w4a4_bf16(None, None, None, None, None, 0, 8, 64, None) == 0
    assert L.kc_gemm_mxfp4_bf16(None, None, None, None, 8, 0, 64, None) == 0
    assert L.kc_kv_cache_write_bf16(None, 0, None, 0, None, 0, _cache(), None) == 0
    assert L.kc_kv_cache_read_bf16(_cache(), None, 0, None, 0, 9, None, None, None) == 0
    assert L.kc_qk_norm_rope_bf16(None, 0, None, 0, None, None, _rp(), 1e-6, 0, 2, 2, 64, None, None, None) == 0
    assert L.kc_get_last_error() == 0


def test_plain_forms_agree():
    """The tests' restatement of the format against its definition by hand."""
    import numpy as np
    x = np.zeros((1, 64))
    x[0, :8] = [7.9, 6, 5, 4.99, 2.5, 1.75, -0.25, -0.26]
    x[0, 32:36] = [0.001, -0.0007, 0.00025, 0]
    codes, scales = ref.quantize(x)
    assert list(scales[0]) == [127, 115]      # 7.9 -> 2^2 - 2 = 0; 0.001 -> 2^-10 - 2 = -12
    v = ref.values(codes, scales)[0]
    assert list(v[:8]) == [6, 6, 4, 4, 2, 2, 0, -0.5]
    assert list(v[32:36] * 2 ** 12) == [4, -3, 1, 0]
    x[0, 40] = np.nan
    codes, scales = ref.quantize(x)
    assert list(scales[0]) == [127, 255] and not codes[0, 16:].any()


@pytest.mark.parametrize("call,why", [
    (lambda L: L.kc_gemm_mxfp4_bf16(P, P, P, P, 1048561, 4, 64, None), "at most 1048560"),
    (lambda L: L.kc_gemm_mxfp4_bf16(P, P, P, P, 16, (1 << 28) + 1, 64, None), "too large"),
    (lambda L: L.kc_gemm_mxfp4_w4a4_bf16(P, P, P, P, P, 16 << 13, (16 << 13) + 1, 64, None), "too large"),
    (lambda L: L.kc_gemm_mxfp4_w4a4_f32(P, P, P, P, P, 4, 4, (1 << 24) + 32, None), "too large"),
])
def test_products_refuse_what_is_just_past_their_limits(call, why):
    """The limits that the header names."""
    L = kc_abi.lib()
    L.kc_get_last_error()
    assert call(L) == 1
    assert why in L.kc_last_error_string().decode()
    assert L.kc_get_last_error() == 1
