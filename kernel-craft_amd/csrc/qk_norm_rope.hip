// qk_norm_rope.hip -- the heads of a fused QKV projection on gfx950: RMSNorm of
// each query and key head, the rotation by the token's position, and the
// quantization of keys and values as they are written into a paged cache.  No
// counterpart in the reference, whose RMSNorm takes whole rows
// (rmsnorm.cu:40-70) and whose caches are fp32 (paged_attention.cu:135-142).
//
// Per head x of D values:
//   y_i = (gamma_i * x_i) * rms_inv,  rms_inv = 1 / sqrtf(sum x^2 / D + eps)
//   (a, b) -> (a c - b s, b c + a s) for the pairs of the first R values,
//   paired (i, i + R/2) or, interleaved, (2i, 2i + 1); c, s from the token's row
//   of the fp32 tables
// in fp32, rounded to the output type once.  A cached row is the quantization of
// that rounded key, and of the value as it is:
//   FP8    one fp32 scale per token and head and E4M3 codes, as the per-token
//          quantizer (fp8_quant.hip) gives them for a row of D values
//   MXFP4  blocks of 32 along D (mxfp4.hpp)
//
// Everything here is bound by memory: a head goes in once and out once.
//
// Vector kernel.  A slot is 8 values (16 bytes of bf16).  Lane j of the
// lanes that share a head takes two slots: those of its rotation pairs, j and
// j + R/16 (interleaved and past R: 2j and 2j + 1), so that both partners of
// every pair are in one lane and no value crosses lanes but in the sum of
// squares.  D = 128 needs 8 lanes: a wave holds 8 heads of one token at a time
// and keeps the token's 8 cos and sin per lane in registers over its heads.
//
// The sum of squares runs over the lane's first slot, then its second, one FMA
// a value, then over the lanes (xor butterfly).  The general kernel (any D up to
// 1024, strides and alignment; one wave per head, the row in LDS) adds in the
// same order where the slots exist, so both give the same bits.
#include <algorithm>
#include <type_traits>

#include "kv_cache.hpp"

namespace {

using kc::kWave;
using namespace kc::mx;
using kc::fp8::RowDiv;

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;

template <bool BF16>
using Elem = std::conditional_t<BF16, uint16_t, float>;

enum Sink { kPlain, kFp8, kMx };

struct Args {
    const void *q, *k, *v;            // heads of a token are D apart
    int64_t q_stride, k_stride, v_stride;
    const void *q_gamma, *k_gamma;
    const float *cos_t, *sin_t;       // [table_rows, R / 2]
    const int32_t* positions;
    const int64_t* slots;
    void *q_out, *k_out;
    uint8_t *k_codes, *v_codes;
    void *k_scales, *v_scales;
    int64_t tokens, table_rows, n_slots;
    int q_heads, kv_heads, D, R;
    float eps;
    bool interleaved;
    int lanes_log2;                   // lanes of a head
    int groups, splits, per_split;    // waves of a token and the head groups of each
};

// 8 values of a row, as fp32.
template <bool BF16>
__device__ __forceinline__ void load8(const void* base, int64_t at, float (&v)[8]) {
    if constexpr (BF16) {
        const u32x4 d = *reinterpret_cast<const u32x4*>(static_cast<const uint16_t*>(base) + at);
        const uint32_t w[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        }
    } else {
        const f32x4* p = reinterpret_cast<const f32x4*>(static_cast<const float*>(base) + at);
        const f32x4 a = p[0], b = p[1];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[i] = a[i];
            v[4 + i] = b[i];
        }
    }
}

template <bool BF16>
__device__ __forceinline__ void store8(void* base, int64_t at, const float (&v)[8]) {
    if constexpr (BF16) {
        u32x4 d;
        d.x = kc::pack_bf16x2(v[0], v[1]);
        d.y = kc::pack_bf16x2(v[2], v[3]);
        d.z = kc::pack_bf16x2(v[4], v[5]);
        d.w = kc::pack_bf16x2(v[6], v[7]);
        *reinterpret_cast<u32x4*>(static_cast<uint16_t*>(base) + at) = d;
    } else {
        f32x4* p = reinterpret_cast<f32x4*>(static_cast<float*>(base) + at);
        p[0] = f32x4{v[0], v[1], v[2], v[3]};
        p[1] = f32x4{v[4], v[5], v[6], v[7]};
    }
}

template <bool BF16>
__device__ __forceinline__ float rounded(float v) {
    if constexpr (BF16) return kc::bf16_to_f32(kc::f32_to_bf16(v));
    else return v;
}

__device__ __forceinline__ float rms_inverse(float ss, int D, float eps) {
    return 1.0f / sqrtf(ss / static_cast<float>(D) + eps);
}

__device__ __forceinline__ void rotate(float& a, float& b, float c, float s) {
    const float ra = fmaf(a, c, -(b * s)), rb = fmaf(b, c, a * s);
    a = ra;
    b = rb;
}

// What becomes of a token: its position's row of the tables, or the row
// that it writes in place of a rotation.
struct Token {
    bool in_table, cached;
    int64_t row, slot;
    float fill;  // of q and k where the position is not in the table
};

template <bool NORM, int SINK>
__device__ __forceinline__ Token token_of(const Args& p, int64_t t) {
    Token k{true, false, 0, 0, 0.0f};
    if constexpr (NORM) {
        const int32_t pos = p.positions[t];
        k.in_table = pos >= 0 && pos < p.table_rows;
        k.fill = pos < 0 ? 0.0f : __uint_as_float(0x7FC00000u);
        k.row = k.in_table ? pos : 0;
    }
    if constexpr (SINK != kPlain) {
        const int64_t s = p.slots[t];
        k.cached = k.in_table && s >= 0 && s < p.n_slots;
        k.slot = k.cached ? s : 0;
    }
    return k;
}

// 8 values -> 8 E4M3 codes.
template <bool FAST>
__device__ __forceinline__ u32x2 fp8_codes(const float (&v)[8], const RowDiv& d) {
    using kc::fp8::e4m3x4_div;
    return u32x2{e4m3x4_div<FAST>(kc::fp8::f32x4{v[0], v[1], v[2], v[3]}, d),
                 e4m3x4_div<FAST>(kc::fp8::f32x4{v[4], v[5], v[6], v[7]}, d)};
}

__device__ __forceinline__ uint32_t absmax_bits8(const float (&v)[8]) {
    return absmax_bits_f32(f32x4{v[0], v[1], v[2], v[3]}, f32x4{v[4], v[5], v[6], v[7]});
}

__device__ __forceinline__ uint32_t mx_codes(const float (&v)[8], uint32_t b) {
    return b == kNaN ? 0u : encode8_f32(f32x4{v[0], v[1], v[2], v[3]}, f32x4{v[4], v[5], v[6], v[7]}, b);
}

template <bool BF16, bool NORM, int SINK>
__global__ __launch_bounds__(kThreads) void heads_kernel(const Args p) {
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t w = static_cast<int64_t>(blockIdx.x) * kWaves + (threadIdx.x >> 6);
    const int64_t t = w / p.splits;
    if (t >= p.tokens) return;
    const int part = static_cast<int>(w - t * p.splits);
    const int D = p.D, half = p.R >> 4;  // slots of half a rotation
    const int lg = p.lanes_log2, hp = kWave >> lg, j = lane & ((1 << lg) - 1);
    const Token tok = token_of<NORM, SINK>(p, t);
    const int n_q = NORM ? p.q_heads : 0, n_all = n_q + p.kv_heads + (SINK != kPlain ? p.kv_heads : 0);
    const bool has = j < (D >> 4);

    float c[8] = {}, s[8] = {};
    if constexpr (NORM) {
        if (has && j < half && tok.in_table) {
            load8<false>(p.cos_t, tok.row * (p.R >> 1) + 8 * j, c);
            load8<false>(p.sin_t, tok.row * (p.R >> 1) + 8 * j, s);
        }
    }
    const int g_end = min(p.groups, (part + 1) * p.per_split);
    for (int g = part * p.per_split; g < g_end; ++g) {
        const int h = g * hp + (lane >> lg);
        const bool live = has && h < n_all;
        const bool is_q = h < n_q, is_v = SINK != kPlain && h >= n_q + p.kv_heads;
        const int hh = is_q ? h : is_v ? h - n_q - p.kv_heads : h - n_q;
        const bool turns = NORM && !is_v && j < half;
        const bool apart = turns && !p.interleaved;  // slots j and j + half
        const int sa = apart ? j : 2 * j, sb = apart ? j + half : 2 * j + 1;
        const void* src = is_q ? p.q : is_v ? p.v : p.k;
        const int64_t at = t * (is_q ? p.q_stride : is_v ? p.v_stride : p.k_stride) + static_cast<int64_t>(hh) * D;
        float a[8], b[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) a[i] = b[i] = 0.0f;
        if (live) {
            load8<BF16>(src, at + 8 * sa, a);
            load8<BF16>(src, at + 8 * sb, b);
        }
        if constexpr (NORM) {
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = fmaf(a[i], a[i], ss);
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = fmaf(b[i], b[i], ss);
            for (int off = (1 << lg) >> 1; off >= 1; off >>= 1) ss += __shfl_xor(ss, off, kWave);
            const float inv = rms_inverse(ss, D, p.eps);
            if (live && !is_v) {
                float ga[8], gb[8];
                load8<BF16>(is_q ? p.q_gamma : p.k_gamma, 8 * sa, ga);
                load8<BF16>(is_q ? p.q_gamma : p.k_gamma, 8 * sb, gb);
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    a[i] = (ga[i] * a[i]) * inv;
                    b[i] = (gb[i] * b[i]) * inv;
                }
                if (turns) {
                    if (apart) {
#pragma unroll
                        for (int i = 0; i < 8; ++i) rotate(a[i], b[i], c[i], s[i]);
                    } else {
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            rotate(a[2 * i], a[2 * i + 1], c[i], s[i]);
                            rotate(b[2 * i], b[2 * i + 1], c[4 + i], s[4 + i]);
                        }
                    }
                }
                if (!tok.in_table) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) a[i] = b[i] = tok.fill;
                }
            }
        }
        if (live && (is_q || SINK == kPlain)) {
            void* out = is_q ? p.q_out : p.k_out;
            const int64_t o = (t * (is_q ? p.q_heads : p.kv_heads) + hh) * D;
            store8<BF16>(out, o + 8 * sa, a);
            store8<BF16>(out, o + 8 * sb, b);
        }
        if constexpr (SINK == kPlain) continue;
        // keys as they would be stored; a value is of the type already
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            a[i] = kc::fp8::quiet(rounded<BF16>(a[i]));
            b[i] = kc::fp8::quiet(rounded<BF16>(b[i]));
        }
        const bool out = live && !is_q && tok.cached;
        const int64_t row = tok.slot * p.kv_heads + hh;
        uint8_t* codes = is_v ? p.v_codes : p.k_codes;
        void* scales = is_v ? p.v_scales : p.k_scales;
        if constexpr (SINK == kFp8) {
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) m = fmaxf(m, fmaxf(fabsf(a[i]), fabsf(b[i])));
            for (int off = (1 << lg) >> 1; off >= 1; off >>= 1) m = fmaxf(m, __shfl_xor(m, off, kWave));
            if (out) {
                const RowDiv d = kc::fp8::row_div(m);
                u32x2 ca, cb;
                if (d.fast) {
                    ca = fp8_codes<true>(a, d);
                    cb = fp8_codes<true>(b, d);
                } else {
                    ca = fp8_codes<false>(a, d);
                    cb = fp8_codes<false>(b, d);
                }
                u32x2* dst = reinterpret_cast<u32x2*>(codes + row * D);
                dst[sa] = ca;
                dst[sb] = cb;
                if (j == 0) static_cast<float*>(scales)[row] = d.s;
            }
        } else {
            // A block is four slots: four lanes' first (second) slots where
            // they lie apart, two lanes' slot pairs elsewhere.
            const uint32_t ma = absmax_bits8(a), mb = absmax_bits8(b);
            const uint32_t qa = max_quad(ma), qb = max_quad(mb), pr = max_pair(max(ma, mb));
            const uint32_t ba = scale_byte(apart ? qa : pr), bb = scale_byte(apart ? qb : pr);
            if (out) {
                uint32_t* dst = reinterpret_cast<uint32_t*>(codes + row * (D / 2));
                dst[sa] = mx_codes(a, ba);
                dst[sb] = mx_codes(b, bb);
                uint8_t* sc = static_cast<uint8_t*>(scales) + row * (D / kBlock);
                if ((sa & 3) == 0) sc[sa >> 2] = static_cast<uint8_t>(ba);
                if (apart && (sb & 3) == 0) sc[sb >> 2] = static_cast<uint8_t>(bb);
            }
        }
    }
}

// Any D up to 1024, any alignment: one wave per head, the row in LDS as fp32.
template <bool BF16, bool NORM, int SINK>
__global__ __launch_bounds__(kThreads) void heads_general_kernel(const Args p, int64_t rows, bool slotted) {
    using T = Elem<BF16>;
    __shared__ float lds[kWaves][kc::kv::kMaxHeadDim];
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
    const int n_q = NORM ? p.q_heads : 0, n_all = n_q + p.kv_heads + (SINK != kPlain ? p.kv_heads : 0);
    const int64_t r = static_cast<int64_t>(blockIdx.x) * kWaves + wave;
    const bool live = r < rows;
    const int64_t t = live ? r / n_all : 0;
    const int h = live ? static_cast<int>(r - t * n_all) : 0, D = p.D, R = p.R;
    const Token tok = token_of<NORM, SINK>(p, t);
    const bool is_q = h < n_q, is_v = SINK != kPlain && h >= n_q + p.kv_heads;
    const int hh = is_q ? h : is_v ? h - n_q - p.kv_heads : h - n_q;
    const T* src = static_cast<const T*>(is_q ? p.q : is_v ? p.v : p.k) +
                   t * (is_q ? p.q_stride : is_v ? p.v_stride : p.k_stride) + static_cast<int64_t>(hh) * D;
    float* row = lds[wave];
    auto get = [](const T* a, int i) {
        if constexpr (BF16) return kc::bf16_to_f32(a[i]);
        else return a[i];
    };
    for (int i = lane; i < D; i += kWave) row[i] = get(src, i);
    __syncthreads();
    if constexpr (NORM) {
        float ss = 0.0f;
        if (slotted) {  // the vector kernel's order
            const int half = R >> 4;
            if (lane < (D >> 4)) {
                const bool apart = lane < half && !p.interleaved;
                const int sa = apart ? lane : 2 * lane, sb = apart ? lane + half : 2 * lane + 1;
                for (int i = 0; i < 8; ++i) ss = fmaf(row[8 * sa + i], row[8 * sa + i], ss);
                for (int i = 0; i < 8; ++i) ss = fmaf(row[8 * sb + i], row[8 * sb + i], ss);
            }
        } else {
            for (int i = lane; i < D; i += kWave) ss = fmaf(row[i], row[i], ss);
        }
        const float inv = rms_inverse(kc::wave_sum(ss), D, p.eps);
        __syncthreads();
        if (!is_v) {
            const T* gamma = static_cast<const T*>(is_q ? p.q_gamma : p.k_gamma);
            for (int i = lane; i < D; i += kWave) row[i] = tok.in_table ? (get(gamma, i) * row[i]) * inv : tok.fill;
        }
        __syncthreads();
        if (!is_v && tok.in_table) {
            const int half = R >> 1;
            for (int i = lane; i < half; i += kWave) {
                const int ia = p.interleaved ? 2 * i : i, ib = p.interleaved ? 2 * i + 1 : i + half;
                float a = row[ia], b = row[ib];
                rotate(a, b, p.cos_t[tok.row * half + i], p.sin_t[tok.row * half + i]);
                row[ia] = a;
                row[ib] = b;
            }
        }
        __syncthreads();
    }
    if (!live) return;
    if (is_q || SINK == kPlain) {
        T* out = static_cast<T*>(is_q ? p.q_out : p.k_out) + (t * (is_q ? p.q_heads : p.kv_heads) + hh) * D;
        for (int i = lane; i < D; i += kWave) {
            if constexpr (BF16) out[i] = kc::f32_to_bf16(row[i]);
            else out[i] = row[i];
        }
        return;
    }
    if (SINK == kPlain || !tok.cached) return;
    const int64_t to = tok.slot * p.kv_heads + hh;
    uint8_t* codes = is_v ? p.v_codes : p.k_codes;
    void* scales = is_v ? p.v_scales : p.k_scales;
    auto value = [&](int i) { return kc::fp8::quiet(rounded<BF16>(row[i])); };
    if constexpr (SINK == kFp8) {
        float m = 0.0f;
        for (int i = lane; i < D; i += kWave) m = fmaxf(m, fabsf(value(i)));
        const RowDiv d = kc::fp8::row_div(kc::wave_max(m));
        for (int i = lane; i < D; i += kWave)
            codes[to * D + i] = kc::fp8::e4m3x1(d.fast ? kc::fp8::div_scale<true>(value(i), d)
                                                       : kc::fp8::div_scale<false>(value(i), d));
        if (lane == 0) static_cast<float*>(scales)[to] = d.s;
    } else if constexpr (SINK == kMx) {
        // Lane l of 16 holds values 2l, 2l + 1 of a block; D is a multiple of 32.
        for (int i = 2 * lane; i < D; i += 2 * kWave) {
            const float a = value(i), b = value(i + 1);
            uint32_t m = max(__float_as_uint(a) & 0x7FFFFFFFu, __float_as_uint(b) & 0x7FFFFFFFu);
            for (int off = 8; off >= 1; off >>= 1) m = max(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), off, kWave)));
            const uint32_t sb = scale_byte(m);
            const uint32_t c = sb == kNaN ? 0u : __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0, a, b, scale_operand(sb), 0);
            codes[to * (D / 2) + i / 2] = static_cast<uint8_t>(c);
            if ((i & 31) == 0) static_cast<uint8_t*>(scales)[to * (D / kBlock) + i / kBlock] = static_cast<uint8_t>(sb);
        }
    }
}

template <bool BF16, bool NORM, int SINK>
int launch(const char* fn, Args& p, hipStream_t stream) {
    const int heads = (NORM ? p.q_heads : 0) + p.kv_heads + (SINK != kPlain ? p.kv_heads : 0);
    const int D = p.D, align_elems = BF16 ? 8 : 4;
    const bool slotted = D % 16 == 0 && D <= 512 && p.R % 16 == 0;
    auto rows_ok = [&](const void* ptr, int64_t stride) { return kc::aligned(ptr, 16) && stride % align_elems == 0; };
    bool vec = slotted && rows_ok(p.k, p.k_stride);
    if (NORM)
        vec = vec && rows_ok(p.q, p.q_stride) && kc::aligned(p.q_gamma, 16) && kc::aligned(p.k_gamma, 16) &&
              kc::aligned(p.cos_t, 16) && kc::aligned(p.sin_t, 16) && kc::aligned(p.q_out, 16);
    if (SINK == kPlain) vec = vec && kc::aligned(p.k_out, 16);
    else vec = vec && rows_ok(p.v, p.v_stride);
    if (SINK == kFp8) vec = vec && kc::aligned(p.k_codes, 8) && kc::aligned(p.v_codes, 8);
    if (SINK == kMx)  // whole blocks in the lanes that share a maximum
        vec = vec && kc::aligned(p.k_codes, 4) && kc::aligned(p.v_codes, 4) &&
              (!NORM || p.interleaved || p.R % 64 == 0);
    if (vec) {
        p.lanes_log2 = 0;
        while ((1 << p.lanes_log2) * 16 < D) ++p.lanes_log2;
        const int hp = kWave >> p.lanes_log2;
        p.groups = (heads + hp - 1) / hp;
        // A wave per token once that fills the chip (8 waves on each of 1024
        // SIMDs); fewer tokens split their heads over more waves.
        p.splits = static_cast<int>(std::clamp<int64_t>((8192 + p.tokens - 1) / p.tokens, 1, p.groups));
        p.per_split = (p.groups + p.splits - 1) / p.splits;
        const int64_t grid = (p.tokens * p.splits + kWaves - 1) / kWaves;
        if (grid > kc::kv::kMaxGrid) return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: too many tokens", fn);
        heads_kernel<BF16, NORM, SINK><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(p);
    } else {
        const int64_t rows = p.tokens * heads, grid = (rows + kWaves - 1) / kWaves;
        if (grid > kc::kv::kMaxGrid) return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: too many tokens", fn);
        heads_general_kernel<BF16, NORM, SINK><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(p, rows, slotted);
    }
    return kc::check_launch(fn);
}

int check_rope(const char* fn, const kc_rope* r, int head_dim, int64_t tokens) {
    if (!r) return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: null rope", fn);
    if (r->rotary_dim < 0 || r->rotary_dim % 2 != 0 || r->rotary_dim > head_dim)
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: rotary_dim=%d must be even and at most head_dim=%d", fn,
                             r->rotary_dim, head_dim);
    if (r->table_rows < 0) return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: negative table_rows", fn);
    if (tokens > 0 && (!r->positions || (r->rotary_dim > 0 && r->table_rows > 0 && (!r->cos_table || !r->sin_table))))
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: null device pointer", fn);
    return KC_SUCCESS;
}

int check_heads(const char* fn, int64_t tokens, int q_heads, int kv_heads, int head_dim) {
    if (tokens < 0 || q_heads < 0 || kv_heads < 0 || head_dim < 0)
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: negative shape", fn);
    if (head_dim > kc::kv::kMaxHeadDim)
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: head_dim=%d is over %d", fn, head_dim, kc::kv::kMaxHeadDim);
    if (q_heads > (1 << 16) || kv_heads > (1 << 16) || tokens > (int64_t{1} << 40))
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: shape too large", fn);
    return KC_SUCCESS;
}

void set_rope(Args& p, const kc_rope* r, const void* q_gamma, const void* k_gamma, float eps) {
    p.q_gamma = q_gamma;
    p.k_gamma = k_gamma;
    p.cos_t = r->cos_table;
    p.sin_t = r->sin_table;
    p.positions = r->positions;
    p.table_rows = r->table_rows;
    p.R = r->rotary_dim;
    p.interleaved = r->interleaved != 0;
    p.eps = eps;
}

void set_cache(Args& p, const kc_kv_cache* c, const int64_t* slots) {
    p.slots = slots;
    p.k_codes = static_cast<uint8_t*>(c->k_codes);
    p.v_codes = static_cast<uint8_t*>(c->v_codes);
    p.k_scales = c->k_scales;
    p.v_scales = c->v_scales;
    p.n_slots = c->num_pages * c->page_size;
    p.kv_heads = c->kv_heads;
    p.D = c->head_dim;
}

template <bool BF16>
int norm_rope(const char* fn, const Elem<BF16>* q, int64_t q_stride, const Elem<BF16>* k, int64_t k_stride,
              const Elem<BF16>* q_gamma, const Elem<BF16>* k_gamma, const kc_rope* rope, float eps, int64_t tokens,
              int q_heads, int kv_heads, int head_dim, Elem<BF16>* q_out, Elem<BF16>* k_out, hipStream_t stream) {
    int st = check_heads(fn, tokens, q_heads, kv_heads, head_dim);
    if (st == KC_SUCCESS) st = check_rope(fn, rope, head_dim, tokens);
    if (st != KC_SUCCESS) return st;
    if (tokens == 0 || head_dim == 0 || q_heads + kv_heads == 0) return KC_SUCCESS;
    if ((q_heads && (!q || !q_gamma || !q_out)) || (kv_heads && (!k || !k_gamma || !k_out)))
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: null device pointer", fn);
    Args p{};
    p.q = q;
    p.k = k;
    p.q_stride = q_stride;
    p.k_stride = k_stride;
    p.q_out = q_out;
    p.k_out = k_out;
    p.tokens = tokens;
    p.q_heads = q_heads;
    p.kv_heads = kv_heads;
    p.D = head_dim;
    set_rope(p, rope, q_gamma, k_gamma, eps);
    return launch<BF16, true, kPlain>(fn, p, stream);
}

template <bool BF16>
int norm_rope_cache(const char* fn, const Elem<BF16>* q, int64_t q_stride, const Elem<BF16>* k, int64_t k_stride,
                    const Elem<BF16>* v, int64_t v_stride, const Elem<BF16>* q_gamma, const Elem<BF16>* k_gamma,
                    const kc_rope* rope, float eps, int64_t tokens, int q_heads, const int64_t* slots,
                    const kc_kv_cache* cache, Elem<BF16>* q_out, hipStream_t stream) {
    int st = kc::kv::check_cache(fn, cache);
    if (st == KC_SUCCESS) st = check_heads(fn, tokens, q_heads, cache->kv_heads, cache->head_dim);
    if (st == KC_SUCCESS) st = check_rope(fn, rope, cache->head_dim, tokens);
    if (st != KC_SUCCESS || tokens == 0) return st;
    if ((q_heads && (!q || !q_gamma || !q_out)) || !k || !v || !k_gamma || !slots)
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: null device pointer", fn);
    Args p{};
    p.q = q;
    p.k = k;
    p.v = v;
    p.q_stride = q_stride;
    p.k_stride = k_stride;
    p.v_stride = v_stride;
    p.q_out = q_out;
    p.tokens = tokens;
    p.q_heads = q_heads;
    set_rope(p, rope, q_gamma, k_gamma, eps);
    set_cache(p, cache, slots);
    return cache->format == KC_KV_FP8 ? launch<BF16, true, kFp8>(fn, p, stream) : launch<BF16, true, kMx>(fn, p, stream);
}

template <bool BF16>
int cache_write(const char* fn, const Elem<BF16>* k, int64_t k_stride, const Elem<BF16>* v, int64_t v_stride,
                const int64_t* slots, int64_t tokens, const kc_kv_cache* cache, hipStream_t stream) {
    int st = kc::kv::check_cache(fn, cache);
    if (st == KC_SUCCESS) st = check_heads(fn, tokens, 0, cache->kv_heads, cache->head_dim);
    if (st != KC_SUCCESS || tokens == 0) return st;
    if (!k || !v || !slots) return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: null device pointer", fn);
    Args p{};
    p.k = k;
    p.v = v;
    p.k_stride = k_stride;
    p.v_stride = v_stride;
    p.tokens = tokens;
    set_cache(p, cache, slots);
    return cache->format == KC_KV_FP8 ? launch<BF16, false, kFp8>(fn, p, stream)
                                      : launch<BF16, false, kMx>(fn, p, stream);
}

}  // namespace

extern "C" int kc_qk_norm_rope_bf16(const uint16_t* d_q, int64_t q_stride, const uint16_t* d_k, int64_t k_stride,
                                    const uint16_t* d_q_gamma, const uint16_t* d_k_gamma, const kc_rope* rope, float eps,
                                    int64_t tokens, int q_heads, int kv_heads, int head_dim, uint16_t* d_q_out,
                                    uint16_t* d_k_out, kc_stream_t stream) {
    return norm_rope<true>("kc_qk_norm_rope_bf16", d_q, q_stride, d_k, k_stride, d_q_gamma, d_k_gamma, rope, eps, tokens,
                           q_heads, kv_heads, head_dim, d_q_out, d_k_out, stream);
}

extern "C" int kc_qk_norm_rope_f32(const float* d_q, int64_t q_stride, const float* d_k, int64_t k_stride,
                                   const float* d_q_gamma, const float* d_k_gamma, const kc_rope* rope, float eps,
                                   int64_t tokens, int q_heads, int kv_heads, int head_dim, float* d_q_out,
                                   float* d_k_out, kc_stream_t stream) {
    return norm_rope<false>("kc_qk_norm_rope_f32", d_q, q_stride, d_k, k_stride, d_q_gamma, d_k_gamma, rope, eps, tokens,
                            q_heads, kv_heads, head_dim, d_q_out, d_k_out, stream);
}

extern "C" int kc_qk_norm_rope_cache_bf16(const uint16_t* d_q, int64_t q_stride, const uint16_t* d_k, int64_t k_stride,
                                          const uint16_t* d_v, int64_t v_stride, const uint16_t* d_q_gamma,
                                          const uint16_t* d_k_gamma, const kc_rope* rope, float eps, int64_t tokens,
                                          int q_heads, const int64_t* d_slots, const kc_kv_cache* cache,
                                          uint16_t* d_q_out, kc_stream_t stream) {
    return norm_rope_cache<true>("kc_qk_norm_rope_cache_bf16", d_q, q_stride, d_k, k_stride, d_v, v_stride, d_q_gamma,
                                 d_k_gamma, rope, eps, tokens, q_heads, d_slots, cache, d_q_out, stream);
}

extern "C" int kc_qk_norm_rope_cache_f32(const float* d_q, int64_t q_stride, const float* d_k, int64_t k_stride,
                                         const float* d_v, int64_t v_stride, const float* d_q_gamma,
                                         const float* d_k_gamma, const kc_rope* rope, float eps, int64_t tokens,
                                         int q_heads, const int64_t* d_slots, const kc_kv_cache* cache, float* d_q_out,
                                         kc_stream_t stream) {
    return norm_rope_cache<false>("kc_qk_norm_rope_cache_f32", d_q, q_stride, d_k, k_stride, d_v, v_stride, d_q_gamma,
                                  d_k_gamma, rope, eps, tokens, q_heads, d_slots, cache, d_q_out, stream);
}

extern "C" int kc_kv_cache_write_bf16(const uint16_t* d_k, int64_t k_stride, const uint16_t* d_v, int64_t v_stride,
                                      const int64_t* d_slots, int64_t tokens, const kc_kv_cache* cache,
                                      kc_stream_t stream) {
    return cache_write<true>("kc_kv_cache_write_bf16", d_k, k_stride, d_v, v_stride, d_slots, tokens, cache, stream);
}

extern "C" int kc_kv_cache_write_f32(const float* d_k, int64_t k_stride, const float* d_v, int64_t v_stride,
                                     const int64_t* d_slots, int64_t tokens, const kc_kv_cache* cache,
                                     kc_stream_t stream) {
    return cache_write<false>("kc_kv_cache_write_f32", d_k, k_stride, d_v, v_stride, d_slots, tokens, cache, stream);
}
