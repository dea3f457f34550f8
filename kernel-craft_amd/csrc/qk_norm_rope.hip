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
// Vector kernel.  A slot is W neighbouring values, 16 bytes where R allows (8 bf16,
// 4 fp32), else 4 bf16.  Lane j of the lanes that share a head takes two slots:
// those of its rotation pairs, j and j + R / 2W, so that both partners of every pair
// are in one lane and no value crosses lanes but in the sum of squares.  Where no
// pair asks for it (interleaved heads, values past R, cached values) the lanes of a
// head read two runs of neighbouring slots (fp32, interleaved, 16384 tokens of 40
// heads 192 -> 129 us against slots 2j and 2j + 1), or 2j and 2j + 1 where they store
// both as one and for heads that are no multiple of 64 values, whose blocks of 32
// then stay in neighbouring lanes.  bf16 D = 128 needs 8 lanes: a wave holds 8 heads of one token
// at a time, loads the next 8 while it works on them, and keeps the token's 8 cos and
// sin and the gammas of its two slots in registers over its heads.
//
// The sum of squares runs over the lane's first slot, then its second, one FMA
// a value, then over the lanes (lane ^ 1, ^ 2, ^ 4, ...).  The general kernel (any D up
// to 1024, strides and alignment; one wave per head, the row in LDS) adds in the
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

enum Sink { kPlain, kFp8, kMx, kMxAcross };  // kMxAcross: blocks of 32 in any lanes' slots

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
    int width;                        // values of a slot, 0: no slots
    bool runs;                        // two runs of slots a head, not pairs
    int lanes_log2;                   // lanes of a head
    int groups, splits, per_split;    // waves of a token and the head groups of each
};

// A slot as it lies in memory, and as fp32 values.
template <bool BF16, int W>
struct Slot {
    static constexpr int kWords = W * (BF16 ? 2 : 4) / 4;
    typedef uint32_t Vec __attribute__((ext_vector_type(kWords)));
    Vec raw;
    template <bool STREAM = false>
    __device__ __forceinline__ void load(const Elem<BF16>* base, uint32_t at) {
        const Vec* p = reinterpret_cast<const Vec*>(base + at);
        if constexpr (STREAM) raw = __builtin_nontemporal_load(p);
        else raw = *p;
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kWords; ++i) raw[i] = 0;
    }
    __device__ __forceinline__ void get(float (&v)[W]) const {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            const uint32_t w = raw[i];
            if constexpr (BF16) {
                v[2 * i] = __uint_as_float(w << 16);
                v[2 * i + 1] = __uint_as_float(w & 0xFFFF0000u);
            } else {
                v[i] = __uint_as_float(w);
            }
        }
    }
    __device__ __forceinline__ void set(const float (&v)[W]) {
#pragma unroll
        for (int i = 0; i < kWords; ++i) {
            if constexpr (BF16) raw[i] = kc::pack_bf16x2(v[2 * i], v[2 * i + 1]);
            else raw[i] = __float_as_uint(v[i]);
        }
    }
    __device__ __forceinline__ void store(Elem<BF16>* base, uint32_t at) const {
        __builtin_nontemporal_store(raw, reinterpret_cast<Vec*>(base + at));
    }
};

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __uint_as_float(static_cast<uint32_t>(
        __builtin_amdgcn_mov_dpp(static_cast<int>(__float_as_uint(v)), CTRL, 0xF, 0xF, true)));
}

// op over the 2^lg lanes of a head, lane ^ 1 first (once 4 (8) lanes agree, the
// mirror of 8 (16) lanes is lane ^ 4 (^ 8)).
template <typename Op>
__device__ __forceinline__ float over_head(float v, int lg, Op op) {
    if (lg >= 1) v = op(v, dpp<0xB1>(v));
    if (lg >= 2) v = op(v, dpp<0x4E>(v));
    if (lg >= 3) v = op(v, dpp<0x141>(v));
    if (lg >= 4) v = op(v, dpp<0x140>(v));
    if (lg >= 5) v = op(v, __shfl_xor(v, 16, kWave));
    if (lg >= 6) v = op(v, __shfl_xor(v, 32, kWave));
    return v;
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

// W values -> W E4M3 codes.
template <int W>
__device__ __forceinline__ void store_fp8(uint8_t* dst, const float (&v)[W], const RowDiv& d) {
    using kc::fp8::e4m3x4_div;
    uint32_t c[W / 4];
#pragma unroll
    for (int i = 0; i < W / 4; ++i) {
        const kc::fp8::f32x4 q{v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]};
        c[i] = d.fast ? e4m3x4_div<true>(q, d) : e4m3x4_div<false>(q, d);
    }
    if constexpr (W == 16) *reinterpret_cast<u32x4*>(dst) = u32x4{c[0], c[1], c[2], c[3]};
    else if constexpr (W == 8) *reinterpret_cast<u32x2*>(dst) = u32x2{c[0], c[1]};
    else *reinterpret_cast<uint32_t*>(dst) = c[0];
}

template <int W>
__device__ __forceinline__ uint32_t absmax_bits(const float (&v)[W]) {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) m = max(m, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    return m;
}

template <int W>
__device__ __forceinline__ void store_mx(uint8_t* dst, const float (&v)[W], uint32_t b) {
    if constexpr (W == 8) {
        *reinterpret_cast<uint32_t*>(dst) =
            b == kNaN ? 0u : encode8_f32(f32x4{v[0], v[1], v[2], v[3]}, f32x4{v[4], v[5], v[6], v[7]}, b);
    } else {
        const uint32_t c = encode4_f32(u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]),
                                             __float_as_uint(v[3])}, b);
        *reinterpret_cast<uint16_t*>(dst) = static_cast<uint16_t>(b == kNaN ? 0u : c);
    }
}

// What the lanes of a wave wrote to its LDS before, they read behind it (LDS takes a wave's
// accesses in order).
__device__ __forceinline__ void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

// The two slots of lane j of `lanes`: `apart`, the head's pairs are half a rotation
// apart (`half` slots).
struct Slots {
    int a, b;
};
__device__ __forceinline__ Slots slots_of(int j, int lanes, int half, bool apart, bool runs) {
    if (apart && j < half) return {j, j + half};
    if (!runs) return {2 * j, 2 * j + 1};
    return {apart ? j + half : j, j + lanes};  // past a rotation that takes slots 0 .. 2 half - 1, or none
}

// What lane j has of head group g: head `hh` of its tensor (EVEN: the first lane's) and `sub`
// more, two slots.
struct Place {
    bool live, is_q, is_v, apart;
    int hh, sub;
    Slots s;
};

// Five waves a SIMD: the fused kernels would take registers for four otherwise (8000
// tokens with an 8-bit cache 44 -> 40 us).
// STREAM: nontemporal loads of the heads.  EVEN: a group is of one tensor, so that its
// addresses and what becomes of it are the wave's and not each lane's (8000 tokens, FP8
// cache 41 -> 37 us, 4-bit cache 36 -> 33: two thirds of the clocks went to vector
// instructions).
template <bool BF16, int W, bool NORM, int SINK, bool STREAM, bool EVEN>
__global__ __launch_bounds__(kThreads, 5) void heads_kernel(const Args p) {
    using S = Slot<BF16, W>;
    __shared__ __align__(16) uint32_t slot_tops[SINK == kMxAcross ? kWaves : 1][2 * kWave];
    const int lane = threadIdx.x & (kWave - 1);
    const int64_t w = static_cast<int64_t>(blockIdx.x) * kWaves + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int64_t t = w / p.splits;
    if (t >= p.tokens) return;
    const int part = static_cast<int>(w - t * p.splits);
    const int D = p.D, half = p.R / (2 * W);  // slots of half a rotation
    const int lg = p.lanes_log2, hp = kWave >> lg, j = lane & ((1 << lg) - 1);
    const Token tok = token_of<NORM, SINK>(p, t);
    const int n_q = NORM ? p.q_heads : 0, n_all = n_q + p.kv_heads + (SINK != kPlain ? p.kv_heads : 0);
    const int lanes = D / (2 * W);
    const bool has = j < lanes, pairs_apart = NORM && !p.interleaved;

    using E = Elem<BF16>;
    auto place = [&](int g) {
        Place o;
        const int h = g * hp + (EVEN ? 0 : lane >> lg);
        o.live = has && (EVEN || h < n_all);
        o.is_q = h < n_q;
        o.is_v = SINK != kPlain && h >= n_q + p.kv_heads;
        o.hh = o.is_q ? h : o.is_v ? h - n_q - p.kv_heads : h - n_q;
        o.sub = EVEN ? lane >> lg : 0;
        o.apart = pairs_apart && !o.is_v;
        o.s = slots_of(j, lanes, half, o.apart, p.runs);
        return o;
    };
    auto fetch = [&](int g, S& a, S& b) {
        const Place o = place(g);
        a.clear();
        b.clear();
        if (o.live) {
            const E* src = static_cast<const E*>(o.is_q ? p.q : o.is_v ? p.v : p.k);
            src += t * (o.is_q ? p.q_stride : o.is_v ? p.v_stride : p.k_stride) + static_cast<int64_t>(o.hh) * D;
            const uint32_t at = o.sub * D;
            a.template load<STREAM>(src, at + W * o.s.a);
            b.template load<STREAM>(src, at + W * o.s.b);
        }
    };
    S na, nb;  // the next group's slots
    const int g0 = part * p.per_split, g_end = min(p.groups, g0 + p.per_split);
    if (g0 < g_end) fetch(g0, na, nb);

    float c[W] = {}, s[W] = {};
    S qa, qb, ka, kb;  // gammas of a query's and a key's slots
    if constexpr (NORM) {
        // angles: W of the lane's pairs, or W / 2 of each slot's
        const int turned = p.R / W;
        const Slots qs = slots_of(j, lanes, half, pairs_apart, p.runs);
        if (has && tok.in_table) {
            const float *ct = p.cos_t + tok.row * (p.R >> 1), *st = p.sin_t + tok.row * (p.R >> 1);
            auto angles = [&](int to, int from, auto n) {
                constexpr int kN = decltype(n)::value;
                typedef float Vec __attribute__((ext_vector_type(kN)));
                const Vec cv = *reinterpret_cast<const Vec*>(ct + from), sv = *reinterpret_cast<const Vec*>(st + from);
#pragma unroll
                for (int e = 0; e < kN; ++e) {
                    c[to + e] = cv[e];
                    s[to + e] = sv[e];
                }
            };
            if (pairs_apart) {
                if (j < half) {
                    angles(0, W * j, std::integral_constant<int, 4>{});
                    if constexpr (W == 8) angles(4, W * j + 4, std::integral_constant<int, 4>{});
                }
            } else {
                if (qs.a < turned) angles(0, W / 2 * qs.a, std::integral_constant<int, W / 2>{});
                if (qs.b < turned) angles(W / 2, W / 2 * qs.b, std::integral_constant<int, W / 2>{});
            }
        }
        qa.clear(), qb.clear(), ka.clear(), kb.clear();
        if (has) {
            if (p.q_heads > 0) {
                qa.load(static_cast<const E*>(p.q_gamma), W * qs.a);
                qb.load(static_cast<const E*>(p.q_gamma), W * qs.b);
            }
            if (p.kv_heads > 0) {
                ka.load(static_cast<const E*>(p.k_gamma), W * qs.a);
                kb.load(static_cast<const E*>(p.k_gamma), W * qs.b);
            }
        }
    }
    for (int g = g0; g < g_end; ++g) {
        const S ra = na, rb = nb;
        if (g + 1 < g_end) fetch(g + 1, na, nb);
        const Place o = place(g);
        float a[W], b[W];
        ra.get(a);
        rb.get(b);
        if constexpr (NORM) {
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < W; ++i) ss = fmaf(a[i], a[i], ss);
#pragma unroll
            for (int i = 0; i < W; ++i) ss = fmaf(b[i], b[i], ss);
            ss = over_head(ss, lg, [](float u, float v) { return u + v; });
            const float inv = rms_inverse(ss, D, p.eps);
            if (!o.is_v) {
                float ga[W], gb[W];
                S xa = ka, xb = kb;
                if (o.is_q) xa = qa, xb = qb;
                xa.get(ga);
                xb.get(gb);
#pragma unroll
                for (int i = 0; i < W; ++i) {
                    a[i] = (ga[i] * a[i]) * inv;
                    b[i] = (gb[i] * b[i]) * inv;
                }
                if (pairs_apart) {
                    if (p.R == D || j < half) {
#pragma unroll
                        for (int i = 0; i < W; ++i) rotate(a[i], b[i], c[i], s[i]);
                    }
                } else {
                    if (o.s.a < p.R / W) {
#pragma unroll
                        for (int i = 0; i < W / 2; ++i) rotate(a[2 * i], a[2 * i + 1], c[i], s[i]);
                    }
                    if (o.s.b < p.R / W) {
#pragma unroll
                        for (int i = 0; i < W / 2; ++i) rotate(b[2 * i], b[2 * i + 1], c[W / 2 + i], s[W / 2 + i]);
                    }
                }
                if (!tok.in_table) {
#pragma unroll
                    for (int i = 0; i < W; ++i) a[i] = b[i] = tok.fill;
                }
            }
        }
        if (SINK == kPlain || (NORM && o.is_q)) {
            if (o.live) {
                S out;
                E* base = static_cast<E*>(o.is_q ? p.q_out : p.k_out) + (t * (o.is_q ? p.q_heads : p.kv_heads) + o.hh) * D;
                const uint32_t to = o.sub * D;
                out.set(a);
                out.store(base, to + W * o.s.a);
                out.set(b);
                out.store(base, to + W * o.s.b);
            }
        }
        if constexpr (SINK == kPlain) continue;
        if (NORM && (g + 1) * hp <= n_q) continue;  // queries only
        // keys as they would be stored; a value is of the type already
        if constexpr (NORM && BF16) {
            S v;
            v.set(a);
            v.get(a);
            v.set(b);
            v.get(b);
        }
#pragma unroll
        for (int i = 0; i < W; ++i) {
            a[i] = kc::fp8::quiet(a[i]);
            b[i] = kc::fp8::quiet(b[i]);
        }
        const bool out = o.live && !o.is_q && tok.cached;
        const int64_t row = tok.slot * p.kv_heads + o.hh + o.sub;
        uint8_t* codes = o.is_v ? p.v_codes : p.k_codes;
        void* scales = o.is_v ? p.v_scales : p.k_scales;
        if constexpr (SINK == kFp8) {
            float m = 0.0f;
#pragma unroll
            for (int i = 0; i < W; ++i) m = fmaxf(m, fmaxf(fabsf(a[i]), fabsf(b[i])));
            m = over_head(m, lg, [](float u, float v) { return fmaxf(u, v); });
            if (out) {
                const RowDiv d = kc::fp8::row_div(m);
                if constexpr (NORM) {
                    store_fp8<W>(codes + row * D + W * o.s.a, a, d);
                    store_fp8<W>(codes + row * D + W * o.s.b, b, d);
                } else {  // neighbouring slots
                    float v[2 * W];
#pragma unroll
                    for (int i = 0; i < W; ++i) {
                        v[i] = a[i];
                        v[W + i] = b[i];
                    }
                    store_fp8<2 * W>(codes + row * D + W * o.s.a, v, d);
                }
                if (j == 0) static_cast<float*>(scales)[row] = d.s;
            }
        } else {
            constexpr int kSlots = kBlock / W;
            const uint32_t ma = absmax_bits<W>(a), mb = absmax_bits<W>(b);
            uint32_t ba, bb;
            bool run;
            if constexpr (SINK == kMxAcross) {
                // Half a rotation is no whole number of blocks: the slots' maxima meet
                // in the wave's own LDS, in the head's order (8000 tokens of 32 + 8 bf16
                // heads of 96, all of them turned, 31.5 us, of 128 with a quarter turned
                // 38.6; by one wave a head 196 and 204).
                uint32_t* tops = slot_tops[threadIdx.x >> 6] + (lane >> lg << (lg + 1));
                if (has) {
                    tops[o.s.a] = ma;
                    tops[o.s.b] = mb;
                }
                wave_sync();
                auto top = [&](int slot) {
                    const u32x4* q = reinterpret_cast<const u32x4*>(tops + slot / kSlots * kSlots);
                    uint32_t m = 0;
#pragma unroll
                    for (int i = 0; i < kSlots / 4; ++i) m = max(m, max(max(q[i].x, q[i].y), max(q[i].z, q[i].w)));
                    return m;
                };
                ba = scale_byte(has ? top(o.s.a) : 0u);
                bb = scale_byte(has ? top(o.s.b) : 0u);
                run = true;
                wave_sync();
            } else {
                // A block is 32 / W slots: of so many lanes' first (second) slots in a run,
                // of half as many lanes' slot pairs.
                run = p.runs || (o.apart && j < half);
                const uint32_t mab = max(ma, mb);
                const uint32_t ra2 = W == 8 ? max_quad(ma) : max_oct(ma), rb2 = W == 8 ? max_quad(mb) : max_oct(mb);
                const uint32_t pr = W == 8 ? max_pair(mab) : max_quad(mab);
                ba = scale_byte(run ? ra2 : pr);
                bb = scale_byte(run ? rb2 : pr);
            }
            if (out) {
                uint8_t* dst = codes + row * (D / 2);
                store_mx<W>(dst + W / 2 * o.s.a, a, ba);
                store_mx<W>(dst + W / 2 * o.s.b, b, bb);
                uint8_t* sc = static_cast<uint8_t*>(scales) + row * (D / kBlock);
                if (o.s.a % kSlots == 0) sc[o.s.a / kSlots] = static_cast<uint8_t>(ba);
                if (run && o.s.b % kSlots == 0) sc[o.s.b / kSlots] = static_cast<uint8_t>(bb);
            }
        }
    }
}

// Any D up to 1024, any alignment: one wave per head, the row in LDS as fp32.
template <bool BF16, bool NORM, int SINK>
__global__ __launch_bounds__(kThreads) void heads_general_kernel(const Args p, int64_t rows) {
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
        if (p.width > 0) {  // the vector kernel's order
            const int W = p.width, half = R / (2 * W);
            if (lane < D / (2 * W)) {
                const Slots s = slots_of(lane, D / (2 * W), half, !p.interleaved && !is_v, p.runs);
                for (int i = 0; i < W; ++i) ss = fmaf(row[W * s.a + i], row[W * s.a + i], ss);
                for (int i = 0; i < W; ++i) ss = fmaf(row[W * s.b + i], row[W * s.b + i], ss);
            }
        } else {
            for (int i = lane; i < D; i += kWave) ss = fmaf(row[i], row[i], ss);
        }
        for (int off = 1; off < kWave; off <<= 1) ss += __shfl_xor(ss, off, kWave);
        const float inv = rms_inverse(ss, D, p.eps);
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

// As many tokens as one launch holds.
template <bool BF16, bool NORM, int SINK>
int launch_part(const char* fn, Args& p, int heads, hipStream_t stream) {
    const int D = p.D;
    // 16-byte slots where both halves of the rotation are whole slots, else 4 bf16
    const int wide = BF16 ? 8 : 4;
    p.width = D % (2 * wide) == 0 && p.R % (2 * wide) == 0 ? wide : D % 8 == 0 && p.R % 8 == 0 ? 4 : 0;
    if (p.width > 0 && D / (2 * p.width) > kWave) p.width = 0;
    p.runs = NORM && D % 64 == 0;  // without a rotation neighbouring slots, stored as one
    const uintptr_t bytes = p.width * sizeof(Elem<BF16>);
    auto whole = [&](const void* ptr) { return kc::aligned(ptr, bytes); };
    auto rows_ok = [&](const void* ptr, int64_t stride) { return whole(ptr) && stride % p.width == 0; };
    bool vec = p.width > 0 && rows_ok(p.k, p.k_stride);
    if (NORM)
        vec = vec && rows_ok(p.q, p.q_stride) && whole(p.q_gamma) && whole(p.k_gamma) && kc::aligned(p.cos_t, 16) &&
              kc::aligned(p.sin_t, 16) && whole(p.q_out);
    if (SINK == kPlain) vec = vec && whole(p.k_out);
    else vec = vec && rows_ok(p.v, p.v_stride);
    if (SINK == kFp8) vec = vec && kc::aligned(p.k_codes, (NORM ? 1 : 2) * p.width) && kc::aligned(p.v_codes, (NORM ? 1 : 2) * p.width);
    if (SINK == kMx) vec = vec && kc::aligned(p.k_codes, 4) && kc::aligned(p.v_codes, 4);
    if (vec) {
        p.lanes_log2 = 0;
        while ((1 << p.lanes_log2) * 2 * p.width < D) ++p.lanes_log2;
        const int hp = kWave >> p.lanes_log2;
        p.groups = (heads + hp - 1) / hp;
        // A wave per token once that fills the chip (8 waves on each of 1024
        // SIMDs); fewer tokens split their heads over more waves.
        p.splits = static_cast<int>(std::clamp<int64_t>((8192 + p.tokens - 1) / p.tokens, 1, p.groups));
        p.per_split = (p.groups + p.splits - 1) / p.splits;
        const int64_t grid = (p.tokens * p.splits + kWaves - 1) / kWaves;
        // Nontemporal loads gain 3 to 8 % where the heads cannot lie in the Infinity Cache
        // (256 MB), in which a projection has just left them, and lose where they do (32 + 8
        // bf16 heads of 128: 2048 tokens 11.7 us against 10.3 with plain loads, 4096 17.9 and
        // 16.2, 8192 33.6 and 35.7), or where a load of a head's lanes is no whole 128-byte
        // lines: heads of 96 (20.9 -> 28.8 us for 8192 tokens of 32), half rotations of 64
        // bytes (heads of 64 18.4 -> 21.9).
        const int64_t line = 128 / sizeof(Elem<BF16>);
        const bool stream_heads = p.tokens * heads * D * static_cast<int64_t>(sizeof(Elem<BF16>)) > (int64_t{64} << 20) &&
                                  D % line == 0 && (!NORM || p.interleaved || p.R % (2 * line) == 0);
        const unsigned blocks = static_cast<unsigned>(grid);
        constexpr int kWide = BF16 ? 8 : 4;
        const bool even = (NORM ? p.q_heads : 0) % hp == 0 && p.kv_heads % hp == 0;
        auto run = [&](auto sink) {
            constexpr int kTo = decltype(sink)::value;
            if (p.width < wide) heads_kernel<BF16, 4, NORM, kTo, false, false><<<blocks, kThreads, 0, stream>>>(p);
            else if (stream_heads && even) heads_kernel<BF16, kWide, NORM, kTo, true, true><<<blocks, kThreads, 0, stream>>>(p);
            else if (stream_heads) heads_kernel<BF16, kWide, NORM, kTo, true, false><<<blocks, kThreads, 0, stream>>>(p);
            else if (even) heads_kernel<BF16, kWide, NORM, kTo, false, true><<<blocks, kThreads, 0, stream>>>(p);
            else heads_kernel<BF16, kWide, NORM, kTo, false, false><<<blocks, kThreads, 0, stream>>>(p);
        };
        if constexpr (NORM && SINK == kMx) {
            if (!p.interleaved && p.R % 64 != 0) run(std::integral_constant<int, kMxAcross>{});
            else run(std::integral_constant<int, kMx>{});
        } else {
            run(std::integral_constant<int, SINK>{});
        }
    } else {
        const int64_t rows = p.tokens * heads, grid = (rows + kWaves - 1) / kWaves;
        heads_general_kernel<BF16, NORM, SINK><<<static_cast<unsigned>(grid), kThreads, 0, stream>>>(p, rows);
    }
    return kc::check_launch(fn);
}

// A wave takes one head at least, so a launch holds every batch of up to kMaxGrid kWaves
// heads; more are further launches.
template <bool BF16, bool NORM, int SINK>
int launch(const char* fn, Args& p, hipStream_t stream) {
    using E = Elem<BF16>;
    const int heads = (NORM ? p.q_heads : 0) + p.kv_heads + (SINK != kPlain ? p.kv_heads : 0);
    const int64_t most = kc::kv::kMaxGrid * kWaves / heads, tokens = p.tokens;
    for (int64_t t = 0; t < tokens; t += most) {
        Args part = p;
        part.tokens = std::min(most, tokens - t);
        auto input = [&](const void*& x, int64_t stride) {
            if (x) x = static_cast<const E*>(x) + t * stride;
        };
        auto output = [&](void*& y, int64_t n) {
            if (y) y = static_cast<E*>(y) + t * n * p.D;
        };
        input(part.q, p.q_stride);
        input(part.k, p.k_stride);
        input(part.v, p.v_stride);
        output(part.q_out, p.q_heads);
        output(part.k_out, p.kv_heads);
        if (part.positions) part.positions += t;
        if (part.slots) part.slots += t;
        const int st = launch_part<BF16, NORM, SINK>(fn, part, heads, stream);
        if (st != KC_SUCCESS) return st;
    }
    return KC_SUCCESS;
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
