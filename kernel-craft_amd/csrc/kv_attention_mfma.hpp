// kv_attention_mfma.hpp -- attention of each sequence's newest token over the
// quantized paged cache on gfx950's matrix cores, for head_dims up to 256 whose rows of codes
// are whole 16 bytes.
//
// A wave takes a set of query heads of one key/value head and a stretch of tiles of 32
// positions (kv_attention.hpp).  Keys and values are turned from codes into bf16, which
// holds every E4M3 and E2M1 value (times a power of two) exactly, in registers: no tile
// goes through LDS.  With lane = 16 g + c:
//   S^T = K Q^T    16 positions x 16 columns a product; a lane's 8 scores are those of
//                  column c at positions 4g .. 4g + 3 of both halves of the tile
//   O^T = V^T P^T  the sum over positions may take them in any order: with the values of
//                  just those 8 positions in a lane, its own 8 weights are its operand,
//                  and nothing crosses lanes but the maximum
// so that a column's maximum, sum and output all live in the lanes of column c.
//
// The 16 columns are N query heads in 16 / N pieces.  bf16 queries: 8 heads, the weights
// as the sum of two bf16 values (2^-17), one in each piece.  fp32 queries: 4 heads, queries
// and weights as sums of three bf16 values (exact, and 2^-25).  The pieces cost no product more,
// since groups of up to 8 (4) query heads leave those columns empty.
//
// Two waves a SIMD, each with the next tile's codes, scales and row numbers in flight (the
// loads are counted, never drained), fill the chip.  Bound by memory where there is much to
// read: 4 sequences of up to 131072 tokens, 32 query heads on 8 of 128 in FP8: 430 MB in 78 us,
// 5.5 TB/s, the same time with the arithmetic left out, and 5.9 TB/s is what rows of a
// paged cache can be read at in this order at all.  64 of up to 2000: 92 MB in 21 us, of which
// the split, the first trips to memory and the last tiles are 5.  In MXFP4 a trip to memory
// brings half the bytes: 4 of up to 131072 take 51 us for 222 MB, and leaving the decoding out
// changes nothing.  The join is 4 to 7 us more.  Three or four waves a SIMD, a barrier a tile
// and two tiles in flight were no faster.
#pragma once

#include <type_traits>

#include "kv_attention.hpp"

namespace {

using namespace kc::kv;
using namespace kc::mx;
using kc::kWave;

typedef short bf16x8 __attribute__((ext_vector_type(8)));  // as the matrix instructions take it
typedef int i32x4 __attribute__((ext_vector_type(4)));

template <bool BF16>
using Elem = std::conditional_t<BF16, uint16_t, float>;

constexpr float kLazy = 8.0f;  // a maximum may be passed by 2^8 before the sums are scaled down to a new one

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xF, 0xF, true));
}
constexpr int kRor4 = 0x124, kRor8 = 0x128;  // within 16 lanes

// Codes of w times a power of two.
__device__ __forceinline__ uint32_t fp8_pair(uint32_t w, bool high, float power = 1.0f) {
    const bf16x2 r = high ? __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(static_cast<int>(w), power, true)
                          : __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(static_cast<int>(w), power, false);
    return __builtin_bit_cast(uint32_t, r);
}

// An FP8 key's scale as power * rest: the power of two goes into its values as they are decoded,
// so that products with the query are past fp32 only where those with the key are, and the rest,
// from 1 to 2 (past 2^126 to 4, below 2^-100 less than 1), is the score's.  Between the bounds
// every E4M3 value times the power is no denormal bf16, and the power's inverse a normal fp32.
// Codes decoded alone, and the whole scale in the score, are 0.1 us less of 25 for 64 sequences
// of up to 2000 tokens and the same elsewhere, but overflow from queries of 7.6e35 on.
__device__ __forceinline__ float power_of(float scale) {
    const uint32_t e = __float_as_uint(scale) & 0x7F800000u;
    return __uint_as_float(min(max(e, 0x0D800000u), 0x7E800000u));
}
__device__ __forceinline__ float inverse(float power) { return __uint_as_float(0x7F000000u - __float_as_uint(power)); }

// Lanes 0 .. 15 and 16 .. 31 of v, to all four rows of 16 lanes each.
__device__ __forceinline__ void spread_rows(float v, float& first, float& second) {
    const uint32_t b = __float_as_uint(v);
    const auto low = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    const auto rows = __builtin_amdgcn_permlane16_swap(low[0], low[0], false, false);
    first = __uint_as_float(rows[0]);
    second = __uint_as_float(rows[1]);
}

// The value's first 8 significant bits: fp32 is the sum of three such pieces, exactly, and none
// of them is past the largest bf16 value where the fp32 is.
__device__ __forceinline__ float top_half(float v) { return __uint_as_float(__float_as_uint(v) & 0xFFFF0000u); }

// Codes 2 BYTE and 2 BYTE + 1 of w times the scale 2^(b - 127), b's value as scale_operand gives it.
template <int BYTE>
__device__ __forceinline__ uint32_t fp4_pair(uint32_t w, float scale) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, BYTE));
}

__device__ __forceinline__ bf16x8 operand(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_bit_cast(bf16x8, u32x4{a, b, c, d});
}

__device__ __forceinline__ f32x4 product(bf16x8 a, bf16x8 b, f32x4 c) {
    typedef __bf16 v8 __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
}

// A row of RB bytes spread over LANES lanes in pieces, each of L bytes per lane one after
// the other: as many of the largest L as fit, then one of each smaller power of two that
// is left.
template <int RB, int LANES, int MOST>
struct Cut {
    static constexpr int kLane = RB / LANES;
    static constexpr int pieces() {
        int n = kLane / MOST;
        for (int l = MOST / 2; l > 0; l /= 2) n += (kLane % MOST & l) != 0;
        return n;
    }
    static constexpr int lane_bytes(int i) {
        if (i < kLane / MOST) return MOST;
        i -= kLane / MOST;
        for (int l = MOST / 2; l > 0; l /= 2)
            if ((kLane % MOST & l) != 0 && i-- == 0) return l;
        return 0;
    }
    static constexpr int start(int i) {  // byte of the row
        int at = 0;
        for (int j = 0; j < i; ++j) at += LANES * lane_bytes(j);
        return at;
    }
    static constexpr int dword(int i) {  // of the lane's registers
        int at = 0;
        for (int j = 0; j < i; ++j) at += (lane_bytes(j) + 3) / 4;
        return at;
    }
    static constexpr int dwords() { return dword(pieces()); }
};

template <typename F, int... I>
__device__ __forceinline__ void each_of(F&& f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void each(F&& f) {
    each_of(f, std::make_integer_sequence<int, N>{});
}

template <int BYTES>
__device__ __forceinline__ void load_bytes(const uint8_t* from, uint32_t* to) {
    if constexpr (BYTES == 16) {
        const u32x4 v = *reinterpret_cast<const u32x4*>(from);
        to[0] = v.x, to[1] = v.y, to[2] = v.z, to[3] = v.w;
    } else if constexpr (BYTES == 8) {
        const u32x2 v = *reinterpret_cast<const u32x2*>(from);
        to[0] = v.x, to[1] = v.y;
    } else if constexpr (BYTES == 4) {
        to[0] = *reinterpret_cast<const uint32_t*>(from);
    } else if constexpr (BYTES == 2) {
        to[0] = *reinterpret_cast<const uint16_t*>(from);
    } else {
        to[0] = *from;
    }
}

// out[k]: byte k of t0 .. t3.
__device__ __forceinline__ void transpose4(uint32_t t0, uint32_t t1, uint32_t t2, uint32_t t3, uint32_t (&out)[4]) {
    const uint32_t a = __builtin_amdgcn_perm(t1, t0, 0x05010400), b = __builtin_amdgcn_perm(t3, t2, 0x05010400);
    const uint32_t c = __builtin_amdgcn_perm(t1, t0, 0x07030602), d = __builtin_amdgcn_perm(t3, t2, 0x07030602);
    out[0] = __builtin_amdgcn_perm(b, a, 0x05040100);
    out[1] = __builtin_amdgcn_perm(b, a, 0x07060302);
    out[2] = __builtin_amdgcn_perm(d, c, 0x05040100);
    out[3] = __builtin_amdgcn_perm(d, c, 0x07060302);
}
__device__ __forceinline__ uint32_t low_halves(uint32_t a, uint32_t b) {
    return __builtin_amdgcn_perm(b, a, 0x05040100);
}
__device__ __forceinline__ uint32_t high_halves(uint32_t a, uint32_t b) {
    return __builtin_amdgcn_perm(b, a, 0x07060302);
}

// N values at any alignment of their type.
template <bool BF16, int N>
__device__ __forceinline__ void store_values(Elem<BF16>* to, const float (&v)[N]) {
    if constexpr (BF16) {
        uint32_t w[(N + 1) / 2];
#pragma unroll
        for (int i = 0; i < N; i += 2) w[i / 2] = kc::pack_bf16x2(v[i], i + 1 < N ? v[i + 1] : 0.0f);
        __builtin_memcpy(to, w, 2 * N);
    } else {
        __builtin_memcpy(to, v, 4 * N);
    }
}

template <bool FP8, int D>
struct Shape {
    static constexpr int kRow = FP8 ? D : D / 2;   // bytes
    static constexpr int kBlocks = D / 32;         // MXFP4 scales of a row
    using K = Cut<kRow, 4, 16>;                    // 16 positions by up to 64 bytes a load
    using V = Cut<kRow, 16, 16>;                   // 4 positions by up to 256 bytes a load
    // a lane's K dwords: two are a step of 32 products (FP8; an odd last one has zeros behind it), or one (MXFP4)
    static constexpr int kSteps = FP8 ? (K::dwords() + 1) / 2 : K::dwords();
    static constexpr int kTiles = D / 16;          // of O^T
};

// LDS of a wave: slots of two tiles in turn, where the rows of the coming one lie (in 16
// bytes; the first row for positions without a slot), scales of one.
template <bool FP8, int D>
struct WaveShared {
    int slots[2][kTile];
    uint32_t rows[kTile];
    union {
        float f[2][kTile];                                        // FP8: keys, values
        uint8_t b[2][FP8 ? 1 : Shape<FP8, D>::kBlocks][kTile];    // MXFP4
    } scales;
};

template <bool BF16, bool FP8, int D>
__global__ __launch_bounds__(512) void attention_mfma_kernel(const Attention p) {
    using S = Shape<FP8, D>;
    using KC = typename S::K;
    using VC = typename S::V;
    constexpr int kN = BF16 ? 8 : 4;  // query heads of a set
    constexpr int kRow = D + 4;       // floats of a head in LDS: heads begin at different banks
    __shared__ PlanShared plan;
    __shared__ WaveShared<FP8, D> shared[kMaxWaves];
    __shared__ float joint_ml[kMaxWaves][2][kN];
    extern __shared__ float joint[];  // [waves][kN][kRow], for whole sequences
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int c = lane & 15, g = lane >> 4, t = lane & (kTile - 1), part = c / kN;
    WaveShared<FP8, D>& lds = shared[wave];
    const int set = blockIdx.y * p.wg_sets + wave % p.wg_sets;
    const Stretch s = find_stretch(p, plan, blockIdx.x, wave / p.wg_sets, blockIdx.x == 0 && blockIdx.y == 0);
    if (s.b < 0 || set >= p.sets) return;
    const int per_kv = (p.group + kN - 1) / kN, h = set / per_kv, q0 = (set - h * per_kv) * kN;
    const int heads = min(kN, p.group - q0), qi = c & (kN - 1);
    const int64_t head0 = static_cast<int64_t>(h) * p.group + q0;
    const float nan = __uint_as_float(0x7FC00000u), inf = __uint_as_float(0x7F800000u);
    const uint32_t row_units = static_cast<uint32_t>(p.kv_heads) * (S::kRow / 16);  // 16 bytes
    const uint8_t* kbase = p.k_codes + static_cast<int64_t>(h) * S::kRow;
    const uint8_t* vbase = p.v_codes + static_cast<int64_t>(h) * S::kRow;
    // lanes 0 .. 31 fetch the scales of keys, the others those of values
    const uint8_t* sbase = static_cast<const uint8_t*>(lane < kTile ? p.k_scales : p.v_scales) +
                           static_cast<int64_t>(h) * (FP8 ? 4 : S::kBlocks);
    const uint32_t scale_bytes = static_cast<uint32_t>(p.kv_heads) * (FP8 ? 4 : S::kBlocks);

    // ---- a tile's place: sequence b, positions from base on, of which [first, end) are seen ----
    struct Place {
        int b, base, first, end;
    };
    int seq = s.b, seq_end = s.first + s.vis.tiles();  // the sequence that find() is at, the tile behind its last
    Visible vis = s.vis;
    int shift = tile_of(vis.first) - s.first;
    auto find = [&](int tile) {
        if (tile >= s.end) return Place{-1, kTile, 1, 1};
        while (tile >= seq_end && seq + 1 < p.seqs) {  // tile < s.end ends it
            vis = visible_scalar(p, ++seq);
            shift = tile_of(vis.first) - seq_end;
            seq_end += vis.tiles();
        }
        return Place{seq, (tile + shift) * kTile, vis.first, vis.end};
    };

    // ---- queries: the operand of every step ----
    bf16x8 q[S::kSteps];
    auto load_queries = [&](int b) {
        const Elem<BF16>* from =
            static_cast<const Elem<BF16>*>(p.q) + b * p.q_stride + (head0 + (qi < heads ? qi : 0)) * D;
        each<KC::pieces()>([&](auto piece) {
            constexpr int kP = piece, kBytes = KC::lane_bytes(kP), kAt = KC::dword(kP);
            constexpr int kValues = FP8 ? kBytes : 2 * kBytes, kStep = kValues < 8 ? kValues : 8;
            const int d0 = (FP8 ? 1 : 2) * (KC::start(kP) + g * kBytes);
#pragma unroll
            for (int i = 0; i < kValues / kStep; ++i) {
                uint32_t w[4] = {0, 0, 0, 0};
                if constexpr (BF16) {
                    __builtin_memcpy(w, from + d0 + 8 * i, 2 * kStep);
                } else {
#pragma unroll
                    for (int e = 0; e < kStep; e += 2) {
                        float x[2];
#pragma unroll
                        for (int k = 0; k < 2; ++k) {  // the piece of the value that this column holds
                            x[k] = from[d0 + 8 * i + e + k];
                            const float hi = top_half(x[k]), r = x[k] - hi, mid = top_half(r);
                            x[k] = part == 0 ? hi : part == 1 ? mid : part == 2 ? r - mid : 0.0f;
                        }
                        w[e / 2] = kc::pack_bf16x2(x[0], x[1]);
                    }
                }
                q[(FP8 ? kAt / 2 : kAt) + i] = operand(w[0], w[1], w[2], w[3]);
            }
        });
    };

    // ---- the pipeline's steps ----
    // Every load of the loop is unconditional, and its order is that of the lines before the
    // loop, so that the waits in it count loads instead of draining them.
    int entry, offset;  // of this lane's position t, two tiles ahead; offset < 0: not seen, or past the table
    auto fetch = [&](const Place& at) {
        const int pos = at.base + t, near = min(max(pos, at.first), at.end - 1);
        const int page = p.page_shift >= 0 ? near >> p.page_shift : static_cast<uint32_t>(near) / p.page;
        const int32_t* row = p.table + static_cast<int64_t>(max(at.b, 0)) * p.max_pages;
        entry = row[static_cast<uint32_t>(min(page, p.max_pages - 1))];
        offset = near == pos && page < p.max_pages ? near - page * p.page : -1;
    };
    uint32_t k[2][KC::dwords()], v[8][VC::dwords()];
    constexpr int kScaleUnit = S::kBlocks % 4 == 0 ? 4 : S::kBlocks % 2 == 0 ? 2 : 1;  // MXFP4 scales of a load
    uint32_t sc[FP8 ? 1 : S::kBlocks / kScaleUnit];
    uint32_t krow[2];
    u32x4 vrow[2];
    auto place = [&](int buffer) {  // slots of the fetched tile, and where their rows lie
        const bool there = offset >= 0 && static_cast<uint32_t>(entry) < static_cast<uint32_t>(p.num_pages);
        const int slot = there ? entry * p.page + offset : -1;
        lds.slots[buffer][t] = slot;
        lds.rows[t] = there ? static_cast<uint32_t>(slot) * row_units : 0u;
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            krow[half] = lds.rows[16 * half + c];
            vrow[half] = *reinterpret_cast<const u32x4*>(&lds.rows[16 * half + 4 * g]);
        }
        __builtin_amdgcn_wave_barrier();
        return slot;
    };
    auto load_keys = [&](int slot) {
        const uint8_t* at = sbase + static_cast<uint64_t>(static_cast<uint32_t>(max(slot, 0))) * scale_bytes;
        if constexpr (FP8) {
            sc[0] = *reinterpret_cast<const uint32_t*>(at);
        } else {
#pragma unroll
            for (int i = 0; i < S::kBlocks / kScaleUnit; ++i) load_bytes<kScaleUnit>(at + i * kScaleUnit, &sc[i]);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const uint8_t* from = kbase + (static_cast<uint64_t>(krow[half]) << 4);
            each<KC::pieces()>([&](auto piece) {
                constexpr int kP = piece;
                load_bytes<KC::lane_bytes(kP)>(from + KC::start(kP) + g * KC::lane_bytes(kP),
                                               &k[half][KC::dword(kP)]);
            });
        }
    };
    auto load_values = [&]() {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint8_t* from = vbase + (static_cast<uint64_t>(vrow[i / 4][i % 4]) << 4);
            each<VC::pieces()>([&](auto piece) {
                constexpr int kP = piece;
                load_bytes<VC::lane_bytes(kP)>(from + VC::start(kP) + c * VC::lane_bytes(kP), &v[i][VC::dword(kP)]);
            });
        }
    };

    f32x4 o[S::kTiles];
    float m = -inf, l = 0.0f, at = 0.0f;  // at: m, or 0 while that is -inf
    const float off1 = part >= 1 ? -1.0f : 0.0f, off2 = part >= 2 ? -1.0f : 0.0f;

    Place here = find(s.tile), next = find(s.tile + s.step);
    if (here.b >= 0) load_queries(here.b);
    fetch(here);
    int slot = place(0), next_slot, buffer = 0;
    fetch(next);
    __builtin_amdgcn_sched_barrier(0);
    load_keys(slot);
    __builtin_amdgcn_sched_barrier(0);
    load_values();
    __builtin_amdgcn_sched_barrier(0);
    int from = here.base;  // the first tile of this sequence here
#pragma unroll
    for (int i = 0; i < S::kTiles; ++i) o[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (int tile = s.tile; here.b >= 0; tile += s.step, buffer ^= 1, slot = next_slot) {
        const bool holes = __any(slot < 0);  // a position of the tile is not there, or not seen
        // the next tile's slots
        next_slot = place(buffer ^ 1);
        const Place after = find(tile + 2 * s.step);
        fetch(after);
        __builtin_amdgcn_sched_barrier(0);
        // this tile's scales; without a slot 0, or 2^0 for the zeros there
        float power[2];
        if constexpr (FP8) {
            const float scale = __uint_as_float(sc[0]), own = power_of(scale);
            spread_rows(own, power[0], power[1]);
            const float rest = lane < kTile ? scale * inverse(own) * p.scale : scale;
            lds.scales.f[lane / kTile][t] = slot < 0 ? 0.0f : rest;
        } else {
#pragma unroll
            for (int i = 0; i < S::kBlocks; ++i)
                lds.scales.b[lane / kTile][i][t] =
                    static_cast<uint8_t>(slot < 0 ? kOne : sc[i / kScaleUnit] >> (8 * (i % kScaleUnit)));
        }
        __builtin_amdgcn_wave_barrier();

        // ---- scores ----
        float x[8];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            f32x4 a{0.0f, 0.0f, 0.0f, 0.0f};
            if constexpr (FP8) {
#pragma unroll
                for (int i = 0; i < S::kSteps; ++i) {
                    const uint32_t w0 = k[half][2 * i];
                    const bool pair = 2 * i + 1 < KC::dwords();
                    const uint32_t w1 = pair ? k[half][pair ? 2 * i + 1 : 0] : 0u;
                    a = product(operand(fp8_pair(w0, false, power[half]), fp8_pair(w0, true, power[half]),
                                        pair ? fp8_pair(w1, false, power[half]) : 0u,
                                        pair ? fp8_pair(w1, true, power[half]) : 0u),
                                q[i], a);
                }
            } else {
                each<KC::pieces()>([&](auto piece) {
                    constexpr int kP = piece, kBytes = KC::lane_bytes(kP);
                    const int block = (2 * KC::start(kP) + g * 2 * kBytes) / kBlock;
                    const float f = scale_operand(lds.scales.b[0][block][16 * half + c]);
#pragma unroll
                    for (int i = 0; i < kBytes / 4; ++i) {
                        const uint32_t w = k[half][KC::dword(kP) + i];
                        a = product(operand(fp4_pair<0>(w, f), fp4_pair<1>(w, f), fp4_pair<2>(w, f),
                                            fp4_pair<3>(w, f)),
                                    q[KC::dword(kP) + i], a);
                    }
                });
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                float v = a[i];
                if constexpr (!BF16) {  // the same sum in every piece, bit for bit
                    v += dpp<kRor8>(v);
                    v += dpp<kRor4>(v);
                }
                x[4 * half + i] = FP8 ? v : v * p.scale;
            }
            if constexpr (FP8) {
                const f32x4 f = *reinterpret_cast<const f32x4*>(&lds.scales.f[0][16 * half + 4 * g]);
#pragma unroll
                for (int i = 0; i < 4; ++i) x[4 * half + i] *= f[i];
            }
        }
        if (holes) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const i32x4 at = *reinterpret_cast<const i32x4*>(&lds.slots[buffer][16 * half + 4 * g]);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int pos = here.base + 16 * half + 4 * g + i;
                    const float y = at[i] < 0 ? nan : x[4 * half + i];
                    x[4 * half + i] = pos >= here.first && pos < here.end ? y : -inf;
#pragma unroll
                    for (int w = 0; w < VC::dwords(); ++w) v[4 * half + i][w] &= ~(at[i] >> 31);
                }
            }
        }
        float vs[8];
        if constexpr (FP8) {
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const f32x4 f = *reinterpret_cast<const f32x4*>(&lds.scales.f[1][16 * half + 4 * g]);
#pragma unroll
                for (int i = 0; i < 4; ++i) vs[4 * half + i] = f[i];
            }
        }
        // in front of the keys that will meet them: the wait for those is the wait for both
        __builtin_amdgcn_sched_barrier(0);
        if (next.b != here.b && next.b >= 0) load_queries(next.b);
        __builtin_amdgcn_sched_barrier(0);
        load_keys(next_slot);  // behind the last tile: the first row
        __builtin_amdgcn_sched_barrier(0);

        // ---- weights ----
        const float most = fmaxf(fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3])),
                                 fmaxf(fmaxf(x[4], x[5]), fmaxf(x[6], x[7])));
        if (__any(most > m + kLazy)) {
            float to = fmaxf(most, __shfl_xor(most, 16, kWave));
            to = fmaxf(to, __shfl_xor(to, 32, kWave));
            to = to > m + kLazy ? to : m;  // a column's own decision: the others go on by 1
            const float by = to == m ? 1.0f : __builtin_amdgcn_exp2f(m - to);
            m = to;
            at = m == -inf ? 0.0f : m;
            l *= by;
#pragma unroll
            for (int i = 0; i < S::kTiles; ++i) o[i] *= by;
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __builtin_amdgcn_exp2f(x[i] - at);
        l += ((x[0] + x[1]) + (x[2] + x[3])) + ((x[4] + x[5]) + (x[6] + x[7]));
        if constexpr (FP8) {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] *= vs[i];
        }
        uint32_t pw[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            float a = x[2 * i], e = x[2 * i + 1];
#pragma unroll
            for (int n = 1; n < (BF16 ? 2 : 3); ++n) {  // what the pieces before this column's hold is taken off
                const uint32_t w = kc::pack_bf16x2(a, e);
                const float off = n == 1 ? off1 : off2;
                a = fmaf(off, __uint_as_float(w << 16), a);
                e = fmaf(off, __uint_as_float(w & 0xFFFF0000u), e);
            }
            pw[i] = kc::pack_bf16x2(a, e);
            if (!BF16 && part == 3) pw[i] = 0;
        }
        const bf16x8 weights = operand(pw[0], pw[1], pw[2], pw[3]);

        // ---- output ----
        each<VC::pieces()>([&](auto piece) {
            constexpr int kP = piece, kBytes = VC::lane_bytes(kP), kAt = VC::dword(kP);
            constexpr int kTile0 = (FP8 ? 1 : 2) * VC::start(kP) / 16;
            if constexpr (FP8) {
#pragma unroll
                for (int w = 0; w < (kBytes + 3) / 4; ++w) {
                    uint32_t lo[4], hi[4];
                    transpose4(v[0][kAt + w], v[1][kAt + w], v[2][kAt + w], v[3][kAt + w], lo);
                    transpose4(v[4][kAt + w], v[5][kAt + w], v[6][kAt + w], v[7][kAt + w], hi);
#pragma unroll
                    for (int j = 0; j < (kBytes < 4 ? kBytes : 4); ++j)
                        o[kTile0 + 4 * w + j] =
                            product(operand(fp8_pair(lo[j], false), fp8_pair(lo[j], true), fp8_pair(hi[j], false),
                                            fp8_pair(hi[j], true)),
                                    weights, o[kTile0 + 4 * w + j]);
                }
            } else {
                const int block = 2 * (VC::start(kP) + c * kBytes) / kBlock;
                float f[8];
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    const uint32_t w = *reinterpret_cast<const uint32_t*>(&lds.scales.b[1][block][16 * half + 4 * g]);
#pragma unroll
                    for (int i = 0; i < 4; ++i) f[4 * half + i] = scale_operand((w >> (8 * i)) & 255u);
                }
                each<kBytes>([&](auto byte) {
                    constexpr int kB = byte;
                    uint32_t e[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) e[i] = fp4_pair<kB % 4>(v[i][kAt + kB / 4], f[i]);
                    o[kTile0 + 2 * kB] = product(operand(low_halves(e[0], e[1]), low_halves(e[2], e[3]),
                                                         low_halves(e[4], e[5]), low_halves(e[6], e[7])),
                                                 weights, o[kTile0 + 2 * kB]);
                    o[kTile0 + 2 * kB + 1] = product(operand(high_halves(e[0], e[1]), high_halves(e[2], e[3]),
                                                             high_halves(e[4], e[5]), high_halves(e[6], e[7])),
                                                     weights, o[kTile0 + 2 * kB + 1]);
                });
            }
        });
        __builtin_amdgcn_sched_barrier(0);
        load_values();
        __builtin_amdgcn_sched_barrier(0);

        // ---- the sequence's end here ----
        if (next.b != here.b) {
            l += __shfl_xor(l, 16, kWave);
            l += __shfl_xor(l, 32, kWave);
            const bool whole = from == tile_of(here.first) * kTile && here.base == tile_of(here.end - 1) * kTile;
            const int64_t row = (int64_t{2} * s.unit + (here.b == s.b ? 0 : 1)) * p.q_heads + head0 + qi;
            const float by = p.units != 0 && whole ? 1.0f / l : 1.0f;
            each<VC::pieces()>([&](auto piece) {
                constexpr int kP = piece, kValues = (FP8 ? 1 : 2) * VC::lane_bytes(kP);
                constexpr int kTile0 = (FP8 ? 1 : 2) * VC::start(kP) / 16, kD0 = (FP8 ? 1 : 2) * VC::start(kP);
                // a column's pieces share its rows out
#pragma unroll
                for (int i = 0; i < 4 * kN / 16; ++i) {
                    const int r = part * (4 * kN / 16) + i;
                    float y[kValues];
#pragma unroll
                    for (int j = 0; j < kValues; ++j) {
                        f32x4 a = o[kTile0 + j];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            a[e] += dpp<kRor8>(a[e]);
                            if constexpr (!BF16) a[e] += dpp<kRor4>(a[e]);
                        }
                        y[j] = (r == 0 ? a[0] : r == 1 ? a[1] : r == 2 ? a[2] : a[3]) * by;
                    }
                    const int d = kD0 + (4 * g + r) * kValues;
                    if (qi >= heads) continue;
                    if (p.units == 0) store_values<false, kValues>(joint + (wave * kN + qi) * kRow + d, y);
                    else if (!whole) store_values<false, kValues>(p.part_o + row * D + d, y);
                    else
                        store_values<BF16, kValues>(static_cast<Elem<BF16>*>(p.out) +
                                                        (static_cast<int64_t>(here.b) * p.q_heads + head0 + qi) * D + d,
                                                    y);
                }
            });
            if (lane < heads) {
                if (p.units == 0) {
                    joint_ml[wave][0][lane] = m;
                    joint_ml[wave][1][lane] = l;
                } else if (!whole) {
                    p.part_ml[row * 2] = m;
                    p.part_ml[row * 2 + 1] = l;
                }
            }
            from = next.base;
#pragma unroll
            for (int i = 0; i < S::kTiles; ++i) o[i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            m = -inf;
            l = at = 0.0f;
        }
        here = next;
        next = after;
    }
    if (p.units != 0) return;

    // ---- a whole sequence: all waves' parts; the workgroup has one set ----
    __syncthreads();
    Elem<BF16>* out = static_cast<Elem<BF16>*>(p.out) + (static_cast<int64_t>(s.b) * p.q_heads + head0) * D;
    const int parts = min(p.streams, s.end);
    for (int i = threadIdx.x; i < heads * (D / 4); i += blockDim.x) {
        const int head = i / (D / 4), d = (i - head * (D / 4)) * 4;
        float most = -inf, sum = 0.0f;
        for (int w = 0; w < parts; ++w) most = fmaxf(most, joint_ml[w][0][head]);
        const float at = most == -inf ? 0.0f : most;
        f32x4 y{0.0f, 0.0f, 0.0f, 0.0f};
        for (int w = 0; w < parts; ++w) {
            const float by = __builtin_amdgcn_exp2f(joint_ml[w][0][head] - at);
            sum = fmaf(by, joint_ml[w][1][head], sum);
            const f32x4 a = *reinterpret_cast<const f32x4*>(joint + (w * kN + head) * kRow + d);
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = fmaf(by, a[e], y[e]);
        }
        const float by = parts == 0 ? 0.0f : 1.0f / sum;  // no position: zeros
        const float r[4] = {y.x * by, y.y * by, y.z * by, y.w * by};
        store_values<BF16, 4>(out + head * D + d, r);
    }
}

template <bool BF16, bool FP8, int D>
void launch(const Attention& p, dim3 grid, hipStream_t stream) {
    constexpr int kStep = FP8 ? 16 : 32;
    if constexpr (D > kMaxMfmaD) {
        return;
    } else if (p.D != D) {
        launch<BF16, FP8, D + kStep>(p, grid, stream);
    } else {
        const int waves = p.wg_sets * p.streams;
        const unsigned lds = p.units == 0 ? waves * (BF16 ? 8 : 4) * (D + 4) * 4 : 0;
        attention_mfma_kernel<BF16, FP8, D><<<grid, waves * kWave, lds, stream>>>(p);
    }
}

}  // namespace
