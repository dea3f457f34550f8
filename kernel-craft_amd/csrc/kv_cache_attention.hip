// kv_cache_attention.hip -- attention of each sequence's newest token over the quantized
// paged cache on gfx950 (what qk_norm_rope.hip wrote):
//     out[b, h] = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q[b, h] . k_t - max)
// over the visible positions t of sequence b, k and v the rows' values in fp32.  Here the
// vector kernel for any head_dim and alignment, the join and the entry points; kv_attention.hpp
// says how the work is split.
//
// The vector kernel is for what the matrix cores' does not take (heads over 256, rows of codes
// that are no whole 16 bytes, unaligned pools, keys past 64 GiB).  It decodes value by value and
// is bound by that: 4 sequences of up to 30000 tokens, 16 query heads on 8 of 72 in FP8: 71 us for
// 57 MB, 7 of them the join; 16 on one of 576: 184 us for 54 MB, 23 of them the join.
#include <algorithm>
#include <type_traits>

#include "kv_attention.hpp"

namespace {

using namespace kc::kv;
using namespace kc::mx;
using kc::kWave;

template <bool BF16>
using Elem = std::conditional_t<BF16, uint16_t, float>;

template <bool BF16>
__device__ __forceinline__ float get(const Elem<BF16>* p, int64_t i) {
    if constexpr (BF16) return kc::bf16_to_f32(p[i]);
    else return p[i];
}
template <bool BF16>
__device__ __forceinline__ void put(Elem<BF16>* p, int64_t i, float v) {
    if constexpr (BF16) p[i] = kc::f32_to_bf16(v);
    else p[i] = v;
}

__device__ __forceinline__ int wave_max_int(int v) {
#pragma unroll
    for (int off = kWave / 2; off > 0; off >>= 1) v = max(v, __shfl_xor(v, off, kWave));
    return v;
}

constexpr int kHeads = 4;  // query heads of a wave of the vector kernel

// Values d .. d + W - 1 of the row `row` (slot * kv_heads + head); FP8 without its scale.
template <bool FP8, int W>
__device__ __forceinline__ void values(const uint8_t* codes, const void* scales, int64_t row, int D, int d,
                                       float (&v)[W]) {
    if constexpr (W == 1) {
        static_assert(FP8, "rows of MXFP4 are whole blocks");
        v[0] = __builtin_amdgcn_cvt_f32_fp8(codes[row * D + d], 0);
    } else if constexpr (FP8) {
        int w;
        __builtin_memcpy(&w, codes + row * D + d, 4);
        const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
        v[0] = lo[0], v[1] = lo[1], v[2] = hi[0], v[3] = hi[1];
    } else {
        uint16_t w;
        __builtin_memcpy(&w, codes + (row * D + d) / 2, 2);
        const f32x4 f = decode4_f32(w, scale_value(static_cast<const uint8_t*>(scales)[(row * D + d) / kBlock]));
        v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
    }
}

// A workgroup is one wave: kHeads query heads of one key/value head.  Scores: a lane per
// position and half of the head, W values at a time; output: a lane per NI times W values.
template <bool BF16, bool FP8, int W, int NI>
__global__ __launch_bounds__(kWave) void attention_kernel(const Attention p) {
    __shared__ PlanShared plan;
    __shared__ float ql[kHeads * NI * W * kWave], pl[kHeads * kTile];
    __shared__ int sl[kTile];
    const int lane = threadIdx.x;
    const int set = blockIdx.y;
    Stretch s = find_stretch(p, plan, blockIdx.x, 0, blockIdx.x == 0 && set == 0);
    if (s.b < 0) return;
    const int per_kv = (p.group + kHeads - 1) / kHeads, h = set / per_kv, q0 = (set - h * per_kv) * kHeads;
    const int heads = min(kHeads, p.group - q0);
    const int64_t head0 = static_cast<int64_t>(h) * p.group + q0;
    const float nan = __uint_as_float(0x7FC00000u), inf = __uint_as_float(0x7F800000u);
    int64_t segment = static_cast<int64_t>(s.unit) * 2 * p.q_heads + head0;

    for (int b = s.b; b < p.seqs; ++b) {
        const Visible vis = visible(p, b);
        const int tiles = vis.tiles(), end = min(s.end, s.first + tiles);
        Elem<BF16>* out = static_cast<Elem<BF16>*>(p.out) + (static_cast<int64_t>(b) * p.q_heads + head0) * p.D;
        if (tiles == 0) {
            if (p.units != 0) continue;  // the join's
            for (int i = lane; i < heads * p.D; i += kWave) put<BF16>(out, i, 0.0f);
            return;
        }
        const Elem<BF16>* q = static_cast<const Elem<BF16>*>(p.q) + b * p.q_stride + head0 * p.D;
        for (int i = lane; i < kHeads * p.D; i += kWave) ql[i] = i < heads * p.D ? get<BF16>(q, i) : 0.0f;
        float m[kHeads], l[kHeads], acc[kHeads][NI][W];
#pragma unroll
        for (int j = 0; j < kHeads; ++j) {
            m[j] = -inf;
            l[j] = 0.0f;
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int e = 0; e < W; ++e) acc[j][i][e] = 0.0f;
        }
        __syncthreads();
        for (int tile = s.tile; tile < end; ++tile) {
            const int base = (vis.first / kTile + (tile - s.first)) * kTile;
            const int t = lane & (kTile - 1), half = lane / kTile, pos = base + t;
            const bool seen = pos >= vis.first && pos < vis.end;
            const int slot = seen ? slot_of(p, b, pos) : -1;
            float sc[kHeads] = {}, vs = 1.0f;
            if (slot >= 0) {
                const int64_t row = static_cast<int64_t>(slot) * p.kv_heads + h;
                float ks = 1.0f;
                if constexpr (FP8) {
                    ks = static_cast<const float*>(p.k_scales)[row];
                    vs = static_cast<const float*>(p.v_scales)[row];
                }
#pragma unroll 4
                for (int d = half * W; d < p.D; d += 2 * W) {
                    float k[W];
                    values<FP8, W>(p.k_codes, p.k_scales, row, p.D, d, k);
                    if constexpr (FP8) {  // before the products: those with the codes may be past fp32
#pragma unroll
                        for (int e = 0; e < W; ++e) k[e] *= ks;
                    }
#pragma unroll
                    for (int j = 0; j < kHeads; ++j)
#pragma unroll
                        for (int e = 0; e < W; ++e) sc[j] = fmaf(ql[j * p.D + d + e], k[e], sc[j]);
                }
#pragma unroll
                for (int j = 0; j < kHeads; ++j) sc[j] *= p.scale;
            }
            // positions without a row read another's: a weight of zero, or NaN, is all they have
            const int some = wave_max_int(slot);
            if (half == 0) sl[t] = slot >= 0 ? slot : some;
#pragma unroll
            for (int j = 0; j < kHeads; ++j) {
                float v = sc[j] + __shfl_xor(sc[j], kTile, kWave);
                if (slot < 0) v = nan;
                const float most = fmaxf(m[j], kc::wave_max(seen ? v : -inf));
                const float at = most == -inf ? 0.0f : most, by = __builtin_amdgcn_exp2f(m[j] - at);
                const float e = seen ? __builtin_amdgcn_exp2f(v - at) : 0.0f;
                m[j] = most;
                l[j] = fmaf(l[j], by, kc::wave_sum(half == 0 ? e : 0.0f));
                if (half == 0) pl[j * kTile + t] = seen ? e * vs : 0.0f;
#pragma unroll
                for (int i = 0; i < NI; ++i)
#pragma unroll
                    for (int e = 0; e < W; ++e) acc[j][i][e] *= by;
            }
            __syncthreads();
            if (some >= 0) {  // else the sums of the weights say it all
#pragma unroll 4
                for (int u = 0; u < kTile; ++u) {
                    const int64_t row = static_cast<int64_t>(__builtin_amdgcn_readfirstlane(sl[u])) * p.kv_heads + h;
#pragma unroll
                    for (int i = 0; i < NI; ++i) {
                        const int d = (lane + i * kWave) * W;
                        float v[W] = {};
                        if (d < p.D) values<FP8, W>(p.v_codes, p.v_scales, row, p.D, d, v);
#pragma unroll
                        for (int j = 0; j < kHeads; ++j)
#pragma unroll
                            for (int e = 0; e < W; ++e) acc[j][i][e] = fmaf(pl[j * kTile + u], v[e], acc[j][i][e]);
                    }
                }
            }
            __syncthreads();
        }
        const bool whole = s.tile == s.first && end == s.first + tiles;
#pragma unroll
        for (int j = 0; j < kHeads; ++j) {
            if (j >= heads) break;
#pragma unroll
            for (int i = 0; i < NI; ++i) {
                const int d = (lane + i * kWave) * W;
                if (d >= p.D) break;
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    if (whole) put<BF16>(out, j * p.D + d + e, acc[j][i][e] / l[j]);
                    else p.part_o[(segment + j) * p.D + d + e] = acc[j][i][e];
                }
            }
            if (!whole && lane == 0) {
                p.part_ml[(segment + j) * 2] = m[j];
                p.part_ml[(segment + j) * 2 + 1] = l[j];
            }
        }
        if (b == s.b) segment += p.q_heads;  // what follows begins behind the stretch's first tile
        s.first += tiles;
        s.tile = end;
        if (p.units == 0 || end == s.end) return;
    }
}

// What parts of a sum have come to: maximum, sum and W values of the output.
template <int W>
struct Joined {
    float m, l, o[W];

    __device__ __forceinline__ void add(float m1, float l1, const float (&o1)[W]) {
        const float most = fmaxf(m, m1), at = most == -__builtin_inff() ? 0.0f : most;
        const float by = __builtin_amdgcn_exp2f(m - at), by1 = __builtin_amdgcn_exp2f(m1 - at);
        m = most;
        l = fmaf(l, by, l1 * by1);
#pragma unroll
        for (int e = 0; e < W; ++e) o[e] = fmaf(o[e], by, o1[e] * by1);
    }
};

// blockDim.x / 64 waves, `split` of them for a query head of a sequence.  A row of a segment
// takes D / W lanes (at most 64), so that a wave loads several segments at once, kAhead
// times; the lanes of a value then join theirs, and the waves in LDS.
template <bool BF16, int W>
__global__ __launch_bounds__(512) void join_kernel(const Attention p, int split) {
    constexpr int kAhead = 8;
    __shared__ float part_ml[8][2];
    extern __shared__ float part_o[];  // [waves][D] where split > 1
    const int lane = threadIdx.x & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int b = blockIdx.x, head = blockIdx.y * (blockDim.x / kWave / split) + wave / split, sub = wave % split;
    const int tile = scalar_load(p.starts, b), end = scalar_load(p.starts, b + 1);
    const int per = scalar_load(p.starts, p.seqs + 1);
    const bool mine = head < p.q_heads;
    Elem<BF16>* out = static_cast<Elem<BF16>*>(p.out) + (static_cast<int64_t>(b) * p.q_heads + head) * p.D;
    if (tile == end) {
        if (mine && sub == 0)
            for (int d = lane; d < p.D; d += kWave) put<BF16>(out, d, 0.0f);
        return;
    }
    const int unit = tile / per, n = (end - 1) / per - unit + 1;
    if (n == 1) return;  // the same for the whole workgroup
    int row_lanes = kWave;
    while (row_lanes / 2 * W >= p.D) row_lanes /= 2;
    const int groups = kWave / row_lanes, group = lane / row_lanes, at = lane - group * row_lanes;
    if (mine) {
        for (int d0 = 0; d0 < p.D; d0 += row_lanes * W) {
            const int d = d0 + at * W, from = min(d, p.D - W);
            Joined<W> j{-__builtin_inff(), 0.0f, {}};
            for (int i0 = sub * groups + group; i0 < n; i0 += kAhead * split * groups) {
                float sm[kAhead], sl[kAhead], so[kAhead][W];
#pragma unroll
                for (int i = 0; i < kAhead; ++i) {  // behind the last segment: that one again, without weight
                    const int seg = i0 + i * split * groups;
                    const int slot = 2 * (unit + min(seg, n - 1)) + (min(seg, n - 1) == 0 && tile % per != 0);
                    const int64_t row = static_cast<int64_t>(slot) * p.q_heads + head;
                    sm[i] = p.part_ml[row * 2];
                    sl[i] = p.part_ml[row * 2 + 1];
                    __builtin_memcpy(so[i], __builtin_assume_aligned(p.part_o + row * p.D + from, 4 * W), 4 * W);
                }
#pragma unroll
                for (int i = 0; i < kAhead; ++i)
                    if (i0 + i * split * groups < n) j.add(sm[i], sl[i], so[i]);
            }
            for (int off = row_lanes; off < kWave; off *= 2) {
                float o1[W];
                const float m1 = __shfl_xor(j.m, off, kWave), l1 = __shfl_xor(j.l, off, kWave);
#pragma unroll
                for (int e = 0; e < W; ++e) o1[e] = __shfl_xor(j.o[e], off, kWave);
                j.add(m1, l1, o1);
            }
            if (group == 0 && d < p.D) {
#pragma unroll
                for (int e = 0; e < W; ++e) {
                    if (split > 1) part_o[wave * p.D + d + e] = j.o[e];
                    else put<BF16>(out, d + e, j.o[e] / j.l);
                }
            }
            if (lane == 0) {
                part_ml[wave][0] = j.m;
                part_ml[wave][1] = j.l;
            }
        }
    }
    if (split == 1) return;
    __syncthreads();
    if (!mine) return;
    // the waves of a head share its values out
    const int w0 = wave - sub;
    for (int d = lane + sub * kWave; d < p.D; d += kWave * split) {
        Joined<1> j{-__builtin_inff(), 0.0f, {}};
        for (int w = w0; w < w0 + split; ++w) {
            const float o1[1] = {part_o[w * p.D + d]};
            j.add(part_ml[w][0], part_ml[w][1], o1);
        }
        put<BF16>(out, d, j.o[0] / j.l);
    }
}

// Whether the matrix-core kernel takes this cache.
bool mfma_takes(const kc_kv_cache& c, int64_t max_pages) {
    const bool fp8 = c.format == KC_KV_FP8;
    const int blocks = c.head_dim / 32, row = fp8 ? c.head_dim : c.head_dim / 2;
    // rows of codes in whole 16 bytes, scales in the units that they are loaded in
    const uintptr_t unit = fp8 ? 4 : blocks % 4 == 0 ? 4 : blocks % 2 == 0 ? 2 : 1;
    return row % 16 == 0 && c.head_dim <= kMaxMfmaD && c.num_pages > 0 && max_pages > 0 &&
           kc::aligned(c.k_codes, 16) && kc::aligned(c.v_codes, 16) && kc::aligned(c.k_scales, unit) &&
           kc::aligned(c.v_scales, unit) &&
           // rows are found by 32 bits of 16 bytes
           c.num_pages * c.page_size * (row / 16) * c.kv_heads <= UINT32_MAX;
}

struct Plan {
    int sets, units, wg_sets, streams;
    dim3 grid;
};

constexpr int kMinTiles = 2;      // of a stretch
constexpr int kDirectTiles = 5;   // of a sequence for each wave of a workgroup that takes all of it

// Sets of `heads` query heads, workgroups of up to `waves` waves, `resident` waves at once.
Plan plan_of(int heads, int waves, int resident, const kc_kv_cache* c, int64_t max_pages, int seqs, int q_heads, int window) {
    Plan p{};
    const int group = q_heads / c->kv_heads;
    p.sets = c->kv_heads * ((group + heads - 1) / heads);
    // most tiles of a sequence
    const int64_t room = std::min<int64_t>(max_pages * c->page_size, INT32_MAX);
    const int64_t seen = window > 0 ? std::min<int64_t>(room, int64_t{window} + kTile - 1) : room;
    const int64_t tiles = (seen + kTile - 1) / kTile;
    // A workgroup per sequence and set where all of them run at once and none has many tiles:
    // its waves end at different times and it reads heads apart, but nothing is joined.  FP8, 8
    // sets: one sequence of 22 tiles 9.9 us against 12.8 split and joined, 24 of 33 in fp32 11.9
    // (17.8), one of 63 17.6 (13.3); in two rounds, 64 of up to 32 21.7 (18.1).  A table's width
    // is what the host knows: the one of 22 tiles in a table of 4096 is split, 13.2.
    const int64_t rounds = (int64_t{seqs} * p.sets * waves + resident - 1) / resident;
    if (tiles * std::max<int64_t>(rounds, 1) <= kDirectTiles * waves) {
        p.wg_sets = 1;
        p.streams = static_cast<int>(std::clamp<int64_t>(tiles, 1, waves));
        p.grid = dim3(seqs, p.sets);
        return p;
    }
    const int rows = (p.sets + waves - 1) / waves;
    p.wg_sets = (p.sets + rows - 1) / rows;
    p.streams = waves / p.wg_sets;
    const int64_t most = (tiles * seqs + kMinTiles - 1) / kMinTiles;
    const int at_once = std::max(1, resident / (p.wg_sets * p.streams * rows));
    const int64_t wgs = std::min<int64_t>(at_once, (most + p.streams - 1) / p.streams);
    p.grid = dim3(static_cast<unsigned>(std::clamp<int64_t>(wgs, 1, kMaxUnits / p.streams)), rows);
    p.units = static_cast<int>(p.grid.x) * p.streams;
    return p;
}

Plan plan_for(const kc_kv_cache* c, bool bf16, int64_t max_pages, int seqs, int q_heads, int window) {
    // waves at once: of the matrix cores' kernel two a SIMD, of the vector kernel four (heads
    // past 256, three of which fit, take no longer with them), or the two that fit
    if (mfma_takes(*c, max_pages)) return plan_of(bf16 ? 8 : 4, kMaxWaves, 2048, c, max_pages, seqs, q_heads, window);
    const int resident = c->head_dim <= 512 ? 4096 : 2048;
    return plan_of(kHeads, 1, resident, c, max_pages, seqs, q_heads, window);
}

int64_t starts_bytes(int seqs) { return (int64_t{seqs} + 2) * 4; }

int64_t round16(int64_t bytes) { return (bytes + 15) / 16 * 16; }

int64_t workspace_bytes(const Plan& p, int seqs, int q_heads, int D) {
    const int64_t rows = int64_t{p.units} * 2 * q_heads;
    return p.units == 0 ? 0 : round16(starts_bytes(seqs)) + round16(rows * 8) + rows * D * 4;
}

int check(const char* fn, const kc_kv_cache* cache, int64_t max_pages, int seqs, int q_heads) {
    const int st = check_cache(fn, cache);
    if (st != KC_SUCCESS) return st;
    if (max_pages < 0 || seqs < 0 || q_heads < 0)
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: negative shape", fn);
    if (q_heads % cache->kv_heads != 0)
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: q_heads=%d must be a multiple of kv_heads=%d", fn, q_heads,
                             cache->kv_heads);
    if (max_pages > INT32_MAX || q_heads > (1 << 16) - 1 || int64_t{seqs} * q_heads > kMaxGrid)
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: max_pages=%lld seqs=%d q_heads=%d too large", fn,
                             (long long)max_pages, seqs, q_heads);
    if (cache->num_pages * cache->page_size > INT32_MAX)
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: the cache has over 2^31 - 1 slots", fn);
    const int64_t tiles = (std::min<int64_t>(max_pages * cache->page_size, INT32_MAX) + kTile - 1) / kTile;
    if (tiles * seqs > (1 << 30))
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: seqs=%d max_pages=%lld page_size=%d too large", fn, seqs,
                             (long long)max_pages, cache->page_size);
    return KC_SUCCESS;
}

// Four values at a time where a head is whole fours (every MXFP4 one is).
template <bool BF16, bool FP8>
void launch_vector(const Attention& p, dim3 grid, hipStream_t stream) {
    if (p.D % 4 == 0) {
        if (p.D <= 256) attention_kernel<BF16, FP8, 4, 1><<<grid, kWave, 0, stream>>>(p);
        else if (p.D <= 512) attention_kernel<BF16, FP8, 4, 2><<<grid, kWave, 0, stream>>>(p);
        else attention_kernel<BF16, FP8, 4, 4><<<grid, kWave, 0, stream>>>(p);
    } else if constexpr (FP8) {
        if (p.D <= 256) attention_kernel<BF16, FP8, 1, 4><<<grid, kWave, 0, stream>>>(p);
        else attention_kernel<BF16, FP8, 1, 16><<<grid, kWave, 0, stream>>>(p);
    }
}

template <bool BF16>
int attention(const char* fn, const Elem<BF16>* q, int64_t q_stride, int q_heads, const kc_kv_cache* cache,
              const int32_t* table, int64_t max_pages, const int32_t* lens, int seqs, float scale, int window,
              void* workspace, int64_t bytes, Elem<BF16>* out, hipStream_t stream) {
    const int st = check(fn, cache, max_pages, seqs, q_heads);
    if (st != KC_SUCCESS) return st;
    if (window < 0) return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: window=%d is negative", fn, window);
    if (seqs == 0 || q_heads == 0) return KC_SUCCESS;
    if (!q || !lens || !out || (max_pages > 0 && !table))
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: null device pointer", fn);
    Attention p{};
    p.q = q;
    p.out = out;
    p.k_codes = static_cast<const uint8_t*>(cache->k_codes);
    p.v_codes = static_cast<const uint8_t*>(cache->v_codes);
    p.k_scales = cache->k_scales;
    p.v_scales = cache->v_scales;
    p.table = table;
    p.lens = lens;
    p.q_stride = q_stride;
    p.max_pages = static_cast<int>(max_pages);
    p.num_pages = static_cast<int>(cache->num_pages);
    p.page = cache->page_size;
    p.page_shift = kc::is_pow2(p.page) ? kc::ilog2(p.page) : -1;
    p.room = static_cast<int>(std::min<int64_t>(max_pages * p.page, INT32_MAX));
    p.kv_heads = cache->kv_heads;
    p.D = cache->head_dim;
    p.q_heads = q_heads;
    p.group = q_heads / cache->kv_heads;
    p.seqs = seqs;
    p.window = window;
    p.scale = scale * 1.44269504088896340736f;
    const bool fp8 = cache->format == KC_KV_FP8;
    const Plan plan = plan_for(cache, BF16, max_pages, seqs, q_heads, window);
    p.units = plan.units;
    p.min_tiles = kMinTiles;
    p.sets = plan.sets;
    p.wg_sets = plan.wg_sets;
    p.streams = plan.streams;
    const int64_t needs = workspace_bytes(plan, seqs, q_heads, p.D);
    if (bytes < needs || (plan.units > 0 && (!workspace || !kc::aligned(workspace, 16))))
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: the workspace has %lld bytes, needs %lld, 16-byte aligned",
                             fn, (long long)bytes, (long long)needs);
    p.starts = static_cast<int*>(workspace);
    char* parts = static_cast<char*>(workspace) + round16(starts_bytes(seqs));
    p.part_ml = reinterpret_cast<float*>(parts);
    p.part_o = reinterpret_cast<float*>(parts + round16(int64_t{plan.units} * 2 * q_heads * 8));
    if (mfma_takes(*cache, max_pages)) (BF16 ? launch_mfma_bf16 : launch_mfma_f32)(p, fp8, plan.grid, stream);
    else if (fp8) launch_vector<BF16, true>(p, plan.grid, stream);
    else launch_vector<BF16, false>(p, plan.grid, stream);
    const int launched = kc::check_launch(fn);
    if (launched != KC_SUCCESS || plan.units == 0) return launched;
    // One wave per query head of a sequence where that makes waves enough, else 4 or 8.  The join
    // with 1, 4 and 8 of them: 128 pairs (4 sequences of up to 131072 tokens) 16.2, 7.2 and 7.5 us,
    // 512 5.4, 4.5 and 5.7, 1024 4.3, 5.2 and 8.4, 2048 (64 of up to 2000) 4.3, 7.4 and 12.6.
    // Lengths are not looked at: one of 100000 among 63 of 100 takes 20.8, 18.1 and 17.6.
    const int64_t pairs = int64_t{seqs} * q_heads;
    const int split = pairs >= 2048 ? 1 : pairs >= 512 ? 4 : 8, waves = std::max(split, 4), per_wg = waves / split;
    const dim3 join_grid(seqs, (q_heads + per_wg - 1) / per_wg);
    const unsigned lds = split > 1 ? waves * p.D * sizeof(float) : 0;
    if (p.D % 4 == 0) join_kernel<BF16, 4><<<join_grid, waves * kWave, lds, stream>>>(p, split);
    else join_kernel<BF16, 1><<<join_grid, waves * kWave, lds, stream>>>(p, split);
    return kc::check_launch(fn);
}

}  // namespace

extern "C" int64_t kc_kv_cache_attention_workspace(const kc_kv_cache* cache, int64_t max_pages, int seqs,
                                                   int q_heads) {
    const char* fn = "kc_kv_cache_attention_workspace";
    if (check(fn, cache, max_pages, seqs, q_heads) != KC_SUCCESS) return -1;
    if (seqs == 0 || q_heads == 0) return 0;
    const int D = cache->head_dim;
    return std::max(workspace_bytes(plan_for(cache, true, max_pages, seqs, q_heads, 0), seqs, q_heads, D),
                    workspace_bytes(plan_for(cache, false, max_pages, seqs, q_heads, 0), seqs, q_heads, D));
}

extern "C" int kc_kv_cache_attention_bf16(const uint16_t* d_q, int64_t q_stride, int q_heads, const kc_kv_cache* cache,
                                          const int32_t* d_block_table, int64_t max_pages, const int32_t* d_seq_lens,
                                          int seqs, float scale, int window, void* d_workspace,
                                          int64_t workspace_bytes, uint16_t* d_out, kc_stream_t stream) {
    return attention<true>("kc_kv_cache_attention_bf16", d_q, q_stride, q_heads, cache, d_block_table, max_pages,
                           d_seq_lens, seqs, scale, window, d_workspace, workspace_bytes, d_out, stream);
}

extern "C" int kc_kv_cache_attention_f32(const float* d_q, int64_t q_stride, int q_heads, const kc_kv_cache* cache,
                                         const int32_t* d_block_table, int64_t max_pages, const int32_t* d_seq_lens,
                                         int seqs, float scale, int window, void* d_workspace,
                                         int64_t workspace_bytes, float* d_out, kc_stream_t stream) {
    return attention<false>("kc_kv_cache_attention_f32", d_q, q_stride, q_heads, cache, d_block_table, max_pages,
                            d_seq_lens, seqs, scale, window, d_workspace, workspace_bytes, d_out, stream);
}
