// kv_cache_read.hip -- the quantized paged key/value cache back to rows of
// bf16 or fp32 on gfx950 (what qk_norm_rope.hip wrote): for token t of the
// packed batch, sequence b with cu_seqlens[b] <= t < cu_seqlens[b + 1] and
// position t - cu_seqlens[b] in it, page block_table[b][position / page_size].
//
// Bound by memory: 1 (FP8) or 0.53 (MXFP4) bytes in and 2 or 4 out per value (45 000
// tokens of 8 heads of 128, keys and values: FP8 to bf16 50 to 54 us, 5.2 to 5.6 TB/s,
// MXFP4 35 to 36; FP8 to fp32 84).  A workgroup takes a tile of tokens: its first threads find one
// token's slot each (a binary search of cu_seqlens, in LDS up to 1023 sequences, all
// searches of the tile at once instead of one before every row), then all threads walk
// the rows in units of 16 bytes of output, four keys and four values in flight each
// (keys and values in workgroups of their own, each with its search: 53.5 us).
#include <algorithm>
#include <type_traits>

#include "kv_cache.hpp"

namespace {

using namespace kc::mx;
using kc::kWave;

constexpr int kThreads = 256;
constexpr int kMaxTile = 64;
constexpr int kAhead = 4;  // rows of keys, and of values, in flight per thread

template <bool BF16>
using Elem = std::conditional_t<BF16, uint16_t, float>;

struct Args {
    const uint8_t* codes[2];   // keys, values
    const void* scales[2];
    void* out[2];
    const int32_t *table, *cu;
    int64_t max_pages, num_pages, total;
    int page_size, kv_heads, D, seqs, tile;
};

constexpr int64_t kBad = -1, kOutside = -2;

constexpr int kStarts = 1024;  // starts of sequences held in LDS

// Slot of token t, the starts of the sequences at cu; kBad where its page is missing, kOutside where it belongs to
// no sequence.
__device__ __forceinline__ int64_t slot_of(const Args& p, const int32_t* cu, int64_t t) {
    if (t >= p.total || t < cu[0] || t >= cu[p.seqs]) return kOutside;
    int lo = 0, hi = p.seqs - 1;  // first b with cu[b + 1] > t
    while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (cu[mid + 1] > t) hi = mid;
        else lo = mid + 1;
    }
    const int64_t pos = t - cu[lo];
    if (pos < 0) return kBad;  // cu_seqlens that do not ascend
    const int64_t page_at = pos / p.page_size;
    if (page_at >= p.max_pages) return kBad;
    const int32_t page = p.table[lo * p.max_pages + page_at];
    if (page < 0 || page >= p.num_pages) return kBad;
    return static_cast<int64_t>(page) * p.page_size + (pos - page_at * p.page_size);
}

template <bool BF16, bool FP8, bool VEC>
__global__ __launch_bounds__(kThreads) void kv_read_kernel(const Args p) {
    __shared__ int64_t slot[kMaxTile];
    const int tid = threadIdx.x;
    const int64_t t0 = static_cast<int64_t>(blockIdx.x) * p.tile;
    if (p.seqs < kStarts) {
        __shared__ int32_t starts[kStarts];
        for (int i = tid; i <= p.seqs; i += kThreads) starts[i] = p.cu[i];
        __syncthreads();
        if (tid < p.tile) slot[tid] = slot_of(p, starts, t0 + tid);
    } else if (tid < p.tile) {
        slot[tid] = slot_of(p, p.cu, t0 + tid);
    }
    __syncthreads();
    constexpr int W = !VEC ? 1 : BF16 ? 8 : 4;     // values per unit: a lane writes 16 bytes
    const int units = p.kv_heads * p.D / W, per_head = p.D / W;
    // A thread keeps its unit of the row and walks the tile's tokens: the head and
    // the place in it cost two divisions a thread.
    const int together = max(1, kThreads / units);  // tokens side by side
    const int first = tid / units;
    if (units <= kThreads && first >= together) return;
    const float nan = __uint_as_float(0x7FC00000u);
    for (int u = units <= kThreads ? tid - first * units : tid; u < units; u += kThreads) {
        const int h = u / per_head, d = (u - h * per_head) * W;
        for (int tt = units <= kThreads ? first : 0; tt < p.tile; tt += kAhead * together) {
            int64_t s[kAhead];
            u32x2 c[2][kAhead];
            float sc[2][kAhead];
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                const int at = tt + i * together;
                s[i] = at < p.tile ? slot[at] : kOutside;
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    c[w][i] = u32x2{0u, 0u};
                    sc[w][i] = nan;
                }
                if (s[i] < 0) continue;
                const int64_t row = s[i] * p.kv_heads + h;
                const int64_t v = row * p.D + d;
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const uint8_t* codes = p.codes[w];
                    if constexpr (FP8) {
                        if constexpr (W == 8) c[w][i] = *reinterpret_cast<const u32x2*>(codes + v);
                        else if constexpr (W == 4) c[w][i].x = *reinterpret_cast<const uint32_t*>(codes + v);
                        else c[w][i].x = codes[v];
                        sc[w][i] = static_cast<const float*>(p.scales[w])[row];
                    } else {
                        if constexpr (W == 8) c[w][i].x = *reinterpret_cast<const uint32_t*>(codes + v / 2);
                        else if constexpr (W == 4) c[w][i].x = *reinterpret_cast<const uint16_t*>(codes + v / 2);
                        else c[w][i].x = codes[v / 2] >> (4 * (d & 1));
                        sc[w][i] = scale_value(static_cast<const uint8_t*>(p.scales[w])[v / kBlock]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < kAhead; ++i) {
                if (s[i] == kOutside) continue;
                const int64_t to = ((t0 + tt + i * together) * p.kv_heads + h) * p.D + d;
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    Elem<BF16>* out = static_cast<Elem<BF16>*>(p.out[w]);
                    const u32x2 cw = c[w][i];
                    const float f = sc[w][i];
                    f32x4 lo, hi;
                    if constexpr (FP8) {
                        const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(cw.x), false);
                        const auto b = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(cw.x), true);
                        const auto e = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(cw.y), false);
                        const auto g = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(cw.y), true);
                        lo = f32x4{a[0] * f, a[1] * f, b[0] * f, b[1] * f};
                        hi = f32x4{e[0] * f, e[1] * f, g[0] * f, g[1] * f};
                    } else {
                        decode8_f32(cw.x, f, lo, hi);
                    }
                    if constexpr (!VEC) {
                        if constexpr (BF16) out[to] = kc::f32_to_bf16(lo.x);
                        else out[to] = lo.x;
                    } else if constexpr (BF16) {
                        __builtin_nontemporal_store(u32x4{kc::pack_bf16x2(lo.x, lo.y), kc::pack_bf16x2(lo.z, lo.w),
                                                          kc::pack_bf16x2(hi.x, hi.y), kc::pack_bf16x2(hi.z, hi.w)},
                                                    reinterpret_cast<u32x4*>(out + to));
                    } else {
                        __builtin_nontemporal_store(lo, reinterpret_cast<f32x4*>(out + to));
                    }
                }
            }
        }
    }
}

template <bool BF16>
int cache_read(const char* fn, const kc_kv_cache* cache, const int32_t* table, int64_t max_pages, const int32_t* cu,
               int seqs, int64_t total, Elem<BF16>* k, Elem<BF16>* v, hipStream_t stream) {
    const int st = kc::kv::check_cache(fn, cache);
    if (st != KC_SUCCESS) return st;
    if (max_pages < 0 || seqs < 0 || total < 0)
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: negative shape", fn);
    if (seqs == 0 || total == 0) return KC_SUCCESS;
    if (!cu || !k || !v || (max_pages > 0 && !table))
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: null device pointer", fn);
    Args p{};
    p.codes[0] = static_cast<const uint8_t*>(cache->k_codes);
    p.codes[1] = static_cast<const uint8_t*>(cache->v_codes);
    p.scales[0] = cache->k_scales;
    p.scales[1] = cache->v_scales;
    p.out[0] = k;
    p.out[1] = v;
    p.table = table;
    p.cu = cu;
    p.max_pages = max_pages;
    p.num_pages = cache->num_pages;
    p.total = total;
    p.page_size = cache->page_size;
    p.kv_heads = cache->kv_heads;
    p.D = cache->head_dim;
    p.seqs = seqs;
    const bool fp8 = cache->format == KC_KV_FP8;
    const uintptr_t in = fp8 ? 8 : 4;
    const bool vec = p.D % 8 == 0 && kc::aligned(k, 16) && kc::aligned(v, 16) && kc::aligned(p.codes[0], in) &&
                     kc::aligned(p.codes[1], in);
    // Tokens of a workgroup: what its threads take at once where 512 workgroups are left,
    // more while 4096 are (larger ones end unevenly: 43 000 tokens 60.8 us at 32, 54 at 8,
    // keys and values apart; one head of 128 11.0 us at 8,
    // 8.3 at 64).
    const int units = p.kv_heads * p.D / (!vec ? 1 : BF16 ? 8 : 4), at_once = kAhead * std::max(1, kThreads / units);
    p.tile = 4;
    while (p.tile < kMaxTile && total / (2 * p.tile) >= (2 * p.tile <= at_once ? 512 : 4096)) p.tile *= 2;
    const int64_t grid = (total + p.tile - 1) / p.tile;
    if (grid > kc::kv::kMaxGrid) return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: too many tokens", fn);
    const unsigned g = static_cast<unsigned>(grid);
    if (fp8 && vec) kv_read_kernel<BF16, true, true><<<g, kThreads, 0, stream>>>(p);
    else if (fp8) kv_read_kernel<BF16, true, false><<<g, kThreads, 0, stream>>>(p);
    else if (vec) kv_read_kernel<BF16, false, true><<<g, kThreads, 0, stream>>>(p);
    else kv_read_kernel<BF16, false, false><<<g, kThreads, 0, stream>>>(p);
    return kc::check_launch(fn);
}

}  // namespace

extern "C" int kc_kv_cache_read_bf16(const kc_kv_cache* cache, const int32_t* d_block_table, int64_t max_pages,
                                     const int32_t* d_cu_seqlens, int seqs, int64_t total_tokens, uint16_t* d_k,
                                     uint16_t* d_v, kc_stream_t stream) {
    return cache_read<true>("kc_kv_cache_read_bf16", cache, d_block_table, max_pages, d_cu_seqlens, seqs, total_tokens,
                            d_k, d_v, stream);
}

extern "C" int kc_kv_cache_read_f32(const kc_kv_cache* cache, const int32_t* d_block_table, int64_t max_pages,
                                    const int32_t* d_cu_seqlens, int seqs, int64_t total_tokens, float* d_k, float* d_v,
                                    kc_stream_t stream) {
    return cache_read<false>("kc_kv_cache_read_f32", cache, d_block_table, max_pages, d_cu_seqlens, seqs, total_tokens,
                             d_k, d_v, stream);
}
