// kv_attention.hpp -- how attention of one token per sequence over the quantized cache is
// split: shared by its kernels (kv_cache_attention.hip, kv_cache_attention_mfma.hip).
//
// The visible positions of a sequence are cut into tiles of 32 (at multiples of 32), the
// tiles of all sequences stand in one row, and `units` waves per group of heads take
// equal stretches of that row, whatever the lengths are: no wave waits for a longest
// sequence, and the host need not know the lengths.  A stretch that holds all tiles of a
// sequence writes its output; the others write sums and their maximum to the workspace
// (segment number: unit + sequence, which no two segments share), and a second launch
// joins them:  m = max m_i,  l = sum l_i 2^(m_i - m),  o = sum o_i 2^(m_i - m) / l.
// Scores are kept times log2(e).  A stretch without a finite score has m = -inf, l = 0,
// o = 0.
#pragma once

#include "kv_cache.hpp"

namespace kc {
namespace kv {

constexpr int kTile = 32;          // positions
constexpr int kMaxUnits = 4096;    // stretches of a group of heads
constexpr int kMaxWaves = 8;       // of a workgroup

struct Attention {
    const void* q;
    void* out;
    const uint8_t *k_codes, *v_codes;
    const void *k_scales, *v_scales;
    const int32_t *table, *lens;
    int64_t q_stride, max_pages, num_pages;
    int page, page_shift;  // page_shift: its logarithm, or -1
    int kv_heads, D, q_heads, group, seqs, window;
    float scale;       // times log2(e)
    int units;         // stretches; 0: a stretch per sequence, and no join
    int min_tiles;     // of a stretch
    int streams;       // stretches per workgroup
    int sets, wg_sets; // sets of query heads that share a key/value head and a wave; of a workgroup
    int64_t* starts;   // workspace: first tile of each sequence, their number, tiles per stretch
    float* part_o;     // [units + seqs][q_heads][D]
    float* part_ml;    // [units + seqs][q_heads][2]
};

// Visible positions [first, end) of a sequence.  A length past the table sees a page that
// is missing, hence one position there in place of all.
struct Visible {
    int first, end;
    __device__ __forceinline__ int tiles() const { return end > first ? (end - 1) / kTile - first / kTile + 1 : 0; }
};

__device__ __forceinline__ Visible visible(const Attention& p, int b) {
    const int len = max(p.lens[b], 0);
    const int64_t room = p.max_pages * p.page;
    if (len > room) return {static_cast<int>(room), static_cast<int>(room) + 1};
    return {p.window > 0 && p.window < len ? len - p.window : 0, len};
}

// Slot of a position; -1 where its page is missing.  num_pages * page_size is below 2^31.
__device__ __forceinline__ int slot_of(const Attention& p, int b, int pos) {
    const int at = pos / p.page;
    if (at >= p.max_pages) return -1;
    const int32_t page = p.table[b * p.max_pages + at];
    return page < 0 || page >= p.num_pages ? -1 : page * p.page + (pos - at * p.page);
}

// A stretch: tiles [tile, end) of the row of all tiles, beginning in sequence b, whose
// first tile is `first`.
struct Stretch {
    int64_t tile, end, first;
    int b, unit;
};

struct PlanShared {
    int64_t part[kMaxWaves], tile[kMaxWaves], first[kMaxWaves];
    int b[kMaxWaves];
};

// The stretch of this wave (wave-uniform), found by the whole workgroup: thread i counts
// the tiles of its own sequences, a scan puts them in a row, and the thread whose
// sequences hold a stretch's first tile says so.
__device__ __forceinline__ Stretch find_stretch(const Attention& p, PlanShared& s, int stream) {
    if (p.units == 0) {
        const int b = blockIdx.x * p.streams + stream;
        return {0, b < p.seqs ? visible(p, b).tiles() : 0, 0, b < p.seqs ? b : -1, b};
    }
    const int threads = blockDim.x, tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    const int each = (p.seqs + threads - 1) / threads;
    const int b0 = min(tid * each, p.seqs), b1 = min(b0 + each, p.seqs);
    int64_t mine = 0;
    for (int b = b0; b < b1; ++b) mine += visible(p, b).tiles();
    int64_t up = mine;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
        const int64_t below = __shfl_up(up, off, kWave);
        if (lane >= off) up += below;
    }
    if (lane == kWave - 1) s.part[wave] = up;
    if (tid < kMaxWaves) s.b[tid] = -1;
    __syncthreads();
    int64_t before = 0, total = 0;
    for (int w = 0; w < threads / kWave; ++w) {
        if (w < wave) before += s.part[w];
        total += s.part[w];
    }
    before += up - mine;
    const int64_t per = max((total + p.units - 1) / p.units, static_cast<int64_t>(p.min_tiles));
    for (int i = 0; i < p.streams; ++i) {
        const int64_t t = (static_cast<int64_t>(blockIdx.x) * p.streams + i) * per;
        if (t < before || t >= before + mine) continue;
        int64_t at = before;
        int b = b0, n = visible(p, b).tiles();
        for (; t >= at + n; n = visible(p, ++b).tiles()) at += n;
        s.b[i] = b;
        s.tile[i] = t;
        s.first[i] = at;
    }
    if (blockIdx.x == 0 && blockIdx.y == 0) {  // for the join
        int64_t at = before;
        for (int b = b0; b < b1; ++b) {
            p.starts[b] = at;
            at += visible(p, b).tiles();
        }
        if (tid == 0) {
            p.starts[p.seqs] = total;
            p.starts[p.seqs + 1] = per;
        }
    }
    __syncthreads();
    Stretch r;
    r.unit = blockIdx.x * p.streams + stream;
    r.b = __builtin_amdgcn_readfirstlane(s.b[stream]);
    r.tile = s.tile[stream];
    r.first = s.first[stream];
    r.end = min(r.tile + per, total);
    return r;
}

// Where a stretch's result for a sequence goes: the output where it holds all of its
// tiles, else a segment of the workspace.
__device__ __forceinline__ bool holds_all(const Stretch& s, int64_t tile, int64_t end, int tiles) {
    return tile == s.first && end == s.first + tiles;
}

// The matrix-core kernel (kv_cache_attention_mfma.hip): sets of 8 query heads in bf16, 4 in fp32.
bool mfma_takes(const kc_kv_cache& cache);
bool launch_mfma(const Attention& p, bool bf16, bool fp8, dim3 grid, int threads, hipStream_t stream);

}  // namespace kv
}  // namespace kc
