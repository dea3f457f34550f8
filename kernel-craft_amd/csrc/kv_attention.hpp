// kv_attention.hpp -- how attention of one token per sequence over the quantized cache is
// split: shared by its kernels (kv_cache_attention.hip, kv_cache_attention_mfma.hip).
//
// The visible positions of a sequence are cut into tiles of 32 (at multiples of 32), the
// tiles of all sequences stand in one row, and `units` waves for each set of query heads
// take equal stretches of that row, whatever the lengths are: no wave waits for a longest
// sequence, and the host need not know the lengths.  A stretch that holds all tiles of a
// sequence writes its output; the others write sums and their maximum to the workspace
// (segment number: unit + sequence, which no two segments share), and a second launch
// joins them:  m = max m_i,  l = sum l_i 2^(m_i - m),  o = sum o_i 2^(m_i - m) / l.
// Scores are kept times log2(e).  A part without a finite score has m = -inf, l = 0, o = 0.
//
// Where the block table has few tiles a row, a workgroup takes whole sequences instead, its
// waves their tiles in turn, and joins them in LDS: one launch.
#pragma once

#include "kv_cache.hpp"

namespace kc {
namespace kv {

constexpr int kTile = 32;          // positions
constexpr int kMaxUnits = 4096;    // stretches of a set of query heads
constexpr int kMaxWaves = 8;       // of a workgroup
constexpr int kXcds = 8;           // workgroups go round them in turn

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
    int units;         // stretches; 0: whole sequences, and no join
    int min_tiles;     // of a stretch
    int sets;          // of query heads that share a key/value head and a wave
    int wg_sets, streams;  // sets of a workgroup, and its waves for each of them
    int* starts;       // workspace: first tile of each sequence, their number, tiles per stretch
    float* part_o;     // [units + seqs][q_heads][D]
    float* part_ml;    // [units + seqs][q_heads][2]
};

// Visible positions [first, end) of a sequence.  A length past the table sees a page that
// is missing, hence one position there in place of all.
struct Visible {
    int first, end;
    __device__ __forceinline__ int tiles() const { return end > first ? (end - 1) / kTile - first / kTile + 1 : 0; }
};

__device__ __forceinline__ Visible visible_of(const Attention& p, int len) {
    len = max(len, 0);
    const int64_t room = p.max_pages * p.page;
    if (len > room) return {static_cast<int>(room), static_cast<int>(room) + 1};
    return {p.window > 0 && p.window < len ? len - p.window : 0, len};
}

__device__ __forceinline__ Visible visible(const Attention& p, int b) { return visible_of(p, p.lens[b]); }

// The same for a wave-uniform b: a scalar load, which vector loads in flight do not hold up.
__device__ __forceinline__ Visible visible_scalar(const Attention& p, int b) {
    typedef const __attribute__((address_space(4))) int32_t* Constant;
    return visible_of(p, reinterpret_cast<Constant>(reinterpret_cast<uintptr_t>(p.lens))[__builtin_amdgcn_readfirstlane(b)]);
}

// Slot of a position; -1 where its page is missing.  num_pages * page_size is below 2^31.
__device__ __forceinline__ int slot_of(const Attention& p, int b, int pos) {
    const int at = pos / p.page;
    if (at >= p.max_pages) return -1;
    const int32_t page = p.table[b * p.max_pages + at];
    return page < 0 || page >= p.num_pages ? -1 : page * p.page + (pos - at * p.page);
}

// Tiles [tile, end) of the row of all tiles, `step` apart, beginning in sequence b, whose
// first tile is `first`.  b < 0: nothing.
struct Stretch {
    int tile, end, step, first, b, unit;
};

struct PlanShared {
    int part[kMaxWaves], first[kMaxWaves], b[kMaxWaves];
};

// The stretch of this wave (wave-uniform), found by the whole workgroup `at` (of those with
// the same sets): thread i counts the tiles of its own sequences, a scan puts them in a
// row, and the thread whose sequences hold a stretch's first tile says so.
__device__ __forceinline__ Stretch find_stretch(const Attention& p, PlanShared& s, int at, int stream, bool says_starts) {
    Stretch r;
    if (p.units == 0) {
        r.unit = at;
        r.b = at < p.seqs ? at : -1;
        r.first = 0;
        r.tile = stream;
        r.step = p.streams;
        r.end = at < p.seqs ? visible_scalar(p, at).tiles() : 0;
        return r;
    }
    const int threads = blockDim.x, tid = threadIdx.x, lane = tid & (kWave - 1), wave = tid / kWave;
    const int each = (p.seqs + threads - 1) / threads;
    const int b0 = min(tid * each, p.seqs), b1 = min(b0 + each, p.seqs);
    const int n0 = b0 < b1 ? visible(p, b0).tiles() : 0;  // most often all
    int mine = n0;
    for (int b = b0 + 1; b < b1; ++b) mine += visible(p, b).tiles();
    int up = mine;
#pragma unroll
    for (int off = 1; off < kWave; off <<= 1) {
        const int below = __shfl_up(up, off, kWave);
        if (lane >= off) up += below;
    }
    if (lane == kWave - 1) s.part[wave] = up;
    if (tid < kMaxWaves) s.b[tid] = -1;
    __syncthreads();
    int before = 0, total = 0;
    for (int w = 0; w < threads / kWave; ++w) {
        if (w < wave) before += s.part[w];
        total += s.part[w];
    }
    before += up - mine;
    const int per = max((total + p.units - 1) / p.units, p.min_tiles);
    for (int i = 0; i < p.streams; ++i) {
        const int t = (at * p.streams + i) * per;  // below 2^30 + units * min_tiles
        if (t < before || t >= before + mine) continue;
        int to = before, b = b0;
        for (int n = n0; t >= to + n; n = visible(p, ++b).tiles()) to += n;
        s.b[i] = b;
        s.first[i] = to;
    }
    if (says_starts) {  // for the join
        int to = before;
        for (int b = b0; b < b1; ++b) {
            p.starts[b] = to;
            to += b == b0 ? n0 : visible(p, b).tiles();
        }
        if (tid == 0) {
            p.starts[p.seqs] = total;
            p.starts[p.seqs + 1] = per;
        }
    }
    __syncthreads();
    r.unit = at * p.streams + stream;
    r.b = __builtin_amdgcn_readfirstlane(s.b[stream]);
    r.first = __builtin_amdgcn_readfirstlane(s.first[stream]);
    r.tile = r.unit * per;
    r.step = 1;
    r.end = min(r.tile + per, total);
    return r;
}

// The matrix-core kernel (kv_cache_attention_mfma.hip): sets of 8 query heads in bf16, 4 in fp32.
bool mfma_takes(const kc_kv_cache& cache, int64_t max_pages);
void launch_mfma(const Attention& p, bool bf16, bool fp8, dim3 grid, hipStream_t stream);

}  // namespace kv
}  // namespace kc
