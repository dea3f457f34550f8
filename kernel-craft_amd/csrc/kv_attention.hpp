// kv_attention.hpp -- how attention of one token per sequence over the quantized cache is
// split: shared by its kernels (kv_cache_attention.hip, kv_attention_mfma.hpp).
//
// The visible positions of a sequence are cut into tiles of 32 (at multiples of 32), the
// tiles of all sequences stand in one row, and `units` waves for each set of query heads
// take equal stretches of that row, whatever the lengths are: no wave waits for a longest
// sequence, and the host need not know the lengths.  A stretch that holds all tiles of a
// sequence writes its output; the others write sums and their maximum to the workspace
// (segment 2 unit where it begins with the stretch, 2 unit + 1 where it ends with it: a
// stretch cuts two sequences at most), and a second launch joins them:
//     m = max m_i,  l = sum l_i 2^(m_i - m),  o = sum o_i 2^(m_i - m) / l
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

struct Attention {
    const void* q;
    void* out;
    const uint8_t *k_codes, *v_codes;
    const void *k_scales, *v_scales;
    const int32_t *table, *lens;
    int64_t q_stride;
    int max_pages, num_pages, page, page_shift;  // page_shift: its logarithm, or -1
    int room;              // positions of a row of the table, at most 2^31 - 1
    int kv_heads, D, q_heads, group, seqs, window;
    float scale;       // times log2(e)
    int units;         // stretches; 0: whole sequences, and no join
    int min_tiles;     // of a stretch
    int sets;          // of query heads that share a key/value head and a wave
    int wg_sets, streams;  // sets of a workgroup, and its waves for each of them
    int* starts;       // workspace: first tile of each sequence, their number, tiles per stretch
    float* part_o;     // [2 units][q_heads][D]
    float* part_ml;    // [2 units][q_heads][2]
};

__device__ __forceinline__ int tile_of(int pos) { return static_cast<uint32_t>(pos) / kTile; }

// Visible positions [first, end) of a sequence.  A length past the table sees a page that
// is missing, hence one position there in place of all.
struct Visible {
    int first, end;
    __device__ __forceinline__ int tiles() const { return end > first ? tile_of(end - 1) - tile_of(first) + 1 : 0; }
};

__device__ __forceinline__ Visible visible_of(const Attention& p, int len) {
    len = max(len, 0);
    if (len > p.room) return {p.room, p.room + 1};
    return {p.window > 0 && p.window < len ? len - p.window : 0, len};
}

__device__ __forceinline__ Visible visible(const Attention& p, int b) { return visible_of(p, p.lens[b]); }

// An element of memory that nothing writes while the kernel runs, at a wave-uniform index: a
// scalar load, which vector loads in flight do not hold up.
template <typename T>
__device__ __forceinline__ T scalar_load(const T* from, int64_t i) {
    typedef const __attribute__((address_space(4))) T* Constant;
    return reinterpret_cast<Constant>(reinterpret_cast<uintptr_t>(from))[i];
}

__device__ __forceinline__ Visible visible_scalar(const Attention& p, int b) {
    return visible_of(p, scalar_load(p.lens, __builtin_amdgcn_readfirstlane(b)));
}

// Inclusive scan over the 64 lanes.
__device__ __forceinline__ int wave_scan(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, true);   // from 1, 2, 4, 8 lanes below in a row of 16
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, true);   // the row below's last lane, in rows 1 and 3
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, true);   // lane 31's, in the upper half
    return v;
}

// Slot of a position; -1 where its page is missing.  num_pages * page_size is below 2^31.
__device__ __forceinline__ int slot_of(const Attention& p, int b, int pos) {
    const int at = pos / p.page;
    if (at >= p.max_pages) return -1;
    const int32_t page = p.table[static_cast<int64_t>(b) * p.max_pages + at];
    return page < 0 || page >= p.num_pages ? -1 : page * p.page + (pos - at * p.page);
}

// Tiles [tile, end) of the row of all tiles, `step` apart, beginning in sequence b, whose
// first tile is `first`.  b < 0: nothing.
struct Stretch {
    int tile, end, step, first, b, unit;
    Visible vis;  // of sequence b
};

struct PlanShared {
    int part[kMaxWaves], first[kMaxWaves], b[kMaxWaves];
};

// The stretch of this wave (wave-uniform) of workgroup `at` of those with the same sets.  Up
// to 64 sequences, every wave counts all tiles by itself: a load, a scan and no barrier.
// Beyond, the workgroup does: thread i counts the tiles of its own sequences, a scan puts
// them in a row, and the thread whose sequences hold a stretch's first tile says so.
__device__ __forceinline__ Stretch find_stretch(const Attention& p, PlanShared& s, int at, int stream,
                                                bool says_starts) {
    Stretch r;
    if (p.units == 0) {
        r.unit = at;
        r.b = at < p.seqs ? at : -1;
        r.vis = at < p.seqs ? visible_scalar(p, at) : Visible{0, 0};
        r.first = 0;
        r.tile = stream;
        r.step = p.streams;
        r.end = r.vis.tiles();
        return r;
    }
    r.unit = at * p.streams + stream;
    r.step = 1;
    const int tid = threadIdx.x, lane = tid & (kWave - 1), wave = __builtin_amdgcn_readfirstlane(tid / kWave);
    if (p.seqs <= kWave) {
        const Visible mine = lane < p.seqs ? visible(p, lane) : Visible{0, 0};
        const int n = mine.tiles(), up = wave_scan(n), total = __builtin_amdgcn_readlane(up, kWave - 1);
        const int per = max((total + p.units - 1) / p.units, p.min_tiles);
        r.tile = r.unit * per;  // below 2^30 + units * min_tiles
        r.end = min(r.tile + per, total);
        if (says_starts && wave == 0) {  // for the join
            if (lane < p.seqs) p.starts[lane] = up - n;
            if (lane == 0) {
                p.starts[p.seqs] = total;
                p.starts[p.seqs + 1] = per;
            }
        }
        // the first sequence that ends behind the stretch's first tile
        const int b = __builtin_popcountll(__ballot(up <= r.tile));
        r.b = r.tile < total ? b : -1;
        const int from = b < kWave ? b : 0;
        r.vis.first = __builtin_amdgcn_readlane(mine.first, from);
        r.vis.end = __builtin_amdgcn_readlane(mine.end, from);
        r.first = __builtin_amdgcn_readlane(up - n, from);
        return r;
    }
    const int threads = blockDim.x, each = (p.seqs + threads - 1) / threads;
    const int b0 = min(tid * each, p.seqs), b1 = min(b0 + each, p.seqs);
    const int n0 = b0 < b1 ? visible(p, b0).tiles() : 0;  // most often all
    int mine = n0;
    for (int b = b0 + 1; b < b1; ++b) mine += visible(p, b).tiles();
    const int up = wave_scan(mine);
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
        const int t = (at * p.streams + i) * per;
        if (t < before || t >= before + mine) continue;
        int to = before, b = b0;
        for (int n = n0; t >= to + n && b + 1 < b1; n = visible(p, ++b).tiles()) to += n;
        s.b[i] = b;
        s.first[i] = to;
    }
    if (says_starts) {
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
    r.b = __builtin_amdgcn_readfirstlane(s.b[stream]);
    r.first = __builtin_amdgcn_readfirstlane(s.first[stream]);
    r.vis = r.b >= 0 ? visible_scalar(p, r.b) : Visible{0, 0};
    r.tile = r.unit * per;
    r.end = min(r.tile + per, total);
    return r;
}

constexpr int kMaxMfmaD = 256;

// The matrix-core kernel (kv_attention_mfma.hpp): sets of 8 query heads in bf16, 4 in fp32.
void launch_mfma_bf16(const Attention& p, bool fp8, dim3 grid, hipStream_t stream);
void launch_mfma_f32(const Attention& p, bool fp8, dim3 grid, hipStream_t stream);

}  // namespace kv
}  // namespace kc
