// mxfp4_gemm_tile.hip -- the MXFP4 x MXFP4 product for more rows than a decode
// batch has.  Y[m, n] = sum_b 2^(sx + sw - 254) sum_{k in b} e2m1(qx) e2m1(qw).
//
// The matrix core takes 128 values of K at a time and the scale of each block of
// 32 with them: lane (i, kb) of an operand holds 16 bytes, one block, of row i,
// and that block's scale byte in a byte of another register.
//
// Tiling.  A workgroup of WGM x WGN waves computes 16 TM WGM x 16 TN WGN outputs;
// a wave owns TM x TN tiles of 16 x 16.  K advances in steps of 128 bytes (256
// values), which go from global memory straight into LDS (rows of 128 bytes,
// 16-byte chunks XOR-swizzled by the row) through a ring of ST buffers.  A step
// is two halves, chunk 2 kb + h of a row in half h: half 1 is read into
// registers while half 0 is multiplied, and half 0 of the next step while half 1
// is, so that no MFMA waits for LDS.  One barrier a step, between the halves:
// after it step s + 1 has landed and step s's buffer is free for step s + ST.
//
// LDS sets the wave tile: per half step a wave reads TM + TN operands (8 clocks
// each) for TM TN MFMAs of 16 clocks on its own SIMD, and the tile's bytes are
// written there too (128 a clock).  8 x 8 on four waves needs three quarters of the LDS
// clocks that its MFMAs take, 8 x 4 on eight waves all of them, 4 x 2 on eight waves
// (128 x 128) about 910 (counted) for 512 of MFMAs, of the 1290 that a step takes there.
//
// Scales.  Four steps need 32 scale bytes of every row.  Their bytes come one group of
// four steps ahead; each thread sorts its rows' so that a lane's bytes are neighbours
// ([row][kb][step, half]) and leaves them in LDS; a lane then holds the 16 bytes a block
// of rows needs for four steps in two registers, and the MFMA picks its byte by number.
// They come through registers where two buffers make every step wait for all loads
// anyway.  With more (SDMA) they go straight into LDS as the operands do: the
// compiler's wait for a load into registers would be for every load in flight, once a
// group (M 1000, N 4096, K 14336 45.6 -> 42.3 us, K 16384 50.7 -> 46.6).
//
// Tails.  Rows past M (N) load the last row and feed outputs that are not stored.
// K past the last group of four steps runs in a loop without the overlap; chunks
// past K load the last valid chunk, and the scale bytes of their blocks are 0 on
// both sides: a factor 2^-254 on products of at most 36, none of which reaches
// the smallest fp32 number (E2M1 has no NaN and no infinity).
#include <algorithm>
#include <type_traits>

#include "mxfp4_gemm.hpp"

namespace {

using namespace kc::mx;

typedef __attribute__((address_space(3))) void lds_void;

constexpr int kBK = 128;      // bytes of K per step
constexpr int kGroup = 4;     // steps per group of scales
constexpr int kGroupM = 4;    // row tiles walked together

// A 128-bit read of LDS serves lanes 0-3, 12-15, 20-23 and 24-27 together, then the same of
// the upper half, then the others (rows 0-3 and 12-15 of chunk c with rows 4-11 of chunk
// c + 2): the pairs of rows take the eight slots in an order that gives each such sixteen
// different banks.  With row / 2 for the order they meet two by two: M 1000, N 4096, K 14336
// 5.6e6 clocks of conflicts against 1.9e6 (on four waves; 2.7e6 on eight), and the prefill product 0.6 % slower.
__device__ __forceinline__ int swizzle(int row) {
    const int j = row >> 1;
    return (j & 1) | (j >> 1 & 2) | ((j << 1 ^ j) & 4);
}

template <int TM_, int TN_, int WGM, int WGN, int ST, bool SDMA>
struct Shape {
    static constexpr int kRowsM = 16 * TM_ * WGM, kRowsN = 16 * TN_ * WGN, kRows = kRowsM + kRowsN;
    static constexpr int kWaves = WGM * WGN, kThreads = 64 * kWaves;
    static constexpr int kPerM = kRowsM / 8 / kWaves, kPerN = kRowsN / 8 / kWaves;  // loads of a wave and step
    static constexpr int kLoads = kPerM + kPerN;
    static constexpr int kStage = kRows * kBK;
    static constexpr int kScaleOff = ST * kStage;                // [row][kb][8 bytes]
    static constexpr int kRawOff = kScaleOff + kRows * 32;       // [row][32 bytes] as they come
    static constexpr int kLds = SDMA ? kRawOff + kRows * 32 : kRawOff;
    static constexpr int kScaleLoads = (kRows / 32 + kWaves - 1) / kWaves;  // of a wave and group
    static constexpr int kRowsPerThread = (kRows + kThreads - 1) / kThreads;
    static_assert(kPerM * 8 * kWaves == kRowsM && kPerN * 8 * kWaves == kRowsN, "whole loads per wave");
    static_assert(kLds <= 160 * 1024, "LDS");
    static_assert(!SDMA || (ST <= 4 && kRows % 32 == 0), "scales have landed two steps on; whole loads");
};

template <int TM, int TN, int WGM, int WGN, int ST, bool SDMA, bool YBF16>
__global__ __launch_bounds__(64 * WGM * WGN) void gemm_mxfp4_tile_kernel(
    const uint8_t* __restrict__ qx, const uint8_t* __restrict__ sx, const uint8_t* __restrict__ qw,
    const uint8_t* __restrict__ sw, void* __restrict__ y, int64_t M, int64_t N, int K, int tiles_m, int tiles_n,
    bool vec) {
    using S = Shape<TM, TN, WGM, WGN, ST, SDMA>;
    extern __shared__ __align__(16) uint8_t lds[];
    const int lane = threadIdx.x & 63, tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave / WGN, wn = wave % WGN;
    const int i16 = lane & 15, kb = lane >> 4;

    // Workgroup b runs on XCD b % 8; each XCD takes a contiguous share of the tile
    // list, ordered in groups of kGroupM row tiles walked column by column.
    const int wg = blockIdx.x, nb = gridDim.x;
    const int xcd = wg % 8, q8 = nb / 8, r8 = nb % 8;
    const int lin = xcd * q8 + min(xcd, r8) + wg / 8;
    const int per_group = kGroupM * tiles_n;
    const int first_m = (lin / per_group) * kGroupM;
    const int group_m = min(tiles_m - first_m, kGroupM);
    const int tm = first_m + (lin % per_group) % group_m;
    const int tn = (lin % per_group) / group_m;
    const int64_t m0 = static_cast<int64_t>(tm) * S::kRowsM, n0 = static_cast<int64_t>(tn) * S::kRowsN;

    const int kbytes = K / 2, blocks = K / kBlock;
    const int steps = (kbytes + kBK - 1) / kBK, full = kbytes / kBK;
    const int groups = full / kGroup;  // groups of four whole steps
    const uint8_t* xbase = qx + m0 * kbytes;
    const uint8_t* wbase = qw + n0 * kbytes;
    const int xrows = static_cast<int>(min(M - m0, int64_t{S::kRowsM})), wrows = static_cast<int>(min(N - n0, int64_t{S::kRowsN}));
    // load i of a wave carries rows 8 (kPer wave + i) .. + 7, lane l row l / 8 of
    // them, chunk (l % 8) ^ swizzle(row)
    auto row_in = [&](int per, int i) { return 8 * (per * wave + i) + (lane >> 3); };
    uint32_t xo[S::kPerM], wo[S::kPerN];
#pragma unroll
    for (int i = 0; i < S::kPerM; ++i) {
        const int row = row_in(S::kPerM, i);
        xo[i] = static_cast<uint32_t>(min(row, xrows - 1)) * kbytes + 16 * ((lane & 7) ^ swizzle(row));
    }
#pragma unroll
    for (int i = 0; i < S::kPerN; ++i) {
        const int row = row_in(S::kPerN, i);
        wo[i] = static_cast<uint32_t>(min(row, wrows - 1)) * kbytes + 16 * ((lane & 7) ^ swizzle(row));
    }
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<size_t>((lds_void*)lds));
    auto stage_at = [&](int s) { return lds + (s % ST) * S::kStage; };
    auto dma_one = [&](int u, int k0, uint32_t st) {
        if (u < S::kPerM) kc::lds_dma16(xo[u], xbase + k0, st + 1024 * (S::kPerM * wave + u));
        else kc::lds_dma16(wo[u - S::kPerM], wbase + k0, st + S::kRowsM * kBK + 1024 * (S::kPerN * wave + u - S::kPerM));
    };
    auto stage_lds = [&](int s) { return __builtin_amdgcn_readfirstlane(lds0 + (s % ST) * S::kStage); };
    auto dma = [&](int s) {  // a whole step
        const uint32_t st = stage_lds(s);
#pragma unroll
        for (int u = 0; u < S::kLoads; ++u) dma_one(u, s * kBK, st);
    };
    auto dma_partial = [&](int s) {  // chunks past K load the last one
        const uint32_t st = stage_lds(s);
        const uint32_t last = kbytes - 16;
#pragma unroll
        for (int u = 0; u < S::kLoads; ++u) {
            const bool m = u < S::kPerM;
            const int per = m ? S::kPerM : S::kPerN, v = m ? u : u - S::kPerM;
            const int row = row_in(per, v);
            const uint32_t at = static_cast<uint32_t>(min(row, (m ? xrows : wrows) - 1)) * kbytes +
                                min(static_cast<uint32_t>(s) * kBK + 16 * ((lane & 7) ^ swizzle(row)), last);
            kc::lds_dma16(at, m ? xbase : wbase, st + (m ? 0 : S::kRowsM * kBK) + 1024 * (per * wave + v));
        }
    };

    // scale bytes of group g of this thread's rows
    u32x4 sreg[S::kRowsPerThread][2];
    auto scale_row = [&](int r) {
        return r < S::kRowsM ? sx + (m0 + min(r, xrows - 1)) * blocks : sw + (n0 + min(r - S::kRowsM, wrows - 1)) * blocks;
    };
    auto fetch_scales = [&](int g) {
#pragma unroll
        for (int t = 0; t < S::kRowsPerThread; ++t) {
            const int r = tid + t * S::kThreads;
            if (r < S::kRows) {
                const uint8_t* p = scale_row(r) + 32 * g;
                __builtin_memcpy(&sreg[t][0], p, 16);
                __builtin_memcpy(&sreg[t][1], p + 16, 16);
            }
        }
    };
    // SDMA: the same straight into LDS, 32 rows a load, half a row per lane
    auto dma_scales = [&](int g) {
#pragma unroll
        for (int u = 0; u < S::kScaleLoads; ++u) {
            const int first = 32 * (wave + S::kWaves * u);
            if (first >= S::kRows) continue;
            const bool m = first < S::kRowsM;
            const int r = first + (lane >> 1) - (m ? 0 : S::kRowsM);
            const uint32_t at = static_cast<uint32_t>(min(r, (m ? xrows : wrows) - 1)) * static_cast<uint32_t>(blocks) + 16 * (lane & 1);
            kc::lds_dma16(at, (m ? sx + m0 * blocks : sw + n0 * blocks) + 32 * g,
                      __builtin_amdgcn_readfirstlane(lds0 + S::kRawOff + 32 * first));
        }
    };
    auto raw_scales = [&] {
#pragma unroll
        for (int t = 0; t < S::kRowsPerThread; ++t) {
            const int r = tid + t * S::kThreads;
            if (r < S::kRows) {
                const u32x4* p = reinterpret_cast<const u32x4*>(lds + S::kRawOff + 32 * r);
                sreg[t][0] = p[0];
                sreg[t][1] = p[1];
            }
        }
    };
    auto fetch_scales_partial = [&](int g) {
#pragma unroll
        for (int t = 0; t < S::kRowsPerThread; ++t) {
            const int r = tid + t * S::kThreads;
            uint32_t d[8];
            const uint8_t* p = scale_row(min(r, S::kRows - 1)) + 32 * g;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                d[j] = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (32 * g + 4 * j + e < blocks) d[j] |= static_cast<uint32_t>(p[4 * j + e]) << (8 * e);
            }
            sreg[t][0] = u32x4{d[0], d[1], d[2], d[3]};
            sreg[t][1] = u32x4{d[4], d[5], d[6], d[7]};
        }
    };
    // step s of the group has bytes 8 s .. 8 s + 7; lane kb takes 2 kb and 2 kb + 1
    auto store_scales = [&] {
#pragma unroll
        for (int t = 0; t < S::kRowsPerThread; ++t) {
            const int r = tid + t * S::kThreads;
            if (r < S::kRows) {
                const u32x4 p = sreg[t][0], q = sreg[t][1];
                auto lo = [](uint32_t u, uint32_t v) { return (u & 0xFFFFu) | (v << 16); };
                auto hi = [](uint32_t u, uint32_t v) { return (u >> 16) | (v & 0xFFFF0000u); };
                u32x4* d = reinterpret_cast<u32x4*>(lds + S::kScaleOff + 32 * r);
                d[0] = u32x4{lo(p.x, p.z), lo(q.x, q.z), hi(p.x, p.z), hi(q.x, q.z)};
                d[1] = u32x4{lo(p.y, p.w), lo(q.y, q.w), hi(p.y, p.w), hi(q.y, q.w)};
            }
        }
    };

    u32x4 a[TM], b[2][TN];  // A of the half at hand, replaced row by row; B of both halves
    uint32_t sa[TM][2], sb[TN][2];  // scales of the group: steps 0, 1 and 2, 3
    const int arow = 16 * TM * wm + i16, brow = 16 * TN * wn + i16;
    auto read_scales = [&](int w) {
        const uint8_t* base = lds + S::kScaleOff + 8 * kb + 4 * w;
#pragma unroll
        for (int i = 0; i < TM; ++i) sa[i][w] = *reinterpret_cast<const uint32_t*>(base + 32 * (arow + 16 * i));
#pragma unroll
        for (int j = 0; j < TN; ++j)
            sb[j][w] = *reinterpret_cast<const uint32_t*>(base + 32 * (S::kRowsM + brow + 16 * j));
    };
    // operands of half h from a step's buffer (16-row blocks start at multiples of 16)
    auto read_a = [&](int i, const uint8_t* st, int h) {
        a[i] = *reinterpret_cast<const u32x4*>(st + (arow + 16 * i) * kBK + 16 * ((2 * kb + h) ^ swizzle(i16)));
    };
    auto read_b = [&](int j, const uint8_t* st, int h) {
        b[h][j] = *reinterpret_cast<const u32x4*>(st + (S::kRowsM + brow + 16 * j) * kBK + 16 * ((2 * kb + h) ^ swizzle(i16)));
    };
    f32x4 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    start(acc);
    // scalar loads still in flight would make every LDS wait a full drain
    asm volatile("" ::"s"(y), "s"(M), "s"(N));

    auto mfma_row = [&](auto pc, auto hc, int i, auto between) {
        constexpr int p = decltype(pc)::value, h = decltype(hc)::value, w = p >> 1, byte = 2 * (p & 1) + h;
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            mfma<byte>(acc[i][j], b[h][j], a[i], sb[j][w], sa[i][w]);
            between(j);
        }
        __builtin_amdgcn_sched_barrier(0);
    };

    if (groups > 0) {
        const int last = kGroup * groups - 1;
        if constexpr (SDMA) {
            dma_scales(0);
        } else {
            fetch_scales(0);
            store_scales();
        }
#pragma unroll
        for (int s = 0; s < ST; ++s) dma(min(s, last));
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(S::kLoads * (ST - 1)) : "memory");
        if constexpr (SDMA) {
            raw_scales();
            store_scales();
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        }
        read_scales(0);
#pragma unroll
        for (int j = 0; j < TN; ++j) read_b(j, stage_at(0), 0);
#pragma unroll
        for (int i = 0; i < TM; ++i) read_a(i, stage_at(0), 0);
        // Step s, at place p of its group.  Half 0: as soon as a row of MFMAs has
        // taken its A operand the register gets the row's operand of half 1.  Half 1
        // opens with kWait rows, in which the last of those reads land; then the
        // barrier (step s + 1 is here, and nobody reads step s's buffer any more), the
        // loads of step s + ST and the reads of half 0 of step s + 1.
        constexpr int kWait = TM >= 8 ? 2 : 1, kOpen = (TM - kWait) * TN;
        auto step = [&](auto pc, int g) {
            constexpr int p = decltype(pc)::value;
            constexpr std::integral_constant<int, 0> first{};
            constexpr std::integral_constant<int, 1> second{};
            const int s = kGroup * g + p;
            const uint8_t* cur = stage_at(s);
            const uint8_t* nxt = stage_at(s + 1);
            if constexpr (p == 0) read_scales(1);
#pragma unroll
            for (int i = 0; i < TM; ++i) {
                mfma_row(pc, first, i, [&](int j) {
                    if (i == 0) read_b(j, cur, 1);
                });
                read_a(i, cur, 1);
            }
#pragma unroll
            for (int i = 0; i < kWait; ++i) mfma_row(pc, second, i, [](int) {});
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(S::kLoads * (ST - 2)) : "memory");
            if constexpr (SDMA) {  // two barriers on the loads are among the waited for
                if constexpr (p == 0) dma_scales(min(g + 1, groups - 1));
                if constexpr (p == 2) {
                    raw_scales();
                    store_scales();
                }
                if constexpr (p == 3) read_scales(0);
            } else {
                if constexpr (p == 0) {
                    if (g + 1 < groups) fetch_scales(g + 1);
                }
                if constexpr (p == 1) {
                    if (g + 1 < groups) store_scales();
                }
                if constexpr (p == 2) read_scales(0);
            }
            const int k0 = min(s + ST, last) * kBK;
            const uint32_t st = stage_lds(s);
#pragma unroll
            for (int i = kWait; i < TM; ++i) {
                mfma_row(pc, second, i, [&](int j) {
                    const int q = (i - kWait) * TN + j;
                    if (i == kWait) read_b(j, nxt, 0);
#pragma unroll
                    for (int u = q * S::kLoads / kOpen; u < (q + 1) * S::kLoads / kOpen; ++u) dma_one(u, k0, st);
                });
                if (i == kWait) {
#pragma unroll
                    for (int v = 0; v < kWait; ++v) read_a(v, nxt, 0);
                }
                read_a(i, nxt, 0);
            }
        };
        for (int g = 0; g < groups; ++g) {
            step(std::integral_constant<int, 0>{}, g);
            step(std::integral_constant<int, 1>{}, g);
            step(std::integral_constant<int, 2>{}, g);
            step(std::integral_constant<int, 3>{}, g);
        }
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }
    if (kGroup * groups < steps) {
        // the last steps, ST at a time
        fetch_scales_partial(groups);
        store_scales();
        for (int s0 = kGroup * groups; s0 < steps; s0 += ST) {
            const int n = min(ST, steps - s0);
            for (int t = 0; t < n; ++t) {
                if (s0 + t < full) dma(s0 + t);
                else dma_partial(s0 + t);
            }
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
            for (int t = 0; t < n; ++t) {
                const uint8_t* st = stage_at(s0 + t);
                const uint8_t* sc = lds + S::kScaleOff + 8 * kb + 2 * ((s0 + t) % kGroup);
                uint32_t ta[TM], tb[TN];
#pragma unroll
                for (int i = 0; i < TM; ++i) ta[i] = *reinterpret_cast<const uint16_t*>(sc + 32 * (arow + 16 * i));
#pragma unroll
                for (int j = 0; j < TN; ++j) tb[j] = *reinterpret_cast<const uint16_t*>(sc + 32 * (S::kRowsM + brow + 16 * j));
                auto one = [&](auto hc) {
                    constexpr int h = decltype(hc)::value;
#pragma unroll
                    for (int j = 0; j < TN; ++j) read_b(j, st, h);
#pragma unroll
                    for (int i = 0; i < TM; ++i) read_a(i, st, h);
#pragma unroll
                    for (int i = 0; i < TM; ++i)
#pragma unroll
                        for (int j = 0; j < TN; ++j)
                            mfma<h>(acc[i][j], b[h][j], a[i], tb[j], ta[i]);
                };
                one(std::integral_constant<int, 0>{});
                one(std::integral_constant<int, 1>{});
            }
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        }
    }

    // D of a 16 x 16 tile: lane (j, g) holds columns n = 4 g + v of row m = j.
    // bf16 rows are put together in the wave's own LDS, 16 rows of 16 TN columns at a
    // time, and leave in pieces of 16 bytes per lane.
    settle(acc);
    const int64_t mw = m0 + 16 * TM * wm, nw = n0 + 16 * TN * wn;
    if constexpr (YBF16 && TN > 1) {
        if (vec) {
            constexpr int kChunks = 2 * TN;              // 16-byte chunks of a row
            constexpr int kPasses = 16 * kChunks / 64;   // of the wave
            static_assert(kPasses * 64 == 16 * kChunks, "whole passes");
            uint8_t* wl = lds + wave * (16 * 32 * TN);
#pragma unroll
            for (int i = 0; i < TM; ++i) {
#pragma unroll
                for (int j = 0; j < TN; ++j) {
                    const f32x4 v = acc[i][j];
                    const int c = (2 * j + (kb >> 1)) ^ (i16 & (kChunks - 1));
                    *reinterpret_cast<u32x2*>(wl + i16 * 32 * TN + 16 * c + 8 * (kb & 1)) =
                        u32x2{kc::pack_bf16x2(v.x, v.y), kc::pack_bf16x2(v.z, v.w)};
                }
#pragma unroll
                for (int t = 0; t < kPasses; ++t) {
                    const int row = (64 * t + lane) / kChunks, c = (64 * t + lane) % kChunks;
                    const u32x4 v = *reinterpret_cast<const u32x4*>(wl + row * 32 * TN + 16 * (c ^ (row & (kChunks - 1))));
                    const int64_t m = mw + 16 * i + row, n = nw + 8 * c;
                    if (m < M && n < N)
                        __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(static_cast<uint16_t*>(y) + m * N + n));
                }
            }
            return;
        }
    }
#pragma unroll
    for (int i = 0; i < TM; ++i) {
        const int64_t m = mw + 16 * i + i16;
        if (m >= M) continue;
#pragma unroll
        for (int j = 0; j < TN; ++j) {
            const int64_t n = nw + 16 * j + 4 * kb;
            const f32x4 v = acc[i][j];
            if (vec && n < N) {
                if constexpr (YBF16)
                    *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(y) + m * N + n) =
                        u32x2{kc::pack_bf16x2(v.x, v.y), kc::pack_bf16x2(v.z, v.w)};
                else *reinterpret_cast<f32x4*>(static_cast<float*>(y) + m * N + n) = v;
                continue;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if (n + e >= N) break;
                if constexpr (YBF16) static_cast<uint16_t*>(y)[m * N + n + e] = kc::f32_to_bf16(v[e]);
                else static_cast<float*>(y)[m * N + n + e] = v[e];
            }
        }
    }
}

template <int TM, int TN, int WGM, int WGN, int ST, bool SDMA, bool YBF16>
int launch_tile(const char* fn, const uint8_t* qx, const uint8_t* sx, const uint8_t* qw, const uint8_t* sw, void* y, int64_t M,
                int64_t N, int64_t K, hipStream_t stream) {
    using S = Shape<TM, TN, WGM, WGN, ST, SDMA>;
    const int st = raise_lds_limit<gemm_mxfp4_tile_kernel<TM, TN, WGM, WGN, ST, SDMA, YBF16>>(fn, S::kLds);
    if (st != KC_SUCCESS) return st;
    const int64_t tm = (M + S::kRowsM - 1) / S::kRowsM, tn = (N + S::kRowsN - 1) / S::kRowsN;
    const bool vec = YBF16 ? N % 8 == 0 && kc::aligned(y, 16) : N % 4 == 0 && kc::aligned(y, 16);
    gemm_mxfp4_tile_kernel<TM, TN, WGM, WGN, ST, SDMA, YBF16><<<static_cast<unsigned>(tm * tn), S::kThreads, S::kLds, stream>>>(
        qx, sx, qw, sw, y, M, N, static_cast<int>(K), static_cast<int>(tm), static_cast<int>(tn), vec);
    return kc::check_launch(fn);
}

template <int TM, int TN, int WGM, int WGN, int ST, bool YBF16>
int launch(const char* fn, const uint8_t* qx, const uint8_t* sx, const uint8_t* qw, const uint8_t* sw, void* y, int64_t M,
           int64_t N, int64_t K, hipStream_t stream) {
    if constexpr (ST > 2) {
        if (K % (4 * kBlock) == 0 && kc::aligned(sx, 4) && kc::aligned(sw, 4))
            return launch_tile<TM, TN, WGM, WGN, ST, true, YBF16>(fn, qx, sx, qw, sw, y, M, N, K, stream);
    }
    return launch_tile<TM, TN, WGM, WGN, ST, false, YBF16>(fn, qx, sx, qw, sw, y, M, N, K, stream);
}

// Tiles, and what one costs a CU in hundredths of a microsecond: per step of 256
// values, and beside the steps (start, first loads, stores), alone on its CU and
// as one of two.  Measured with K 1024 to 14336 on grids of 64 to 1024 tiles; the
// least expected time wins (22 shapes of 64 to 8192 rows: the fastest tile on 18, 8 % from it on
// one, 3 % at most on the others).  Against
// the 256 x 256 tile: M 128, N 4096, K 4096 29.1 -> 6.8 us (32 x 64); M 1000, N 4096,
// K 14336 103 -> 41.5 (128 x 128, eight waves and four buffers, one a CU; four waves 43.1);
// M 500, N 6144, K 4096 32.9 -> 14.8 (the same); M 64, N 28672, K 4096 32.0 -> 15.1 (64 x 128); M 2048, N 4096, K 4096 34.2 ->
// 26.0 (256 x 128, eight waves; four 27.2); M 3000, N 4096 34.6 and M 300, N 28672 38.1 stay (256 x 128: 43.5 and 46.6).
struct TileCost {
    int rows_m, rows_n, step, fixed, step2, fixed2;  // step2, fixed2: two of them (0: one a CU)
};
constexpr int kCus = 256;
constexpr TileCost kTiles[] = {{256, 256, 205, 300, 0, 0},
                               {256, 128, 140, 200, 0, 0},
                               {128, 128, 91, 300, 145, 240},
                               {128, 128, 65, 500, 0, 0},
                               {64, 64, 35, 260, 62, 210},
                               {64, 128, 52, 340, 0, 0},
                               {32, 64, 30, 190, 45, 150}};

int best_tile(int64_t M, int64_t N, int64_t K) {
    const int64_t steps = (K + 2 * kBK - 1) / (2 * kBK);
    int best = 0;
    int64_t least = INT64_MAX;
    for (int i = 0; i < static_cast<int>(sizeof(kTiles) / sizeof(kTiles[0])); ++i) {
        const TileCost& t = kTiles[i];
        const int64_t tiles = ((M + t.rows_m - 1) / t.rows_m) * ((N + t.rows_n - 1) / t.rows_n);
        const int64_t per_cu = (tiles + kCus - 1) / kCus;
        const int64_t one = steps * t.step + t.fixed, two = steps * t.step2 + t.fixed2;
        const int64_t cost = t.step2 ? per_cu / 2 * two + per_cu % 2 * one : per_cu * one;
        if (cost < least) least = cost, best = i;
    }
    return best;
}

}  // namespace

namespace kc {
namespace mx {

template <bool YBF16>
int gemm_tile(const char* fn, const uint8_t* qx, const uint8_t* sx, const uint8_t* qw, const uint8_t* sw, void* y, int64_t M,
              int64_t N, int64_t K, hipStream_t stream) {
    switch (best_tile(M, N, K)) {
        case 0: return launch<8, 8, 2, 2, 2, YBF16>(fn, qx, sx, qw, sw, y, M, N, K, stream);
        case 1: return launch<4, 4, 4, 2, 2, YBF16>(fn, qx, sx, qw, sw, y, M, N, K, stream);
        case 2: return launch<4, 4, 2, 2, 2, YBF16>(fn, qx, sx, qw, sw, y, M, N, K, stream);
        case 3: return launch<4, 2, 2, 4, 4, YBF16>(fn, qx, sx, qw, sw, y, M, N, K, stream);
        case 4: return launch<2, 2, 2, 2, 4, YBF16>(fn, qx, sx, qw, sw, y, M, N, K, stream);
        case 5: return launch<4, 2, 1, 4, 4, YBF16>(fn, qx, sx, qw, sw, y, M, N, K, stream);
        default: return launch<2, 1, 1, 4, 4, YBF16>(fn, qx, sx, qw, sw, y, M, N, K, stream);
    }
}

template int gemm_tile<true>(const char*, const uint8_t*, const uint8_t*, const uint8_t*, const uint8_t*, void*, int64_t,
                             int64_t, int64_t, hipStream_t);
template int gemm_tile<false>(const char*, const uint8_t*, const uint8_t*, const uint8_t*, const uint8_t*, void*, int64_t,
                              int64_t, int64_t, hipStream_t);

}  // namespace mx
}  // namespace kc
