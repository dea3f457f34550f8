// mxfp4_gemm_a16_tile.hip -- bf16 activations times MXFP4 weights on gfx950 for
// batches of tokens on layers of many rows, where the kernel of mxfp4_gemm_a16.hip
// reads X too often.  Y[m, n] = sum_k x[m, k] e2m1(qw[n, k]) 2^(sw[n, k / 32] - 127).
//
// A workgroup computes 16 MT tokens x 128 rows of W with eight waves: wave (g, w)
// takes rows 32 w .. 32 w + 31 and blocks 4 g .. 4 g + 3 of every step of 256 values; the
// two halves of K meet in LDS at the end.  X, the codes and the scales of a step go
// from global memory straight into LDS through a ring of ST buffers, so every byte
// of X is fetched once per 128 rows and no register holds a load in flight.  Rows are
// whole in LDS (512 bytes of X, 128 of codes) with their 16-byte chunks XOR-swizzled
// by the row: lane (i, g) then reads 16 bytes of X row i and the dword g of a block of
// W row i, 8 values of K each, without bank conflicts, decodes the codes with their
// scale (v_cvt_scalef32_pk_bf16_fp4) and multiplies on the bf16 matrix cores.
//
// Bound by the arrival of the steps in LDS (512 bytes of X a token and 128 of codes a
// row): M 64, N 28672, K 4096 24 us, the weights alone 10.5.
//
// Rows past M or N load the last row and feed outputs that are not stored.  K is a
// multiple of 128: in a last half step the second half of the waves has nothing to
// do, and what lies past K loads the last valid chunk and is not read.
#include <algorithm>
#include <type_traits>

#include "mxfp4_gemm.hpp"

namespace {

using namespace kc::mx;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) void lds_void;

constexpr int kStep = 256;                 // values of K per step
constexpr int kRowsN = 128, kThreads = 512, kWaves = 8;
constexpr int kRT = 2;                     // tiles of 16 rows of a wave

template <int MT>
struct Shape {
    static constexpr int kX = 16 * MT * 512, kW = kRowsN * 128, kS = kRowsN * 8;
    static constexpr int kStage = kX + kW + kS;
    static constexpr int ST = std::min(6, 160 * 1024 / kStage);
    static constexpr int kLds = ST * kStage;
    static constexpr int kXLoads = kX / 1024 / kWaves, kWLoads = kW / 1024 / kWaves;  // of a wave and step
    static constexpr int kLoads = kXLoads + kWLoads + 1;
    static_assert(kXLoads * 1024 * kWaves == kX && kWLoads * 1024 * kWaves == kW, "whole loads per wave");
};

// 16 (4) bytes per lane from sbase + voff into LDS at lds_base + 16 (4) * lane.
__device__ __forceinline__ void lds_dma16(uint32_t voff, const void* sbase, uint32_t lds_base) {
    asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(sbase), "s"(lds_base)
                 : "memory", "m0");
}
__device__ __forceinline__ void lds_dma4(uint32_t voff, const void* sbase, uint32_t lds_base) {
    asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dword %0, %1" ::"v"(voff), "s"(sbase), "s"(lds_base)
                 : "memory", "m0");
}

__device__ __forceinline__ bf16x8 decode(uint32_t c, uint32_t b) {
    const float s = scale_operand(b);
    const bf16x2 p = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0), q = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1);
    const bf16x2 r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2), t = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3);
    return bf16x8{p.x, p.y, q.x, q.y, r.x, r.y, t.x, t.y};
}

template <int MT>
__global__ __launch_bounds__(kThreads) void gemm_mxfp4_a16_tile_kernel(const uint8_t* __restrict__ qw,
                                                                       const uint8_t* __restrict__ sw,
                                                                       const uint16_t* __restrict__ x,
                                                                       uint16_t* __restrict__ y, int M, int N, int K,
                                                                       bool vec) {
    using S = Shape<MT>;
    extern __shared__ __align__(16) uint8_t lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const int kg = wave >> 2, wn = wave & 3;
    const int i = lane & 15, g = lane >> 4;
    const int n0 = static_cast<int>(blockIdx.x) * kRowsN, m0 = static_cast<int>(blockIdx.y) * 16 * MT;
    const uint32_t kbytes = K / 2, blocks = K / kBlock;
    const int steps = (K + kStep - 1) / kStep;
    const uint8_t* xbase = reinterpret_cast<const uint8_t*>(x + static_cast<int64_t>(m0) * K);
    const uint8_t* wbase = qw + static_cast<int64_t>(n0) * kbytes;
    const uint8_t* sbase = sw + static_cast<int64_t>(n0) * blocks;
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<size_t>((lds_void*)lds));

    // A wave's loads of a step: 2 rows of X each, 8 rows of W each, and the scales of
    // 16 rows; chunk c of row r lies in slot c ^ (r % 16) (X) or c ^ (r / 2 % 8) (W).
    uint32_t xrow[S::kXLoads], xchunk[S::kXLoads], wrow[S::kWLoads], wchunk[S::kWLoads];
#pragma unroll
    for (int u = 0; u < S::kXLoads; ++u) {
        const int r = 2 * (S::kXLoads * wave + u) + (lane >> 5), slot = lane & 31;
        xrow[u] = static_cast<uint32_t>(min(m0 + r, M - 1) - m0) * (2u * K);
        xchunk[u] = 16u * (slot ^ (r & 15));
    }
#pragma unroll
    for (int u = 0; u < S::kWLoads; ++u) {
        const int r = 8 * (S::kWLoads * wave + u) + (lane >> 3), slot = lane & 7;
        wrow[u] = static_cast<uint32_t>(min(n0 + r, N - 1) - n0) * kbytes;
        wchunk[u] = 16u * (slot ^ ((r >> 1) & 7));
    }
    const uint32_t srow = static_cast<uint32_t>(min(n0 + 16 * wave + (lane >> 1), N - 1) - n0) * blocks;
    auto load = [&](int s) {
        const uint32_t st = __builtin_amdgcn_readfirstlane(lds0 + (s % S::ST) * S::kStage);
        const uint32_t k0 = static_cast<uint32_t>(s) * kStep;
#pragma unroll
        for (int u = 0; u < S::kXLoads; ++u)
            lds_dma16(xrow[u] + min(2 * k0 + xchunk[u], 2u * K - 16), xbase, st + 1024 * (S::kXLoads * wave + u));
#pragma unroll
        for (int u = 0; u < S::kWLoads; ++u)
            lds_dma16(wrow[u] + min(k0 / 2 + wchunk[u], kbytes - 16), wbase, st + S::kX + 1024 * (S::kWLoads * wave + u));
        if (lane < 32)
            lds_dma4(srow + min(k0 / kBlock + 4 * (lane & 1), blocks - 4), sbase, st + S::kX + S::kW + 128 * wave);
    };

    f32x4 acc[kRT][MT];
#pragma unroll
    for (int r = 0; r < kRT; ++r)
#pragma unroll
        for (int c = 0; c < MT; ++c) acc[r][c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    asm volatile("" ::"s"(y), "s"(M), "s"(N));

    constexpr int kAhead = S::ST - 1;  // steps on their way while one is multiplied
#pragma unroll
    for (int p = 0; p < kAhead; ++p) load(min(p, steps - 1));
    for (int s = 0; s < steps; ++s) {
        // step s has landed, and everyone has read step s - 1, whose buffer is next
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(S::kLoads * (kAhead - 1)) : "memory");
        load(min(s + kAhead, steps - 1));
        if (kg == 1 && static_cast<uint32_t>(s) * kStep + kStep / 2 >= static_cast<uint32_t>(K)) continue;  // nothing past K
        const uint8_t* st = lds + (s % S::ST) * S::kStage;
        uint32_t sc[kRT];
#pragma unroll
        for (int r = 0; r < kRT; ++r)
            sc[r] = *reinterpret_cast<const uint32_t*>(st + S::kX + S::kW + 8 * (32 * wn + 16 * r + i) + 4 * kg);
        // every read of the step ahead of its first use
        uint32_t code[4][kRT];
        bf16x8 xv[4][MT];
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            const int blk = 4 * kg + b;
#pragma unroll
            for (int r = 0; r < kRT; ++r) {
                const int row = 32 * wn + 16 * r + i;
                code[b][r] = *reinterpret_cast<const uint32_t*>(st + S::kX + row * 128 + 16 * (blk ^ ((row >> 1) & 7)) + 4 * g);
            }
#pragma unroll
            for (int c = 0; c < MT; ++c)
                xv[b][c] = *reinterpret_cast<const bf16x8*>(st + (16 * c + i) * 512 + 16 * ((4 * blk + g) ^ i));
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int b = 0; b < 4; ++b)
#pragma unroll
            for (int r = 0; r < kRT; ++r) {
                const bf16x8 wv = decode(code[b][r], (sc[r] >> (8 * b)) & 255);
#pragma unroll
                for (int c = 0; c < MT; ++c) acc[r][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv, xv[b][c], acc[r][c], 0, 0, 0);
            }
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    f32x4* red = reinterpret_cast<f32x4*>(lds);  // [wn][tile][lane]
    if (kg == 1) {
#pragma unroll
        for (int r = 0; r < kRT; ++r)
#pragma unroll
            for (int c = 0; c < MT; ++c) red[((wn * kRT + r) * MT + c) * 64 + lane] = acc[r][c];
    }
    __syncthreads();
    if (kg == 1) return;
    // D: lane (i, g) holds rows n = 4 g + v of token i
#pragma unroll
    for (int c = 0; c < MT; ++c) {
        const int m = m0 + 16 * c + i;
        if (m >= M) continue;
#pragma unroll
        for (int r = 0; r < kRT; ++r) {
            const f32x4 o = red[((wn * kRT + r) * MT + c) * 64 + lane];
            const f32x4 v = {acc[r][c].x + o.x, acc[r][c].y + o.y, acc[r][c].z + o.z, acc[r][c].w + o.w};
            const int n = n0 + 32 * wn + 16 * r + 4 * g;
            uint16_t* out = y + static_cast<int64_t>(m) * N + n;
            if (vec && n < N) {
                *reinterpret_cast<u32x2*>(out) = u32x2{kc::pack_bf16x2(v.x, v.y), kc::pack_bf16x2(v.z, v.w)};
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (n + e < N) out[e] = kc::f32_to_bf16(v[e]);
            }
        }
    }
}

template <int MT>
int launch(const char* fn, const uint8_t* qw, const uint8_t* sw, const uint16_t* x, uint16_t* y, int M, int N, int K,
           hipStream_t stream) {
    using S = Shape<MT>;
    const int st = raise_lds_limit<gemm_mxfp4_a16_tile_kernel<MT>>(fn, S::kLds);
    if (st != KC_SUCCESS) return st;
    const dim3 grid((N + kRowsN - 1) / kRowsN, (M + 16 * MT - 1) / (16 * MT));
    gemm_mxfp4_a16_tile_kernel<MT><<<grid, kThreads, S::kLds, stream>>>(qw, sw, x, y, M, N, K,
                                                                        N % 4 == 0 && kc::aligned(y, 8));
    return kc::check_launch(fn);
}

}  // namespace

namespace kc {
namespace mx {

int gemm_a16_tile(const char* fn, int mt, const uint8_t* qw, const uint8_t* sw, const uint16_t* x, uint16_t* y, int M, int N,
                  int K, hipStream_t stream) {
    switch (mt) {
        case 2: return launch<2>(fn, qw, sw, x, y, M, N, K, stream);
        case 3: return launch<3>(fn, qw, sw, x, y, M, N, K, stream);
        default: return launch<4>(fn, qw, sw, x, y, M, N, K, stream);
    }
}

}  // namespace mx
}  // namespace kc
