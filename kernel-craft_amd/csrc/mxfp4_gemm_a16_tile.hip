// mxfp4_gemm_a16_tile.hip -- bf16 activations times MXFP4 weights on gfx950 for
// batches of tokens on layers of many rows, where the kernel of mxfp4_gemm_a16.hip
// reads X too often.  Y[m, n] = sum_k x[m, k] e2m1(qw[n, k]) 2^(sw[n, k / 32] - 127).
//
// A workgroup computes 16 MT TG tokens x 128 rows of W with eight waves: half of them
// take the first blocks of every step of STEP values of K and half the others, and the
// two halves meet in LDS at the end; the four waves of a half share the tokens in TG
// groups and the rows.  X, the codes and the scales of a step go from global memory
// straight into LDS through a ring of ST buffers, so every byte of X is fetched once per
// 128 rows and no register holds a load in flight.  Rows are whole in LDS (512 bytes of
// X, 128 of codes) with their 16-byte chunks XOR-swizzled by the row: lane (i, g) then
// reads 16 bytes of X row i and the dword g of a block of W row i, 8 values of K each,
// without bank conflicts, decodes the codes with their scale
// (v_cvt_scalef32_pk_bf16_fp4) and multiplies on the bf16 matrix cores.
//
// A step's operands are read, and the loads of a later one issued, between the matrix
// instructions of the step before: all of them ahead of the matrix instructions keep a
// wave, which issues in order, from those until LDS has taken them (M 128, N 4096,
// K 4096 in tiles of 64 tokens 21.8 -> 17.8 us, of 128 36 -> 30.5).  Full grids are bound by
// the arrival of the steps (512 bytes of X a token and 128 of codes a row, 10 TB/s): M 64,
// N 28672, K 4096 24 us, the weights alone 10.5; M 128 38.  128 tokens take half the
// reads of W and its decoding, and steps of 128 values, since 256 leave one buffer.
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

constexpr int kRowsN = 128, kThreads = 512, kWaves = 8;

// TG groups of MT tiles of 16 tokens, steps of STEP values of K.
template <int TG, int MT, int STEP>
struct Shape {
    static constexpr int kTokens = 16 * MT * TG;
    static constexpr int kWn = kWaves / 2 / TG, kRT = kRowsN / 16 / kWn;  // groups of rows, tiles of 16 of each
    static constexpr int kXRow = 2 * STEP, kWRow = STEP / 2, kSRow = STEP / kBlock;  // bytes of a row and step
    static constexpr int kX = kTokens * kXRow, kW = kRowsN * kWRow, kS = kRowsN * kSRow;
    static constexpr int kStage = kX + kW + kS;
    static constexpr int ST = std::min(6, 160 * 1024 / kStage);
    static constexpr int kLds = ST * kStage;
    static constexpr int kXLoads = kX / 1024 / kWaves, kWLoads = kW / 1024 / kWaves;  // of a wave and step
    static constexpr int kLoads = kXLoads + kWLoads + 1;
    static_assert(kXLoads * 1024 * kWaves == kX && kWLoads * 1024 * kWaves == kW, "whole loads per wave");
    static_assert(ST >= 3 && kWn * TG * kRT * MT * 1024 <= kLds, "LDS");
};

__device__ __forceinline__ bf16x8 decode(uint32_t c, uint32_t b) {
    const float s = scale_operand(b);
    const bf16x2 p = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0), q = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1);
    const bf16x2 r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2), t = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3);
    return bf16x8{p.x, p.y, q.x, q.y, r.x, r.y, t.x, t.y};
}

template <int TG, int MT, int STEP>
__global__ __launch_bounds__(kThreads) void gemm_mxfp4_a16_tile_kernel(const uint8_t* __restrict__ qw,
                                                                       const uint8_t* __restrict__ sw,
                                                                       const uint16_t* __restrict__ x,
                                                                       uint16_t* __restrict__ y, int M, int N, int K,
                                                                       bool vec) {
    using S = Shape<TG, MT, STEP>;
    constexpr int kRT = S::kRT, kHalf = STEP / 2 / kBlock;  // blocks of a wave's half step
    extern __shared__ __align__(16) uint8_t lds[];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const int kg = wave >> 2, tile = wave & 3, wn = tile % S::kWn, tg = tile / S::kWn;
    const int i = lane & 15, g = lane >> 4;
    const int n0 = static_cast<int>(blockIdx.x) * kRowsN, m0 = static_cast<int>(blockIdx.y) * S::kTokens;
    const uint32_t kbytes = K / 2, blocks = K / kBlock;
    const int steps = (K + STEP - 1) / STEP;
    const uint8_t* xbase = reinterpret_cast<const uint8_t*>(x + static_cast<int64_t>(m0) * K);
    const uint8_t* wbase = qw + static_cast<int64_t>(n0) * kbytes;
    const uint8_t* sbase = sw + static_cast<int64_t>(n0) * blocks;
    const uint32_t lds0 = static_cast<uint32_t>(reinterpret_cast<size_t>((lds_void*)lds));

    // A wave's loads of a step: 1 KB of whole rows of X or W each, and the scales of 16
    // rows; chunk c of row r lies in slot c ^ x_swizzle(r) (X) or c ^ w_swizzle(r) (W).
    constexpr int kXChunks = S::kXRow / 16, kWChunks = S::kWRow / 16, kSWords = S::kSRow / 4;
    auto x_swizzle = [](int r) { return r & 15; };
    auto w_swizzle = [](int r) { return kWChunks == 8 ? (r >> 1) & 7 : (r >> 2) & 3; };
    uint32_t xrow[S::kXLoads], xchunk[S::kXLoads], wrow[S::kWLoads], wchunk[S::kWLoads];
#pragma unroll
    for (int u = 0; u < S::kXLoads; ++u) {
        const int r = 64 / kXChunks * (S::kXLoads * wave + u) + lane / kXChunks, slot = lane % kXChunks;
        xrow[u] = static_cast<uint32_t>(min(m0 + r, M - 1) - m0) * (2u * K);
        xchunk[u] = 16u * (slot ^ x_swizzle(r));
    }
#pragma unroll
    for (int u = 0; u < S::kWLoads; ++u) {
        const int r = 64 / kWChunks * (S::kWLoads * wave + u) + lane / kWChunks, slot = lane % kWChunks;
        wrow[u] = static_cast<uint32_t>(min(n0 + r, N - 1) - n0) * kbytes;
        wchunk[u] = 16u * (slot ^ w_swizzle(r));
    }
    const uint32_t srow = static_cast<uint32_t>(min(n0 + 16 * wave + lane / kSWords, N - 1) - n0) * blocks;
    // load u of step s; then all of them
    auto load_one = [&](int u, int s, uint32_t st) {
        const uint32_t k0 = static_cast<uint32_t>(s) * STEP;
        if (u < S::kXLoads) {
            kc::lds_dma16(xrow[u] + min(2 * k0 + xchunk[u], 2u * K - 16), xbase, st + 1024 * (S::kXLoads * wave + u));
        } else if (u < S::kXLoads + S::kWLoads) {
            const int v = u - S::kXLoads;
            kc::lds_dma16(wrow[v] + min(k0 / 2 + wchunk[v], kbytes - 16), wbase, st + S::kX + 1024 * (S::kWLoads * wave + v));
        } else if (lane < 16 * kSWords) {
            kc::lds_dma4(srow + min(k0 / kBlock + 4 * (lane % kSWords), blocks - 4), sbase,
                     st + S::kX + S::kW + 16 * S::kSRow * wave);
        }
    };
    auto buffer = [&](int s) { return __builtin_amdgcn_readfirstlane(lds0 + (s % S::ST) * S::kStage); };

    f32x4 acc[kRT][MT];
#pragma unroll
    for (int r = 0; r < kRT; ++r)
#pragma unroll
        for (int c = 0; c < MT; ++c) acc[r][c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    asm volatile("" ::"s"(y), "s"(M), "s"(N));

    // What a wave multiplies of a step, its half: read from LDS between the matrix
    // instructions of the step before.
    struct Operands {
        uint32_t sc[kRT];  // bytes of the half's blocks
        uint32_t code[kHalf][kRT];
        bf16x8 xv[kHalf][MT];
    };
    auto read = [&](int b, int r, const uint8_t* st, Operands& o) {  // a share of block b
        const int blk = kHalf * kg + b, row = 16 * kRT * wn + 16 * r + i;
        if (b == 0)
            o.sc[r] = *reinterpret_cast<const uint32_t*>(st + S::kX + S::kW + S::kSRow * row + (kSWords == 2 ? 4 * kg : 0));
        o.code[b][r] = *reinterpret_cast<const uint32_t*>(st + S::kX + row * S::kWRow + 16 * (blk ^ w_swizzle(row)) + 4 * g);
#pragma unroll
        for (int c = r * MT / kRT; c < (r + 1) * MT / kRT; ++c)
            o.xv[b][c] = *reinterpret_cast<const bf16x8*>(st + (16 * (MT * tg + c) + i) * S::kXRow + 16 * ((4 * blk + g) ^ i));
    };
    auto multiply = [&](int b, int r, const Operands& o) {
        const bf16x8 wv = decode(o.code[b][r], (o.sc[r] >> (8 * b + (kSWords == 2 ? 0 : 16 * kg))) & 255);
#pragma unroll
        for (int c = 0; c < MT; ++c) acc[r][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wv, o.xv[b][c], acc[r][c], 0, 0, 0);
    };
    const int last = steps - 1;
    Operands even, odd;
#pragma unroll
    for (int p = 0; p < S::ST; ++p)
#pragma unroll
        for (int u = 0; u < S::kLoads; ++u) load_one(u, min(p, last), buffer(p));
    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"(S::kLoads * (S::ST - 1)) : "memory");
#pragma unroll
    for (int b = 0; b < kHalf; ++b)
#pragma unroll
        for (int r = 0; r < kRT; ++r) read(b, r, lds, even);
    // Step s + 1 has landed and everyone holds step s in registers, so its buffer takes
    // step s + ST.  Steps past the last load the last one.
    auto step = [&](int s, Operands& now, Operands& next) {
        // the compiler's wait for these reads stands here, and not behind the next ones
#pragma unroll
        for (int b = 0; b < kHalf; ++b) {
#pragma unroll
            for (int r = 0; r < kRT; ++r) asm volatile("" : "+v"(now.code[b][r]));
#pragma unroll
            for (int c = 0; c < MT; ++c) asm volatile("" : "+v"(now.xv[b][c]));
        }
#pragma unroll
        for (int r = 0; r < kRT; ++r) asm volatile("" : "+v"(now.sc[r]));
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(S::kLoads * (S::ST - 2)) : "memory");
        const uint8_t* nxt = lds + ((s + 1) % S::ST) * S::kStage;
        const uint32_t st = buffer(s);
        constexpr int kParts = kHalf * kRT;
#pragma unroll
        for (int b = 0; b < kHalf; ++b)
#pragma unroll
            for (int r = 0; r < kRT; ++r) {
                const int q = b * kRT + r;
                read(b, r, nxt, next);
                multiply(b, r, now);
#pragma unroll
                for (int u = q * S::kLoads / kParts; u < (q + 1) * S::kLoads / kParts; ++u) load_one(u, min(s + S::ST, last), st);
                __builtin_amdgcn_sched_barrier(0);
            }
    };
    auto finish = [&](int s, const Operands& now) {
        if (kg == 1 && static_cast<uint32_t>(s) * STEP + STEP / 2 >= static_cast<uint32_t>(K)) return;  // nothing past K
#pragma unroll
        for (int b = 0; b < kHalf; ++b)
#pragma unroll
            for (int r = 0; r < kRT; ++r) multiply(b, r, now);
    };
    int s = 0;
    for (; s + 2 < steps; s += 2) {
        step(s, even, odd);
        step(s + 1, odd, even);
    }
    if (s + 1 < steps) {
        step(s, even, odd);
        finish(s + 1, odd);
    } else {
        finish(s, even);
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
    f32x4* red = reinterpret_cast<f32x4*>(lds);  // [tile of the wave][16 x 16 tile][lane]
    if (kg == 1) {
#pragma unroll
        for (int r = 0; r < kRT; ++r)
#pragma unroll
            for (int c = 0; c < MT; ++c) red[((tile * kRT + r) * MT + c) * 64 + lane] = acc[r][c];
    }
    __syncthreads();
    if (kg == 1) return;
    // D: lane (i, g) holds rows n = 4 g + v of token i
#pragma unroll
    for (int c = 0; c < MT; ++c) {
        const int m = m0 + 16 * (MT * tg + c) + i;
        if (m >= M) continue;
#pragma unroll
        for (int r = 0; r < kRT; ++r) {
            const f32x4 o = red[((tile * kRT + r) * MT + c) * 64 + lane];
            const f32x4 v = {acc[r][c].x + o.x, acc[r][c].y + o.y, acc[r][c].z + o.z, acc[r][c].w + o.w};
            const int n = n0 + 16 * kRT * wn + 16 * r + 4 * g;
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

template <int TG, int MT, int STEP>
int launch(const char* fn, const uint8_t* qw, const uint8_t* sw, const uint16_t* x, uint16_t* y, int M, int N, int K,
           hipStream_t stream) {
    using S = Shape<TG, MT, STEP>;
    const int st = raise_lds_limit<gemm_mxfp4_a16_tile_kernel<TG, MT, STEP>>(fn, S::kLds);
    if (st != KC_SUCCESS) return st;
    const dim3 grid((N + kRowsN - 1) / kRowsN, (M + S::kTokens - 1) / S::kTokens);
    gemm_mxfp4_a16_tile_kernel<TG, MT, STEP><<<grid, kThreads, S::kLds, stream>>>(qw, sw, x, y, M, N, K,
                                                                        N % 4 == 0 && kc::aligned(y, 8));
    return kc::check_launch(fn);
}

}  // namespace

namespace kc {
namespace mx {

int gemm_a16_tile(const char* fn, int mt, const uint8_t* qw, const uint8_t* sw, const uint16_t* x, uint16_t* y, int M, int N,
                  int K, hipStream_t stream) {
    switch (mt) {
        case 2: return launch<1, 2, 256>(fn, qw, sw, x, y, M, N, K, stream);
        case 3: return launch<1, 3, 256>(fn, qw, sw, x, y, M, N, K, stream);
        case 4: return launch<1, 4, 256>(fn, qw, sw, x, y, M, N, K, stream);
        default: return launch<2, 4, 128>(fn, qw, sw, x, y, M, N, K, stream);
    }
}

}  // namespace mx
}  // namespace kc
