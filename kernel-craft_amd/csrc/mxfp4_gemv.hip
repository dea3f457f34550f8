// mxfp4_gemv.hip -- one token of bf16 activations times MXFP4 weights on gfx950
// (more tokens: mxfp4_gemm_a16.hip).
//
//   y[n] = sum_b 2^(sw[n, b] - 127) sum_{k in b} x[k] e2m1(qw[n, k])
//
// Bound by the weight stream.  A lane owns a block of 32 values of K for all of its
// wave's rows, so x stays in 16 registers and a wave's load is 1 KB of one row, whole
// cache lines; all four rows of a wave are on their way before the first is used.  K is
// split over kw waves of 64 blocks; the workgroup's 8 / kw groups of waves take four
// rows each.  A block is decoded to bf16 with its scale
// (v_cvt_scalef32_pk_bf16_fp4), as for more tokens, so that one token's terms leave
// fp32's range (and its weights bf16's) where many tokens' do, and multiplied with
// v_dot2_f32_bf16.  The lanes meet in DPP sums, the waves in LDS.
//
// Measured (us, against the matrix-core kernel for one token): N 28672, K 4096 11.9
// and 13.5 (62 MB; 10.4 at 6 TB/s); K 8192 22.6 and 29.6; K 2048 7.2 and 9.6; N 4096, K 4096
// 3.9 and 5.1, K 14336 7.9 and 10.2 (with the scale on the block's fp32 sum 12.0, 23.8, 7.6,
// 4.3 and 8.5); with a block per lane missing (K 1024) 3.2 and 2.4, so
// K under 2048 stays there, and so do two tokens (15.8 and 13.2 us: the sums over lanes
// cost as much as the dot products).  Two rows a wave 12.4 us, eight 13.3, sixteen 16.9.
#include "mxfp4_gemm.hpp"

namespace {

using namespace kc::mx;
using kc::kWave;

constexpr int kRows = 4;    // of a wave
constexpr int kWaves = 8;

template <int CTRL>
__device__ __forceinline__ float dpp_add(float v) {
    return v + __uint_as_float(static_cast<uint32_t>(
                   __builtin_amdgcn_mov_dpp(static_cast<int>(__float_as_uint(v)), CTRL, 0xF, 0xF, true)));
}

// Sum over the wave, in every lane.
__device__ __forceinline__ float sum_all(float v) {
    v = dpp_add<0xB1>(v);
    v = dpp_add<0x4E>(v);
    v = dpp_add<0x141>(v);
    v = dpp_add<0x140>(v);
    v += __shfl_xor(v, 16, kWave);
    return v + __shfl_xor(v, 32, kWave);
}

__device__ __forceinline__ float dot8(uint32_t c, float s, const uint32_t (&x)[4], float a) {
    const bf16x2 w0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0), w1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1);
    const bf16x2 w2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2), w3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3);
    a = __builtin_amdgcn_fdot2_f32_bf16(w0, __builtin_bit_cast(bf16x2, x[0]), a, false);
    a = __builtin_amdgcn_fdot2_f32_bf16(w1, __builtin_bit_cast(bf16x2, x[1]), a, false);
    a = __builtin_amdgcn_fdot2_f32_bf16(w2, __builtin_bit_cast(bf16x2, x[2]), a, false);
    return __builtin_amdgcn_fdot2_f32_bf16(w3, __builtin_bit_cast(bf16x2, x[3]), a, false);
}

__global__ __launch_bounds__(kWaves * 64) void gemv_mxfp4_kernel(const uint8_t* __restrict__ qw, const uint8_t* __restrict__ sw,
                                                                 const uint16_t* __restrict__ x, uint16_t* __restrict__ y,
                                                                 int N, int K, int kw) {
    __shared__ float red[kWaves][kRows];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const int groups = kWaves / kw, group = wave / kw, part = wave - group * kw;
    const int blocks = K / kBlock, b = 64 * part + lane;
    const bool has = group < groups && b < blocks;
    const int n0 = (static_cast<int>(blockIdx.x) * groups + group) * kRows;

    u32x4 w[kRows];
    uint32_t s[kRows];
    u32x4 xv[4];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        const int64_t at = static_cast<int64_t>(min(n0 + r, N - 1)) * blocks + (has ? b : 0);
        w[r] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(qw) + at);
        s[r] = sw[at];
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) xv[q] = reinterpret_cast<const u32x4*>(x)[4 * (has ? b : 0) + q];
#pragma unroll
    for (int r = 0; r < kRows; ++r) {
        const uint32_t c[4] = {w[r].x, w[r].y, w[r].z, w[r].w};
        const float scale = scale_operand(s[r]);
        float a = 0.0f;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const uint32_t xq[4] = {xv[q].x, xv[q].y, xv[q].z, xv[q].w};
            a = dot8(c[q], scale, xq, a);
        }
        a = sum_all(has ? a : 0.0f);
        if (lane == 0) red[wave][r] = a;
    }
    __syncthreads();
    const int t = threadIdx.x, n = static_cast<int>(blockIdx.x) * groups * kRows + t;
    if (t < groups * kRows && n < N) {
        const int g = t / kRows, r = t % kRows;
        float v = red[g * kw][r];
        for (int p = 1; p < kw; ++p) v += red[g * kw + p][r];
        y[n] = kc::f32_to_bf16(v);
    }
}

}  // namespace

namespace kc {
namespace mx {

bool gemv(const char* fn, const uint8_t* qw, const uint8_t* sw, const uint16_t* x, uint16_t* y, int N, int K,
          hipStream_t stream, int* status) {
    constexpr int kWaveK = 64 * kBlock;
    if (K < kWaveK || K > kWaves * kWaveK) return false;
    const int kw = (K + kWaveK - 1) / kWaveK, rows = kWaves / kw * kRows;
    gemv_mxfp4_kernel<<<(N + rows - 1) / rows, kWaves * 64, 0, stream>>>(qw, sw, x, y, N, K, kw);
    *status = check_launch(fn);
    return true;
}

}  // namespace mx
}  // namespace kc
