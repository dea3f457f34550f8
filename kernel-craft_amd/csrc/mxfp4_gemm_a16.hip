// mxfp4_gemm_a16.hip -- bf16 activations times MXFP4 weights on gfx950:
//   Y[m, n] = sum_k x[m, k] * e2m1(qw[n, k]) 2^(sw[n, k / 32] - 127)
#include <algorithm>

#include "mxfp4_gemm.hpp"

namespace {

using namespace kc::mx;
using kc::kWave;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256;

// One wave per 16 x 16 tile of Y.
__global__ __launch_bounds__(kThreads) void gemm_mxfp4_a16_kernel(const uint8_t* __restrict__ qw,
                                                                  const uint8_t* __restrict__ sw,
                                                                  const uint16_t* __restrict__ x,
                                                                  uint16_t* __restrict__ y, int64_t M, int64_t N,
                                                                  int64_t K, int64_t tiles_n, int64_t tiles) {
    const int lane = threadIdx.x & 63;
    const int64_t tile = static_cast<int64_t>(blockIdx.x) * (kThreads / kWave) + (threadIdx.x >> 6);
    if (tile >= tiles) return;
    const int i = lane & 15, g = lane >> 4;
    const int64_t m0 = tile / tiles_n * 16, n0 = tile % tiles_n * 16, blocks = K / kBlock;
    const int64_t xr = min(m0 + i, M - 1), wr = min(n0 + i, N - 1);
    f32x4 acc = {0, 0, 0, 0};
    for (int64_t b = 0; b < blocks; ++b) {
        const u32x4 xv = *reinterpret_cast<const u32x4*>(x + xr * K + b * 32 + 8 * g);
        const uint32_t c = *reinterpret_cast<const uint32_t*>(qw + (wr * blocks + b) * 16 + 4 * g);
        const u32x4 wv = decode8_bf16(c, scale_value(sw[wr * blocks + b]));
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, wv), __builtin_bit_cast(bf16x8, xv),
                                                      acc, 0, 0, 0);
    }
    const int64_t m = m0 + i;
    if (m >= M) return;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
        const int64_t n = n0 + 4 * g + v;
        if (n < N) y[m * N + n] = kc::f32_to_bf16(acc[v]);
    }
}

}  // namespace

extern "C" int kc_gemm_mxfp4_bf16(const uint8_t* d_qw, const uint8_t* d_sw, const uint16_t* d_x, uint16_t* d_y,
                                  int64_t M, int64_t N, int64_t K, kc_stream_t stream) {
    const char* fn = "kc_gemm_mxfp4_bf16";
    const int st = kc::mx::check_gemm(fn, M, N, K, d_y);
    if (st != KC_SUCCESS || M == 0 || N == 0) return st;
    if (K == 0) return kc::mx::fill_zero<true>(fn, d_y, M * N, stream);
    if (!d_qw || !d_sw || !d_x) return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: null device pointer", fn);
    if (!kc::aligned(d_qw, 16) || !kc::aligned(d_x, 16))
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: the codes and x must be 16-byte aligned", fn);
    const int64_t tn = (N + 15) / 16, tiles = tn * ((M + 15) / 16);
    gemm_mxfp4_a16_kernel<<<static_cast<unsigned>((tiles + 3) / 4), kThreads, 0, stream>>>(d_qw, d_sw, d_x, d_y, M, N, K,
                                                                                          tn, tiles);
    return kc::check_launch(fn);
}
