// mxfp4_gemm.hip -- products of MXFP4 matrices on gfx950's scaled matrix cores.
//
//   Y[m, n] = sum_b 2^(sx[m, b] + sw[n, b] - 254) sum_{k in block b} e2m1(qx[m, k]) e2m1(qw[n, k])
#include <algorithm>

#include "mxfp4_gemm.hpp"

namespace {

using namespace kc::mx;
using kc::kWave;

typedef int32_t i32x8 __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256;

__device__ __forceinline__ i32x8 operand(u32x4 v) {
    return i32x8{static_cast<int32_t>(v.x), static_cast<int32_t>(v.y), static_cast<int32_t>(v.z),
                 static_cast<int32_t>(v.w), 0, 0, 0, 0};
}

// One wave per 16 x 16 tile of Y.  Lane (i, g) of an operand holds block g of a
// 128-value step of row i and its scale byte; blocks past K read as zeros.
template <bool YBF16>
__global__ __launch_bounds__(kThreads) void gemm_mxfp4_kernel(const uint8_t* __restrict__ qx, const uint8_t* __restrict__ sx,
                                                              const uint8_t* __restrict__ qw, const uint8_t* __restrict__ sw,
                                                              void* __restrict__ y, int64_t M, int64_t N, int64_t K,
                                                              int64_t tiles_n, int64_t tiles) {
    const int lane = threadIdx.x & 63;
    const int64_t tile = static_cast<int64_t>(blockIdx.x) * (kThreads / kWave) + (threadIdx.x >> 6);
    if (tile >= tiles) return;
    const int i = lane & 15, g = lane >> 4;
    const int64_t m0 = tile / tiles_n * 16, n0 = tile % tiles_n * 16, blocks = K / kBlock;
    const int64_t xr = min(m0 + i, M - 1), wr = min(n0 + i, N - 1);
    f32x4 acc = {0, 0, 0, 0};
    for (int64_t b0 = 0; b0 < blocks; b0 += 4) {
        const int64_t b = b0 + g;
        u32x4 xv = {0, 0, 0, 0}, wv = {0, 0, 0, 0};
        int xs = kOne, ws = kOne;
        if (b < blocks) {
            xv = *reinterpret_cast<const u32x4*>(qx + (xr * blocks + b) * 16);
            wv = *reinterpret_cast<const u32x4*>(qw + (wr * blocks + b) * 16);
            xs = sx[xr * blocks + b];
            ws = sw[wr * blocks + b];
        }
        acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(operand(wv), operand(xv), acc, 4, 4, 0, ws, 0, xs);
    }
    const int64_t m = m0 + i;
    if (m >= M) return;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
        const int64_t n = n0 + 4 * g + v;
        if (n >= N) break;
        if constexpr (YBF16) static_cast<uint16_t*>(y)[m * N + n] = kc::f32_to_bf16(acc[v]);
        else static_cast<float*>(y)[m * N + n] = acc[v];
    }
}

template <bool YBF16>
int gemm(const char* fn, const uint8_t* qx, const uint8_t* sx, const uint8_t* qw, const uint8_t* sw, void* y, int64_t M,
         int64_t N, int64_t K, hipStream_t stream) {
    const int st = kc::mx::check_gemm(fn, M, N, K, y);
    if (st != KC_SUCCESS || M == 0 || N == 0) return st;
    if (K == 0) return kc::mx::fill_zero<YBF16>(fn, y, M * N, stream);
    if (!qx || !sx || !qw || !sw) return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: null device pointer", fn);
    if (!kc::aligned(qx, 16) || !kc::aligned(qw, 16))
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: the codes must be 16-byte aligned", fn);
    const int64_t tn = (N + 15) / 16, tiles = tn * ((M + 15) / 16);
    gemm_mxfp4_kernel<YBF16><<<static_cast<unsigned>((tiles + 3) / 4), kThreads, 0, stream>>>(qx, sx, qw, sw, y, M, N, K,
                                                                                             tn, tiles);
    return kc::check_launch(fn);
}

// Y = 0 for an empty contraction.
template <typename T>
__global__ void fill_zero_kernel(T* y, int64_t n) {
    const int64_t stride = static_cast<int64_t>(gridDim.x) * blockDim.x;
    for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < n; i += stride) y[i] = T(0);
}

}  // namespace

namespace kc {
namespace mx {

int check_gemm(const char* fn, int64_t M, int64_t N, int64_t K, const void* y) {
    if (M < 0 || N < 0 || K < 0) return set_error(KC_ERR_INVALID_ARGUMENT, "%s: negative shape", fn);
    if (K % kBlock != 0)
        return set_error(KC_ERR_INVALID_ARGUMENT, "%s: K=%lld must be a multiple of 32", fn, (long long)K);
    if (M == 0 || N == 0) return KC_SUCCESS;
    if (!y) return set_error(KC_ERR_INVALID_ARGUMENT, "%s: null device pointer", fn);
    if (((M + 15) / 16) > (int64_t{1} << 26) / ((N + 15) / 16))
        return set_error(KC_ERR_INVALID_ARGUMENT, "%s: M=%lld N=%lld too large", fn, (long long)M, (long long)N);
    return KC_SUCCESS;
}

template <bool YBF16>
int fill_zero(const char* fn, void* y, int64_t n, hipStream_t stream) {
    const unsigned blocks = static_cast<unsigned>(std::min<int64_t>((n + 255) / 256, 4096));
    if constexpr (YBF16) fill_zero_kernel<<<blocks, 256, 0, stream>>>(static_cast<uint16_t*>(y), n);
    else fill_zero_kernel<<<blocks, 256, 0, stream>>>(static_cast<float*>(y), n);
    return check_launch(fn);
}
template int fill_zero<true>(const char*, void*, int64_t, hipStream_t);
template int fill_zero<false>(const char*, void*, int64_t, hipStream_t);

}  // namespace mx
}  // namespace kc

extern "C" int kc_gemm_mxfp4_w4a4_bf16(const uint8_t* d_qx, const uint8_t* d_sx, const uint8_t* d_qw,
                                       const uint8_t* d_sw, uint16_t* d_y, int64_t M, int64_t N, int64_t K,
                                       kc_stream_t stream) {
    return gemm<true>("kc_gemm_mxfp4_w4a4_bf16", d_qx, d_sx, d_qw, d_sw, d_y, M, N, K, stream);
}

extern "C" int kc_gemm_mxfp4_w4a4_f32(const uint8_t* d_qx, const uint8_t* d_sx, const uint8_t* d_qw,
                                      const uint8_t* d_sw, float* d_y, int64_t M, int64_t N, int64_t K,
                                      kc_stream_t stream) {
    return gemm<false>("kc_gemm_mxfp4_w4a4_f32", d_qx, d_sx, d_qw, d_sw, d_y, M, N, K, stream);
}
