// mxfp4_gemm.hpp -- host helpers shared by the MXFP4 products.
#pragma once

#include "mxfp4.hpp"

namespace kc {
namespace mx {

// Shapes of Y [M, N] = X [M, K] W [N, K]^T; y checked where Y has elements.
int check_gemm(const char* fn, int64_t M, int64_t N, int64_t K, const void* y);

// Y = 0 (an empty contraction).
template <bool YBF16>
int fill_zero(const char* fn, void* y, int64_t n, hipStream_t stream);

// M > 64 (mxfp4_gemm_tile.hip); arguments checked by the caller, K > 0.
template <bool YBF16>
int gemm_tile(const char* fn, const uint8_t* qx, const uint8_t* sx, const uint8_t* qw, const uint8_t* sw, void* y, int64_t M,
              int64_t N, int64_t K, hipStream_t stream);

// One token of bf16 activations (mxfp4_gemv.hip); false, nothing launched, for
// shapes that are left to the matrix cores.
bool gemv(const char* fn, const uint8_t* qw, const uint8_t* sw, const uint16_t* x, uint16_t* y, int N, int K,
          hipStream_t stream, int* status);

}  // namespace mx
}  // namespace kc
