// mxfp4_gemm.hpp -- host helpers shared by the MXFP4 products.
#pragma once

#include <atomic>

#include "lds_dma.hpp"
#include "mxfp4.hpp"

namespace kc {
namespace mx {

// acc += a b^T of one 16 x 16 x 128 tile, the scales in byte BYTE of sa and sb.
// In assembly for the accumulator's "a" and the operands' four registers: with 256
// accumulator registers and most of the others in use, the compiler's allocation keeps
// moving accumulators between the two halves of the register file (640 moves per 512
// of these), and the builtin's eight-register operands spill where loads fill most
// registers.  Nothing but these instructions touches the accumulators between
// start() and settle().  NOP: the operands may come from the instruction just before
// (the wait states that the compiler adds between a vector instruction and a matrix one
// that reads its result); operands that LDS or memory wrote need none.
template <int BYTE, bool NOP = false>
__device__ __forceinline__ void mfma(f32x4& acc, u32x4 a, u32x4 b, uint32_t sa, uint32_t sb) {
    if constexpr (NOP) asm volatile("s_nop 3" : "+v"(a), "+v"(b), "+v"(sa), "+v"(sb));
#define KC_MFMA(sel)                                                                                        \
    asm("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 " sel " cbsz:4 blgp:4" \
        : "+a"(acc)                                                                                         \
        : "v"(a), "v"(b), "v"(sa), "v"(sb))
    if constexpr (BYTE == 0) KC_MFMA("op_sel_hi:[0,0,0]");
    else if constexpr (BYTE == 1) KC_MFMA("op_sel:[1,1,0] op_sel_hi:[0,0,0]");
    else if constexpr (BYTE == 2) KC_MFMA("op_sel_hi:[1,1,0]");
    else KC_MFMA("op_sel:[1,1,0] op_sel_hi:[1,1,0]");
#undef KC_MFMA
}

// Ties every accumulator to this place: what made it comes before, its uses behind.
template <int I, int J>
__device__ __forceinline__ void tie(f32x4 (&acc)[I][J]) {
#pragma unroll
    for (int i = 0; i < I; ++i)
#pragma unroll
        for (int j = 0; j < J; ++j) asm volatile("" : "+a"(acc[i][j]));
}

// Behind the accumulators' first values: vector instructions write them, and a matrix
// instruction that reads one has to be two wait states behind.
template <int I, int J>
__device__ __forceinline__ void start(f32x4 (&acc)[I][J]) {
    tie(acc);
    asm volatile("s_nop 1" ::: "memory");
    tie(acc);
}

// Waits until the last results are in their registers (the compiler does not know the
// latency of the assembly above): every instruction that makes an accumulator comes
// before the wait, every later use of one behind it.
template <int I, int J>
__device__ __forceinline__ void settle(f32x4 (&acc)[I][J]) {
    tie(acc);
    asm volatile("s_nop 15\n\ts_nop 15" ::: "memory");
    tie(acc);
}

// Lets KERNEL use `bytes` of dynamic LDS on the current device (once per device: the
// limit is the loaded function's).
template <auto KERNEL>
int raise_lds_limit(const char* fn, int bytes) {
    static std::atomic<uint64_t> done{0};
    int device = 0;
    if (hipGetDevice(&device) != hipSuccess) return set_error(KC_ERR_HIP, "%s: no current device", fn);
    const uint64_t bit = uint64_t{1} << (device & 63);
    if (done.load(std::memory_order_acquire) & bit) return KC_SUCCESS;
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(KERNEL), hipFuncAttributeMaxDynamicSharedMemorySize, bytes) !=
        hipSuccess)
        return set_error(KC_ERR_HIP, "%s: cannot raise the LDS limit", fn);
    done.fetch_or(bit, std::memory_order_release);
    return KC_SUCCESS;
}

// Shapes of Y [M, N] = X [M, K] W [N, K]^T; y checked where Y has elements.
int check_gemm(const char* fn, int64_t M, int64_t N, int64_t K, const void* y);

// Y = 0 (an empty contraction).
template <bool YBF16>
int fill_zero(const char* fn, void* y, int64_t n, hipStream_t stream);

// More rows than a decode batch (mxfp4_gemm_tile.hip); arguments checked by the caller,
// K > 0.
template <bool YBF16>
int gemm_tile(const char* fn, const uint8_t* qx, const uint8_t* sx, const uint8_t* qw, const uint8_t* sw, void* y, int64_t M,
              int64_t N, int64_t K, hipStream_t stream);

// One token of bf16 activations (mxfp4_gemv.hip); false, nothing launched, for
// shapes that are left to the matrix cores.
bool gemv(const char* fn, const uint8_t* qw, const uint8_t* sw, const uint16_t* x, uint16_t* y, int N, int K,
          hipStream_t stream, int* status);

// bf16 activations in tiles of 16 mt tokens x 128 rows (mxfp4_gemm_a16_tile.hip): K a
// multiple of 128, sw 4-byte aligned.
int gemm_a16_tile(const char* fn, int mt, const uint8_t* qw, const uint8_t* sw, const uint16_t* x, uint16_t* y, int M, int N,
                  int K, hipStream_t stream);

}  // namespace mx
}  // namespace kc
