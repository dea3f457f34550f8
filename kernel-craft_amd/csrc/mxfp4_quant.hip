// mxfp4_quant.hip -- MXFP4 quantization and dequantization on gfx950 (the
// format: mxfp4.hpp).  No counterpart in the reference, whose 4-bit weights
// are integers with fp32 scales (quant_int4.cu:5-13).
//
// Rows are whole blocks of 32, so both kernels see the tensor as one list of
// units of 8 values: lane l of a wave holds units l, l + 64, l + 128, l + 192 of
// the wave's 256, four neighbouring lanes hold a block, and its largest
// magnitude is two DPP maxima on the bits (no LDS).  Both are bound by memory.
#include <algorithm>

#include "mxfp4.hpp"

namespace {

using namespace kc::mx;
using kc::kWave;

constexpr int kThreads = 256;
constexpr int kUnits = 4;                          // units of 8 values per lane
constexpr int kWaveUnits = kUnits * kWave;
constexpr int kBlockUnits = kUnits * kThreads;
constexpr int kMaxGrid = (1 << 24) - 1;            // workgroups: a launch holds fewer than 2^32 threads

// VEC: x 16-byte aligned (codes always are 4-byte aligned).
template <bool BF16, bool VEC>
struct Unit;
template <bool VEC>
struct Unit<true, VEC> {
    using T = uint16_t;
    u32x4 v;
    __device__ void load(const T* x, int64_t u) {
        if constexpr (VEC) {
            v = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(x) + u);
        } else {
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = x[8 * u + 2 * i] | static_cast<uint32_t>(x[8 * u + 2 * i + 1]) << 16;
            v = u32x4{w[0], w[1], w[2], w[3]};
        }
    }
    __device__ uint32_t absmax() const { return absmax_bits_bf16(v); }
    __device__ uint32_t encode(uint32_t b) const { return encode8_bf16(v, b); }
};
template <bool VEC>
struct Unit<false, VEC> {
    using T = float;
    f32x4 a, b;
    __device__ void load(const T* x, int64_t u) {
        if constexpr (VEC) {
            const f32x4* p = reinterpret_cast<const f32x4*>(x) + 2 * u;
            a = p[0];
            b = p[1];
        } else {
            const float* p = x + 8 * u;
            a = f32x4{p[0], p[1], p[2], p[3]};
            b = f32x4{p[4], p[5], p[6], p[7]};
        }
    }
    __device__ uint32_t absmax() const { return absmax_bits_f32(a, b); }
    __device__ uint32_t encode(uint32_t s) const { return encode8_f32(a, b, s); }
};

template <bool BF16, bool VEC>
__global__ __launch_bounds__(kThreads) void quantize_mxfp4_kernel(const typename Unit<BF16, VEC>::T* __restrict__ x,
                                                                  uint32_t* __restrict__ codes,
                                                                  uint8_t* __restrict__ scales, int64_t units) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
    const int64_t base = static_cast<int64_t>(blockIdx.x) * kBlockUnits + wave * kWaveUnits;
    Unit<BF16, VEC> v[kUnits];
    // units is a multiple of 4, so the four lanes of a block are live together
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
        const int64_t u = base + i * kWave + lane;
        v[i].load(x, u < units ? u : 0);
    }
    uint32_t mine = 0;  // scale byte of the block that this lane writes
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
        const int64_t u = base + i * kWave + lane;
        const uint32_t b = scale_byte(max_quad(v[i].absmax()));
        const uint32_t c = b == kNaN ? 0u : v[i].encode(b);
        if (u < units) __builtin_nontemporal_store(c, codes + u);
        if ((lane & 3) == i) mine = b;
    }
    // Lane 4 q + i writes the scale of the wave's block q of units i: one byte
    // store for all four.
    const int64_t u = base + (lane & 3) * kWave + (lane & ~3);
    if (u < units) scales[u >> 2] = static_cast<uint8_t>(mine);
}

template <bool BF16, bool VEC>
__global__ __launch_bounds__(kThreads) void dequantize_mxfp4_kernel(const uint32_t* __restrict__ codes,
                                                                    const uint8_t* __restrict__ scales,
                                                                    typename Unit<BF16, VEC>::T* __restrict__ out,
                                                                    int64_t units) {
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
    const int64_t base = static_cast<int64_t>(blockIdx.x) * kBlockUnits + wave * kWaveUnits;
    uint32_t c[kUnits], b[kUnits];
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
        const int64_t u = min(base + i * kWave + lane, units - 1);
        c[i] = __builtin_nontemporal_load(codes + u);
        b[i] = scales[u >> 2];
    }
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
        const int64_t u = base + i * kWave + lane;
        if (u >= units) return;
        if constexpr (BF16) {
            const u32x4 v = decode8_bf16(c[i], scale_value(b[i]));
            if constexpr (VEC) {
                __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(out) + u);
            } else {
                const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                for (int j = 0; j < 8; ++j) out[8 * u + j] = static_cast<uint16_t>(w[j >> 1] >> (16 * (j & 1)));
            }
        } else {
            f32x4 lo, hi;
            decode8_f32(c[i], scale_value(b[i]), lo, hi);
            if constexpr (VEC) {
                f32x4* p = reinterpret_cast<f32x4*>(out) + 2 * u;
                p[0] = lo;
                p[1] = hi;
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    out[8 * u + j] = lo[j];
                    out[8 * u + 4 + j] = hi[j];
                }
            }
        }
    }
}

// Shape and pointer checks of both directions; *units = 0 where there is
// nothing to do.
int check(const char* fn, const void* values, const void* codes, const void* scales, int64_t rows, int64_t cols,
          int64_t* units) {
    *units = 0;
    if (rows < 0 || cols < 0)
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: negative shape rows=%lld cols=%lld", fn, (long long)rows,
                             (long long)cols);
    if (cols % kBlock != 0)
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: cols=%lld must be a multiple of 32", fn, (long long)cols);
    if (rows == 0 || cols == 0) return KC_SUCCESS;
    if (!values || !codes || !scales) return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: null device pointer", fn);
    if (!kc::aligned(codes, 4))
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: codes must be 4-byte aligned", fn);
    if (rows > (int64_t{kMaxGrid} * kBlockUnits) / (cols / 8))
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: rows=%lld cols=%lld too large", fn, (long long)rows,
                             (long long)cols);
    *units = rows * (cols / 8);
    return KC_SUCCESS;
}

unsigned grid_of(int64_t units) { return static_cast<unsigned>((units + kBlockUnits - 1) / kBlockUnits); }

template <bool BF16>
int quantize(const char* fn, const typename Unit<BF16, true>::T* x, uint8_t* codes, uint8_t* scales, int64_t rows,
             int64_t cols, hipStream_t stream) {
    int64_t units;
    const int st = check(fn, x, codes, scales, rows, cols, &units);
    if (st != KC_SUCCESS || units == 0) return st;
    uint32_t* c = reinterpret_cast<uint32_t*>(codes);
    if (kc::aligned(x, 16))
        quantize_mxfp4_kernel<BF16, true><<<grid_of(units), kThreads, 0, stream>>>(x, c, scales, units);
    else
        quantize_mxfp4_kernel<BF16, false><<<grid_of(units), kThreads, 0, stream>>>(x, c, scales, units);
    return kc::check_launch(fn);
}

template <bool BF16>
int dequantize(const char* fn, const uint8_t* codes, const uint8_t* scales, typename Unit<BF16, true>::T* out,
               int64_t rows, int64_t cols, hipStream_t stream) {
    int64_t units;
    const int st = check(fn, out, codes, scales, rows, cols, &units);
    if (st != KC_SUCCESS || units == 0) return st;
    const uint32_t* c = reinterpret_cast<const uint32_t*>(codes);
    if (kc::aligned(out, 16))
        dequantize_mxfp4_kernel<BF16, true><<<grid_of(units), kThreads, 0, stream>>>(c, scales, out, units);
    else
        dequantize_mxfp4_kernel<BF16, false><<<grid_of(units), kThreads, 0, stream>>>(c, scales, out, units);
    return kc::check_launch(fn);
}

}  // namespace

extern "C" int kc_quantize_mxfp4_bf16(const uint16_t* d_input, uint8_t* d_codes, uint8_t* d_scales, int64_t rows,
                                      int64_t cols, kc_stream_t stream) {
    return quantize<true>("kc_quantize_mxfp4_bf16", d_input, d_codes, d_scales, rows, cols, stream);
}

extern "C" int kc_quantize_mxfp4_f32(const float* d_input, uint8_t* d_codes, uint8_t* d_scales, int64_t rows,
                                     int64_t cols, kc_stream_t stream) {
    return quantize<false>("kc_quantize_mxfp4_f32", d_input, d_codes, d_scales, rows, cols, stream);
}

extern "C" int kc_dequantize_mxfp4_bf16(const uint8_t* d_codes, const uint8_t* d_scales, uint16_t* d_output,
                                        int64_t rows, int64_t cols, kc_stream_t stream) {
    return dequantize<true>("kc_dequantize_mxfp4_bf16", d_codes, d_scales, d_output, rows, cols, stream);
}

extern "C" int kc_dequantize_mxfp4_f32(const uint8_t* d_codes, const uint8_t* d_scales, float* d_output,
                                       int64_t rows, int64_t cols, kc_stream_t stream) {
    return dequantize<false>("kc_dequantize_mxfp4_f32", d_codes, d_scales, d_output, rows, cols, stream);
}
