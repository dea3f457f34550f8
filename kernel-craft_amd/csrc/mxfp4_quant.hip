// mxfp4_quant.hip -- MXFP4 quantization and dequantization on gfx950 (the
// format: mxfp4.hpp).  No counterpart in the reference, whose 4-bit weights
// are integers with fp32 scales (quant_int4.cu:5-13).
//
// Rows are whole blocks of 32, so every kernel sees the tensor as one list of
// units of 16 bytes of values (8 bf16, 4 fp32), each load and store of a wave taking
// 64 neighbouring ones.  A block is 4 (8) neighbouring lanes, and its largest
// magnitude two (three) DPP maxima on the bits; no LDS.  All are bound by memory:
// 28672 x 8192 bf16 (595 MB) quantized in 95 us (6.2 TB/s), dequantized in 101 (5.9), where
// streams of two parts read and one written reach 6.0 to 6.3.
#include <algorithm>
#include <type_traits>

#include "mxfp4.hpp"

namespace {

using namespace kc::mx;
using kc::kWave;

constexpr int kThreads = 256;
constexpr int kMaxGrid = (1 << 24) - 1;  // workgroups: a launch holds fewer than 2^32 threads

template <bool BF16>
using Elem = std::conditional_t<BF16, uint16_t, float>;
template <bool BF16>
constexpr int kUnits = BF16 ? 4 : 8;     // units per lane
template <bool BF16>
constexpr int kPerUnit = BF16 ? 8 : 4;   // values per unit
template <bool BF16>
constexpr int kBlockUnits = kUnits<BF16> * kThreads;

// A unit as packed words; VEC: x is 16-byte aligned.
template <bool BF16, bool VEC>
__device__ __forceinline__ u32x4 load_unit(const Elem<BF16>* x, int64_t u) {
    if constexpr (VEC) {
        return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(x) + u);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (BF16) w[i] = x[8 * u + 2 * i] | static_cast<uint32_t>(x[8 * u + 2 * i + 1]) << 16;
            else w[i] = __float_as_uint(x[4 * u + i]);
        }
        return u32x4{w[0], w[1], w[2], w[3]};
    }
}

template <bool BF16, bool VEC>
__device__ __forceinline__ void store_unit(Elem<BF16>* out, int64_t u, u32x4 v) {
    if constexpr (VEC) {
        __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(out) + u);
    } else {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (BF16) {
                out[8 * u + 2 * i] = static_cast<uint16_t>(w[i]);
                out[8 * u + 2 * i + 1] = static_cast<uint16_t>(w[i] >> 16);
            } else {
                out[4 * u + i] = __uint_as_float(w[i]);
            }
        }
    }
}

__device__ __forceinline__ uint32_t swap_pair(uint32_t v) {  // lane l reads lane l ^ 1
    return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xB1, 0xF, 0xF, true));
}

// fp32: the 4 codes of a unit are 2 bytes.  An even lane puts its unit of row A (64
// units) and its neighbour's together, an odd lane those of the next row, B, so
// that every lane stores one word.
__device__ __forceinline__ uint32_t join(uint32_t a, uint32_t b, bool even) {
    const uint32_t other = swap_pair(even ? b : a);
    return even ? a | other << 16 : other | b << 16;
}
__device__ __forceinline__ void part(uint32_t w, bool even, uint32_t& a, uint32_t& b) {
    const uint32_t other = swap_pair(even ? w >> 16 : w & 0xFFFFu);
    a = even ? w & 0xFFFFu : other;
    b = even ? other : w >> 16;
}

template <bool BF16, bool VEC>
__global__ __launch_bounds__(kThreads) void quantize_mxfp4_kernel(const Elem<BF16>* __restrict__ x,
                                                                  uint32_t* __restrict__ codes,
                                                                  uint8_t* __restrict__ scales, int64_t units) {
    constexpr int U = kUnits<BF16>, kLanes = BF16 ? 4 : 8;  // lanes of a block: U, which the last store uses
    static_assert(U == kLanes, "one scale byte per lane");
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
    const bool even = (lane & 1) == 0;
    const int64_t base = static_cast<int64_t>(blockIdx.x) * kBlockUnits<BF16> + wave * (U * kWave);
    u32x4 v[U];
    // units is a multiple of the lanes of a block: they are live together
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int64_t u = base + i * kWave + lane;
        v[i] = load_unit<BF16, VEC>(x, u < units ? u : 0);
    }
    uint32_t mine = 0, held = 0;
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int64_t u = base + i * kWave + lane;
        uint32_t b, c = 0;
        if constexpr (BF16) {
            b = scale_byte(max_quad(absmax_bits_bf16(v[i])));
            if (b != kNaN) c = encode8_bf16(v[i], b);
            if (u < units) __builtin_nontemporal_store(c, codes + u);
        } else {
            b = scale_byte(max_oct(absmax_bits_f32(v[i])));
            if (b != kNaN) c = encode4_f32(v[i], b);
            if (i & 1) {
                // an even lane holds units u - 64 and u - 63, an odd lane u - 1 and u
                const int64_t first = even ? u - kWave : u - 1;
                const uint32_t w = join(held, c, even);
                if (first < units) __builtin_nontemporal_store(w, codes + (first >> 1));
            }
            held = c;
        }
        if ((lane & (kLanes - 1)) == i) mine = b;
    }
    // Lane kLanes q + i writes the scale of block q of the wave's row i of units: one
    // byte store for all of them.
    const int64_t u = base + (lane & (kLanes - 1)) * kWave + (lane & ~(kLanes - 1));
    if (u < units) scales[u / kLanes] = static_cast<uint8_t>(mine);
}

template <bool BF16, bool VEC>
__global__ __launch_bounds__(kThreads) void dequantize_mxfp4_kernel(const uint32_t* __restrict__ codes,
                                                                    const uint8_t* __restrict__ scales,
                                                                    Elem<BF16>* __restrict__ out, int64_t units) {
    constexpr int U = kUnits<BF16>, kLanes = BF16 ? 4 : 8;
    const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x >> 6;
    const bool even = (lane & 1) == 0;
    const int64_t base = static_cast<int64_t>(blockIdx.x) * kBlockUnits<BF16> + wave * (U * kWave);
    uint32_t c[U], b[U];
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int64_t u = min(base + i * kWave + lane, units - 1);
        if constexpr (BF16) {
            c[i] = __builtin_nontemporal_load(codes + u);
        } else if (i & 1) {
            const int64_t at = base + i * kWave + lane, first = even ? at - kWave : at - 1;
            part(__builtin_nontemporal_load(codes + (min(first, units - 2) >> 1)), even, c[i - 1], c[i]);
        }
        b[i] = scales[u / kLanes];
    }
#pragma unroll
    for (int i = 0; i < U; ++i) {
        const int64_t u = base + i * kWave + lane;
        if (u >= units) return;
        if constexpr (BF16) store_unit<BF16, VEC>(out, u, decode8_bf16(c[i], scale_value(b[i])));
        else store_unit<BF16, VEC>(out, u, __builtin_bit_cast(u32x4, decode4_f32(c[i], scale_value(b[i]))));
    }
}

// Shape and pointer checks of both directions; *units = 0 where there is
// nothing to do.
template <bool BF16>
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
    if (rows > (int64_t{kMaxGrid} * kBlockUnits<BF16>) / (cols / kPerUnit<BF16>))
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: rows=%lld cols=%lld too large", fn, (long long)rows,
                             (long long)cols);
    *units = rows * (cols / kPerUnit<BF16>);
    return KC_SUCCESS;
}

template <bool BF16>
unsigned grid_of(int64_t units) {
    return static_cast<unsigned>((units + kBlockUnits<BF16> - 1) / kBlockUnits<BF16>);
}

template <bool BF16>
int quantize(const char* fn, const Elem<BF16>* x, uint8_t* codes, uint8_t* scales, int64_t rows,
             int64_t cols, hipStream_t stream) {
    int64_t units;
    const int st = check<BF16>(fn, x, codes, scales, rows, cols, &units);
    if (st != KC_SUCCESS || units == 0) return st;
    uint32_t* c = reinterpret_cast<uint32_t*>(codes);
    if (kc::aligned(x, 16))
        quantize_mxfp4_kernel<BF16, true><<<grid_of<BF16>(units), kThreads, 0, stream>>>(x, c, scales, units);
    else
        quantize_mxfp4_kernel<BF16, false><<<grid_of<BF16>(units), kThreads, 0, stream>>>(x, c, scales, units);
    return kc::check_launch(fn);
}

template <bool BF16>
int dequantize(const char* fn, const uint8_t* codes, const uint8_t* scales, Elem<BF16>* out,
               int64_t rows, int64_t cols, hipStream_t stream) {
    int64_t units;
    const int st = check<BF16>(fn, out, codes, scales, rows, cols, &units);
    if (st != KC_SUCCESS || units == 0) return st;
    const uint32_t* c = reinterpret_cast<const uint32_t*>(codes);
    if (kc::aligned(out, 16))
        dequantize_mxfp4_kernel<BF16, true><<<grid_of<BF16>(units), kThreads, 0, stream>>>(c, scales, out, units);
    else
        dequantize_mxfp4_kernel<BF16, false><<<grid_of<BF16>(units), kThreads, 0, stream>>>(c, scales, out, units);
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
