// mxfp4.hpp -- the MXFP4 format (OCP microscaling, 4-bit floating point) on
// gfx950, shared by its quantizers, products and the 4-bit cache.
//
// A row is cut into blocks of 32 neighbouring values.  A block holds one
// scale byte b, the factor 2^(b - 127) (255: NaN), and 32 E2M1 codes, sign in
// bit 3, magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6; two codes to a byte, the
// even value in the low nibble.
//
// Quantization of a block with largest magnitude a:
//   b    = clamp(floor(log2(a)) - 2, -127, 127) + 127   (127, i.e. 1, for a == 0)
//   code = E2M1_rne(x * 2^(127 - b)), at most 6 in magnitude
// With the exponent field E of a (fp32 or bf16, the same field) that is
// b = max(E - 2, 0): a subnormal a is below 2^-126 and clamps to b = 0.  A block that
// holds a NaN or an infinity gets b = 255 and codes 0, so that every value of
// it reads back as NaN.
#pragma once

#include "kc_common.hpp"

namespace kc {
namespace mx {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

constexpr int kBlock = 32;       // values per scale
constexpr uint32_t kOne = 127;   // scale byte of 2^0
constexpr uint32_t kNaN = 255;

// Scale byte of a block from the bits of its largest magnitude as fp32.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
    if (amax_bits == 0) return kOne;
    const uint32_t e = amax_bits >> 23;
    return e == 255 ? kNaN : (e > 2 ? e - 2 : 0u);
}

// 2^(b - 127) as fp32 (2^-127 is subnormal), NaN for b == 255.
__device__ __forceinline__ float scale_value(uint32_t b) {
    return __uint_as_float(b == 0 ? 0x00400000u : b == kNaN ? 0x7FC00000u : b << 23);
}

// The fp32 value whose exponent field is b, for the operand of the scaled
// conversions, which look at the exponent field alone (checked for every
// field over every code and bf16 value on the GPU).
__device__ __forceinline__ float scale_operand(uint32_t b) { return __uint_as_float(b << 23); }

// Bits of the largest magnitude in 8 packed bf16 values, as fp32 bits.
__device__ __forceinline__ uint32_t absmax_bits_bf16(u32x4 v) {
    typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
    auto mag = [](uint32_t w) { return __builtin_bit_cast(u16x2, w & 0x7FFF7FFFu); };
    const u16x2 m = __builtin_elementwise_max(__builtin_elementwise_max(mag(v.x), mag(v.y)),
                                              __builtin_elementwise_max(mag(v.z), mag(v.w)));
    return static_cast<uint32_t>(m.x > m.y ? m.x : m.y) << 16;
}

// The same of 4 fp32 values as words.
__device__ __forceinline__ uint32_t absmax_bits_f32(u32x4 v) {
    constexpr uint32_t m = 0x7FFFFFFFu;
    return max(max(v.x & m, v.y & m), max(v.z & m, v.w & m));
}

// Largest of v over the lanes that differ in bits 0 (to 1, to 2) of their number.
__device__ __forceinline__ uint32_t max_pair(uint32_t v) {
    return max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xB1, 0xF, 0xF, true)));
}
__device__ __forceinline__ uint32_t max_quad(uint32_t v) {
    v = max_pair(v);
    return max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x4E, 0xF, 0xF, true)));
}

__device__ __forceinline__ uint32_t max_oct(uint32_t v) {
    v = max_quad(v);  // four lanes agree: the mirror of 8 lanes is lane ^ 4
    return max(v, static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0x141, 0xF, 0xF, true)));
}

// 8 values -> 8 codes (value i in nibble i) at scale byte b != 255.
__device__ __forceinline__ uint32_t encode8_bf16(u32x4 v, uint32_t b) {
    const float s = scale_operand(b);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, w[0]), s, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, w[1]), s, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, w[2]), s, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2, w[3]), s, 3);
}

__device__ __forceinline__ uint32_t encode8_f32(f32x4 a, f32x4 b, uint32_t sb) {
    const float s = scale_operand(sb);
    uint32_t r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, a.x, a.y, s, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, a.z, a.w, s, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, b.x, b.y, s, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, b.z, b.w, s, 3);
}

// 4 fp32 values as words -> 4 codes in 16 bits.
__device__ __forceinline__ uint32_t encode4_f32(u32x4 v, uint32_t sb) {
    const float s = scale_operand(sb);
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __uint_as_float(w[0]), __uint_as_float(w[1]), s, 0);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, __uint_as_float(w[2]), __uint_as_float(w[3]), s, 1);
}

// 8 codes -> 8 fp32 values times s: the conversion gives the E2M1 value, the
// multiplication is exact but where it leaves fp32's range.
__device__ __forceinline__ void decode8_f32(uint32_t c, float s, f32x4& a, f32x4& b) {
    const f32x2 p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 0);
    const f32x2 q = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 1);
    const f32x2 r = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 2);
    const f32x2 t = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 3);
    a = f32x4{p.x * s, p.y * s, q.x * s, q.y * s};
    b = f32x4{r.x * s, r.y * s, t.x * s, t.y * s};
}

// The same of 4 codes in the low 16 bits.
__device__ __forceinline__ f32x4 decode4_f32(uint32_t c, float s) {
    const f32x2 p = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 0);
    const f32x2 q = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, 1.0f, 1);
    return f32x4{p.x * s, p.y * s, q.x * s, q.y * s};
}

// 8 codes as packed bf16 (every E2M1 value times a power of two is a bf16
// value, but where it leaves the range).
__device__ __forceinline__ u32x4 decode8_bf16(uint32_t c, float s) {
    f32x4 a, b;
    decode8_f32(c, s, a, b);
    return u32x4{pack_bf16x2(a.x, a.y), pack_bf16x2(a.z, a.w), pack_bf16x2(b.x, b.y), pack_bf16x2(b.z, b.w)};
}

}  // namespace mx
}  // namespace kc
