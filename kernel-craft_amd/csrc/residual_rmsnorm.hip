// residual_rmsnorm.hip -- the residual sum between two blocks of a decoder with the norms
// on both of its sides on gfx950: for a token's block output y and residual stream h,
//     b  = post_gamma ? post_gamma y / sqrt(mean(y^2) + eps) : y
//     h' = h + alpha gate b                     (gate: 1, per channel, or per value)
//     n  = gamma h' / sqrt(mean(h'^2) + eps)    of the h' that is not rounded yet
// in fp32, each output rounded once; or n as E4M3 codes with a scale per token, quantized
// from fp32 as the row quantizer does (absmax / 448, a NaN to +448).
//
// Bound by memory: y, h and a gate per value once in, h' and n (or codes) once out.  A
// workgroup holds a row in registers, W units of 8 values per thread; its gammas and a
// channel gate stay in registers from row to row.  8000 rows of 4096 in bf16 with both norms
// and a channel gate, to codes: 229 MB in 44 us, 5.2 TB/s (a copy of 1 GiB 5.0); 2003 of 5120 on
// an fp32 stream: 144 MB in 25 us, 5.8 TB/s, part of it from cache; one row 3.2 us, all of it the
// launch, the trip to memory and the row's sums.
#include <algorithm>
#include <type_traits>

#include "fp8_common.hpp"

namespace {

using kc::kWave;
using kc::fp8::f32x4;
using kc::fp8::u32x2;
using kc::fp8::u32x4;

constexpr int kUnit = 8;
constexpr int kMaxCols = 32768;

template <bool BF16>
using Elem = std::conditional_t<BF16, uint16_t, float>;

// 8 values as they lie in memory.
template <bool BF16>
struct Unit {
    u32x4 w[BF16 ? 1 : 2];
};

template <bool BF16>
__device__ __forceinline__ void unpack(const Unit<BF16>& u, float (&v)[kUnit]) {
    if constexpr (BF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(u.w[0][i] << 16);
            v[2 * i + 1] = __uint_as_float(u.w[0][i] & 0xFFFF0000u);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(u.w[i / 4][i % 4]);
    }
}

template <bool BF16>
__device__ __forceinline__ Unit<BF16> pack(const float (&v)[kUnit]) {
    Unit<BF16> u;
    if constexpr (BF16) {
#pragma unroll
        for (int i = 0; i < 4; ++i) u.w[0][i] = kc::pack_bf16x2(v[2 * i], v[2 * i + 1]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) u.w[i / 4][i % 4] = __float_as_uint(v[i]);
    }
    return u;
}

// How rows lie: kWhole in whole units, every one aligned to 16 bytes; kAny of at least a unit's
// values, at any address; kShort of fewer than that.  Any address costs no loads value by value:
// the memory unit takes 16 bytes as they come (4000 rows of 4097 in bf16, to codes: 29 us; value
// by value 114, and 21 for 4096).
enum Lie { kWhole, kAny, kShort };
typedef uint32_t u32x4_any __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x2_any __attribute__((ext_vector_type(2), aligned(1)));

// Where a unit begins in a row of D values.  The last one of kAny is moved back to end with the
// row: its first `again` values are the unit's before too, come out the same and are stored
// twice, but count once in sums.
struct Place {
    int at, again;  // again >= kUnit: past the row
};

template <Lie LIE>
__device__ __forceinline__ Place place(int unit, int D) {
    const int at = unit * kUnit;
    if (LIE != kAny) return {at, at < D ? 0 : kUnit};
    const int back = max(0, at + kUnit - D);
    return {at - back, back};
}

// The values of a unit's that count in sums, the others as zeros.
template <Lie LIE>
__device__ __forceinline__ float counted(float v, int e, Place a) {
    return LIE != kAny || e >= a.again ? v : 0.0f;
}

// A row's unit; zeros past its end.
template <bool BF16, Lie LIE>
__device__ __forceinline__ Unit<BF16> load(const Elem<BF16>* row, int unit, int D) {
    using Load = std::conditional_t<LIE == kWhole, u32x4, u32x4_any>;
    const Place a = place<LIE>(unit, D);
    Unit<BF16> r{};
    if constexpr (LIE != kShort) {
        const Load* p = reinterpret_cast<const Load*>(row + a.at);
#pragma unroll
        for (int k = 0; k < (BF16 ? 1 : 2); ++k) r.w[k] = a.again < kUnit ? u32x4(p[k]) : u32x4{0u, 0u, 0u, 0u};
    } else if (a.again == 0) {
#pragma unroll
        for (int e = 0; e < kUnit; ++e) {
            if (e >= D) break;
            if constexpr (BF16) r.w[0][e / 2] |= static_cast<uint32_t>(row[e]) << (16 * (e % 2));
            else r.w[e / 4][e % 4] = __float_as_uint(row[e]);
        }
    }
    return r;
}

template <bool BF16, Lie LIE>
__device__ __forceinline__ void store(Elem<BF16>* row, int unit, int D, const float (&v)[kUnit]) {
    using Store = std::conditional_t<LIE == kWhole, u32x4, u32x4_any>;
    const Place a = place<LIE>(unit, D);
    const Unit<BF16> r = pack<BF16>(v);
    if (a.again >= kUnit) return;
    if constexpr (LIE != kShort) {
#pragma unroll
        for (int k = 0; k < (BF16 ? 1 : 2); ++k)
            __builtin_nontemporal_store(Store(r.w[k]), reinterpret_cast<Store*>(row + a.at) + k);
    } else {
#pragma unroll
        for (int e = 0; e < kUnit; ++e) {
            if (e >= D) break;
            if constexpr (BF16) row[e] = static_cast<uint16_t>(r.w[0][e / 2] >> (16 * (e % 2)));
            else row[e] = v[e];
        }
    }
}

struct Args {
    const void *y, *h, *gate, *post, *gamma;
    int64_t y_stride, h_stride, gate_stride, rows;
    int D;
    float alpha, eps;
    void *h_out, *out;
    float* scales;
};

// Sum, or largest, over the workgroup, in an order that the number of threads fixes.
template <int THREADS, bool MAX>
__device__ __forceinline__ float over_row(float v, float* part) {
    v = MAX ? kc::wave_max(v) : kc::wave_sum(v);
    if constexpr (THREADS == kWave) return v;
    const int wave = threadIdx.x / kWave;
    if ((threadIdx.x & (kWave - 1)) == 0) part[wave] = v;
    __syncthreads();
    float r = part[0];
#pragma unroll
    for (int w = 1; w < THREADS / kWave; ++w) r = MAX ? fmaxf(r, part[w]) : r + part[w];
    return r;
}

template <bool YB, bool HB, bool FP8, Lie LIE, int THREADS, int W>
__global__ __launch_bounds__(THREADS, 4) void residual_kernel(const Args p) {
    using namespace kc::fp8;
    constexpr int kParts = THREADS / kWave;
    __shared__ float part[2][3][kParts];
    using Y = Elem<YB>;
    using H = Elem<HB>;
    const int tid = threadIdx.x;
    const Y* y = static_cast<const Y*>(p.y);
    const H* h = static_cast<const H*>(p.h);
    const Y* gate = static_cast<const Y*>(p.gate);
    const bool channel = gate && p.gate_stride == 0;
    Unit<YB> gamma[W], post[W], cgate[W];
#pragma unroll
    for (int i = 0; i < W; ++i) {
        gamma[i] = load<YB, LIE>(static_cast<const Y*>(p.gamma), tid + i * THREADS, p.D);
        if (p.post) post[i] = load<YB, LIE>(static_cast<const Y*>(p.post), tid + i * THREADS, p.D);
        if (channel) cgate[i] = load<YB, LIE>(gate, tid + i * THREADS, p.D);
    }
    int turn = 0;  // rows take the two sets of partial results in turn
    for (int64_t row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
        Unit<YB> yv[W], gv[W];
        Unit<HB> hv[W];
#pragma unroll
        for (int i = 0; i < W; ++i) {
            yv[i] = load<YB, LIE>(y + row * p.y_stride, tid + i * THREADS, p.D);
            hv[i] = load<HB, LIE>(h + row * p.h_stride, tid + i * THREADS, p.D);
            if (gate && !channel) gv[i] = load<YB, LIE>(gate + row * p.gate_stride, tid + i * THREADS, p.D);
        }
        float inv = 1.0f;
        if (p.post) {
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const Place a = place<LIE>(tid + i * THREADS, p.D);
                float v[kUnit];
                unpack<YB>(yv[i], v);
#pragma unroll
                for (int e = 0; e < kUnit; ++e) ss = fmaf(v[e], counted<LIE>(v[e], e, a), ss);
            }
            ss = over_row<THREADS, false>(ss, part[turn][0]);
            inv = 1.0f / sqrtf(ss / static_cast<float>(p.D) + p.eps);
        }
        float x[W][kUnit], ss = 0.0f;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            const Place a = place<LIE>(tid + i * THREADS, p.D);
            float b[kUnit], g[kUnit];
            unpack<YB>(yv[i], b);
            unpack<HB>(hv[i], x[i]);
            if (p.post) {
                unpack<YB>(post[i], g);
#pragma unroll
                for (int e = 0; e < kUnit; ++e) b[e] = (g[e] * b[e]) * inv;
            }
            if (gate) {
                unpack<YB>(channel ? cgate[i] : gv[i], g);
#pragma unroll
                for (int e = 0; e < kUnit; ++e) b[e] *= g[e];
            }
#pragma unroll
            for (int e = 0; e < kUnit; ++e) {
                x[i][e] = fmaf(p.alpha, b[e], x[i][e]);
                ss = fmaf(x[i][e], counted<LIE>(x[i][e], e, a), ss);
            }
            store<HB, LIE>(static_cast<H*>(p.h_out) + row * p.D, tid + i * THREADS, p.D, x[i]);
        }
        ss = over_row<THREADS, false>(ss, part[turn][1]);
        inv = 1.0f / sqrtf(ss / static_cast<float>(p.D) + p.eps);
        float most = 0.0f;
#pragma unroll
        for (int i = 0; i < W; ++i) {
            float g[kUnit];
            unpack<YB>(gamma[i], g);
#pragma unroll
            for (int e = 0; e < kUnit; ++e) {
                x[i][e] = (g[e] * x[i][e]) * inv;
                if constexpr (FP8) most = fmaxf(most, fabsf(x[i][e]));
            }
            if constexpr (!FP8) store<YB, LIE>(static_cast<Y*>(p.out) + row * p.D, tid + i * THREADS, p.D, x[i]);
        }
        if constexpr (FP8) {
            const RowDiv d = row_div(over_row<THREADS, true>(most, part[turn][2]));
            if (tid == 0) p.scales[row] = d.s;
            uint8_t* codes = static_cast<uint8_t*>(p.out) + row * p.D;
#pragma unroll
            for (int i = 0; i < W; ++i) {
                const Place a = place<LIE>(tid + i * THREADS, p.D);
                if (a.again >= kUnit) break;
                const f32x4 lo{x[i][0], x[i][1], x[i][2], x[i][3]}, hi{x[i][4], x[i][5], x[i][6], x[i][7]};
                const u32x2 c = d.fast ? u32x2{e4m3x4_div<true>(lo, d), e4m3x4_div<true>(hi, d)}
                                       : u32x2{e4m3x4_div<false>(lo, d), e4m3x4_div<false>(hi, d)};
                if constexpr (LIE != kShort) {
                    using Store = std::conditional_t<LIE == kWhole, u32x2, u32x2_any>;
                    __builtin_nontemporal_store(Store(c), reinterpret_cast<Store*>(codes + a.at));
                } else {
#pragma unroll
                    for (int e = 0; e < kUnit; ++e)
                        if (e < p.D) codes[e] = static_cast<uint8_t>(c[e / 4] >> (8 * (e % 4)));
                }
            }
        }
    }
}

// One thread per unit while a row fits 256 of them, two units per thread to 16384 values; small
// rows get small workgroups (32000 rows of 512 24 us, 256 threads 36), and 4 waves stay on a SIMD
// with two units held.  Four units, for rows past 16384, spill (1000 rows of 28672 in bf16 72 us,
// 3.2 TB/s); 1000 of 14336 took 49 us that way and take 19 with two.
template <bool YB, bool HB, bool FP8, Lie LIE>
void launch(const Args& p, hipStream_t stream) {
    const unsigned grid = static_cast<unsigned>(std::min<int64_t>(p.rows, 2048));
    const int units = (p.D + kUnit - 1) / kUnit;
    if constexpr (LIE == kShort) residual_kernel<YB, HB, FP8, LIE, 64, 1><<<grid, 64, 0, stream>>>(p);
    else if (units <= 64) residual_kernel<YB, HB, FP8, LIE, 64, 1><<<grid, 64, 0, stream>>>(p);
    else if (units <= 128) residual_kernel<YB, HB, FP8, LIE, 128, 1><<<grid, 128, 0, stream>>>(p);
    else if (units <= 256) residual_kernel<YB, HB, FP8, LIE, 256, 1><<<grid, 256, 0, stream>>>(p);
    else if (units <= 512) residual_kernel<YB, HB, FP8, LIE, 256, 2><<<grid, 256, 0, stream>>>(p);
    else if (units <= 1024) residual_kernel<YB, HB, FP8, LIE, 512, 2><<<grid, 512, 0, stream>>>(p);
    else if (units <= 2048) residual_kernel<YB, HB, FP8, LIE, 1024, 2><<<grid, 1024, 0, stream>>>(p);
    else residual_kernel<YB, HB, FP8, LIE, 1024, 4><<<grid, 1024, 0, stream>>>(p);
}

template <bool YB, bool HB, bool FP8>
int residual(const char* fn, const kc_residual* a, void* h_out, void* out, float* scales, hipStream_t stream) {
    if (!a) return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: null arguments", fn);
    if (a->rows < 0 || a->cols < 0)
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: negative shape rows=%lld cols=%d", fn, (long long)a->rows,
                             a->cols);
    if (a->cols > kMaxCols)
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: cols=%d is over %d", fn, a->cols, kMaxCols);
    if (a->rows == 0 || a->cols == 0) return KC_SUCCESS;
    if (!a->y || !a->h || !a->gamma || !h_out || !out || (FP8 && !scales))
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: null device pointer", fn);
    const Args p{a->y,    a->h,    a->gate,  a->post_gamma, a->gamma, a->y_stride, a->h_stride, a->gate_stride,
                 a->rows, a->cols, a->alpha, a->eps,        h_out,    out,         scales};
    constexpr int y_step = YB ? 8 : 4, h_step = HB ? 8 : 4;  // values in 16 bytes
    const bool whole = p.D % kUnit == 0 && p.y_stride % y_step == 0 && p.h_stride % h_step == 0 &&
                     (!p.gate || p.gate_stride % y_step == 0) && kc::aligned(p.y, 16) && kc::aligned(p.h, 16) &&
                     kc::aligned(p.gate, 16) && kc::aligned(p.post, 16) && kc::aligned(p.gamma, 16) &&
                     kc::aligned(h_out, 16) && kc::aligned(out, FP8 ? 8 : 16);
    if (whole) launch<YB, HB, FP8, kWhole>(p, stream);
    else if (p.D >= kUnit) launch<YB, HB, FP8, kAny>(p, stream);
    else launch<YB, HB, FP8, kShort>(p, stream);
    return kc::check_launch(fn);
}

}  // namespace

extern "C" int kc_residual_rmsnorm_bf16(const kc_residual* args, uint16_t* d_h_out, uint16_t* d_n,
                                        kc_stream_t stream) {
    return residual<true, true, false>("kc_residual_rmsnorm_bf16", args, d_h_out, d_n, nullptr, stream);
}

extern "C" int kc_residual_rmsnorm_bf16_f32(const kc_residual* args, float* d_h_out, uint16_t* d_n,
                                            kc_stream_t stream) {
    return residual<true, false, false>("kc_residual_rmsnorm_bf16_f32", args, d_h_out, d_n, nullptr, stream);
}

extern "C" int kc_residual_rmsnorm_f32(const kc_residual* args, float* d_h_out, float* d_n, kc_stream_t stream) {
    return residual<false, false, false>("kc_residual_rmsnorm_f32", args, d_h_out, d_n, nullptr, stream);
}

extern "C" int kc_residual_rmsnorm_quantize_fp8_bf16(const kc_residual* args, uint16_t* d_h_out, int8_t* d_codes,
                                                     float* d_scales, kc_stream_t stream) {
    return residual<true, true, true>("kc_residual_rmsnorm_quantize_fp8_bf16", args, d_h_out, d_codes, d_scales,
                                      stream);
}

extern "C" int kc_residual_rmsnorm_quantize_fp8_bf16_f32(const kc_residual* args, float* d_h_out, int8_t* d_codes,
                                                         float* d_scales, kc_stream_t stream) {
    return residual<true, false, true>("kc_residual_rmsnorm_quantize_fp8_bf16_f32", args, d_h_out, d_codes, d_scales,
                                       stream);
}

extern "C" int kc_residual_rmsnorm_quantize_fp8_f32(const kc_residual* args, float* d_h_out, int8_t* d_codes,
                                                    float* d_scales, kc_stream_t stream) {
    return residual<false, false, true>("kc_residual_rmsnorm_quantize_fp8_f32", args, d_h_out, d_codes, d_scales,
                                        stream);
}
