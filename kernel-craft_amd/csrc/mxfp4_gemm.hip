// mxfp4_gemm.hip -- the product of two MXFP4 matrices on gfx950's scaled matrix
// cores: entry points, and the kernel for decode batches (M <= 64).  More rows:
// mxfp4_gemm_tile.hip.  No counterpart in the reference.
//
//   Y[m, n] = sum_b 2^(sx[m, b] + sw[n, b] - 254) sum_{k in block b} e2m1(qx[m, k]) e2m1(qw[n, k])
//
// M <= 64 is bound by the weight stream (0.53 bytes a weight).  A workgroup of KW
// waves owns RT tiles of 16 weight rows and all MT = ceil(M / 16) tiles of X; wave w
// takes K steps w, w + KW, ... of 128 bytes (256 values), D of them in flight in
// registers, and the KW partial sums of every output meet in LDS in a fixed
// order.  No barrier stands in the K loop and no operand goes through LDS:
// with K split over the waves no two of them read the same bytes.
//
// A load carries 8 whole rows of a step (128 bytes, a cache line each): lane l
// takes 16-byte chunk 2 (l / 16) + l % 2 of row 8 h + (l % 16) / 2.  A lane and its
// neighbour l ^ 1 exchange one chunk each, after which lane (i, kb) holds chunks
// 2 kb and 2 kb + 1, two blocks of 32, of row row_of(i) = i / 2 + 8 (i % 2): the
// operands of two matrix-core instructions of 128 values.  The blocks' scale bytes
// are neighbours and come as one 16-bit load.
#include <algorithm>

#include "mxfp4_gemm.hpp"

namespace {

using namespace kc::mx;

typedef int32_t i32x8 __attribute__((ext_vector_type(8)));

constexpr int kBK = 128;       // bytes of K per step
constexpr int kSkinnyM = 64;

struct Frag {
    u32x4 h0, h1;
};

__device__ __forceinline__ uint32_t swap_pair(uint32_t v) {  // lane l reads lane l ^ 1
    return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xB1, 0xF, 0xF, true));
}

// Chunks 2 kb (lo) and 2 kb + 1 (hi) of the lane's operand row.
__device__ __forceinline__ void as_operands(const Frag& f, bool even, i32x8& lo, i32x8& hi) {
    const uint32_t a[4] = {f.h0.x, f.h0.y, f.h0.z, f.h0.w}, b[4] = {f.h1.x, f.h1.y, f.h1.z, f.h1.w};
    lo = hi = i32x8{0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        const uint32_t an = swap_pair(a[d]), bn = swap_pair(b[d]);
        lo[d] = static_cast<int32_t>(even ? a[d] : bn);
        hi[d] = static_cast<int32_t>(even ? an : b[d]);
    }
}

template <int MT, int RT, int KW, int D, bool YBF16>
__global__ __launch_bounds__(KW * 64) void gemm_mxfp4_skinny_kernel(
    const uint8_t* __restrict__ qx, const uint8_t* __restrict__ sx, const uint8_t* __restrict__ qw,
    const uint8_t* __restrict__ sw, void* __restrict__ y, int M, int N, int K, bool vec) {
    __shared__ f32x4 red[KW][RT * MT][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const int i = lane & 15, kb = lane >> 4;
    const bool even = (lane & 1) == 0;
    const int n0 = static_cast<int>(blockIdx.x) * 16 * RT;
    const int kbytes = K / 2, blocks = K / kBlock;
    const uint8_t* wbase = qw + static_cast<int64_t>(n0) * kbytes;
    const uint8_t* wsbase = sw + static_cast<int64_t>(n0) * blocks;
    const int chunk = 2 * kb + (i & 1), r8 = i >> 1, orow = (i >> 1) + 8 * (i & 1);
    uint32_t woff[RT][2], xoff[MT][2], wsoff[RT], xsoff[MT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
            woff[r][h] = static_cast<uint32_t>(min(n0 + 16 * r + 8 * h + r8, N - 1) - n0) * static_cast<uint32_t>(kbytes) + 16u * chunk;
        wsoff[r] = static_cast<uint32_t>(min(n0 + 16 * r + orow, N - 1) - n0) * static_cast<uint32_t>(blocks) + 2u * kb;
    }
#pragma unroll
    for (int c = 0; c < MT; ++c) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
            xoff[c][h] = static_cast<uint32_t>(min(16 * c + 8 * h + r8, M - 1)) * static_cast<uint32_t>(kbytes) + 16u * chunk;
        xsoff[c] = static_cast<uint32_t>(min(16 * c + orow, M - 1)) * static_cast<uint32_t>(blocks) + 2u * kb;
    }

    f32x4 acc[RT][MT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int c = 0; c < MT; ++c) acc[r][c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const int full = kbytes / kBK;
    const int mine = full > wave ? (full - wave + KW - 1) / KW : 0;  // K steps wave, wave + KW, ...

    Frag wf[D][RT], xf[D][MT];
    uint32_t ws[D][RT], xs[D][MT];
    auto pair_at = [](const uint8_t* p) {
        uint16_t v;
        __builtin_memcpy(&v, p, 2);
        return static_cast<uint32_t>(v);
    };
    auto load = [&](int slot, int j) {
        const int step = wave + KW * min(j, mine - 1);
        const uint8_t *wp = wbase + step * kBK, *xp = qx + step * kBK, *wsp = wsbase + 8 * step, *xsp = sx + 8 * step;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            wf[slot][r].h0 = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(wp + woff[r][0]));
            wf[slot][r].h1 = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(wp + woff[r][1]));
            ws[slot][r] = pair_at(wsp + wsoff[r]);
        }
#pragma unroll
        for (int c = 0; c < MT; ++c) {
            xf[slot][c].h0 = *reinterpret_cast<const u32x4*>(xp + xoff[c][0]);
            xf[slot][c].h1 = *reinterpret_cast<const u32x4*>(xp + xoff[c][1]);
            xs[slot][c] = pair_at(xsp + xsoff[c]);
        }
    };
    auto multiply = [&](const Frag (&w)[RT], const Frag (&x)[MT], const uint32_t (&wsc)[RT], const uint32_t (&xsc)[MT]) {
        i32x8 b0[MT], b1[MT];
#pragma unroll
        for (int c = 0; c < MT; ++c) as_operands(x[c], even, b0[c], b1[c]);
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            i32x8 a0, a1;
            as_operands(w[r], even, a0, a1);
#pragma unroll
            for (int c = 0; c < MT; ++c)
                acc[r][c] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                    a0, b0[c], acc[r][c], 4, 4, 0, static_cast<int>(wsc[r]), 0, static_cast<int>(xsc[c]));
#pragma unroll
            for (int c = 0; c < MT; ++c)
                acc[r][c] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(
                    a1, b1[c], acc[r][c], 4, 4, 1, static_cast<int>(wsc[r]), 1, static_cast<int>(xsc[c]));
        }
    };
    if (mine > 0) {
#pragma unroll
        for (int d = 0; d < D; ++d) load(d, d);
        __builtin_amdgcn_sched_barrier(0);
        int j = 0;
        for (; j + D < mine; j += D) {
#pragma unroll
            for (int d = 0; d < D; ++d) {
                multiply(wf[d], xf[d], ws[d], xs[d]);
                load(d, j + D + d);
                __builtin_amdgcn_sched_barrier(0);
            }
        }
#pragma unroll
        for (int d = 0; d < D; ++d)
            if (j + d < mine) multiply(wf[d], xf[d], ws[d], xs[d]);
    }
    if (kbytes % kBK != 0 && wave == full % KW) {
        // The partial last step: no codes and scale bytes 0 past K.
        const int kvalid = kbytes - full * kBK;
        auto tail = [&](const uint8_t* base, const uint32_t (&off)[2]) {
            const u32x4 z{0u, 0u, 0u, 0u};
            Frag f{z, z};
            if (16 * chunk < kvalid) {
                f.h0 = *reinterpret_cast<const u32x4*>(base + full * kBK + off[0]);
                f.h1 = *reinterpret_cast<const u32x4*>(base + full * kBK + off[1]);
            }
            return f;
        };
        auto tail_scales = [&](const uint8_t* p) {
            uint32_t v = 0;
            if (32 * kb < kvalid) v = p[8 * full];
            if (32 * kb + 16 < kvalid) v |= static_cast<uint32_t>(p[8 * full + 1]) << 8;
            return v;
        };
        Frag w[RT], x[MT];
        uint32_t wsc[RT], xsc[MT];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            w[r] = tail(wbase, woff[r]);
            wsc[r] = tail_scales(wsbase + wsoff[r]);
        }
#pragma unroll
        for (int c = 0; c < MT; ++c) {
            x[c] = tail(qx, xoff[c]);
            xsc[c] = tail_scales(sx + xsoff[c]);
        }
        multiply(w, x, wsc, xsc);
    }
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int c = 0; c < MT; ++c) red[wave][r * MT + c][lane] = acc[r][c];
    __syncthreads();
    for (int t = wave; t < RT * MT; t += KW) {
        f32x4 v = red[0][t][lane];
#pragma unroll
        for (int w = 1; w < KW; ++w) {
            const f32x4 o = red[w][t][lane];
            v = f32x4{v.x + o.x, v.y + o.y, v.z + o.z, v.w + o.w};
        }
        // D: lane (i, g) holds operand rows 4 g + v of W, column i of X, that is
        // outputs n = 2 g, 2 g + 8, 2 g + 1, 2 g + 9 (v = 0 .. 3) of row row_of(i)
        const int m = 16 * (t % MT) + orow;
        if (m >= M) continue;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int n = n0 + 16 * (t / MT) + 2 * kb + 8 * h;
            if (n >= N) break;
            const float v0 = h ? v.y : v.x, v1 = h ? v.w : v.z;
            const int64_t at = static_cast<int64_t>(m) * N + n;
            if constexpr (YBF16) {
                uint16_t* o = static_cast<uint16_t*>(y) + at;
                if (vec) {
                    *reinterpret_cast<uint32_t*>(o) = kc::pack_bf16x2(v0, v1);
                } else {
                    o[0] = kc::f32_to_bf16(v0);
                    if (n + 1 < N) o[1] = kc::f32_to_bf16(v1);
                }
            } else {
                float* o = static_cast<float*>(y) + at;
                o[0] = v0;
                if (n + 1 < N) o[1] = v1;
            }
        }
    }
}

template <int MT, int RT, int KW, int D, bool YBF16>
int launch_skinny(const char* fn, const uint8_t* qx, const uint8_t* sx, const uint8_t* qw, const uint8_t* sw, void* y, int M,
                  int N, int K, hipStream_t stream) {
    gemm_mxfp4_skinny_kernel<MT, RT, KW, D, YBF16><<<static_cast<unsigned>((N + 16 * RT - 1) / (16 * RT)), KW * 64, 0, stream>>>(
        qx, sx, qw, sw, y, M, N, K, N % 2 == 0 && kc::aligned(y, 4));
    return kc::check_launch(fn);
}

// Row tiles per workgroup: the fewest that leave at most one workgroup per CU,
// since every workgroup reads all of X (M 32, K 4096: N 6144 8.4 us at one tile, 7.0
// at two, 9.4 at four; N 28672 19.7 at two, 17.8 at four, 16.2 at seven; M 64
// 32.6, 25.0, 20.5); four on two workgroups a CU where X is one tile and N large (M 8,
// N 28672, K 8192 26.1 against 28.6 at seven; M 16, K 4096 15.2 and 15.4).  At one row
// tile eight waves with one tile of X, four with more (M 1, K 4096 3.9 against 4.2
// us; M 64, N 6144 13.3 against 12.5, M 32, K 14336 15.1 against 13.0).
template <int MT, bool YBF16>
int skinny(const char* fn, const uint8_t* qx, const uint8_t* sx, const uint8_t* qw, const uint8_t* sw, void* y, int M, int N,
           int K, hipStream_t stream) {
    constexpr int kRowsPerTile = 16 * 256;
    if (N <= kRowsPerTile)
        return launch_skinny<MT, 1, MT == 1 ? 8 : 4, 2, YBF16>(fn, qx, sx, qw, sw, y, M, N, K, stream);
    if (N <= 2 * kRowsPerTile) return launch_skinny<MT, 2, 8, 2, YBF16>(fn, qx, sx, qw, sw, y, M, N, K, stream);
    if (MT == 1 || N <= 4 * kRowsPerTile) return launch_skinny<MT, 4, 4, 2, YBF16>(fn, qx, sx, qw, sw, y, M, N, K, stream);
    return launch_skinny<MT, 7, 4, 1, YBF16>(fn, qx, sx, qw, sw, y, M, N, K, stream);
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
    if (M > kSkinnyM) return kc::mx::gemm_tile<YBF16>(fn, qx, sx, qw, sw, y, M, N, K, stream);
    const int m = static_cast<int>(M), n = static_cast<int>(N), k = static_cast<int>(K);
    switch ((m + 15) / 16) {
        case 1: return skinny<1, YBF16>(fn, qx, sx, qw, sw, y, m, n, k, stream);
        case 2: return skinny<2, YBF16>(fn, qx, sx, qw, sw, y, m, n, k, stream);
        case 3: return skinny<3, YBF16>(fn, qx, sx, qw, sw, y, m, n, k, stream);
        default: return skinny<4, YBF16>(fn, qx, sx, qw, sw, y, m, n, k, stream);
    }
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
    // 32-bit lane offsets (256 rows of K / 2 bytes), tile counts and launch sizes
    if (K > (1 << 24) || M > (1 << 30) || N > (1 << 30) || ((M + 15) / 16) > (int64_t{1} << 26) / ((N + 15) / 16))
        return set_error(KC_ERR_INVALID_ARGUMENT, "%s: M=%lld N=%lld K=%lld too large", fn, (long long)M, (long long)N,
                         (long long)K);
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
