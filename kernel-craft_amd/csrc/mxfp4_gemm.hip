// mxfp4_gemm.hip -- the product of two MXFP4 matrices on gfx950's scaled matrix
// cores: entry points, and the kernel for decode batches (M <= 16, or 48 and 64 on layers
// of few rows).  More: mxfp4_gemm_tile.hip.  No counterpart in the reference.
//
//   Y[m, n] = sum_b 2^(sx[m, b] + sw[n, b] - 254) sum_{k in block b} e2m1(qx[m, k]) e2m1(qw[n, k])
//
// gemm_mxfp4_skinny_kernel is bound by the weight stream (0.53 bytes a weight).  A workgroup of KW
// waves owns RT tiles of 16 weight rows and all MT = ceil(M / 16) tiles of X; K advances
// in spans of 1024 values, 512 bytes of every row, which the waves take in turn, and
// the KW partial sums of every output meet in LDS in a fixed order.  No barrier
// stands in the K loop and no operand goes through LDS: with K split over the waves no
// two of them read the same bytes.  A step's registers take the next span's as soon as
// they have been multiplied.
//
// A load carries 8 whole rows of a quarter span, a step (128 bytes, a cache line each):
// lane l takes 16-byte chunk 2 (l / 16) + l % 2 of row 8 h + (l % 16) / 2.  A lane and its
// neighbour l ^ 1 exchange one chunk each, after which lane (i, kb) holds chunks
// 2 kb and 2 kb + 1, two blocks of 32, of row row_of(i) = i / 2 + 8 (i % 2): the
// operands of two matrix-core instructions of 128 values.  The 32 scale bytes of a row's
// span come with one load of 8 bytes, step kb's, to lane (i, kb); a 4 x 4 transpose of
// 16-bit pairs over the lanes l % 16 leaves each lane its own two blocks' bytes of all
// four steps (a 16-bit load a step costs the load unit as many lines as the codes).
#include <algorithm>
#include <type_traits>

#include "mxfp4_gemm.hpp"

namespace {

using namespace kc::mx;

constexpr int kBK = 128;       // bytes of K per step
constexpr int kSpan = 4 * kBK;  // and per span
constexpr int kSkinnyM = 64;

struct Frag {
    u32x4 h0, h1;
};

__device__ __forceinline__ uint32_t swap_pair(uint32_t v) {  // lane l reads lane l ^ 1
    return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xB1, 0xF, 0xF, true));
}

// Chunks 2 kb (lo) and 2 kb + 1 (hi) of the lane's operand row.
__device__ __forceinline__ void as_operands(const Frag& f, bool even, u32x4& lo, u32x4& hi) {
#pragma unroll
    for (int d = 0; d < 4; ++d) {
        const uint32_t a = f.h0[d], b = f.h1[d], an = swap_pair(a), bn = swap_pair(b);
        lo[d] = even ? a : bn;
        hi[d] = even ? an : b;
    }
}

// Lane (i, g) holds pairs 0 .. 3 of step g (16 bits each, two to a word); it gets pair g
// of steps 0, 1 (x) and 2, 3 (y).
__device__ __forceinline__ u32x2 transpose_pairs(u32x2 v, uint32_t select) {
    uint32_t a = v.x, b = v.y;
    const auto q = __builtin_amdgcn_permlane32_swap(a, b, false, false);  // lanes 32-63 of a with 0-31 of b
    a = q[0];
    b = q[1];
    const auto r = __builtin_amdgcn_permlane16_swap(a, a, false, false);  // even row's in [0], odd row's in [1]
    const auto s = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    return u32x2{__builtin_amdgcn_perm(r[1], r[0], select), __builtin_amdgcn_perm(s[1], s[0], select)};
}

template <int MT, int RT, int KW, bool YBF16>
__global__ __launch_bounds__(KW * 64) void gemm_mxfp4_skinny_kernel(
    const uint8_t* __restrict__ qx, const uint8_t* __restrict__ sx, const uint8_t* __restrict__ qw,
    const uint8_t* __restrict__ sw, void* __restrict__ y, int M, int N, int K, bool vec) {
    __shared__ f32x4 red[KW][RT * MT][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const int i = lane & 15, kb = lane >> 4;
    const bool even = (lane & 1) == 0;
    const uint32_t select = kb & 1 ? 0x07060302u : 0x05040100u;  // high or low halves of two words
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
        wsoff[r] = static_cast<uint32_t>(min(n0 + 16 * r + orow, N - 1) - n0) * static_cast<uint32_t>(blocks);
    }
#pragma unroll
    for (int c = 0; c < MT; ++c) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
            xoff[c][h] = static_cast<uint32_t>(min(16 * c + 8 * h + r8, M - 1)) * static_cast<uint32_t>(kbytes) + 16u * chunk;
        xsoff[c] = static_cast<uint32_t>(min(16 * c + orow, M - 1)) * static_cast<uint32_t>(blocks);
    }

    f32x4 acc[RT][MT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int c = 0; c < MT; ++c) acc[r][c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    start(acc);
    const int spans = kbytes / kSpan;
    const int mine = spans > wave ? (spans - wave + KW - 1) / KW : 0;  // spans wave, wave + KW, ...

    // acc += W X^T of one step, its scales at `byte` and the next of their words
    auto multiply = [&](const Frag (&w)[RT], const Frag (&x)[MT], const uint32_t (&wsc)[RT], const uint32_t (&xsc)[MT],
                        auto bc) {
        constexpr int byte = decltype(bc)::value;
        u32x4 b0[MT], b1[MT];
#pragma unroll
        for (int c = 0; c < MT; ++c) as_operands(x[c], even, b0[c], b1[c]);
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            u32x4 a0, a1;
            as_operands(w[r], even, a0, a1);
#pragma unroll
            for (int c = 0; c < MT; ++c) mfma<byte, true>(acc[r][c], a0, b0[c], wsc[r], xsc[c]);
#pragma unroll
            for (int c = 0; c < MT; ++c) mfma<byte + 1, true>(acc[r][c], a1, b1[c], wsc[r], xsc[c]);
        }
    };
    Frag wf[4][RT], xf[4][MT];
    u32x2 ws[RT], xs[MT];
    auto load = [&](int s, int span) {
        const uint8_t *wp = wbase + span * kSpan + s * kBK, *xp = qx + span * kSpan + s * kBK;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            wf[s][r].h0 = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(wp + woff[r][0]));
            wf[s][r].h1 = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(wp + woff[r][1]));
        }
#pragma unroll
        for (int c = 0; c < MT; ++c) {
            xf[s][c].h0 = *reinterpret_cast<const u32x4*>(xp + xoff[c][0]);
            xf[s][c].h1 = *reinterpret_cast<const u32x4*>(xp + xoff[c][1]);
        }
    };
    auto load_scales = [&](int span) {
#pragma unroll
        for (int r = 0; r < RT; ++r) __builtin_memcpy(&ws[r], wsbase + 32 * span + wsoff[r] + 8 * kb, 8);
#pragma unroll
        for (int c = 0; c < MT; ++c) __builtin_memcpy(&xs[c], sx + 32 * span + xsoff[c] + 8 * kb, 8);
    };
    if (mine > 0) {
        load_scales(wave);
#pragma unroll
        for (int s = 0; s < 4; ++s) load(s, wave);
        __builtin_amdgcn_sched_barrier(0);
        auto span = [&](int next, auto mc) {
            constexpr bool more = decltype(mc)::value;
            uint32_t wsc[2][RT], xsc[2][MT];
#pragma unroll
            for (int r = 0; r < RT; ++r) {
                const u32x2 v = transpose_pairs(ws[r], select);
                wsc[0][r] = v.x;
                wsc[1][r] = v.y;
            }
#pragma unroll
            for (int c = 0; c < MT; ++c) {
                const u32x2 v = transpose_pairs(xs[c], select);
                xsc[0][c] = v.x;
                xsc[1][c] = v.y;
            }
            if constexpr (more) load_scales(next);
            auto step = [&](auto sc) {
                constexpr int s = decltype(sc)::value;
                multiply(wf[s], xf[s], wsc[s / 2], xsc[s / 2], std::integral_constant<int, 2 * (s % 2)>{});
                if constexpr (more) load(s, next);
                __builtin_amdgcn_sched_barrier(0);
            };
            step(std::integral_constant<int, 0>{});
            step(std::integral_constant<int, 1>{});
            step(std::integral_constant<int, 2>{});
            step(std::integral_constant<int, 3>{});
        };
        for (int j = 1; j < mine; ++j) span(wave + KW * j, std::true_type{});
        span(0, std::false_type{});
    }
    // The steps behind the last whole span, one a wave: no codes and scale bytes 0 past K.
    for (int step = 4 * spans; step * kBK < kbytes; ++step) {
        if (step % KW != wave) continue;
        const int kvalid = kbytes - step * kBK;
        auto tail = [&](const uint8_t* base, const uint32_t (&off)[2]) {
            const u32x4 z{0u, 0u, 0u, 0u};
            Frag f{z, z};
            if (16 * chunk < kvalid) {
                f.h0 = *reinterpret_cast<const u32x4*>(base + step * kBK + off[0]);
                f.h1 = *reinterpret_cast<const u32x4*>(base + step * kBK + off[1]);
            }
            return f;
        };
        auto tail_scales = [&](const uint8_t* p) {
            p += 8 * step + 2 * kb;
            uint32_t v = 0;
            if (32 * kb < kvalid) v = p[0];
            if (32 * kb + 16 < kvalid) v |= static_cast<uint32_t>(p[1]) << 8;
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
        multiply(w, x, wsc, xsc, std::integral_constant<int, 0>{});
    }
    settle(acc);
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

template <int MT, int RT, int KW, bool YBF16>
int launch_skinny(const char* fn, const uint8_t* qx, const uint8_t* sx, const uint8_t* qw, const uint8_t* sw, void* y, int M,
                  int N, int K, hipStream_t stream) {
    gemm_mxfp4_skinny_kernel<MT, RT, KW, YBF16><<<static_cast<unsigned>((N + 16 * RT - 1) / (16 * RT)), KW * 64, 0, stream>>>(
        qx, sx, qw, sw, y, M, N, K, N % 2 == 0 && kc::aligned(y, 4));
    return kc::check_launch(fn);
}

// Row tiles per workgroup, us at 1, 2 and 4 of them: one tile of X N 4096, K 14336 8.4,
// 10.9, 15.7, N 11008, K 5120 7.5, 8.5, 8.7, N 28672, K 4096 15.0, 13.7, 14.7; two tiles
// N 4096, K 14336 10.7, 13.2, 19.6, N 6144, K 4096 7.0, 6.3, 8.4; four N 4096, K 14336 15.1,
// 19.3, 29.8.  Eight waves instead of four: one tile of X 4.2 against 4.1 us (N 4096,
// K 4096) and 8.2 against 8.4 (K 14336), more tiles spill.
template <int MT, bool YBF16>
int skinny(const char* fn, const uint8_t* qx, const uint8_t* sx, const uint8_t* qw, const uint8_t* sw, void* y, int M, int N,
           int K, hipStream_t stream) {
    if constexpr (MT < 4) {  // four tiles come with at most 4096 rows
        if (N > (MT == 1 ? 12288 : 4096)) return launch_skinny<MT, 2, 4, YBF16>(fn, qx, sx, qw, sw, y, M, N, K, stream);
    }
    return launch_skinny<MT, 1, 4, YBF16>(fn, qx, sx, qw, sw, y, M, N, K, stream);
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
    // More than one tile of tokens on layers of many rows read X less often from LDS
    // (M 32, N 28672, K 4096 16.4 -> 14.8 us; M 64 20.5 -> 15.4), and so do four tiles on more
    // than 4096 (M 64, N 6144, K 2048 6.5 -> 4.9, K 4096 8.6 -> 7.9, K 14336 the same; M 48 7.4
    // there, 7.8 in LDS tiles; M 64, N 4096, K 4096 6.6 and 6.5, K 14336 15.1 and 19.4).
    if (M > kSkinnyM || (M > 16 && N > 8192) || (M > 48 && N > 4096)) return kc::mx::gemm_tile<YBF16>(fn, qx, sx, qw, sw, y, M, N, K, stream);
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
    if (K > (1 << 24) || M > (1 << 28) || N > (1 << 28) || ((M + 15) / 16) > (int64_t{1} << 26) / ((N + 15) / 16))
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
