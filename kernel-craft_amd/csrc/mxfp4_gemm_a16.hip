// mxfp4_gemm_a16.hip -- bf16 activations times MXFP4 weights on gfx950, the linear
// layer of decode batches (one token: mxfp4_gemv.hip).  No counterpart in the reference.
//
//   Y[m, n] = sum_k x[m, k] * e2m1(qw[n, k]) 2^(sw[n, k / 32] - 127)
//
// An E2M1 value times a power of two is a bf16 value, so the weights are decoded in
// registers (v_cvt_scalef32_pk_bf16_fp4: two codes and their scale in one
// instruction) and multiplied on the bf16 matrix cores with fp32 accumulation; the
// only rounding is that of Y.  Scale bytes 0 and 1 give subnormal bf16 values, exactly;
// a code times a scale past bf16's range (bytes 253 and 254 with large codes) is an
// infinity, as it is dequantized.
//
// Bound by the weight stream (0.53 bytes a weight) on wide layers (M 13, N 28672, K 4096
// 13.8 us, 4.7 TB/s), by the reads of X, one for every RT tiles of rows, on narrow ones.
// A workgroup of KW waves owns RT tiles of 16 weight rows and MT tiles of 16 tokens; K
// advances in spans of four steps of 256 values, which the waves take in turn, and
// their partial sums meet in LDS in a fixed order.  Tokens past 16 MT are further
// workgroups.  KW is 8 where one or two tiles of rows leave room (M 13, N 4096,
// K 14336 15.7 -> 15.1 us), 4 elsewhere (M 13, N 28672, K 4096 with four tiles 17.2 at
// 8, 15.5 at 4).  The registers hold DX steps of X: two where they fit (N 11008,
// K 5120 13.7 -> 12.5 us), one for the two smallest tiles (no gain) and the largest.
//
// A weight load carries 8 whole rows of a step (128 bytes, a cache line each); a
// lane and its neighbour l ^ 1 exchange one 16-byte chunk, after which lane
// (i, kb) holds blocks 2 kb and 2 kb + 1 of row row_of(i) = i / 2 + 8 (i % 2).  A
// 4 x 4 transpose of dwords over the lanes l % 16 (two permlane swaps) then
// leaves dword g of block b with lane (i, g): the 8 values the matrix core wants from
// it when X is read in its own order, 64 neighbouring bytes of each row.  The 32 scale
// bytes of a row's span come with one load of 8 bytes, step kb's, to lane (i, kb), and
// two more swaps hand a step's to all of the row's lanes (a load of 8 bytes a step
// costs the load unit as many lines as the codes: M 13, N 28672, K 4096 16.5 us).
#include <algorithm>
#include <type_traits>

#include "mxfp4_gemm.hpp"

namespace {

using namespace kc::mx;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kStep = 256;   // values of K per step
constexpr int kBK = 128;     // their bytes

__device__ __forceinline__ uint32_t swap_pair(uint32_t v) {  // lane l reads lane l ^ 1
    return static_cast<uint32_t>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), 0xB1, 0xF, 0xF, true));
}

// v[c] of lane (i, g) becomes v[g] of lane (i, c).
__device__ __forceinline__ void transpose4(uint32_t (&v)[4]) {
    auto swap32 = [](uint32_t& a, uint32_t& b) {  // lanes 32-63 of a with lanes 0-31 of b
        const auto r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
        a = r[0];
        b = r[1];
    };
    auto swap16 = [](uint32_t& a, uint32_t& b) {  // odd rows of 16 lanes of a with even rows of b
        const auto r = __builtin_amdgcn_permlane16_swap(a, b, false, false);
        a = r[0];
        b = r[1];
    };
    swap32(v[0], v[2]);
    swap32(v[1], v[3]);
    swap16(v[0], v[1]);
    swap16(v[2], v[3]);
}

// 8 codes -> 8 bf16 values at scale byte b.
__device__ __forceinline__ bf16x8 decode(uint32_t c, uint32_t b) {
    const float s = scale_operand(b);
    const bf16x2 p = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0), q = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1);
    const bf16x2 r = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2), t = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3);
    return bf16x8{p.x, p.y, q.x, q.y, r.x, r.y, t.x, t.y};
}

// v of the lanes (i, S), in all lanes (i, .).
template <int S>
__device__ __forceinline__ uint32_t of_group(uint32_t v) {
    const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);  // groups 0, 1 twice; 2, 3 twice
    const uint32_t h = r[S >> 1];
    const auto q = __builtin_amdgcn_permlane16_swap(h, h, false, false);
    return q[S & 1];
}

template <int MT, int RT, int KW, int DX>
__global__ __launch_bounds__(KW * 64) void gemm_mxfp4_a16_kernel(const uint8_t* __restrict__ qw, const uint8_t* __restrict__ sw,
                                                                 const uint16_t* __restrict__ x, uint16_t* __restrict__ y,
                                                                 int M, int N, int K, bool vec) {
    // More would not fit a wave's 512 registers, and a variant that spills is not to be
    // used: a spilled half of an address has been left out of its reload.
    static_assert(RT * MT <= 21 && RT * MT * DX <= 28, "more registers than a wave has");
    __shared__ f32x4 red[KW][RT * MT][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x >> 6));
    const int i = lane & 15, kb = lane >> 4;
    const bool even = (lane & 1) == 0;
    const int n0 = static_cast<int>(blockIdx.x) * 16 * RT, m0 = static_cast<int>(blockIdx.y) * 16 * MT;
    const int kbytes = K / 2, blocks = K / kBlock;
    const uint8_t* wbase = qw + static_cast<int64_t>(n0) * kbytes;
    const uint8_t* wsbase = sw + static_cast<int64_t>(n0) * blocks;
    const uint16_t* xbase = x + static_cast<int64_t>(m0) * K;
    const int chunk = 2 * kb + (i & 1), r8 = i >> 1, orow = (i >> 1) + 8 * (i & 1);
    uint32_t woff[RT][2], wsoff[RT], xoff[MT];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
#pragma unroll
        for (int h = 0; h < 2; ++h)
            woff[r][h] = static_cast<uint32_t>(min(n0 + 16 * r + 8 * h + r8, N - 1) - n0) * static_cast<uint32_t>(kbytes) + 16u * chunk;
        wsoff[r] = static_cast<uint32_t>(min(n0 + 16 * r + orow, N - 1) - n0) * static_cast<uint32_t>(blocks);
    }
#pragma unroll
    for (int c = 0; c < MT; ++c)
        xoff[c] = static_cast<uint32_t>(min(m0 + 16 * c + i, M - 1) - m0) * static_cast<uint32_t>(K) + 8u * kb;

    f32x4 acc[RT][MT];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int c = 0; c < MT; ++c) acc[r][c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    const int spans = K / (4 * kStep);
    const int mine = spans > wave ? (spans - wave + KW - 1) / KW : 0;  // spans wave, wave + KW, ...

    // The weights of one step; a tile's registers take the next step's as soon as
    // they have been decoded, so that RT - 1 tiles are always on their way.
    u32x4 wf[RT][2];
    u32x2 ws[RT];                // scales of the span: step kb's
    u32x4 xf[DX][MT][8];
    auto load_w = [&](int r, int step) {
        const uint8_t* wp = wbase + step * kBK;
        wf[r][0] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(wp + woff[r][0]));
        wf[r][1] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(wp + woff[r][1]));
    };
    auto load_scales = [&](int r, int span) { __builtin_memcpy(&ws[r], wsbase + 32 * span + wsoff[r] + 8 * kb, 8); };
    auto load_x = [&](int slot, int step) {
        const uint16_t* xp = xbase + step * kStep;
#pragma unroll
        for (int c = 0; c < MT; ++c)
#pragma unroll
            for (int b = 0; b < 8; ++b) xf[slot][c][b] = *reinterpret_cast<const u32x4*>(xp + xoff[c] + 32 * b);
    };
    auto multiply = [&](int r, const u32x4 (&w)[2], u32x2 sc, const u32x4 (&xv)[MT][8], auto then) {
        const uint32_t a[4] = {w[0].x, w[0].y, w[0].z, w[0].w}, b[4] = {w[1].x, w[1].y, w[1].z, w[1].w};
        uint32_t lo[4], hi[4];
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            const uint32_t an = swap_pair(a[d]), bn = swap_pair(b[d]);
            lo[d] = even ? a[d] : bn;
            hi[d] = even ? an : b[d];
        }
        then();
        transpose4(lo);
        transpose4(hi);
#pragma unroll
        for (int s = 0; s < 4; ++s) {  // blocks 2 s and 2 s + 1
            const uint32_t word = s < 2 ? sc.x : sc.y;
            const bf16x8 w0 = decode(lo[s], (word >> (16 * (s & 1))) & 255);
            const bf16x8 w1 = decode(hi[s], (word >> (16 * (s & 1) + 8)) & 255);
#pragma unroll
            for (int c = 0; c < MT; ++c)
                acc[r][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w0, __builtin_bit_cast(bf16x8, xv[c][2 * s]), acc[r][c], 0, 0, 0);
#pragma unroll
            for (int c = 0; c < MT; ++c)
                acc[r][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w1, __builtin_bit_cast(bf16x8, xv[c][2 * s + 1]), acc[r][c], 0, 0, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    if (mine > 0) {
#pragma unroll
        for (int r = 0; r < RT; ++r) load_scales(r, wave);
#pragma unroll
        for (int d = 0; d < DX; ++d) load_x(d, 4 * wave + d);
#pragma unroll
        for (int r = 0; r < RT; ++r) load_w(r, 4 * wave);
        __builtin_amdgcn_sched_barrier(0);
        // one span; `more`: the next one's loads follow its own
        auto span = [&](int at, auto mc) {
            constexpr bool more = decltype(mc)::value;
            const int next = at + KW;
            auto step = [&](auto sc) {
                constexpr int s = decltype(sc)::value;
#pragma unroll
                for (int r = 0; r < RT; ++r) {
                    const u32x2 scale = {of_group<s>(ws[r].x), of_group<s>(ws[r].y)};
                    multiply(r, wf[r], scale, xf[s % DX], [&] {
                        if constexpr (s < 3) load_w(r, 4 * at + s + 1);
                        else if constexpr (more) load_w(r, 4 * next);
                        if constexpr (s == 3 && more) load_scales(r, next);
                    });
                }
                if constexpr (s + DX < 4) load_x(s % DX, 4 * at + s + DX);
                else if constexpr (more) load_x(s % DX, 4 * next + s + DX - 4);
                __builtin_amdgcn_sched_barrier(0);
            };
            step(std::integral_constant<int, 0>{});
            step(std::integral_constant<int, 1>{});
            step(std::integral_constant<int, 2>{});
            step(std::integral_constant<int, 3>{});
        };
        for (int j = 0; j + 1 < mine; ++j) span(wave + KW * j, std::true_type{});
        span(wave + KW * (mine - 1), std::false_type{});
    }
    // The steps behind the last whole span, one a wave: zeros past K in both operands.
    for (int step = 4 * spans; step * kStep < K; ++step) {
        if (step % KW != wave) continue;
        const int valid = K - step * kStep;
        u32x4 w[RT][2], xv[MT][8];
        u32x2 sc[RT];
        const u32x4 z{0u, 0u, 0u, 0u};
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            w[r][0] = w[r][1] = z;
            if (32 * chunk < valid) {
                w[r][0] = *reinterpret_cast<const u32x4*>(wbase + step * kBK + woff[r][0]);
                w[r][1] = *reinterpret_cast<const u32x4*>(wbase + step * kBK + woff[r][1]);
            }
            uint32_t d[2] = {0, 0};
#pragma unroll
            for (int b = 0; b < 8; ++b)
                if (32 * b < valid) d[b >> 2] |= static_cast<uint32_t>(wsbase[wsoff[r] + 8 * step + b]) << (8 * (b & 3));
            sc[r] = u32x2{d[0], d[1]};
        }
#pragma unroll
        for (int c = 0; c < MT; ++c)
#pragma unroll
            for (int b = 0; b < 8; ++b) {
                xv[c][b] = z;
                if (32 * b < valid) xv[c][b] = *reinterpret_cast<const u32x4*>(xbase + step * kStep + xoff[c] + 32 * b);
            }
#pragma unroll
        for (int r = 0; r < RT; ++r) multiply(r, w[r], sc[r], xv, [] {});
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
        // D: lane (i, g) holds operand rows 4 g + v of W, outputs n = 2 g, 2 g + 8,
        // 2 g + 1, 2 g + 9 (v = 0 .. 3), of token i
        const int m = m0 + 16 * (t % MT) + i;
        if (m >= M) continue;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int n = n0 + 16 * (t / MT) + 2 * kb + 8 * h;
            if (n >= N) break;
            const float v0 = h ? v.y : v.x, v1 = h ? v.w : v.z;
            uint16_t* o = y + static_cast<int64_t>(m) * N + n;
            if (vec) {
                *reinterpret_cast<uint32_t*>(o) = kc::pack_bf16x2(v0, v1);
            } else {
                o[0] = kc::f32_to_bf16(v0);
                if (n + 1 < N) o[1] = kc::f32_to_bf16(v1);
            }
        }
    }
}

template <int MT, int RT, int KW, int DX>
int launch(const char* fn, const uint8_t* qw, const uint8_t* sw, const uint16_t* x, uint16_t* y, int M, int N, int K,
           hipStream_t stream) {
    const dim3 grid((N + 16 * RT - 1) / (16 * RT), (M + 16 * MT - 1) / (16 * MT));
    gemm_mxfp4_a16_kernel<MT, RT, KW, DX><<<grid, KW * 64, 0, stream>>>(qw, sw, x, y, M, N, K,
                                                                       N % 2 == 0 && kc::aligned(y, 4));
    return kc::check_launch(fn);
}

// Tokens (tiles of 16) and weight rows (tiles of 16) per workgroup, and what a
// workgroup takes in hundredths of a microsecond per step of 256 values and beside
// the steps, with every CU holding one (fitted to K 4096, 8192 and 14336).  More rows
// share the reads of X, more tokens those of the weights and their decoding, fewer of
// both fill the CUs: M 13, N 28672, K 4096 14.1 us with 1 and 7, 15.4 with 1 and 4, 29.8
// with 1 and 1; M 13, N 4096, K 14336 14.9 with 1 and 1, 23.2 with 1 and 4; M 64, same
// N and K 24.5 with 1 and 4, 37.0 with 2 and 4, 62 with 3 and 7; M 32, N 28672, K 4096
// 19.8 with 2 and 7, 30.4 with 1 and 4.
// The last four are the kernel of mxfp4_gemm_a16_tile.hip (128 rows; K a multiple of
// 128): M 64, N 28672, K 4096 24 us against 38 with 2 and 7; M 128 39 with 128 tokens, 43
// with 64; M 2048, N 4096 78 and 86; M 64, N 14336 16.9 in tiles of 32 tokens, 21.2 in one
// of 64; M 128, N 6144 15.5 and 19.4 (27 with 1 and 7).  The expected times are up to 10 % over and 30 % under the
// measured ones (most where X comes from L2 many times); on 21 shapes of 2 to 2048 tokens
// the least of them is the fastest.
struct Cost {
    int mt, rt, step, fixed;
};
constexpr int kCus = 256;
constexpr int kTileRt = 8;  // 128 rows: the other kernel
constexpr Cost kCosts[] = {{1, 1, 22, 260}, {1, 2, 27, 265}, {1, 4, 40, 260}, {1, 7, 84, 100}, {2, 4, 64, 310}, {2, 7, 88, 250},
                           {3, 7, 100, 370}, {2, kTileRt, 84, 150}, {3, kTileRt, 84, 250}, {4, kTileRt, 107, 130},
                           {8, kTileRt, 175, 200}};

int best(int M, int N, int K, bool tile) {
    const int64_t steps = (K + kStep - 1) / kStep;
    int which = 0;
    int64_t least = INT64_MAX;
    for (int i = 0; i < static_cast<int>(sizeof(kCosts) / sizeof(kCosts[0])); ++i) {
        const Cost& c = kCosts[i];
        if (c.rt == kTileRt && !tile) continue;
        const int64_t wgs = int64_t{(N + 16 * c.rt - 1) / (16 * c.rt)} * ((M + 16 * c.mt - 1) / (16 * c.mt));
        const int64_t cost = (wgs + kCus - 1) / kCus * steps * c.step + c.fixed;
        if (cost < least) least = cost, which = i;
    }
    return which;
}

}  // namespace

extern "C" int kc_gemm_mxfp4_bf16(const uint8_t* d_qw, const uint8_t* d_sw, const uint16_t* d_x, uint16_t* d_y,
                                  int64_t M, int64_t N, int64_t K, kc_stream_t stream) {
    const char* fn = "kc_gemm_mxfp4_bf16";
    const int st = kc::mx::check_gemm(fn, M, N, K, d_y);
    if (st != KC_SUCCESS || M == 0 || N == 0) return st;
    if (K == 0) return kc::mx::fill_zero<true>(fn, d_y, M * N, stream);
    if (M > 16 * 65535)  // tiles of tokens are the grid's second dimension
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: M=%lld too large, at most %d", fn, (long long)M, 16 * 65535);
    if (!d_qw || !d_sw || !d_x) return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: null device pointer", fn);
    if (!kc::aligned(d_qw, 16) || !kc::aligned(d_x, 16))
        return kc::set_error(KC_ERR_INVALID_ARGUMENT, "%s: the codes and x must be 16-byte aligned", fn);
    const int m = static_cast<int>(M), n = static_cast<int>(N), k = static_cast<int>(K);
    int done = KC_SUCCESS;
    if (m == 1 && kc::mx::gemv(fn, d_qw, d_sw, d_x, d_y, n, k, stream, &done)) return done;
    switch (best(m, n, k, k % 128 == 0 && kc::aligned(d_sw, 4))) {
        case 0: return launch<1, 1, 8, 1>(fn, d_qw, d_sw, d_x, d_y, m, n, k, stream);
        case 1: return launch<1, 2, 8, 1>(fn, d_qw, d_sw, d_x, d_y, m, n, k, stream);
        case 2: return launch<1, 4, 4, 2>(fn, d_qw, d_sw, d_x, d_y, m, n, k, stream);
        case 3: return launch<1, 7, 4, 2>(fn, d_qw, d_sw, d_x, d_y, m, n, k, stream);
        case 4: return launch<2, 4, 4, 2>(fn, d_qw, d_sw, d_x, d_y, m, n, k, stream);
        case 5: return launch<2, 7, 4, 2>(fn, d_qw, d_sw, d_x, d_y, m, n, k, stream);
        case 6: return launch<3, 7, 4, 1>(fn, d_qw, d_sw, d_x, d_y, m, n, k, stream);
        case 7: return kc::mx::gemm_a16_tile(fn, 2, d_qw, d_sw, d_x, d_y, m, n, k, stream);
        case 8: return kc::mx::gemm_a16_tile(fn, 3, d_qw, d_sw, d_x, d_y, m, n, k, stream);
        case 9: return kc::mx::gemm_a16_tile(fn, 4, d_qw, d_sw, d_x, d_y, m, n, k, stream);
        default: return kc::mx::gemm_a16_tile(fn, 8, d_qw, d_sw, d_x, d_y, m, n, k, stream);
    }
}
