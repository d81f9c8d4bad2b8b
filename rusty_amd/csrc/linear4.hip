// Linears with 4-bit affine weights (RQ_Q_AFFINE_U4):
//   Y[m, n] = sum_k X[m, k] W[n, k],  W[n, k] = u[n, k] s[n, k/G] + b[n, k/G],
// u in 0..15, two codes a byte (the even k in the low nibble), an f32 scale and
// bias per G consecutive k of a row.
//
// Bound by the weight's bytes: n k / 2 of codes and 8 n k / G of scales and
// biases, each read once.  Codes enter the products exactly, as fp16 16 + u: a
// nibble at mantissa bits 6..9 under the exponent of 16.0 (one shift and one
// v_and_or per two codes, the pairs k and k + 4 of each 8).  Per group, with
// t = sum (16 + u) x and xs = sum x in f32,
//   sum (u s + b) x = s t + (b - 16 s) xs,
// so a weight is never rounded, and the offset costs f32 rounding of terms at
// most (16 + 15) / 15 times the largest ones.
//  * m <= 2: k_linear4_dot, v_dot2_f32_f16 with the activation rows in registers;
//  * m <= 16: k_linear4_mfma, the rows on the matrix cores;
//  * more: 16 rows at a time, or (many rows) the codes widened to bytes once
//    and the 8-bit GEMM (launch_linear4).
#include <algorithm>
#include <type_traits>

#include "common.hpp"

namespace rq {
namespace {

constexpr int TH = 256;
// More rows than this: launch_widened (us, 16 at a time / widened: 48 rows, 4096x4096 22 / 35,
// 11008x4096 44 / 46, 4096x11008 48 / 47; 64 rows 28 / 35, 60 / 46, 64 / 47; 96 rows 42 / 40, 90 / 56, 97 / 59)
constexpr int kRowsBySixteen = 48;
constexpr uint32_t kOOB = 0x80000000u;  // any offset past a buffer resource reads zero

typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef float f2_t __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ __amdgpu_buffer_rsrc_t make_rsrc(const void *p, uint32_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, bytes, 0x00020000);
}
// aux bit 1 = non-temporal (streamed once), 0 = default caching
template <int AUX>
__device__ __forceinline__ u32x4 bload(__amdgpu_buffer_rsrc_t r, uint32_t off) {
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, AUX));
}
__device__ __forceinline__ float bload1(__amdgpu_buffer_rsrc_t r, uint32_t off) {
    return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, off, 0, 0));
}
__device__ __forceinline__ float dot2(uint32_t a, uint32_t b, float c) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2_t, a), __builtin_bit_cast(h2_t, b), c, false);
}
template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xF, 0xF, false));
}
__device__ __forceinline__ float readlane(float v, int l) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), l));
}
// Sum over the 64 lanes, uniform across the wave.
__device__ __forceinline__ float wave_total(float v) {
    v += dpp<0xB1>(v);   // quad_perm [1,0,3,2]
    v += dpp<0x4E>(v);   // quad_perm [2,3,0,1]
    v += dpp<0x141>(v);  // row_half_mirror
    v += dpp<0x140>(v);  // row_mirror: each 16-lane row holds its sum
    return (readlane(v, 0) + readlane(v, 16)) + (readlane(v, 32) + readlane(v, 48));
}
// 8 codes (a dword) -> fp16 16 + u of codes (0, 4), (1, 5), (2, 6), (3, 7).
__device__ __forceinline__ u32x4 expand8(uint32_t w) {
    const uint32_t m = 0x03C003C0u, e = 0x4C004C00u;
    return u32x4{((w << 6) & m) | e, ((w << 2) & m) | e, ((w >> 2) & m) | e, ((w >> 6) & m) | e};
}
// 8 consecutive halves in that order: (0, 4), (1, 5), (2, 6), (3, 7).
__device__ __forceinline__ u32x4 pair_up(u32x4 x) {
    return u32x4{__builtin_amdgcn_perm(x.z, x.x, 0x05040100u), __builtin_amdgcn_perm(x.z, x.x, 0x07060302u),
                 __builtin_amdgcn_perm(x.w, x.y, 0x05040100u), __builtin_amdgcn_perm(x.w, x.y, 0x07060302u)};
}

// Each lane's x from the lane 8 places on in its row of 16.
__device__ __forceinline__ u32x4 turn8(u32x4 x) {
    u32x4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x[e], 0x128, 0xF, 0xF, false);
    return y;
}

// The largest v of the four lanes l % 16, l % 16 + 16, ... (EIGHT: of the eight l % 8, l % 8 + 8, ...).
template <bool EIGHT>
__device__ __forceinline__ float row_max(float v) {
    const auto p = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    const unsigned p0 = p[0], p1 = p[1];
    v = fmaxf(__builtin_bit_cast(float, p0), __builtin_bit_cast(float, p1));
    const auto q = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    const unsigned q0 = q[0], q1 = q[1];
    v = fmaxf(__builtin_bit_cast(float, q0), __builtin_bit_cast(float, q1));
    return EIGHT ? fmaxf(v, dpp<0x128>(v)) : v;
}

// 8 f32 values (a, b) times 2^-sh -> hi = fp16(v), lo = fp16(v - hi) in the
// codes' pair order: hi + lo is the scaled v to 2^-22 relative from 2^-3 to fp16's largest, and
// to 2^-25 below.
template <bool SC>
__device__ __forceinline__ void split8(floatx4 a, floatx4 b, int sh, u32x4 &hi, u32x4 &lo) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        f2_t v = {a[e], b[e]};
        if constexpr (SC) v = f2_t{__builtin_amdgcn_ldexpf(v.x, -sh), __builtin_amdgcn_ldexpf(v.y, -sh)};
        const h2_t h = __builtin_convertvector(v, h2_t);
        const h2_t l = __builtin_convertvector((f2_t{v.x - (float)h.x, v.y - (float)h.y}), h2_t);
        hi[e] = __builtin_bit_cast(uint32_t, h);
        lo[e] = __builtin_bit_cast(uint32_t, l);
    }
}

// Y[m, n] term by term, each weight as u s + b, across the wave.  For sums s t + (b - 16 s) xs that came out
// infinite or NaN: an infinite activation makes them inf - inf, and t may pass f32's range where
// the result does not.  A wave's trip through both rows per output: 8 rows 11008x4096 12.6 us, one of them
// infinite 58, all 286; the test costs calls without any at most 0.1 us.
template <bool XF>
__device__ __forceinline__ float by_terms(const uint8_t *W, const float *scales, const float *biases, const void *X,
                                          int K, int group, int n, int m) {
    const uint32_t *codes = reinterpret_cast<const uint32_t *>(W + (size_t)n * (K / 2));
    const size_t g0 = (size_t)n * (K / group);
    float y = 0.0f;
    for (int c = threadIdx.x & 63; c < K / 8; c += 64) {
        const uint32_t w = codes[c];
        const float s = scales[g0 + 8 * c / group], b = biases ? biases[g0 + 8 * c / group] : 0.0f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const size_t at = (size_t)m * K + 8 * c + e;
            const float x = XF ? static_cast<const float *>(X)[at] : (float)static_cast<const _Float16 *>(X)[at];
            y = __builtin_fmaf(__builtin_fmaf((float)(w >> (4 * e) & 15u), s, b), x, y);
        }
    }
    return wave_total(y);
}

// m <= M = 1 or 2 rows.  A block owns R * RP weight rows; thread tt of a row
// group (TPR threads) owns the 16-byte chunks (32 codes, one group) tt, tt +
// TPR, ... of each of its R rows, so a wave reads 1 KiB of a row at a time, all
// R * CPT chunks in flight before the first is used.  Rows past N and chunks past K
// are offsets past the resource and read as zero.  The threads' partial sums
// meet in LDS; a wave then finishes whole (row, token) sums.
// XF: f32 rows; each chunk of a row is scaled by the power of two that puts its
// largest magnitude in [2^14, 2^15) and carried as two fp16 terms.
// One row: 4096x4096 4.5 us in a graph (one launch's first bytes and end bound it), 32000x2048 9.0,
// 4.5 TB/s (HBM).
template <int M, int CPT, int TPR, int R, bool XF>
__global__ __launch_bounds__(TH) void k_linear4_dot(const uint8_t *__restrict__ W, const float *__restrict__ scales,
                                                    const float *__restrict__ biases, const void *__restrict__ X,
                                                    void *__restrict__ Y, int y_f16, int m_act, int N, int K, int group) {
    constexpr int RP = TH / TPR, ROWS = R * RP, TASKS = ROWS * M;
    __shared__ float part[TASKS][TPR];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6, rp = t / TPR, tt = t % TPR;
    const int C = K / 32, gk = K / group, row0 = blockIdx.x * ROWS, rows_here = min(ROWS, N - row0);

    const auto rx = make_rsrc(X, (uint32_t)m_act * (uint32_t)K * (XF ? 4u : 2u));
    u32x4 xr[CPT][M][XF ? 8 : 4];
#pragma unroll
    for (int j = 0; j < CPT; ++j)
#pragma unroll
        for (int m = 0; m < M; ++m) {
            const int c = tt + TPR * j;
            const uint32_t off = c < C ? ((uint32_t)m * K + (uint32_t)c * 32) * (XF ? 4u : 2u) : kOOB;
#pragma unroll
            for (int i = 0; i < (XF ? 8 : 4); ++i) xr[j][m][i] = bload<0>(rx, off + 16 * i);
        }
    float sg[R][CPT], bg[R][CPT];
    int cg[CPT];
#pragma unroll
    for (int j = 0; j < CPT; ++j) cg[j] = (int)((unsigned)(tt + TPR * j) * 32u / (unsigned)group);
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < CPT; ++j) {
            // (a chunk or row that is not there takes group 0's: it meets zeros, or is not stored)
            const bool ok = tt + TPR * j < C && r * RP + rp < rows_here;
            const size_t g = ok ? (size_t)(row0 + r * RP + rp) * gk + cg[j] : 0;
            sg[r][j] = scales[g];
            bg[r][j] = biases ? biases[g] : 0.0f;
        }
    const auto rw = make_rsrc(W + (size_t)row0 * (K / 2), (uint32_t)rows_here * (uint32_t)(K / 2));
    u32x4 w[R][CPT];
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
        for (int j = 0; j < CPT; ++j) {
            const int c = tt + TPR * j;
            w[r][j] = bload<2>(rw, c < C ? (uint32_t)(r * RP + rp) * (uint32_t)(K / 2) + (uint32_t)c * 16u : kOOB);
        }

    // the activations in the codes' pair order (XF: two terms and 2^e), and their sums
    u32x4 xh[CPT][M][4], xl[XF ? CPT : 1][XF ? M : 1][4];
    float pe[XF ? CPT : 1][XF ? M : 1], xs[CPT][M];
#pragma unroll
    for (int j = 0; j < CPT; ++j)
#pragma unroll
        for (int m = 0; m < M; ++m) {
            if constexpr (XF) {
                float amax = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const floatx4 f = __builtin_bit_cast(floatx4, xr[j][m][i]);
                    amax = fmaxf(fmaxf(fmaxf(amax, fabsf(f.x)), fmaxf(fabsf(f.y), fabsf(f.z))), fabsf(f.w));
                }
                // amax = f 2^E, f in [0.5, 1); an infinite or NaN one gives E = 0 and stays what it is
                const int ex = max(__builtin_amdgcn_frexp_expf(amax) - 15, -126);
                pe[j][m] = __builtin_amdgcn_ldexpf(1.0f, ex);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    split8<true>(__builtin_bit_cast(floatx4, xr[j][m][2 * i]),
                                 __builtin_bit_cast(floatx4, xr[j][m][2 * i + 1]), ex, xh[j][m][i], xl[j][m][i]);
            } else {
#pragma unroll
                for (int i = 0; i < 4; ++i) xh[j][m][i] = pair_up(xr[j][m][i]);
            }
            float s = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s = dot2(xh[j][m][i][e], 0x3C003C00u, s);
                    if constexpr (XF) s = dot2(xl[j][m][i][e], 0x3C003C00u, s);
                }
            xs[j][m] = XF ? s * pe[j][m] : s;
        }
#pragma unroll
    for (int r = 0; r < R; ++r) {
        float p[M];
#pragma unroll
        for (int m = 0; m < M; ++m) p[m] = 0.0f;
#pragma unroll
        for (int j = 0; j < CPT; ++j) {
            float d[M];
#pragma unroll
            for (int m = 0; m < M; ++m) d[m] = 0.0f;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const u32x4 u = expand8(w[r][j][i]);
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int m = 0; m < M; ++m) {
                        d[m] = dot2(u[e], xh[j][m][i][e], d[m]);
                        if constexpr (XF) d[m] = dot2(u[e], xl[j][m][i][e], d[m]);
                    }
            }
            const float c = __builtin_fmaf(-16.0f, sg[r][j], bg[r][j]);
#pragma unroll
            for (int m = 0; m < M; ++m) {
                p[m] = __builtin_fmaf(sg[r][j], XF ? d[m] * pe[j][m] : d[m], p[m]);
                p[m] = __builtin_fmaf(c, xs[j][m], p[m]);
            }
        }
#pragma unroll
        for (int m = 0; m < M; ++m) part[(r * RP + rp) * M + m][tt] = p[m];
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < (TASKS + 3) / 4; ++i) {
        const int task = wave + 4 * i;
        if (task >= TASKS) break;
        float v = 0.0f;
#pragma unroll
        for (int j = 0; j < TPR / 64; ++j) v += part[task][lane + 64 * j];
        float y = wave_total(v);
        const int row = task / M, m = task % M;
        if (__builtin_expect(!__builtin_isfinite(y) && row < rows_here && m < m_act, 0))
            y = by_terms<XF>(W, scales, biases, X, K, group, row0 + row, m);
        if (lane == 0 && row < rows_here && m < m_act) {
            const size_t o = (size_t)m * N + row0 + row;
            if (y_f16) static_cast<_Float16 *>(Y)[o] = (_Float16)y;
            else static_cast<float *>(Y)[o] = y;
        }
    }
}

// m <= 16 rows on v_mfma_f32_16x16x32_f16: A = 16 rows of X x 32 k, B = 32 k x
// 16 weight rows, so lane l has weight row l % 16 and, of the result, rows 4 (l /
// 16) + r, r < 4, of X.  Per group of GS steps of 32 k: t = X . (16 + U) and (B all ones)
// xs = the rows' sums, then acc += s t + (b - 16 s) xs with the lane's own s and b.
// A block of NW waves has RT tiles of 16 weight rows; wave w takes the batches of 256 k
// w, w + NW, ... (from a per-block rotation: every block reads all of X, and the
// blocks of one XCD should not ask for the same lines at once), and each
// activation fragment it loads serves all RT tiles.  Codes are loaded 8 rows x 128
// bytes per instruction and turned to operand order through the wave's own LDS
// (chunk c of row r at c ^ (r % 8)); no barrier.  The next batch's loads are in flight while
// one is multiplied.  The waves' sums meet in LDS.
// Scales and biases go through LDS too, whole rows of them first (they lie one
// after another), as (s, b - 16 s): read by each lane in place they touch 16 cache
// lines per load, which bounded the kernel (this step alone, 8 rows: 11008x4096 in groups of 64 21.2 ->
// 12.6 us, 4096x11008 in groups of 32 32.3 -> 16.9).  What is left above the bytes' 5.6 and 6.8 us
// is the loads of X, which every block reads whole, and the expansion of the codes (the table of
// shapes at launch_mfma has today's times).  Rows longer than kSegGroups groups take several rounds.
// XF: f32 rows as two fp16 terms.  In a batch where a row's largest magnitude is past fp16's range or
// below 1 (whose low terms reach fp16's subnormals, an error of 2^-25 whatever the row's size)
// every row is scaled by a power of two, so that each keeps f32 accuracy.  Looking at the batch first
// costs up to 7 % (us in a graph, without / with: 8 rows 11008x4096 18.8 / 19.3, 16 rows 27.8 / 28.9, 13 rows
// 4096x11008 25.7 / 27.5), a scaled batch 3 % more, scaling them all 28.3 for the last; multiplying first
// and again where needed spills (37).  Two waves per SIMD are asked for where they fit: with 16 rows and
// one tile the compiler otherwise takes 262 registers and one wave (16 rows 11008x4096 37.4 us, 28.9 with two).
constexpr int kSegGroups = 512;

// M8: up to 8 rows, where half of the lanes would load nothing: lanes 8-15 of each 16 take the
// next 32 k of rows 0-7 instead, whole cache lines per load and half the loads, and a
// rotation by 8 lanes brings those to their place (result rows 8-15 mix both and go unused;
// this step alone, 8 rows: 11008x4096 13.4 -> 12.7 us, f32 32000x2048 29.1 -> 19.8).
template <int RT, int NW, int GS, bool XF, bool M8>
__global__ __launch_bounds__(NW * 64, RT == 1 || M8 ? 2 : 1) void k_linear4_mfma(
    const uint8_t *__restrict__ W, const float *__restrict__ scales, const float *__restrict__ biases,
    const void *__restrict__ X, void *__restrict__ Y, int y_f16, int m_act, int N, int K, int group) {
    constexpr int NG = 8 / GS, NT = NW * 64;  // groups of a batch, threads
    __shared__ floatx4 red[NW][RT][64];
    __shared__ __attribute__((aligned(16))) uint8_t wt[NW][RT][16 * 128];
    extern __shared__ float2 sc[];  // [16 RT][pitch]
    const int t = threadIdx.x, lane = t & 63, wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int fr = lane & 15, q = lane >> 4, n0 = blockIdx.x * 16 * RT;
    const int gk = K / group, pitch = min(gk, kSegGroups) | 1;
    __amdgpu_buffer_rsrc_t rw[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        const int n = n0 + 16 * i, rows = max(0, min(16, N - n));
        rw[i] = make_rsrc(W + (rows ? (size_t)n : 0) * (K / 2), (uint32_t)rows * (uint32_t)(K / 2));
    }
    const auto rx = make_rsrc(X, (uint32_t)m_act * (uint32_t)K * (XF ? 4u : 2u));
    const uint32_t xrow = (uint32_t)(M8 ? fr & 7 : fr) * (uint32_t)K + 8u * (uint32_t)q + (M8 ? 32u * (uint32_t)(fr >> 3) : 0u);
    constexpr int XL = M8 ? 4 : 8;  // activation fragments a lane holds of a batch

    struct Batch {
        u32x4 w[RT][2], x[XF ? 2 * XL : XL];
        int g, r;  // the batch's first k: its group, from the segment's, and how far into it (in 32 k)
    };
    const int g32 = group / 32;
    floatx4 acc[RT];
#pragma unroll
    for (int i = 0; i < RT; ++i) acc[i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    const half8 ones = {1, 1, 1, 1, 1, 1, 1, 1};
    for (int g0 = 0; g0 < gk; g0 += kSegGroups) {
        const int sg = min(kSegGroups, gk - g0), kbeg = g0 * group, klen = sg * group;
        const int nb = (klen + 255) / 256;
        const int rot = (int)((blockIdx.x >> 3) * 5u + (blockIdx.x & 7u)) % nb;
        if (g0) __syncthreads();  // every wave is done with the last segment's scales
        // scales of 4 elements per thread at a time (row and group by division once per element)
        const int rows = min(16 * RT, N - n0), total = rows * sg;
        for (int i0 = t; i0 < total; i0 += 4 * NT) {
            float s[4], b[4];
            int at[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const int i = min(i0 + e * NT, total - 1), row = i / sg, g = i - row * sg;
                const size_t src = (size_t)(n0 + row) * gk + g0 + g;
                s[e] = scales[src];
                b[e] = biases ? biases[src] : 0.0f;
                at[e] = row * pitch + g;
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[at[e]] = make_float2(s[e], __builtin_fmaf(-16.0f, s[e], b[e]));
        }
        auto load = [&](Batch &b, int bi) {
            int bb = bi + rot;
            bb -= bb >= nb ? nb : 0;
            const uint32_t k0 = (uint32_t)kbeg + (uint32_t)bb * 256u;
            b.g = bb * 8 / g32;
            b.r = bb * 8 - b.g * g32;
#pragma unroll
            for (int i = 0; i < RT; ++i)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    // row 8 h + lane / 8, chunk lane % 8 (past K: the next row's codes, which meet zeros)
                    const uint32_t off = (uint32_t)(8 * h + lane / 8) * (uint32_t)(K / 2) + k0 / 2 + 16u * (lane & 7);
                    b.w[i][h] = bload<2>(rw[i], off);
                }
#pragma unroll
            for (int j = 0; j < XL; ++j) {
                const uint32_t k = k0 + 256u / XL * j;
                const bool ok = k + (M8 ? 32u * (uint32_t)(fr >> 3) : 0u) < (uint32_t)(kbeg + klen);
                if constexpr (XF) {
                    b.x[2 * j] = bload<0>(rx, ok ? (xrow + k) * 4u : kOOB);
                    b.x[2 * j + 1] = bload<0>(rx, ok ? (xrow + k) * 4u + 16u : kOOB);
                } else {
                    b.x[j] = bload<0>(rx, ok ? (xrow + k) * 2u : kOOB);
                }
            }
        };
        auto mma = [&](const Batch &b) {
            uint32_t u[RT][8];
            float2 sv[RT][NG];
            // the groups of the batch's NG pieces of GS * 32 k, which divide a group: a group
            // may start and end anywhere in a batch (96, 192, ...)
            int gi[NG], at = b.g, in = b.r;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                gi[g] = min(at, sg - 1);
                in += GS;
                at += in == g32;
                in = in == g32 ? 0 : in;
            }
#pragma unroll
            for (int i = 0; i < RT; ++i) {
                uint8_t *wl = wt[wave][i];
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const int r = 8 * h + lane / 8;
                    *reinterpret_cast<u32x4 *>(wl + r * 128 + (((lane & 7) ^ (r & 7)) << 4)) = b.w[i][h];
                }
                // (groups past the row's end, and rows past the weight, meet zeros or are
                // not stored: any place inside sc does)
                const int r = min(16 * i + fr, rows - 1);
#pragma unroll
                for (int g = 0; g < NG; ++g) sv[i][g] = sc[r * pitch + gi[g]];
#pragma unroll
                for (int j = 0; j < 8; ++j)
                    u[i][j] = *reinterpret_cast<const uint32_t *>(wl + fr * 128 + ((j ^ (fr & 7)) << 4) + 4 * q);
            }
            // sh: power of two of this lane's row of X (scaled)
            auto run = [&](auto scaled, int sh) {
                constexpr bool SC = decltype(scaled)::value;
                int back[4];  // those of the rows 4 q + r that acc holds
#pragma unroll
                for (int r = 0; r < 4; ++r) back[r] = SC ? __shfl(sh, 4 * q + r) : 0;
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    floatx4 tg[RT], xg = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int i = 0; i < RT; ++i) tg[i] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int e = 0; e < GS; ++e) {
                        const int j = g * GS + e;
                        u32x4 hi, lo = {0, 0, 0, 0};
                        const int at = M8 ? j / 2 : j;
                        if constexpr (XF)
                            split8<SC>(__builtin_bit_cast(floatx4, M8 && j % 2 ? turn8(b.x[2 * at]) : b.x[2 * at]),
                                       __builtin_bit_cast(floatx4, M8 && j % 2 ? turn8(b.x[2 * at + 1]) : b.x[2 * at + 1]),
                                       sh, hi, lo);
                        else
                            hi = pair_up(M8 && j % 2 ? turn8(b.x[at]) : b.x[at]);
                        const half8 xh = __builtin_bit_cast(half8, hi), xl = __builtin_bit_cast(half8, lo);
                        xg = __builtin_amdgcn_mfma_f32_16x16x32_f16(xh, ones, xg, 0, 0, 0);
                        if constexpr (XF) xg = __builtin_amdgcn_mfma_f32_16x16x32_f16(xl, ones, xg, 0, 0, 0);
#pragma unroll
                        for (int i = 0; i < RT; ++i) {
                            const half8 wv = __builtin_bit_cast(half8, expand8(u[i][j]));
                            tg[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xh, wv, tg[i], 0, 0, 0);
                            if constexpr (XF) tg[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(xl, wv, tg[i], 0, 0, 0);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < RT; ++i)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const float tv = SC ? __builtin_amdgcn_ldexpf(tg[i][r], back[r]) : tg[i][r];
                            const float xv = SC ? __builtin_amdgcn_ldexpf(xg[r], back[r]) : xg[r];
                            acc[i][r] = __builtin_fmaf(sv[i][g].y, xv, __builtin_fmaf(sv[i][g].x, tv, acc[i][r]));
                        }
                }
            };
            if constexpr (XF) {
                float top = 0.0f;  // the row's largest magnitude in the batch
#pragma unroll
                for (int i = 0; i < 2 * XL; ++i) {
                    const floatx4 f = __builtin_bit_cast(floatx4, b.x[i]);
                    top = fmaxf(fmaxf(fmaxf(top, fabsf(f.x)), fmaxf(fabsf(f.y), fabsf(f.z))), fabsf(f.w));
                }
                top = row_max<M8>(top);
                // sh puts it in [2^14, 2^15) (2^-126 at most, so that the power is a normal number)
                if (__builtin_amdgcn_ballot_w64(top > 65504.0f || (top < 1.0f && top > 0.0f)))
                    run(std::true_type{}, max(__builtin_amdgcn_frexp_expf(top) - 15, -126));
                else run(std::false_type{}, 0);
            } else {
                run(std::false_type{}, 0);
            }
        };
        // two batches alternate; the tail is peeled so that every load sits beside
        // the products of the batch before it
        const int mb = (nb - wave + NW - 1) / NW;  // this wave's batches (uniform)
        Batch A, B;
        if (mb > 0) load(A, wave);
        __syncthreads();  // the scales are there
        if (mb > 0) {
            int b = 0;
            for (; b + 2 < mb; b += 2) {
                load(B, wave + (b + 1) * NW);
                __builtin_amdgcn_sched_barrier(0);
                mma(A);
                load(A, wave + (b + 2) * NW);
                __builtin_amdgcn_sched_barrier(0);
                mma(B);
            }
            if (b + 1 < mb) {
                load(B, wave + (b + 1) * NW);
                __builtin_amdgcn_sched_barrier(0);
                mma(A);
                mma(B);
            } else {
                mma(A);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < RT; ++i) red[wave][i][lane] = acc[i];
    __syncthreads();
    // tile i is finished by wave i % NW: lane l has weight row l % 16, rows 4 q + r of X
#pragma unroll
    for (int i = 0; i < RT; ++i) {
        if (wave != i % NW) continue;
        floatx4 v = red[0][i][lane];
#pragma unroll
        for (int w = 1; w < NW; ++w) v += red[w][i][lane];
        const int n = n0 + 16 * i + fr;
        bool bad = false;
#pragma unroll
        for (int r = 0; r < 4; ++r) bad = bad || !__builtin_isfinite(v[r]);
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(bad) != 0, 0)) {
#pragma unroll 1
            for (int r = 0; r < 4; ++r) {
                const float vr = r == 0 ? v[0] : r == 1 ? v[1] : r == 2 ? v[2] : v[3];
                uint64_t todo = __builtin_amdgcn_ballot_w64(n < N && 4 * q + r < m_act && !__builtin_isfinite(vr));
                while (todo) {
                    const int l = __builtin_ctzll(todo);
                    const float y = by_terms<XF>(W, scales, biases, X, K, group, n0 + 16 * i + l % 16, 4 * (l / 16) + r);
#pragma unroll
                    for (int e = 0; e < 4; ++e) v[e] = e == r && lane == l ? y : v[e];
                    todo &= todo - 1;
                }
            }
        }
        if (n >= N) continue;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int m = 4 * q + r;
            if (m >= m_act) break;
            const size_t o = (size_t)m * N + n;
            if (y_f16) static_cast<_Float16 *>(Y)[o] = (_Float16)v[r];
            else static_cast<float *>(Y)[o] = v[r];
        }
    }
}

// Bytes of the kernel's scales in LDS.
size_t scale_lds(int rt, int64_t gk) { return (size_t)16 * rt * (size_t)(std::min<int64_t>(gk, kSegGroups) | 1) * 8; }

__global__ __launch_bounds__(TH) void k_dequantize4(const uint8_t *__restrict__ codes, const float *__restrict__ scales,
                                                    const float *__restrict__ biases, float *__restrict__ out,
                                                    int64_t pairs, int64_t group) {
    for (int64_t i = (int64_t)blockIdx.x * TH + threadIdx.x; i < pairs; i += (int64_t)gridDim.x * TH) {
#pragma clang fp contract(off)
        const uint32_t c = codes[i];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const int64_t g = (2 * i + e) / group;
            const float p = (float)(e ? c >> 4 : c & 15u) * scales[g];
            out[2 * i + e] = p + (biases ? biases[g] : 0.0f);
        }
    }
}

// Any shape, alignment and dtype: one block per output feature, its threads
// stride over the code bytes of the row, once per token.
__global__ __launch_bounds__(TH) void k_linear4_generic(const uint8_t *__restrict__ codes,
                                                        const float *__restrict__ scales,
                                                        const float *__restrict__ biases, int64_t group,
                                                        const void *__restrict__ X, int x_f16, void *__restrict__ Y,
                                                        int y_f16, int64_t M, int64_t N, int64_t K) {
    __shared__ float red[TH / 64];
    const int64_t n = blockIdx.x, gk = K / group;
    const int t = threadIdx.x;
    const uint8_t *row = codes + n * (K / 2);
    for (int64_t m = 0; m < M; ++m) {
        float acc = 0.0f;
        for (int64_t i = t; i < K / 2; i += TH) {
            const uint32_t c = row[i];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int64_t k = 2 * i + e, g = n * gk + k / group;
                const float x = x_f16 ? (float)static_cast<const _Float16 *>(X)[m * K + k]
                                      : static_cast<const float *>(X)[m * K + k];
                const float w = __builtin_fmaf((float)(e ? c >> 4 : c & 15u), scales[g], biases ? biases[g] : 0.0f);
                acc = __builtin_fmaf(w, x, acc);
            }
        }
        for (int o = 32; o > 0; o >>= 1) acc += __shfl_xor(acc, o, 64);
        if (t % 64 == 0) red[t / 64] = acc;
        __syncthreads();
        if (t == 0) {
            float v = 0.0f;
            for (int i = 0; i < TH / 64; ++i) v += red[i];
            if (y_f16) static_cast<_Float16 *>(Y)[m * N + n] = (_Float16)v;
            else static_cast<float *>(Y)[m * N + n] = v;
        }
        __syncthreads();
    }
}

// 4-bit codes to bytes, 32 of them per thread (bound by its 1.5 bytes per code: 4096x4096 9 us, 11008x4096 15.5, 4.4 TB/s).
__global__ __launch_bounds__(TH) void k_widen4(const u32x4 *__restrict__ codes, u32x4 *__restrict__ out, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * TH + threadIdx.x; i < n; i += (int64_t)gridDim.x * TH) {
        const u32x4 w = codes[i];
        u32x4 o[2];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t lo = w[e] & 0x0F0F0F0Fu, hi = (w[e] >> 4) & 0x0F0F0F0Fu;
            o[e / 2][2 * (e % 2)] = __builtin_amdgcn_perm(hi, lo, 0x05010400u);
            o[e / 2][2 * (e % 2) + 1] = __builtin_amdgcn_perm(hi, lo, 0x07030602u);
        }
        out[2 * i] = o[0];
        out[2 * i + 1] = o[1];
    }
}

using DotFn = void (*)(const uint8_t *, const float *, const float *, const void *, void *, int, int, int, int, int);

// The m <= 2 kernel of a shape and the weight rows of its blocks.
template <int M, bool XF, int CPT, int TPR>
DotFn dot_rows(int *rows) {
    constexpr int R = 4;
    *rows = R * (TH / TPR);
    return k_linear4_dot<M, CPT, TPR, R, XF>;
}
template <int M, bool XF>
DotFn dot_kernel(int64_t K, int *rows) {
    const int64_t C = K / 32;
    if (C <= 64) return dot_rows<M, XF, 1, 64>(rows);
    if (C <= 128) return dot_rows<M, XF, 1, 128>(rows);
    if (C <= 256) return dot_rows<M, XF, 1, 256>(rows);
    if (C <= 512) return dot_rows<M, XF, 2, 256>(rows);
    return nullptr;
}

// m <= 2; RQ_ERR_UNSUPPORTED outside what the kernel serves.
int launch_dot(const rq_qweight &w, const void *x, bool xf, void *y, bool yh, int m, hipStream_t s) {
    int rows = 0;
    const DotFn fn = m == 1 ? (xf ? dot_kernel<1, true>(w.k_in, &rows) : dot_kernel<1, false>(w.k_in, &rows))
                            : (xf ? dot_kernel<2, true>(w.k_in, &rows) : dot_kernel<2, false>(w.k_in, &rows));
    if (!fn) return RQ_ERR_UNSUPPORTED;
    hipLaunchKernelGGL(fn, dim3((unsigned)cdiv(w.n_out, rows)), dim3(TH), 0, s, (const uint8_t *)w.codes, w.scales,
                       w.biases, x, y, yh ? 1 : 0, m, (int)w.n_out, (int)w.k_in, w.group);
    RQ_LAUNCH_CHECK();
    return RQ_OK;
}

// m <= 16
int launch_mfma(const rq_qweight &w, const void *x, bool xf, void *y, bool yh, int m, hipStream_t s) {
    auto go = [&](auto rt, auto nw, auto gs, auto xfc) {
        constexpr int RT = decltype(rt)::value, NW = decltype(nw)::value, GS = decltype(gs)::value;
        constexpr bool XF = decltype(xfc)::value;
        const auto fn = m <= 8 ? k_linear4_mfma<RT, NW, GS, XF, true> : k_linear4_mfma<RT, NW, GS, XF, false>;
        hipLaunchKernelGGL(fn, dim3((unsigned)cdiv(w.n_out, 16 * RT)), dim3(NW * 64),
                           (unsigned)scale_lds(RT, w.k_in / w.group), s, (const uint8_t *)w.codes, w.scales, w.biases, x,
                           y, yh ? 1 : 0, m, (int)w.n_out, (int)w.k_in, w.group);
    };
    auto by_group = [&](auto rt, auto nw, auto xfc) {
        if (w.group % 128 == 0) go(rt, nw, std::integral_constant<int, 4>{}, xfc);
        else if (w.group % 64 == 0) go(rt, nw, std::integral_constant<int, 2>{}, xfc);
        else go(rt, nw, std::integral_constant<int, 1>{}, xfc);
    };
    // Waves and row tiles per block, measured (us in a graph, 1 tile of 4 waves / 1 of 8 / 2 of 4; f32 rows in
    // brackets).  8 rows: 2048x2048 4.6 / 4.8 / 5.6 [6.3 / 6.1 / 7.4], 4096x4096 7.0 / 7.0 / 8.6
    // [10.1 / 10.0 / 12.5], 4096x11008 in groups of 32 18.1 / 14.3 / 25.9 [25.8 / 21.8 / 33.3], 5632x2048
    // 6.2 / 7.0 / 6.0 [9.0 / 11.7 / 8.0], 11008x4096 12.5 / 14.5 / 13.2 [21.0 / 26.8 / 19.2], 32000x2048
    // 17.3 / 23.2 / 14.2 [30.5 / 44.0 / 21.2].  16 rows: 4096x4096 7.9 / 7.8 / 10.2 [13.2 / 12.5 / 15.4],
    // 4096x11008 19.3 / 17.6 / 28.6 [30.6 / 28.2 / 39.1], 5632x2048 7.7 / 9.5 / 7.0 [11.7 / 14.6 / 9.7],
    // 11008x4096 16.3 / 19.6 / 16.1 [28.9 / 34.3 / 29.6], 32000x2048 23.4 / 32.5 / 18.2 [39.8 / 55.2 / 35.3].
    // (f32 past 8 rows keeps one tile below 1024: right at 688 tiles, 2 us off at 352.)
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    using I4 = std::integral_constant<int, 4>;
    using I8 = std::integral_constant<int, 8>;
    const int64_t tiles = cdiv(w.n_out, 16);
    const bool two = tiles >= 1024 || (tiles > 256 && (xf ? m <= 8 : m > 8 || tiles <= 512));
    const bool wide = tiles <= 256 && w.k_in > 2048;
    auto by_shape = [&](auto xfc) {
        if (two) by_group(I2{}, I4{}, xfc);
        else if (wide) by_group(I1{}, I8{}, xfc);
        else by_group(I1{}, I4{}, xfc);
    };
    if (xf) by_shape(std::true_type{});
    else by_shape(std::false_type{});
    RQ_LAUNCH_CHECK();
    return RQ_OK;
}

}  // namespace

int launch_dequantize4(const rq_qweight &w, float *out, hipStream_t s) {
    const int64_t pairs = w.n_out * w.k_in / 2;
    if (pairs == 0) return RQ_OK;
    const int64_t blocks = std::min<int64_t>(cdiv(pairs, TH), 65536);
    hipLaunchKernelGGL(k_dequantize4, dim3((unsigned)blocks), dim3(TH), 0, s, (const uint8_t *)w.codes, w.scales,
                       w.biases, out, pairs, (int64_t)w.group);
    RQ_LAUNCH_CHECK();
    return RQ_OK;
}

// More rows than the kernels above take at once: the codes widened to bytes in the
// preparation area and the 8-bit GEMM (whose weights are rounded to fp16) on them,
// where it serves the shape; RQ_ERR_UNSUPPORTED otherwise.
int launch_widened(const rq_qweight &w, const void *x, rq_dtype xt, void *y, rq_dtype yt, int64_t m, int num_cus,
                   const GemmWorkspace &ws, hipStream_t s) {
    const int64_t N = w.n_out, K = w.k_in;
    const size_t codes = ((size_t)N * (size_t)K + 255) & ~size_t(255);
    // (the GEMM lays its scale table, and f32 rows cast to fp16, behind them)
    if (!ws.prep || K % 64 != 0 || w.group % 64 != 0 || codes > ws.prep_bytes / 4 * 3) return RQ_ERR_UNSUPPORTED;
    rq_qweight wide = w;
    wide.codes = ws.prep;
    wide.format = RQ_Q_AFFINE_U8;
    wide.prep = nullptr;
    if (affine_prep_bytes(wide) == 0 || affine_prep_bytes(wide) > (ws.prep_bytes - codes) / 2) return RQ_ERR_UNSUPPORTED;
    const int64_t chunks = N * K / 32;
    hipLaunchKernelGGL(k_widen4, dim3((unsigned)std::min<int64_t>(cdiv(chunks, TH), 16384)), dim3(TH), 0, s,
                       static_cast<const u32x4 *>(w.codes), static_cast<u32x4 *>(ws.prep), chunks);
    RQ_LAUNCH_CHECK();
    GemmWorkspace rest = ws;
    rest.prep = static_cast<char *>(ws.prep) + codes;
    rest.prep_bytes = ws.prep_bytes - codes;
    return launch_gemm(wide, x, xt, y, yt, m, num_cus, rest, s);
}

int launch_linear4(const rq_qweight &w, const void *x, rq_dtype xt, void *y, rq_dtype yt, int64_t m, int num_cus,
                   const GemmWorkspace &ws, hipStream_t s) {
    const int64_t N = w.n_out, K = w.k_in;
    const bool xf = xt == RQ_F32, yh = yt == RQ_F16;
    // Chunks of 32 codes in one group each, 16-byte loads, 32-bit offsets into 16 rows of X and of W
    const bool fast = K > 0 && w.group % 32 == 0 && K <= (1 << 24) && grid_ok(N, 64) && aligned(w.codes, 16) && aligned(x, 16);
    if (fast) {
        if (m > kRowsBySixteen) {
            const int st = launch_widened(w, x, xt, y, yt, m, num_cus, ws, s);
            if (st != RQ_ERR_UNSUPPORTED) return st;
        }
        const size_t xr = (size_t)K * (xf ? 4 : 2), yr = (size_t)N * (yh ? 2 : 4);
        for (int64_t m0 = 0; m0 < m; m0 += 16) {
            const int mc = (int)std::min<int64_t>(16, m - m0);
            const char *xp = static_cast<const char *>(x) + m0 * xr;
            char *yp = static_cast<char *>(y) + m0 * yr;
            int st = mc <= 2 ? launch_dot(w, xp, xf, yp, yh, mc, s) : RQ_ERR_UNSUPPORTED;
            if (st == RQ_ERR_UNSUPPORTED) st = launch_mfma(w, xp, xf, yp, yh, mc, s);
            if (st != RQ_OK) return st;
        }
        return RQ_OK;
    }
    if (!grid_ok(N, TH)) return fail(RQ_ERR_SHAPE, "n_out too large for the generic kernel");
    hipLaunchKernelGGL(k_linear4_generic, dim3((unsigned)N), dim3(TH), 0, s, (const uint8_t *)w.codes, w.scales,
                       w.biases, (int64_t)w.group, x, xf ? 0 : 1, y, yh ? 1 : 0, m, N, K);
    RQ_LAUNCH_CHECK();
    return RQ_OK;
}

}  // namespace rq
