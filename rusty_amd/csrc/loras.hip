// A quantized Linear with an adapter per row (rq_qmatmul_loras):
//   Y[t] = X[t] . deq(W)^T + factor_i (X[t] . A_i^T) . B_i,  i = ids[t].
//
// Three launches: the rows' t = X . A_i^T (k_loras_in: a narrow product, its k cut
// over blocks, one partial sum per slice), the shared product into f32
// (rq_qmatmul's kernels), and Y = main + factor t . B_i (k_loras_out), rounded
// once.  Small batches are bound by the launches and by the weight's bytes, which
// each used adapter adds (k_in + n_out) rank elements to; prompts by the shared product.
//
// One or two rows of 8-bit codes, and prompts for which the product takes tiles of 128 rows, take
// two launches: the decode GEMV or the GEMM adds its rows' adapters itself.
//
// k_loras_in: rows of X are the rows of a matrix instruction, 16 rows of A_i its
// columns, k runs along both (16-byte loads, no LDS).  Rows of a tile may have
// different adapters: each one's product is formed for all its rows and
// kept for its own, so nothing a foreign adapter holds reaches a row.
//
// k_loras_out has two forms.  Few rows: a block takes one row and a stretch of
// columns, its lanes 8 columns each, the adapter's rank one fma at a time -- no work
// on foreign rows.  Many: a wave takes 16 rows and 64 columns on the matrix
// instructions, an adapter of theirs after another (f32 B: f32 instructions; fp16 B:
// t as two fp16 terms).
//
// Measured (us; X . A / shared product / t . B; in brackets the bytes at 6.9 TB/s or the products at 1157 TFLOP/s):
// one row of 4096 x 4096, 8-bit rows, rank 16: 3.2 / 5.8 with t . B, 8.9 a call (2.5; apart 3.3 / 4.7 / 2.7, 12.3);
// 16 rows of 8 to 10 adapters of rank 16, 11008 x 4096, 4-bit groups: 4.8 / 16.7 / 4.0, 23.4 a call (4.7 to 4.9); 2048 rows
// of 4096 x 4096, 8-bit rows, rank 32: 9.8 / 69 with t . B, 79 a call (60; apart 9.4 / 66 / 18.9, 91).  X . A and the shared product
// of a few rows in one launch took 8 us, 6.1 in two.
#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "lds_dma.hpp"
#include "loras.hpp"

namespace rq {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

constexpr int kMaxRank = 256;
constexpr int kMaxSide = 65535 * 256;  // m, k_in, n_out
// Up to so many rows k_loras_in takes one tile of 16 rows a block (more blocks), else two, so that A's rows are
// read less often (2048 rows, rank 32: one 12.6 us, two 9.4, four 10.6), and the output a row a block, else 16:
// 4096 x 4096, all three launches, row / tile: 128 rows of 64 adapters of rank 16 23.7 / 35.7 us, of one 20.3 / 21.8;
// 256 of 64 32.2 / 43.3, of one 24.6 / 25.7, of rank 64 32.4 / 29.5; 512 of one 35.6 / 35.9, of rank 64 46.6 / 40.4.
constexpr int64_t kFewRows = 256;
// A block's k, a quarter per wave: as much as the registers hold of X and of 32 rows of A.
constexpr int slice(bool f16, int tiles) { return (f16 ? 1024 : 512) / (tiles > 1 ? 2 : 1); }

struct LoraArgs {
    const void *x, *a, *b;
    const float *factors;
    const int *ids, *ranks;
    float *part;        // [m][slices][ranks4]: X . A_i^T, a sum per slice of k
    const float *main;  // [m][n]
    void *y;
    int64_t m, k, n;
    int n_adapters, rank, slices;
    int ranks4;         // rank rounded up to 4
};

// The adapter of row t, -1 for none.
__device__ __forceinline__ int adapter_of(const LoraArgs &p, int64_t t) {
    const int i = p.ids[t];
    return (uint32_t)i < (uint32_t)p.n_adapters ? i : -1;
}
__device__ __forceinline__ int rank_of(const LoraArgs &p, int i) {
    return p.ranks ? min(max(p.ranks[i], 0), p.rank) : p.rank;
}

// N consecutive values at p + e as floats or halves, those at and past `end` zero.  VEC: whole or not at all, aligned;
// otherwise of any alignment (16-byte loads allow it; element by element 1037 rows of 5001 x 2048, rank 100, took 566 us).
template <typename S, int N, bool VEC, typename D>
__device__ __forceinline__ D load_n(const S *p, int64_t e, int64_t end) {
    typedef S vec __attribute__((ext_vector_type(N), aligned(VEC ? sizeof(S) * N : sizeof(S))));
    D r;
    vec v = {};
    if (VEC ? e < end : e + N <= end) {
        v = *reinterpret_cast<const vec *>(p + e);
    } else if constexpr (!VEC) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (e + i < end) v[i] = p[e + i];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) r[i] = (std::remove_reference_t<decltype(r[0] + r[0])>)v[i];
    return r;
}
// The same for stores.
template <typename S, int N, bool VEC, typename D>
__device__ __forceinline__ void store_n(S *p, int64_t e, int64_t end, D d) {
    typedef S vec __attribute__((ext_vector_type(N), aligned(VEC ? sizeof(S) * N : sizeof(S))));
    vec v;
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = (S)d[i];
    if (VEC ? e < end : e + N <= end) {
        *reinterpret_cast<vec *>(p + e) = v;
    } else if constexpr (!VEC) {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (e + i < end) p[e + i] = v[i];
    }
}

// Block (TM tiles of 16 rows, slice of k, z): of the rows' distinct adapters every gridDim.z-th, 16 RT of their
// rows at once.  X is asked for at once.
template <typename X, typename A, int TM, int RT, bool VEC>
__global__ __launch_bounds__(256) void k_loras_in(LoraArgs p) {
    constexpr bool F16 = sizeof(X) == 2 && sizeof(A) == 2;
    constexpr int N = F16 ? 8 : 4, STEP = 4 * N, WAVE = slice(F16, TM) / 4, STEPS = WAVE / STEP;  // k a lane, an instruction, of a wave
    typedef std::conditional_t<F16, half8, floatx4> frag;
    __shared__ float sums[4][16 * TM][16 * RT + 1];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, col = lane & 15, qt = lane >> 4;
    const int64_t t0 = (int64_t)blockIdx.x * 16 * TM;
    const int64_t k0 = (int64_t)blockIdx.y * slice(F16, TM) + wv * WAVE + N * qt;
    const int id = adapter_of(p, min(t0 + lane, p.m - 1));
    frag xf[TM][STEPS];
#pragma unroll
    for (int u = 0; u < TM; ++u) {
        const X *xr = static_cast<const X *>(p.x) + min(t0 + 16 * u + col, p.m - 1) * p.k;
#pragma unroll
        for (int j = 0; j < STEPS; ++j) xf[u][j] = load_n<X, N, VEC, frag>(xr, k0 + j * STEP, p.k);
    }
    const int mine = lane < 16 * TM && t0 + lane < p.m ? id : -1;
    uint64_t left = __builtin_amdgcn_ballot_w64(mine >= 0);
    for (int z = 0; left; ++z) {
        const int i = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
        const uint64_t same = __builtin_amdgcn_ballot_w64(mine == i);
        left &= ~same;
        if (z % (int)gridDim.z != (int)blockIdx.z) continue;
        const int rank = rank_of(p, i);
        const A *a = static_cast<const A *>(p.a) + (int64_t)i * p.rank * p.k;
#pragma unroll 1
        for (int r0 = 0; r0 < rank; r0 += 16 * RT) {
            frag af[RT][STEPS];
#pragma unroll
            for (int u = 0; u < RT; ++u) {
                const A *ar = a + (int64_t)min(r0 + 16 * u + col, rank - 1) * p.k;
#pragma unroll
                for (int j = 0; j < STEPS; ++j) af[u][j] = load_n<A, N, VEC, frag>(ar, k0 + j * STEP, p.k);
            }
            __syncthreads();  // the last sums have been read
#pragma unroll
            for (int t = 0; t < TM; ++t)
#pragma unroll
                for (int u = 0; u < RT; ++u) {
                    floatx4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int j = 0; j < STEPS; ++j) {
                        if constexpr (F16) {
                            acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(xf[t][j], af[u][j], acc, 0, 0, 0);
                        } else {
#pragma unroll
                            for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(xf[t][j][e], af[u][j][e], acc, 0, 0, 0);
                        }
                    }
#pragma unroll
                    for (int e = 0; e < 4; ++e) sums[wv][16 * t + 4 * qt + e][16 * u + col] = acc[e];
                }
            __syncthreads();
#pragma unroll
            for (int e = 0; e < TM * RT; ++e) {
                const int tr = (e / RT) * 16 + (threadIdx.x >> 4), r = 16 * (e % RT) + (threadIdx.x & 15);
                if ((same >> tr & 1) && r0 + r < p.ranks4)
                    p.part[((t0 + tr) * p.slices + blockIdx.y) * p.ranks4 + r0 + r] =
                        r0 + r < rank ? (sums[0][tr][r] + sums[1][tr][r]) + (sums[2][tr][r] + sums[3][tr][r]) : 0.0f;
            }
        }
    }
}

// Few rows: block (row, stretch of 2048 columns).  What does not wait for t is asked for first.
template <typename B, typename Y, bool VEC>
__global__ __launch_bounds__(256) void k_loras_out_row(LoraArgs p) {
    typedef float floatx8 __attribute__((ext_vector_type(8)));
    typedef B vecb __attribute__((ext_vector_type(8)));
    constexpr int RC = sizeof(B) == 2 ? 16 : 8;  // rows of B at once
    const int64_t t = blockIdx.x, c = ((int64_t)blockIdx.y * 256 + threadIdx.x) * 8;
    const int i = adapter_of(p, t);
    const floatx8 main = load_n<float, 8, VEC, floatx8>(p.main + t * p.n, c, p.n);
    const int rank = i < 0 ? 0 : rank_of(p, i);
    const B *b = static_cast<const B *>(p.b) + (int64_t)max(i, 0) * p.rank * p.n;
    const float f = p.factors && i >= 0 ? p.factors[i] : 1.0f;
    const int lane = threadIdx.x & 63, u0 = lane & 15;
    floatx8 acc = {};
#pragma unroll 1
    for (int r0 = 0; r0 < rank; r0 += RC) {
        vecb bv[RC];
#pragma unroll
        for (int u = 0; u < RC; ++u) bv[u] = load_n<B, 8, VEC, vecb>(b + (int64_t)min(r0 + u, rank - 1) * p.n, c, r0 + u < rank ? p.n : 0);
        // t of r0 + lane % 16: the wave's four rows of lanes take every fourth slice
        float s = 0.0f;
        if (u0 < RC && r0 + u0 < rank)
            for (int j = lane >> 4; j < p.slices; j += 4) s += p.part[(t * p.slices + j) * p.ranks4 + r0 + u0];
        s += __shfl_xor(s, 16);
        s += __shfl_xor(s, 32);
        s = r0 + u0 < rank ? f * s : 0.0f;  // (0 past the rank, also with an infinite factor)
#pragma unroll
        for (int u = 0; u < RC; ++u) {
            const float su = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, s), u));
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] = __builtin_fmaf(su, (float)bv[u][e], acc[e]);
        }
    }
    if (c >= p.n) return;
    store_n<Y, 8, VEC>(static_cast<Y *>(p.y) + t * p.n, c, p.n, main + acc);
}

// Many rows: block (16 rows, stretch of 256 columns), a wave 64 of them: B^T . t^T on the matrix instructions, so
// that a lane gets 16 columns side by side of one row (row i of instruction v is column 16 (i / 4) + 4 v + i % 4).
// Bound by the shared product's way in and Y's out.  A load that is waited for alone costs 1 to 2 us here, so all
// that a tile with one adapter of up to 32 ranks reads is asked for together, and what B and the shared product take
// waits in LDS (DMA): few registers, many waves.  B's buffers hold 32 ranks (f32 B: 16); with more ranks there are two,
// else further adapters wait for their turn with one (2048 x 11008, rank 16: two buffers 45 us, one 40).
// fp16 B: t as two fp16 terms (loras.hpp, a scale per row), two instructions of 32 ranks a 16 columns, B's fragments by
// transposing LDS reads; f32 instructions of 4 ranks took 3 us longer at 2048 x 4096, rank 32.
__host__ __device__ constexpr int out_ranks(int rank) { return (rank + 31) / 32 * 32; }
template <typename B, typename Y, bool VEC>
__global__ __launch_bounds__(256, sizeof(B) == 2 ? 4 : 1) void k_loras_out(LoraArgs p) {
    constexpr bool F16 = sizeof(B) == 2;
    constexpr int R = F16 ? 32 : 16;  // ranks of a step
    constexpr int CH = 64 * (int)sizeof(B) / 16, RPU = 64 / CH, UN = R / RPU;  // B: 16-byte pieces of a row, rows of a DMA
    typedef short short4v __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) short4v lds_short4;
    __shared__ __attribute__((aligned(16))) floatx4 main[4][16][16];       // [wave][row][16-byte piece ^ row]
    // [16][out_ranks + 4]: t, fp16 B: its two terms side by side (a row that is low: t as it is), the row's scale and
    // whether it is low; then B [wave][buffer][rank][column]
    extern __shared__ __attribute__((aligned(16))) float ts[];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, col = lane & 15, qt = lane >> 4;
    const int64_t t0 = (int64_t)blockIdx.x * 16, c0 = ((int64_t)blockIdx.y * 4 + wv) * 64;
    const int ranks = out_ranks(p.rank), row4 = ranks + 4, buffers = p.rank > R ? 2 : 1;
    B *bs = reinterpret_cast<B *>(ts + 16 * row4) + wv * buffers * (R * 64);
    int mine = t0 + col < p.m ? adapter_of(p, t0 + col) : -1;
    asm volatile("" : "+v"(mine));  // (waited for here: later the wait would be for the DMA, too)
    const uint64_t all = __builtin_amdgcn_ballot_w64(lane < 16 && mine >= 0);
    // steps: R ranks of one adapter
    struct Step {
        int i, rank, r0;
        uint64_t same, left;  // its rows; those of the adapters after it
    };
    auto adapter = [&](uint64_t left) {
        Step s;
        s.i = __builtin_amdgcn_readlane(mine, left ? __builtin_ctzll(left) : 0);
        s.same = __builtin_amdgcn_ballot_w64(mine == s.i) & left;
        s.left = left & ~s.same;
        s.rank = left ? rank_of(p, s.i) : 0;
        s.r0 = 0;
        return s;
    };
    auto after = [&](Step s) {
        s.r0 += R;
        return s.r0 < s.rank ? s : adapter(s.left);
    };
    auto fetch = [&](const Step &s, int buffer) {
        if constexpr (!VEC) {
            // (DMA takes whole, aligned pieces)
            constexpr int E = 16 / (int)sizeof(B);
            typedef B piece __attribute__((ext_vector_type(E)));
            const B *b = static_cast<const B *>(p.b) + (int64_t)s.i * p.rank * p.n;
            piece v[UN];
#pragma unroll
            for (int u = 0; u < UN; ++u)
                v[u] = load_n<B, E, false, piece>(b + (int64_t)min(s.r0 + u * RPU + lane / CH, max(s.rank - 1, 0)) * p.n,
                                                  c0 + lane % CH * E, p.n);
#pragma unroll
            for (int u = 0; u < UN; ++u) *reinterpret_cast<piece *>(bs + (buffer * R + u * RPU) * 64 + lane * E) = v[u];
            wait_lgkm0();
            return;
        }
        const int64_t c = min(c0 + lane % CH * (16 / (int)sizeof(B)), p.n - 16 / (int)sizeof(B));
        const B *b = static_cast<const B *>(p.b) + (int64_t)s.i * p.rank * p.n + c;
#pragma unroll
        for (int u = 0; u < UN; ++u)
            dma16_kept(reinterpret_cast<const char *>(b + (int64_t)min(s.r0 + u * RPU + lane / CH, max(s.rank - 1, 0)) * p.n),
                       lds_addr(bs + (buffer * R + u * RPU) * 64));
    };
    Step s = adapter(all);
    if (all) fetch(s, 0);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int r = 4 * e + qt;
        const float *from = p.main + min(t0 + r, p.m - 1) * p.n;
        if constexpr (VEC)
            dma16_at(reinterpret_cast<const char *>(from + min(c0 + 4 * (col ^ r), p.n - 4)), lds_addr(&main[wv][4 * e][0]));
        else
            main[wv][r][col] = load_n<float, 4, false, floatx4>(from, c0 + 4 * (col ^ r), p.n);
    }
    {
        // t, 16 threads a row, 4 ranks each: the slices summed in order, times the factor; of rows without an
        // adapter not written, and not used
        const int tr = threadIdx.x >> 4, u = threadIdx.x & 15, i = __shfl(mine, tr);
        float *to = ts + tr * row4;
        float most = 0.0f, least = __builtin_inff();
        if (i >= 0) {
            const float f = p.factors ? p.factors[i] : 1.0f;
            const int rank = rank_of(p, i);
            for (int r = 4 * u; r < ranks; r += 64) {
                const float *q = p.part + (t0 + tr) * p.slices * p.ranks4 + r;
                floatx4 v = {0.0f, 0.0f, 0.0f, 0.0f};
                if (r < p.ranks4) {
#pragma unroll 8
                    for (int j = 0; j < p.slices; ++j) v += *reinterpret_cast<const floatx4 *>(q + (int64_t)j * p.ranks4);
                }
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    v[e] = r + e < rank ? f * v[e] : 0.0f;
                    most = fmaxf(most, __builtin_isfinite(v[e]) ? fabsf(v[e]) : 0.0f);
                    least = fminf(least, v[e] != 0.0f ? fabsf(v[e]) : __builtin_inff());
                }
                *reinterpret_cast<floatx4 *>(to + r) = v;
            }
        }
        if constexpr (F16) {
#pragma unroll
            for (int w = 1; w < 16; w <<= 1) {
                most = fmaxf(most, __shfl_xor(most, w));
                least = fminf(least, __shfl_xor(least, w));
            }
            const int ex = lora_exponent(most);
            const bool low = lora_low(__builtin_ldexpf(least, ex));
            if (u == 0) {
                to[ranks] = __builtin_ldexpf(1.0f, -ex);
                to[ranks + 1] = low ? 1.0f : 0.0f;
            }
            if (i >= 0 && !low)
                for (int r = 4 * u; r < ranks; r += 64) {
                    const floatx4 v = *reinterpret_cast<const floatx4 *>(to + r);
                    typedef _Float16 half4 __attribute__((ext_vector_type(4)));
                    half4 hi, lo;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        _Float16 h, l;
                        lora_split(__builtin_ldexpf(v[e], ex), h, l);
                        hi[e] = h;
                        lo[e] = l;
                    }
                    // (8 ranks: 16 bytes of first terms, 16 of second)
                    half4 *h = reinterpret_cast<half4 *>(to + r / 8 * 8) + r / 4 % 2;
                    __builtin_amdgcn_wave_barrier();  // (both halves of the 8 have been read by these lanes)
                    h[0] = hi;
                    h[2] = lo;
                }
        }
    }
    __syncthreads();
    floatx4 out[4], acc[4], acc_lo[4];
#pragma unroll
    for (int v = 0; v < 4; ++v) out[v] = acc[v] = acc_lo[v] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
    // (of a row without an adapter: whatever was there, and not used)
    const float row_scale = F16 ? ts[col * row4 + ranks] : 1.0f, row_low = F16 ? ts[col * row4 + ranks + 1] : 0.0f;
    auto f32 = [&](const Step &s) { return __builtin_amdgcn_ballot_w64((s.same >> col & 1) && row_low != 0.0f) != 0; };
    wait_vmcnt<0>();
    for (int k = 0; s.same; ++k) {
        const Step next = after(s);
        if (next.same && buffers == 2) {
            wait_lgkm0();  // (the buffer has been read)
            fetch(next, (k + 1) & 1);
            if (k > 0) wait_vmcnt<UN>();
        } else if (k > 0) {
            wait_vmcnt<0>();
        }
        const int count = min(s.rank - s.r0, R);  // of these ranks, those that the adapter has
        B *b = bs + (buffers == 2 ? k & 1 : 0) * (R * 64);
        if constexpr (F16) {
            if (count < R) {
                // (what lies past the rank is another rank's, and may be infinite)
#pragma unroll
                for (int u = 0; u < UN; ++u)
                    if (u * RPU + lane / CH >= count)
                        *reinterpret_cast<half8 *>(b + (u * RPU + lane / CH) * 64 + lane % CH * 8) = half8{};
                wait_lgkm0();
            }
            const half8 *tp = reinterpret_cast<const half8 *>(ts + col * row4 + s.r0 + 8 * qt);
            const half8 hi = tp[0], lo = tp[1];
            auto fragment = [&](int v) {
                // 16 lanes take 4 ranks x 4 x 4 columns; each gets one column's 4 ranks
                lds_short4 *a = (lds_short4 *)(uintptr_t)(lds_addr(b) + (uint32_t)((8 * qt + col / 4) * 128 + (col & 3) * 32 + v * 8));
                const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(a));
                const uint2 y = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(a + 4 * 128 / 8));
                return __builtin_bit_cast(half8, make_uint4(x.x, x.y, y.x, y.y));
            };
            if (f32(s)) {
                floatx4 t[2] = {__builtin_bit_cast(floatx4, hi), __builtin_bit_cast(floatx4, lo)};
                if (row_low == 0.0f) {  // (beside a row that is low)
#pragma unroll
                    for (int e = 0; e < 8; ++e) t[e / 4][e % 4] = __builtin_fmaf((float)lo[e], kLoraLo, (float)hi[e]) * row_scale;
                }
#pragma unroll 1
                for (int v = 0; v < 4; ++v) {
                    const floatx4 sum = lora_add_f32(fragment(v), t, v == 0 ? acc[0] : v == 1 ? acc[1] : v == 2 ? acc[2] : acc[3]);
#pragma unroll
                    for (int w = 0; w < 4; ++w) acc[w] = v == w ? sum : acc[w];
                }
            } else {
#pragma unroll
                for (int v = 0; v < 4; ++v) {
                    const half8 bt = fragment(v);
                    acc[v] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bt, hi, acc[v], 0, 0, 0);
                    acc_lo[v] = __builtin_amdgcn_mfma_f32_16x16x32_f16(bt, lo, acc_lo[v], 0, 0, 0);
                }
            }
        } else {
            float bv[R / 4][4], tv[R / 4];  // (all read before the first is used)
#pragma unroll
            for (int u = 0; u < R / 4; ++u) {
                const int r = 4 * u + qt;
                tv[u] = ts[col * row4 + s.r0 + r];
#pragma unroll
                for (int v = 0; v < 4; ++v) bv[u][v] = r < count ? (float)b[r * 64 + 16 * (col / 4) + 4 * v + col % 4] : 0.0f;
            }
#pragma unroll
            for (int u = 0; u < R / 4; ++u)
#pragma unroll
                for (int v = 0; v < 4; ++v) acc[v] = __builtin_amdgcn_mfma_f32_16x16x4f32(bv[u][v], tv[u], acc[v], 0, 0, 0);
        }
        if (next.i != s.i || !next.same) {
            const bool has = s.same >> col & 1;
            const bool plain = !F16 || f32(s);
#pragma unroll
            for (int v = 0; v < 4; ++v) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float sum = plain ? acc[v][e] : lora_join(acc[v][e], acc_lo[v][e]) * row_scale;
                    out[v][e] = has ? sum : out[v][e];
                }
                acc[v] = acc_lo[v] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
            }
        }
        if (next.same && buffers == 1) {
            wait_lgkm0();
            fetch(next, 0);
        }
        s = next;
    }
    const int64_t t = t0 + col, c = c0 + 16 * qt;
    if (t >= p.m) return;
    typedef float floatx8 __attribute__((ext_vector_type(8)));
#pragma unroll
    for (int h = 0; h < 2; ++h) {  // 8 columns
        const floatx4 a0 = main[wv][col][(4 * qt + 2 * h) ^ col] + out[2 * h], a1 = main[wv][col][(4 * qt + 2 * h + 1) ^ col] + out[2 * h + 1];
        store_n<Y, 8, VEC>(static_cast<Y *>(p.y) + t * p.n, c + 8 * h, p.n,
                           floatx8{a0[0], a0[1], a0[2], a0[3], a1[0], a1[1], a1[2], a1[3]});
    }
}

int check_set(const rq_lora_set *s) {
    if (!s) return fail(RQ_ERR_INVALID_ARGUMENT, "null adapter set");
    if (s->dtype != RQ_F16 && s->dtype != RQ_F32) return fail(RQ_ERR_INVALID_ARGUMENT, "the set's dtype must be RQ_F16 or RQ_F32");
    if (s->reserved != 0) return fail(RQ_ERR_INVALID_ARGUMENT, "reserved field must be 0");
    if (s->n_adapters < 0) return fail(RQ_ERR_SHAPE, "negative n_adapters");
    if (s->rank < 1 || s->rank > kMaxRank) return fail(RQ_ERR_SHAPE, "rank %d outside 1..%d", s->rank, kMaxRank);
    return RQ_OK;
}

int64_t slices_of(int64_t m, int64_t k, bool f16) { return std::max<int64_t>(1, cdiv(k, slice(f16, m > kFewRows ? 2 : 1))); }
int64_t ranks4_of(int rank) { return (rank + 3) / 4 * 4; }

int check_loras(const rq_qweight *w, const rq_lora_set *set, const int32_t *ids, const void *x, rq_dtype xt, void *y,
                rq_dtype yt, int64_t m, void *workspace, size_t workspace_bytes, LoraArgs &p, bool &run) {
    run = false;
    int st = check_qweight(w, true);
    if (st != RQ_OK) return st;
    if ((st = check_set(set)) != RQ_OK) return st;
    if ((xt != RQ_F16 && xt != RQ_F32) || (yt != RQ_F16 && yt != RQ_F32))
        return fail(RQ_ERR_INVALID_ARGUMENT, "dtype must be RQ_F16 or RQ_F32");
    const int64_t K = w->k_in, N = w->n_out;
    // (every grid fits, and every size 64 bits)
    if (m < 0 || m > kMaxSide || K > kMaxSide || N > kMaxSide) return fail(RQ_ERR_SHAPE, "m, k_in and n_out go up to %d", kMaxSide);
    int64_t t;
    if (!mul_ok((int64_t)set->n_adapters * set->rank, std::max(K, N) * 4, &t)) return fail(RQ_ERR_SHAPE, "shape overflows");
    if (m == 0 || N == 0) return RQ_OK;
    if (!y || (K > 0 && !x) || !ids) return fail(RQ_ERR_INVALID_ARGUMENT, "null pointer");
    if (set->n_adapters > 0 && ((K > 0 && !set->a) || !set->b)) return fail(RQ_ERR_INVALID_ARGUMENT, "null adapter pointer");
    const int xs = xt == RQ_F16 ? 2 : 4, ys = yt == RQ_F16 ? 2 : 4, as = set->dtype == RQ_F16 ? 2 : 4;
    if (!aligned(x, xs) || !aligned(y, ys) || !aligned(set->a, as) || !aligned(set->b, as) || !aligned(ids, 4) ||
        !aligned(set->factors, 4) || !aligned(set->ranks, 4))
        return fail(RQ_ERR_UNSUPPORTED, "pointers must be aligned to their elements");
    const size_t need = rq_qmatmul_loras_workspace(set, m, K, N, xt, yt);
    if (!workspace || workspace_bytes < need)
        return fail(RQ_ERR_INVALID_ARGUMENT, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
    if (!aligned(workspace, 256)) return fail(RQ_ERR_UNSUPPORTED, "workspace must be 256-byte aligned");
    p.x = x;
    p.a = set->a;
    p.b = set->b;
    p.factors = set->factors;
    p.ids = ids;
    p.ranks = set->ranks;
    p.y = y;
    p.m = m;
    p.k = K;
    p.n = N;
    p.n_adapters = set->n_adapters;
    p.rank = set->rank;
    p.ranks4 = (int)ranks4_of(set->rank);
    p.slices = (int)slices_of(m, K, xt == RQ_F16 && set->dtype == RQ_F16);
    // workspace: the shared product in f32, where y is not that already, then the partial sums
    char *ws = static_cast<char *>(workspace);
    p.main = yt == RQ_F32 ? static_cast<float *>(y) : reinterpret_cast<float *>(ws);
    p.part = reinterpret_cast<float *>(ws + (yt == RQ_F32 ? 0 : (m * N * 4 + 255) / 256 * 256));
    run = true;
    return RQ_OK;
}

template <typename F>
int by_type(int dtype, F f) {
    return dtype == RQ_F16 ? f((_Float16 *)nullptr) : f((float *)nullptr);
}

int run_in(const LoraArgs &p, rq_dtype xt, int at, int num_cus, hipStream_t s) {
    const bool few = p.m <= kFewRows;
    const int64_t blocks = cdiv(p.m, few ? 16 : 32);
    // A block's adapters side by side while blocks are few.
    const int64_t z = std::max<int64_t>(
        1, std::min<int64_t>({few ? 16 : 32, p.m, (int64_t)p.n_adapters, num_cus / (blocks * p.slices)}));
    const dim3 grid((unsigned)blocks, (unsigned)p.slices, (unsigned)z);
    const int n = xt == RQ_F16 && at == RQ_F16 ? 8 : 4, xs = xt == RQ_F16 ? 2 : 4, as = at == RQ_F16 ? 2 : 4;
    const bool vec = p.k % n == 0 && aligned(p.x, n * xs) && aligned(p.a, n * as);
    return by_type(xt, [&](auto *x) {
        return by_type(at, [&](auto *a) {
            using X = std::remove_pointer_t<decltype(x)>;
            using A = std::remove_pointer_t<decltype(a)>;
            auto go = [&](auto tm, auto rt) {
                constexpr int TM = decltype(tm)::value, RT = decltype(rt)::value;
                if (vec) hipLaunchKernelGGL((k_loras_in<X, A, TM, RT, true>), grid, dim3(256), 0, s, p);
                else hipLaunchKernelGGL((k_loras_in<X, A, TM, RT, false>), grid, dim3(256), 0, s, p);
            };
            using One = std::integral_constant<int, 1>;
            using Two = std::integral_constant<int, 2>;
            if (few) p.rank <= 16 ? go(One{}, One{}) : go(One{}, Two{});
            else p.rank <= 16 ? go(Two{}, One{}) : go(Two{}, Two{});
            RQ_LAUNCH_CHECK();
            return (int)RQ_OK;
        });
    });
}

// Few rows: a row per block; else 16.
int run_out(const LoraArgs &p, int bt, rq_dtype yt, hipStream_t s) {
    const bool vec = p.n % 8 == 0 && aligned(p.b, 16) && aligned(p.y, 16), rows = p.m <= kFewRows;
    const int64_t bx = rows ? p.m : cdiv(p.m, 16), by = cdiv(p.n, rows ? 2048 : 256);
    const dim3 grid((unsigned)bx, (unsigned)by);
    return by_type(bt, [&](auto *b) {
        return by_type(yt, [&](auto *y) {
            using B = std::remove_pointer_t<decltype(b)>;
            using Y = std::remove_pointer_t<decltype(y)>;
            const int r = sizeof(B) == 2 ? 32 : 16;
            const size_t lds = 16 * (out_ranks(p.rank) + 4) * sizeof(float) + (p.rank > r ? 2 : 1) * (size_t)(4 * r * 64) * sizeof(B);
            if (!rows && vec) hipLaunchKernelGGL((k_loras_out<B, Y, true>), grid, dim3(256), lds, s, p);
            else if (!rows) hipLaunchKernelGGL((k_loras_out<B, Y, false>), grid, dim3(256), lds, s, p);
            else if (vec) hipLaunchKernelGGL((k_loras_out_row<B, Y, true>), grid, dim3(256), 0, s, p);
            else hipLaunchKernelGGL((k_loras_out_row<B, Y, false>), grid, dim3(256), 0, s, p);
            RQ_LAUNCH_CHECK();
            return (int)RQ_OK;
        });
    });
}

}  // namespace
}  // namespace rq

using namespace rq;

extern "C" {

size_t rq_qmatmul_loras_workspace(const rq_lora_set *set, int64_t m, int64_t k_in, int64_t n_out, rq_dtype x_dtype,
                                  rq_dtype y_dtype) {
    if (check_set(set) != RQ_OK || m < 1 || k_in < 0 || n_out < 1 || m > kMaxSide || k_in > kMaxSide || n_out > kMaxSide) return 0;
    const int64_t part = m * slices_of(m, k_in, x_dtype == RQ_F16 && set->dtype == RQ_F16) * 4 * ranks4_of(set->rank);
    const int64_t main = y_dtype != RQ_F32 ? (m * n_out * 4 + 255) / 256 * 256 : 0;
    return (size_t)(main + part);
}

int rq_qmatmul_loras(rq_ctx *ctx, const rq_qweight *w, const rq_lora_set *set, const int32_t *ids, const void *x,
                     rq_dtype x_dtype, void *y, rq_dtype y_dtype, int64_t m, void *workspace, size_t workspace_bytes,
                     rq_stream stream) {
    RQ_ENTER(ctx);
    LoraArgs p{};
    bool run;
    int st = check_loras(w, set, ids, x, x_dtype, y, y_dtype, m, workspace, workspace_bytes, p, run);
    if (st != RQ_OK || !run) return st;
    hipStream_t s = pick(ctx, stream);
    const bool adapters = set->n_adapters > 0;
    if (adapters && (st = run_in(p, x_dtype, set->dtype, ctx->num_cus, s)) != RQ_OK) return st;
    if (!adapters) return qmatmul_dispatch(ctx, *w, x, x_dtype, y, y_dtype, m, gemm_workspace(ctx, s), s);
    // One or two rows, and many: the product's kernel adds its rows' adapters itself, where it does.
    if (w->format != RQ_Q_AFFINE_U4 && w->k_in > 0 && (m <= 2 || m > kFewRows)) {
        const LoraDecode ld{p.b, p.factors, p.part, p.ids, p.ranks, p.n_adapters, p.rank, p.slices, set->dtype == RQ_F16};
        st = m <= 2 ? launch_gemv_decode_loras(*w, x, x_dtype, y, y_dtype, (int)m, ld, s)
                    : launch_gemm(*w, x, x_dtype, y, y_dtype, m, ctx->num_cus, gemm_workspace(ctx, s), s, &ld);
        if (st != RQ_ERR_UNSUPPORTED) return st;
    }
    if ((st = qmatmul_dispatch(ctx, *w, x, x_dtype, const_cast<float *>(p.main), RQ_F32, m, gemm_workspace(ctx, s), s)) != RQ_OK)
        return st;
    return run_out(p, set->dtype, y_dtype, s);
}

// For the tests, no part of the C ABI: the argument checks alone.  Host arithmetic.
int rusty_loras_check(const rq_qweight *w, const rq_lora_set *set, const int32_t *ids, const void *x, int x_dtype, void *y,
                      int y_dtype, int64_t m, void *workspace, size_t workspace_bytes) {
    LoraArgs p{};
    bool run;
    return check_loras(w, set, ids, x, (rq_dtype)x_dtype, y, (rq_dtype)y_dtype, m, workspace, workspace_bytes, p, run);
}

}  // extern "C"
