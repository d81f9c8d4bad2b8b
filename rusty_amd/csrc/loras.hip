// A quantized Linear with an adapter per row (rq_qmatmul_loras):
//   Y[t] = X[t] . deq(W)^T + factor_i (X[t] . A_i^T) . B_i,  i = ids[t].
//
// Three launches: the rows' t = X . A_i^T (k_loras_in: a narrow product, its k cut
// over blocks, one partial sum per slice), the shared product into f32
// (rq_qmatmul's kernels), and Y = main + factor t . B_i (k_loras_out), rounded
// once.  Small batches are bound by the launches and by the weight's bytes, which
// each used adapter adds (k_in + n_out) rank elements to; prompts by the shared product.
//
// k_loras_in: 16 rows of X are the rows of a matrix instruction, 16 rows of A_i its
// columns, k runs along both (16-byte loads, no LDS).  Rows of a tile may have
// different adapters: each one's product is formed for all 16 rows and
// kept for its own, so nothing a foreign adapter holds reaches a row.
//
// k_loras_out has two forms.  Few rows: a block takes one row and a stretch of
// columns, its lanes 8 columns each, the adapter's rank one fma at a time -- no work
// on foreign rows.  Many: a wave takes 16 rows and 16 V columns on the f32 matrix
// instructions (t keeps its f32 bits), a B fragment of V columns a load.
#include <algorithm>
#include <type_traits>

#include "common.hpp"

namespace rq {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));

constexpr int kMaxRank = 256;
constexpr int kSlice = 1024;  // k of a k_loras_in block: 256 a wave

struct LoraArgs {
    const void *x, *a, *b;
    const float *factors;
    const int *ids, *ranks;
    float *part;        // [m][slices][rank]
    const float *main;  // [m][n]
    void *y;
    int64_t m, k, n;
    int n_adapters, rank, slices;
};

// The adapter of row t, -1 for none.
__device__ __forceinline__ int adapter_of(const LoraArgs &p, int64_t t) {
    const int i = p.ids[t];
    return (uint32_t)i < (uint32_t)p.n_adapters ? i : -1;
}
__device__ __forceinline__ int rank_of(const LoraArgs &p, int i) {
    return p.ranks ? min(max(p.ranks[i], 0), p.rank) : p.rank;
}

// N consecutive values at p + e as floats or halves, those at and past `end` zero.  VEC: whole or not at all, aligned.
template <typename S, int N, bool VEC, typename D>
__device__ __forceinline__ D load_n(const S *p, int64_t e, int64_t end) {
    typedef S vec __attribute__((ext_vector_type(N)));
    D r;
    if constexpr (VEC) {
        vec v = {};
        if (e < end) v = *reinterpret_cast<const vec *>(p + e);
#pragma unroll
        for (int i = 0; i < N; ++i) r[i] = (std::remove_reference_t<decltype(r[0] + r[0])>)v[i];
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) r[i] = 0;
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (e + i < end) r[i] = p[e + i];
    }
    return r;
}

// Block (tile, slice, z): 16 rows, kSlice of k; of the tile's distinct adapters every gridDim.z-th.
template <typename X, typename A, bool VEC>
__global__ __launch_bounds__(256) void k_loras_in(LoraArgs p) {
    constexpr bool F16 = sizeof(X) == 2 && sizeof(A) == 2;
    constexpr int N = F16 ? 8 : 4, STEP = 4 * N, STEPS = 256 / STEP;  // k a lane, an instruction, of a wave
    typedef std::conditional_t<F16, half8, floatx4> frag;
    __shared__ float sums[4][16][17];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, col = lane & 15, qt = lane >> 4;
    const int64_t t0 = (int64_t)blockIdx.x * 16, row = min(t0 + col, p.m - 1);
    const int64_t k0 = (int64_t)blockIdx.y * kSlice + wv * 256 + N * qt;
    const int mine = t0 + col < p.m ? adapter_of(p, t0 + col) : -1;
    uint64_t left = __builtin_amdgcn_ballot_w64(lane < 16 && mine >= 0);
    if (!left) return;
    const X *xr = static_cast<const X *>(p.x) + row * p.k;
    frag xf[STEPS];
#pragma unroll
    for (int j = 0; j < STEPS; ++j) xf[j] = load_n<X, N, VEC, frag>(xr, k0 + j * STEP, p.k);
    for (int z = 0; left; ++z) {
        const int i = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
        const uint64_t same = __builtin_amdgcn_ballot_w64(mine == i) & left;
        left &= ~same;
        if (z % (int)gridDim.z != (int)blockIdx.z) continue;
        const int rank = rank_of(p, i);
        for (int r0 = 0; r0 < rank; r0 += 16) {
            const A *ar = static_cast<const A *>(p.a) + ((int64_t)i * p.rank + min(r0 + col, rank - 1)) * p.k;
            floatx4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
            frag af[STEPS];
#pragma unroll
            for (int j = 0; j < STEPS; ++j) af[j] = load_n<A, N, VEC, frag>(ar, k0 + j * STEP, p.k);
#pragma unroll
            for (int j = 0; j < STEPS; ++j) {
                if constexpr (F16) {
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_f16(xf[j], af[j], acc, 0, 0, 0);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_16x16x4f32(xf[j][e], af[j][e], acc, 0, 0, 0);
                }
            }
            __syncthreads();  // the last sums have been read
#pragma unroll
            for (int e = 0; e < 4; ++e) sums[wv][4 * qt + e][col] = acc[e];
            __syncthreads();
            const int tr = threadIdx.x >> 4, r = threadIdx.x & 15;  // one (row, r) a thread
            if ((same >> tr & 1) && r0 + r < rank)
                p.part[((t0 + tr) * p.slices + blockIdx.y) * p.rank + r0 + r] =
                    (sums[0][tr][r] + sums[1][tr][r]) + (sums[2][tr][r] + sums[3][tr][r]);
        }
    }
}

// The row's t times its factor into ts[0 .. rank), the slices summed in order; whole block of TH threads or wave.
template <int TH>
__device__ __forceinline__ void sum_slices(const LoraArgs &p, int64_t t, int i, int rank, int thread, float *ts) {
    const float f = p.factors ? p.factors[i] : 1.0f;
    for (int r = thread; r < rank; r += TH) {
        const float *q = p.part + t * p.slices * p.rank + r;
        float s = 0.0f;
        for (int j = 0; j < p.slices; ++j) s += q[(int64_t)j * p.rank];
        ts[r] = f * s;
    }
}

// Few rows: block (row, stretch of 2048 columns).
template <typename B, typename Y, bool VEC>
__global__ __launch_bounds__(256) void k_loras_out_row(LoraArgs p) {
    typedef float floatx8 __attribute__((ext_vector_type(8)));
    __shared__ float ts[kMaxRank];
    const int64_t t = blockIdx.x, c = ((int64_t)blockIdx.y * 256 + threadIdx.x) * 8;
    const int i = adapter_of(p, t), rank = i < 0 ? 0 : rank_of(p, i);
    if (rank > 0) sum_slices<256>(p, t, i, rank, threadIdx.x, ts);
    __syncthreads();
    if (c >= p.n) return;
    floatx8 acc = {};
    const B *b = static_cast<const B *>(p.b) + (int64_t)max(i, 0) * p.rank * p.n;
#pragma unroll 8
    for (int r = 0; r < rank; ++r) {
        const floatx8 v = load_n<B, 8, VEC, floatx8>(b + (int64_t)r * p.n, c, p.n);
        const float s = ts[r];
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = __builtin_fmaf(s, v[e], acc[e]);
    }
    const float *main = p.main + t * p.n;
    const floatx8 v = load_n<float, 8, VEC, floatx8>(main, c, p.n);
    Y *y = static_cast<Y *>(p.y) + t * p.n;
    typedef Y vec __attribute__((ext_vector_type(8)));
    if constexpr (VEC) {
        vec o;
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = (Y)(v[e] + acc[e]);
        *reinterpret_cast<vec *>(y + c) = o;
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (c + e < p.n) y[c + e] = (Y)(v[e] + acc[e]);
    }
}

// Many rows: block (16 rows, stretch of 4 x 16 V columns), a wave 16 V columns.
template <typename B, typename Y, bool VEC>
__global__ __launch_bounds__(256) void k_loras_out(LoraArgs p) {
    constexpr int V = 16 / (int)sizeof(B);  // columns of a lane: V instructions, column col of the v-th is V col + v
    typedef float vecf __attribute__((ext_vector_type(V)));
    __shared__ float ts[16][kMaxRank + 4];
    __shared__ int id[16];
    const int lane = threadIdx.x & 63, wv = threadIdx.x >> 6, col = lane & 15, qt = lane >> 4;
    const int64_t t0 = (int64_t)blockIdx.x * 16, c = ((int64_t)blockIdx.y * 4 + wv) * 16 * V + V * col;
    for (int tr = wv; tr < 16; tr += 4) {
        const int64_t t = t0 + tr;
        const int i = t < p.m ? adapter_of(p, t) : -1, rank = i < 0 ? 0 : rank_of(p, i);
        for (int r = rank + lane; r < ((p.rank + 3) & ~3); r += 64) ts[tr][r] = 0.0f;
        if (rank > 0) sum_slices<64>(p, t, i, rank, lane, ts[tr]);
        if (lane == 0) id[tr] = i;
    }
    __syncthreads();
    const int mine = id[col];
    uint64_t left = __builtin_amdgcn_ballot_w64(lane < 16 && mine >= 0);
    vecf out[4];  // rows 4 qt + e
#pragma unroll
    for (int e = 0; e < 4; ++e) out[e] = {};
    while (left) {
        const int i = __builtin_amdgcn_readlane(mine, __builtin_ctzll(left));
        const uint64_t same = __builtin_amdgcn_ballot_w64(mine == i) & left;
        left &= ~same;
        const int rank = rank_of(p, i);
        const B *b = static_cast<const B *>(p.b) + (int64_t)i * p.rank * p.n;
        floatx4 acc[V];
#pragma unroll
        for (int v = 0; v < V; ++v) acc[v] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
        for (int r0 = 0; r0 < rank; r0 += 4) {
            const int r = r0 + qt;
            const vecf bv = load_n<B, V, VEC, vecf>(b + (int64_t)min(r, rank - 1) * p.n, c, r < rank ? p.n : 0);
            const float s = ts[col][r];
#pragma unroll
            for (int v = 0; v < V; ++v) acc[v] = __builtin_amdgcn_mfma_f32_16x16x4f32(s, bv[v], acc[v], 0, 0, 0);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (same >> (4 * qt + e) & 1)
#pragma unroll
                for (int v = 0; v < V; ++v) out[e][v] = acc[v][e];
    }
    if (c >= p.n) return;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int64_t t = t0 + 4 * qt + e;
        if (t >= p.m) return;
        const vecf v = load_n<float, V, VEC, vecf>(p.main + t * p.n, c, p.n);
        Y *y = static_cast<Y *>(p.y) + t * p.n;
        typedef Y vec __attribute__((ext_vector_type(V)));
        if constexpr (VEC) {
            vec o;
#pragma unroll
            for (int i = 0; i < V; ++i) o[i] = (Y)(v[i] + out[e][i]);
            *reinterpret_cast<vec *>(y + c) = o;
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (c + i < p.n) y[c + i] = (Y)(v[i] + out[e][i]);
        }
    }
}

constexpr int64_t kRowForm = 64;  // rows that k_loras_out_row serves

int check_set(const rq_lora_set *s) {
    if (!s) return fail(RQ_ERR_INVALID_ARGUMENT, "null adapter set");
    if (s->dtype != RQ_F16 && s->dtype != RQ_F32) return fail(RQ_ERR_INVALID_ARGUMENT, "the set's dtype must be RQ_F16 or RQ_F32");
    if (s->reserved != 0) return fail(RQ_ERR_INVALID_ARGUMENT, "reserved field must be 0");
    if (s->n_adapters < 0) return fail(RQ_ERR_SHAPE, "negative n_adapters");
    if (s->rank < 1 || s->rank > kMaxRank) return fail(RQ_ERR_SHAPE, "rank %d outside 1..%d", s->rank, kMaxRank);
    return RQ_OK;
}

int64_t slices_of(int64_t k) { return std::max<int64_t>(1, cdiv(k, kSlice)); }

int check_loras(const rq_qweight *w, const rq_lora_set *set, const int32_t *ids, const void *x, rq_dtype xt, void *y,
                rq_dtype yt, int64_t m, void *workspace, size_t workspace_bytes, LoraArgs &p, bool &run) {
    run = false;
    int st = check_qweight(w, true);
    if (st != RQ_OK) return st;
    if ((st = check_set(set)) != RQ_OK) return st;
    if ((xt != RQ_F16 && xt != RQ_F32) || (yt != RQ_F16 && yt != RQ_F32))
        return fail(RQ_ERR_INVALID_ARGUMENT, "dtype must be RQ_F16 or RQ_F32");
    if (m < 0 || m > 0x7fffffff) return fail(RQ_ERR_SHAPE, "m outside 0..2^31-1");
    const int64_t K = w->k_in, N = w->n_out;
    int64_t t;
    if (!mul_ok(m, K * 4, &t) || !mul_ok(m, N * 4, &t) || K > ((int64_t)1 << 40) || N > ((int64_t)1 << 40) ||
        !mul_ok((int64_t)set->n_adapters * set->rank, std::max(K, N) * 4, &t) || !mul_ok(m, slices_of(K) * set->rank * 4, &t))
        return fail(RQ_ERR_SHAPE, "shape overflows");
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
    p.slices = (int)slices_of(K);
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
    const int64_t tiles = cdiv(p.m, 16);
    // A tile's adapters side by side while blocks are few.
    const int64_t z = std::max<int64_t>(
        1, std::min<int64_t>({16, p.m, (int64_t)p.n_adapters, 4 * num_cus / std::max<int64_t>(1, tiles * p.slices)}));
    if (!grid_ok(tiles, 256) || p.slices > 65535) return fail(RQ_ERR_SHAPE, "too many rows or inputs for one call");
    const dim3 grid((unsigned)tiles, (unsigned)p.slices, (unsigned)z);
    const int n = xt == RQ_F16 && at == RQ_F16 ? 8 : 4, xs = xt == RQ_F16 ? 2 : 4, as = at == RQ_F16 ? 2 : 4;
    const bool vec = p.k % n == 0 && aligned(p.x, n * xs) && aligned(p.a, n * as);
    return by_type(xt, [&](auto *x) {
        return by_type(at, [&](auto *a) {
            using X = std::remove_pointer_t<decltype(x)>;
            using A = std::remove_pointer_t<decltype(a)>;
            if (vec) hipLaunchKernelGGL((k_loras_in<X, A, true>), grid, dim3(256), 0, s, p);
            else hipLaunchKernelGGL((k_loras_in<X, A, false>), grid, dim3(256), 0, s, p);
            RQ_LAUNCH_CHECK();
            return (int)RQ_OK;
        });
    });
}

int run_out(const LoraArgs &p, int bt, rq_dtype yt, hipStream_t s) {
    const bool vec = p.n % 8 == 0 && aligned(p.b, 16) && aligned(p.y, 16);
    return by_type(bt, [&](auto *b) {
        return by_type(yt, [&](auto *y) {
            using B = std::remove_pointer_t<decltype(b)>;
            using Y = std::remove_pointer_t<decltype(y)>;
            const bool rows = p.m <= kRowForm;
            const int64_t bx = rows ? p.m : cdiv(p.m, 16), by = cdiv(p.n, rows ? 2048 : 64 * (16 / (int)sizeof(B)));
            if (!grid_ok(bx, 256) || by > 65535) return fail(RQ_ERR_SHAPE, "too many rows or outputs for one call");
            const dim3 grid((unsigned)bx, (unsigned)by);
            if (rows) {
                if (vec) hipLaunchKernelGGL((k_loras_out_row<B, Y, true>), grid, dim3(256), 0, s, p);
                else hipLaunchKernelGGL((k_loras_out_row<B, Y, false>), grid, dim3(256), 0, s, p);
            } else {
                if (vec) hipLaunchKernelGGL((k_loras_out<B, Y, true>), grid, dim3(256), 0, s, p);
                else hipLaunchKernelGGL((k_loras_out<B, Y, false>), grid, dim3(256), 0, s, p);
            }
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
    (void)x_dtype;
    int64_t part, main = 0, t;
    if (check_set(set) != RQ_OK || m < 1 || k_in < 0 || n_out < 1 || !mul_ok(m, slices_of(k_in), &part) ||
        !mul_ok(part, 4 * set->rank, &part) || !mul_ok(m, n_out, &t) || !mul_ok(t, 4, &t))
        return 0;
    if (y_dtype != RQ_F32) main = (t + 255) / 256 * 256;
    return (size_t)main + (size_t)part;
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
