// Attention entry points: causal attention over packed prompts
// (rq_attn_packed) and of drafted tokens over a KV cache (rq_attn_tree).
//
//   out[t, h] = sum_j p_j v[j] / sum_j p_j,  p_j = 2^(c q.k_j - m),  c = scale log2 e
//
// over the keys j token t sees, with the running maximum m of c q.k and the
// running sum kept in f32 and earlier sums rescaled when m rises.
#include <math.h>

#include "common.hpp"

namespace rq {
namespace {

constexpr int kMaxNodes = 64;

// What both kernels read; strides in elements.
struct AttnArgs {
    const void *q, *k, *v;
    void *out;
    const int *starts, *lengths;
    const uint64_t *mask;
    int64_t q_row, k_row, v_row, out_row;  // packed: rows of consecutive tokens
    int64_t seq_stride, head_stride, pos_stride;  // tree: the cache
    int n_heads, n_kv, n_seqs, capacity, max_nodes;
    int tokens;
    float scale;  // times log2 e
};

__device__ __forceinline__ int seq_start(const AttnArgs &a, int s) { return min(max(a.starts[s], 0), a.tokens); }

// The sequence that holds token t, or -1: the last s with starts[s] <= t, if t
// lies before its end.
__device__ __forceinline__ int seq_of(const AttnArgs &a, int t) {
    int lo = 0, hi = a.n_seqs;  // starts[lo] <= t (if any), starts[hi] > t or hi = n_seqs
    if (seq_start(a, 0) > t) return -1;
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (seq_start(a, mid) <= t) lo = mid;
        else hi = mid;
    }
    return t < seq_start(a, lo + 1) ? lo : -1;
}

// One wave per (token, head): lane l holds dims l, l + 64, ...
template <typename T, int HD, bool TREE>
__global__ __launch_bounds__(64) void k_attn_rows(AttnArgs a) {
    constexpr int E = HD / 64;
    const int t = blockIdx.x / a.n_heads, h = blockIdx.x % a.n_heads, lane = threadIdx.x;
    const int s = seq_of(a, t);
    if (s < 0) return;
    const int g = h / (a.n_heads / a.n_kv), s0 = seq_start(a, s), i = t - s0;
    const T *q = static_cast<const T *>(a.q) + (int64_t)t * a.q_row + (int64_t)h * HD;
    const T *kb, *vb;
    int64_t ks, vs;
    int before, nodes;  // keys 0..before-1, then before + j for the bits j < nodes of see
    uint64_t see;
    if (TREE) {
        nodes = min(seq_start(a, s + 1) - s0, a.max_nodes);
        if (i >= nodes) return;
        before = min(max(a.lengths[s], 0), a.capacity);
        nodes = min(nodes, a.capacity - before);
        see = a.mask ? a.mask[t] : (~0ull >> (63 - i));
        kb = static_cast<const T *>(a.k) + s * a.seq_stride + g * a.head_stride;
        vb = static_cast<const T *>(a.v) + s * a.seq_stride + g * a.head_stride;
        ks = vs = a.pos_stride;
    } else {
        before = i + 1;
        nodes = 0;
        see = 0;
        kb = static_cast<const T *>(a.k) + (int64_t)s0 * a.k_row + (int64_t)g * HD;
        vb = static_cast<const T *>(a.v) + (int64_t)s0 * a.v_row + (int64_t)g * HD;
        ks = a.k_row;
        vs = a.v_row;
    }
    float qv[E], o[E], m = -INFINITY, l = 0.0f;
    for (int e = 0; e < E; ++e) {
        qv[e] = (float)q[lane + 64 * e];
        o[e] = 0.0f;
    }
    for (int j = 0; j < before + nodes; ++j) {
        if (j >= before && !(see >> (j - before) & 1)) continue;
        float sc = 0.0f;
        for (int e = 0; e < E; ++e) sc = __builtin_fmaf(qv[e], (float)kb[j * ks + lane + 64 * e], sc);
        for (int w = 32; w > 0; w >>= 1) sc += __shfl_xor(sc, w, 64);
        sc *= a.scale;
        const float mn = fmaxf(m, sc), base = mn == -INFINITY ? 0.0f : mn;
        const float al = exp2f(m - base), p = exp2f(sc - base);
        m = mn;
        l = l * al + p;
        for (int e = 0; e < E; ++e) o[e] = __builtin_fmaf(p, (float)vb[j * vs + lane + 64 * e], o[e] * al);
    }
    const bool none = TREE && before == 0 && (nodes == 0 || !(see & (~0ull >> (64 - nodes))));
    T *out = static_cast<T *>(a.out) + (int64_t)t * a.out_row + (int64_t)h * HD;
    for (int e = 0; e < E; ++e) out[lane + 64 * e] = (T)(none ? 0.0f : o[e] / l);
}

int launch_rows(const AttnArgs &a, bool tree, int hd, int dtype, hipStream_t s) {
    const int64_t blocks = (int64_t)a.tokens * a.n_heads;
    if (!grid_ok(blocks, 64)) return fail(RQ_ERR_SHAPE, "tokens * n_heads too large");
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(64), 0, s, a); };
    if (dtype == RQ_F16) {
        if (hd == 64) tree ? go(k_attn_rows<_Float16, 64, true>) : go(k_attn_rows<_Float16, 64, false>);
        else tree ? go(k_attn_rows<_Float16, 128, true>) : go(k_attn_rows<_Float16, 128, false>);
    } else {
        if (hd == 64) tree ? go(k_attn_rows<float, 64, true>) : go(k_attn_rows<float, 64, false>);
        else tree ? go(k_attn_rows<float, 128, true>) : go(k_attn_rows<float, 128, false>);
    }
    RQ_LAUNCH_CHECK();
    return RQ_OK;
}

// The checks both entry points share; fills the strides of a.
int check_attn(const rq_attn *at, int64_t tokens, AttnArgs &a) {
    if (!at) return fail(RQ_ERR_INVALID_ARGUMENT, "null attention descriptor");
    if (at->dtype != RQ_F16 && at->dtype != RQ_F32) return fail(RQ_ERR_INVALID_ARGUMENT, "dtype must be RQ_F16 or RQ_F32");
    if (at->reserved != 0) return fail(RQ_ERR_INVALID_ARGUMENT, "reserved field must be 0");
    if (at->head_dim != 64 && at->head_dim != 128) return fail(RQ_ERR_UNSUPPORTED, "head_dim must be 64 or 128");
    if (at->n_heads < 1 || at->n_kv_heads < 1 || at->n_heads % at->n_kv_heads != 0)
        return fail(RQ_ERR_SHAPE, "n_heads %d must be a multiple of n_kv_heads %d", at->n_heads, at->n_kv_heads);
    if (at->n_heads > 65536) return fail(RQ_ERR_SHAPE, "too many heads");
    if (!isfinite(at->scale)) return fail(RQ_ERR_INVALID_ARGUMENT, "scale must be finite");
    if (tokens < 0 || tokens > 0x7fffffff) return fail(RQ_ERR_SHAPE, "tokens outside 0..2^31-1");
    const int64_t qw = (int64_t)at->n_heads * at->head_dim, kw = (int64_t)at->n_kv_heads * at->head_dim;
    const int64_t unit = at->dtype == RQ_F16 ? 8 : 4, most = (int64_t)1 << 40;
    a.q_row = at->q_row ? at->q_row : qw;
    a.k_row = at->k_row ? at->k_row : kw;
    a.v_row = at->v_row ? at->v_row : kw;
    a.out_row = at->out_row ? at->out_row : qw;
    if (a.q_row < qw || a.out_row < qw || a.k_row < kw || a.v_row < kw || a.q_row > most || a.out_row > most ||
        a.k_row > most || a.v_row > most)
        return fail(RQ_ERR_SHAPE, "row stride shorter than a row or out of range");
    if (a.q_row % unit || a.out_row % unit || a.k_row % unit || a.v_row % unit)
        return fail(RQ_ERR_UNSUPPORTED, "row strides must be multiples of 16 bytes");
    a.n_heads = at->n_heads;
    a.n_kv = at->n_kv_heads;
    a.tokens = (int)tokens;
    a.scale = (at->scale != 0.0f ? at->scale : 1.0f / sqrtf((float)at->head_dim)) * 1.4426950408889634f;
    return RQ_OK;
}

// rq_attn_packed's arguments; *a is complete where there is work (*run).
int check_packed(const rq_attn *attn, const void *q, const void *k, const void *v, const int32_t *starts,
                 int32_t n_seqs, int64_t tokens, void *out, AttnArgs &a, bool &run) {
    run = false;
    const int st = check_attn(attn, tokens, a);
    if (st != RQ_OK) return st;
    if (n_seqs < 0) return fail(RQ_ERR_SHAPE, "negative n_seqs");
    if (n_seqs == 0 || tokens == 0) return RQ_OK;
    if (!q || !k || !v || !out || !starts) return fail(RQ_ERR_INVALID_ARGUMENT, "null pointer");
    if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 16) || !aligned(starts, 4))
        return fail(RQ_ERR_UNSUPPORTED, "pointers must be 16-byte aligned");
    a.q = q;
    a.k = k;
    a.v = v;
    a.out = out;
    a.starts = starts;
    a.n_seqs = n_seqs;
    run = true;
    return RQ_OK;
}

// rq_attn_tree's arguments likewise.
int check_tree(const rq_attn *attn, const rq_kv_cache *cache, const void *q, const int32_t *starts,
               const int32_t *lengths, const uint64_t *mask, int64_t tokens, int32_t max_nodes, void *out,
               void *workspace, size_t workspace_bytes, AttnArgs &a, bool &run) {
    run = false;
    const int st = check_attn(attn, tokens, a);
    if (st != RQ_OK) return st;
    if (!cache) return fail(RQ_ERR_INVALID_ARGUMENT, "null cache");
    if (max_nodes < 1 || max_nodes > kMaxNodes) return fail(RQ_ERR_SHAPE, "max_nodes %d outside 1..%d", max_nodes, kMaxNodes);
    if (cache->n_seqs < 0 || cache->capacity < 0) return fail(RQ_ERR_SHAPE, "negative cache size");
    const int64_t hd = attn->head_dim, unit = attn->dtype == RQ_F16 ? 8 : 4, most = (int64_t)1 << 40;
    a.seq_stride = cache->seq_stride;
    a.head_stride = cache->head_stride;
    a.pos_stride = cache->pos_stride;
    if (a.seq_stride == 0 && a.head_stride == 0 && a.pos_stride == 0) {
        a.pos_stride = hd;
        a.head_stride = hd * cache->capacity;
        a.seq_stride = a.head_stride * a.n_kv;
    }
    // (a stride that is never taken, of one head or one sequence, may be 0)
    if (a.head_stride < 0 || a.seq_stride < 0 || a.pos_stride > ((int64_t)1 << 24) || a.head_stride > most ||
        a.seq_stride > most ||
        (cache->capacity > 0 && (a.pos_stride < hd || (a.n_kv > 1 && a.head_stride < hd) ||
                                 (cache->n_seqs > 1 && a.seq_stride < hd))))
        return fail(RQ_ERR_SHAPE, "cache strides shorter than a row or out of range");
    if (a.pos_stride % unit || a.head_stride % unit || a.seq_stride % unit)
        return fail(RQ_ERR_UNSUPPORTED, "cache strides must be multiples of 16 bytes");
    if (cache->n_seqs == 0 || tokens == 0) return RQ_OK;
    if (!q || !out || !starts || !lengths || (cache->capacity > 0 && (!cache->k || !cache->v)))
        return fail(RQ_ERR_INVALID_ARGUMENT, "null pointer");
    if (!aligned(q, 16) || !aligned(cache->k, 16) || !aligned(cache->v, 16) || !aligned(out, 16) ||
        !aligned(starts, 4) || !aligned(lengths, 4) || !aligned(mask, 8))
        return fail(RQ_ERR_UNSUPPORTED, "pointers must be 16-byte aligned");
    const size_t need = rq_attn_tree_workspace(attn, cache->n_seqs, tokens, max_nodes, cache->capacity);
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(RQ_ERR_INVALID_ARGUMENT, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
    if (need > 0 && !aligned(workspace, 16)) return fail(RQ_ERR_UNSUPPORTED, "workspace must be 16-byte aligned");
    a.q = q;
    a.k = cache->k;
    a.v = cache->v;
    a.out = out;
    a.starts = starts;
    a.lengths = lengths;
    a.mask = mask;
    a.n_seqs = cache->n_seqs;
    a.capacity = cache->capacity;
    a.max_nodes = max_nodes;
    run = true;
    return RQ_OK;
}

}  // namespace
}  // namespace rq

using namespace rq;

extern "C" {

int rq_attn_packed(rq_ctx *ctx, const rq_attn *attn, const void *q, const void *k, const void *v,
                   const int32_t *starts, int32_t n_seqs, int64_t tokens, void *out, rq_stream stream) {
    RQ_ENTER(ctx);
    AttnArgs a{};
    bool run;
    const int st = check_packed(attn, q, k, v, starts, n_seqs, tokens, out, a, run);
    if (st != RQ_OK || !run) return st;
    return launch_rows(a, false, attn->head_dim, attn->dtype, pick(ctx, stream));
}

size_t rq_attn_tree_workspace(const rq_attn *attn, int32_t n_seqs, int64_t tokens, int32_t max_nodes,
                              int32_t capacity) {
    return 0;
}

int rq_attn_tree(rq_ctx *ctx, const rq_attn *attn, const rq_kv_cache *cache, const void *q, const int32_t *starts,
                 const int32_t *lengths, const uint64_t *mask, int64_t tokens, int32_t max_nodes, void *out,
                 void *workspace, size_t workspace_bytes, rq_stream stream) {
    RQ_ENTER(ctx);
    AttnArgs a{};
    bool run;
    const int st = check_tree(attn, cache, q, starts, lengths, mask, tokens, max_nodes, out, workspace,
                              workspace_bytes, a, run);
    if (st != RQ_OK || !run) return st;
    return launch_rows(a, true, attn->head_dim, attn->dtype, pick(ctx, stream));
}

// For the tests, no part of the C ABI: the argument checks alone (cache NULL:
// rq_attn_packed's, k and v its pointers).  Host arithmetic.
int rusty_attn_check(const rq_attn *attn, const rq_kv_cache *cache, const void *q, const void *k, const void *v,
                     const int32_t *starts, const int32_t *lengths, const uint64_t *mask, int32_t n_seqs,
                     int64_t tokens, int32_t max_nodes, void *out, void *workspace, size_t workspace_bytes) {
    AttnArgs a{};
    bool run;
    return cache ? check_tree(attn, cache, q, starts, lengths, mask, tokens, max_nodes, out, workspace,
                              workspace_bytes, a, run)
                 : check_packed(attn, q, k, v, starts, n_seqs, tokens, out, a, run);
}

}  // extern "C"
