// Rotary positions as entry points: rows of heads turned by their tokens'
// positions, forward and backward (rq_rope_rows), and a call's q, k and v turned
// and put into a paged cache (rq_rope_append).
//
//   out_a = m (x_a cos t - x_b sin t),  out_b = m (x_b cos t + x_a sin t),  t = position * freq_i
//
// The turn is orthogonal but for m, so the gradient of x is the turn by -t.
//
// A pass reads and writes every element once and is bound by that; all heads of
// a token share its rot / 2 angles.  A block takes a few whole tokens: it asks
// for its first elements, forms the tokens' (cos, sin) once into LDS -- the angle
// in 64 bits, reduced to a fraction of a turn there, then f32 functions of its f32 value, and the
// remainder to first order (without it rows of (1, 0) were off by up to 1.85 2^-24, so by 1.31) -- and turns
// the elements, 16 bytes a load at any alignment: where a head's parts are no
// whole number of such pieces, the last one overlaps the one before it, unless the call
// works in place (4096 tokens of 32 heads of 128, 86 of them turned, fp16: element by element 34 us, so 13.6).
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "paged.hpp"

namespace rq {
namespace {

constexpr int TH = 256;
constexpr int U = 4;           // units in flight per thread
constexpr int kMaxAngles = 2048;  // (cos, sin) pairs of a block's tokens: 16 KiB

struct RopeArgs {
    const double *freqs;
    const int *positions, *starts;
    const char *q, *k, *v;
    char *out;
    int64_t q_row, k_row, v_row, out_row;  // bytes
    Pages pages;
    int64_t tokens;
    int per_block;         // tokens
    int rot, hd;           // elements
    int n_q, n_kv;         // heads of q; APPEND: of k and of v
    int turned, units;     // of a head: units that are turned, all units
    int adjacent;          // V = 1: pairs side by side
    Div by_token, by_units;  // units of a token, of a head
    float magnitude, sign;
};

// The sequence of token t: the largest s with starts[s] <= t, where t < starts[s + 1]; -1 if none.
// Whole wave, t uniform: the 64 lanes probe at once.
__device__ __forceinline__ int seq_of(const int *starts, int n_seqs, int64_t tokens, int64_t t) {
    const int lane = threadIdx.x & 63;
    auto start = [&](int s) { return (int64_t)min(max((int64_t)starts[s], (int64_t)0), tokens); };
    int lo = 0, n = n_seqs;
    while (n > 63) {
        const int step = (n + 63) / 64, i = (lane + 1) * step;
        const bool in = i < n;
        const int c = __builtin_popcountll(__builtin_amdgcn_ballot_w64(in && start(in ? lo + i : 0) <= t));
        lo += c * step;
        n = min(step, n - c * step);
    }
    const bool le = start(lo + min(lane, n)) <= t;
    const int c = __builtin_popcountll(__builtin_amdgcn_ballot_w64(lane < n && le)) - 1;  // its index, the last that is not past t
    const uint64_t past = __builtin_amdgcn_ballot_w64(!le);
    return c >= 0 && (past >> (c + 1) & 1) ? lo + c : -1;
}

// A unit is V consecutive elements (INTER) or V pairs as two vectors (otherwise: of a head's halves; V = 1 and
// `adjacent`, of two elements side by side).  Units past `turned` are up to V elements that are copied.
template <typename T, int V, bool INTER, bool APPEND>
__global__ __launch_bounds__(TH) void k_rope(RopeArgs a) {
    typedef T vec __attribute__((ext_vector_type(V), aligned(sizeof(T))));
    extern __shared__ float2 cs[];  // [tokens][rot / 2]
    __shared__ int64_t place[APPEND ? TH : 1];  // a token's offset in the cache; -1: not cached, -2: no sequence
    const int64_t t0 = (int64_t)blockIdx.x * a.per_block;
    const int nt = (int)min((int64_t)a.per_block, a.tokens - t0), half = a.rot / 2;
    const int heads = APPEND ? a.n_q + 2 * a.n_kv : a.n_q;
    const int per_token = heads * a.units, total = nt * per_token;
    // this part of the block's units
    const int part = (total + (int)gridDim.y - 1) / (int)gridDim.y;
    const int first = (int)blockIdx.y * part, end = min(first + part, total);

    const int rest = a.hd - a.rot;
    struct Unit {
        int token, head, pair, e0, e1;  // its first pair, the elements of its two vectors; e1 < 0: one vector
        bool turn, part;                // part: fewer than V elements, to the head's end
    };
    auto unit = [&](int u) {
        Unit r;
        r.token = a.by_token(u);
        const int w = u - r.token * per_token;
        r.head = a.by_units(w);
        const int i = w - r.head * a.units;
        r.turn = i < a.turned;
        const bool adjacent = V == 1 && a.adjacent;
        r.pair = INTER ? min(i * (V / 2), half - V / 2) : min(i * V, half - V);
        r.e0 = INTER || adjacent ? 2 * r.pair : r.pair;
        r.e1 = INTER ? -1 : r.e0 + (adjacent ? 1 : half);
        r.part = false;
        if (!r.turn) {
            r.part = rest < V;
            r.e0 = r.part ? a.rot : a.rot + min((i - a.turned) * V, rest - V);
            r.e1 = -1;
        }
        if (APPEND && r.head >= a.n_q + a.n_kv) r.turn = false;  // v
        return r;
    };
    auto source = [&](const Unit &r) -> const char * {
        const int64_t t = t0 + r.token;
        if (!APPEND || r.head < a.n_q) return a.q + t * a.q_row + (int64_t)r.head * a.hd * (int)sizeof(T);
        if (r.head < a.n_q + a.n_kv) return a.k + t * a.k_row + (int64_t)(r.head - a.n_q) * a.hd * (int)sizeof(T);
        return a.v + t * a.v_row + (int64_t)(r.head - a.n_q - a.n_kv) * a.hd * (int)sizeof(T);
    };
    vec x[U], y[U];
    auto load = [&](int u0) {
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int u = u0 + i * TH;
            if (u >= end) break;
            const Unit r = unit(u);
            const T *p = reinterpret_cast<const T *>(source(r));
            if (V > 1 && r.part) {
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (e < rest) x[i][e] = p[r.e0 + e];
                continue;
            }
            x[i] = *reinterpret_cast<const vec *>(p + r.e0);
            if constexpr (!INTER)
                if (r.e1 >= 0) y[i] = *reinterpret_cast<const vec *>(p + r.e1);
        }
    };
    load(first + threadIdx.x);

    for (int i = threadIdx.x; i < nt * half; i += TH) {
        const int t = i / half;
        const double turns = (double)a.positions[t0 + t] * (a.freqs[i - t * half] * 0.15915494309189535);  // 1 / 2 pi
        const double turn = turns - rint(turns);
        const float near = (float)turn;
        float s, c;
        sincospif(2.0f * near, &s, &c);
        // what f32 leaves of the angle, up to 2^-26 of a turn (its square does not tell)
        const float off = (float)(turn - (double)near) * 6.2831855f;
        cs[i] = make_float2(__builtin_fmaf(-s, off, c) * a.magnitude, __builtin_fmaf(c, off, s) * (a.magnitude * a.sign));
    }
    if constexpr (APPEND) {
        for (int t = threadIdx.x >> 6; t < nt; t += TH / 64) {
            const int s = a.starts ? seq_of(a.starts, a.pages.n_seqs, a.tokens, t0 + t)
                                   : (t0 + t < a.pages.n_seqs ? (int)(t0 + t) : -1);
            if ((threadIdx.x & 63) == 0) place[t] = s < 0 ? -2 : a.pages.at(s, a.positions[t0 + t]);
        }
    }
    __syncthreads();

    for (int u0 = first + threadIdx.x; u0 < end; u0 += U * TH) {
        if (u0 != first + (int)threadIdx.x) load(u0);
#pragma unroll
        for (int i = 0; i < U; ++i) {
            const int u = u0 + i * TH;
            if (u >= end) break;
            const Unit r = unit(u);
            char *to;
            if (!APPEND || r.head < a.n_q) {
                if (APPEND && place[APPEND ? r.token : 0] == -2) continue;
                to = a.out + (t0 + r.token) * a.out_row + (int64_t)r.head * a.hd * (int)sizeof(T);
            } else {
                const int64_t at = place[APPEND ? r.token : 0];
                if (at < 0) continue;
                const int g = r.head - a.n_q;
                to = (g < a.n_kv ? a.pages.k + g * a.pages.head_stride : a.pages.v + (g - a.n_kv) * a.pages.head_stride) + at;
            }
            vec p = x[i], q = y[i];
            if (r.turn) {
                const float2 *w = cs + r.token * half + r.pair;
                if constexpr (INTER) {
#pragma unroll
                    for (int e = 0; e < V; e += 2) {
                        const float2 z = w[e / 2];
                        const float xa = (float)x[i][e], xb = (float)x[i][e + 1 < V ? e + 1 : e];
                        p[e] = (T)__builtin_fmaf(xa, z.x, -(xb * z.y));
                        p[e + 1 < V ? e + 1 : e] = (T)__builtin_fmaf(xb, z.x, xa * z.y);
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < V; ++e) {
                        const float2 z = w[e];
                        const float xa = (float)x[i][e], xb = (float)y[i][e];
                        p[e] = (T)__builtin_fmaf(xa, z.x, -(xb * z.y));
                        q[e] = (T)__builtin_fmaf(xb, z.x, xa * z.y);
                    }
                }
            }
            T *d = reinterpret_cast<T *>(to);
            if (V > 1 && r.part) {
#pragma unroll
                for (int e = 0; e < V; ++e)
                    if (e < rest) d[r.e0 + e] = p[e];
                continue;
            }
            *reinterpret_cast<vec *>(d + r.e0) = p;
            if constexpr (!INTER)
                if (r.e1 >= 0) *reinterpret_cast<vec *>(d + r.e1) = q;
        }
    }
}

// Launches the kernel over vectors of V elements, up to 16 bytes: of what is turned (HALF: of its half) whole pieces
// in place, else one at least (the last may overlap).
template <typename T, bool APPEND>
int launch(RopeArgs a, bool inter, bool in_place, hipStream_t s) {
    const int half = a.rot / 2, span = inter ? a.rot : half, rest = in_place && !APPEND ? 0 : a.hd - a.rot;
    int v = 16 / (int)sizeof(T);
    while (v > 1 && (in_place ? span % v != 0 : span < v)) v /= 2;
    a.adjacent = inter && v == 1;
    if (v == 1) inter = false;
    a.turned = (int)cdiv(inter ? a.rot : half, v);
    a.units = a.turned + (int)cdiv(rest, v);
    const int64_t heads = APPEND ? a.n_q + 2 * (int64_t)a.n_kv : a.n_q, units = heads * a.units;
    if (units > 0x7fffffff / TH) return fail(RQ_ERR_SHAPE, "too many heads");
    // Tokens per block: a thousand units, as long as that leaves a block for every CU.
    int64_t per = std::max<int64_t>(1, std::min({U * TH / units, (int64_t)kMaxAngles / half, (int64_t)TH, cdiv(a.tokens, 512)}));
    a.per_block = (int)per;
    a.by_token = Div::by(units);
    a.by_units = Div::by(a.units);
    const int64_t blocks = cdiv(a.tokens, per);
    // few tokens: a token's units over several blocks
    const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(cdiv(per * units, TH), 512 / blocks));
    if (!grid_ok(blocks, TH)) return fail(RQ_ERR_SHAPE, "too many tokens for one call");
    const dim3 grid((unsigned)blocks, (unsigned)parts);
    const size_t lds = (size_t)per * half * sizeof(float2);
    auto go = [&](auto vc, auto ic) {
        constexpr int V = decltype(vc)::value;
        constexpr bool I = decltype(ic)::value;
        hipLaunchKernelGGL((k_rope<T, V, I, APPEND>), grid, dim3(TH), lds, s, a);
    };
    auto by_layout = [&](auto vc) {
        if (inter) go(vc, std::true_type{});
        else go(vc, std::false_type{});
    };
    switch (v) {
    case 8:
        if constexpr (sizeof(T) == 2) by_layout(std::integral_constant<int, 8>{});
        break;
    case 4: by_layout(std::integral_constant<int, 4>{}); break;
    case 2: by_layout(std::integral_constant<int, 2>{}); break;
    default: go(std::integral_constant<int, 1>{}, std::false_type{});
    }
    RQ_LAUNCH_CHECK();
    return RQ_OK;
}

int check_rope(const rq_rope *r) {
    if (!r) return fail(RQ_ERR_INVALID_ARGUMENT, "null rotary descriptor");
    if (r->layout != RQ_ROPE_HALF && r->layout != RQ_ROPE_INTERLEAVED)
        return fail(RQ_ERR_INVALID_ARGUMENT, "unknown rotary layout %d", r->layout);
    if (!isfinite(r->magnitude)) return fail(RQ_ERR_INVALID_ARGUMENT, "magnitude must be finite");
    if (r->head_dim < 2 || r->head_dim > 1024) return fail(RQ_ERR_SHAPE, "head_dim %d outside 2..1024", r->head_dim);
    if (r->rot_dim < 2 || r->rot_dim > r->head_dim || r->rot_dim % 2)
        return fail(RQ_ERR_SHAPE, "rot_dim %d must be even and in 2..head_dim", r->rot_dim);
    return RQ_OK;
}

void fill_rope(const rq_rope &r, RopeArgs &a) {
    a.freqs = r.freqs;
    a.rot = r.rot_dim;
    a.hd = r.head_dim;
    a.magnitude = r.magnitude;
    a.sign = 1.0f;
}

// rq_rope_rows' arguments; a is complete where there is work (*run).
int check_rows(const rq_rope *rope, const void *x, int64_t x_row, const int32_t *positions, int64_t tokens,
               int32_t n_heads, rq_dtype dtype, const void *out, int64_t out_row, unsigned flags, RopeArgs &a, bool &run) {
    run = false;
    const int st = check_rope(rope);
    if (st != RQ_OK) return st;
    if (dtype != RQ_F16 && dtype != RQ_F32) return fail(RQ_ERR_INVALID_ARGUMENT, "dtype must be RQ_F16 or RQ_F32");
    if (flags & ~RQ_ROPE_BACKWARD) return fail(RQ_ERR_INVALID_ARGUMENT, "unknown flags 0x%x", flags);
    if (tokens < 0 || tokens > 0x7fffffff) return fail(RQ_ERR_SHAPE, "tokens outside 0..2^31-1");
    if (n_heads < 0 || n_heads > 65536) return fail(RQ_ERR_SHAPE, "n_heads %d outside 0..65536", n_heads);
    const int64_t row = (int64_t)n_heads * rope->head_dim, most = (int64_t)1 << 31;
    const int64_t xr = x_row ? x_row : row, orow = out_row ? out_row : row;
    if (xr < row || orow < row || xr > most || orow > most)
        return fail(RQ_ERR_SHAPE, "row strides must hold a row and be at most 2^31 elements");
    if (tokens == 0 || n_heads == 0) return RQ_OK;
    if (!x || !out || !positions || !rope->freqs) return fail(RQ_ERR_INVALID_ARGUMENT, "null pointer");
    const int size = dtype == RQ_F16 ? 2 : 4;
    if (!aligned(x, size) || !aligned(out, size) || !aligned(positions, 4) || !aligned(rope->freqs, 8))
        return fail(RQ_ERR_UNSUPPORTED, "pointers must be aligned to their elements");
    if (x == out && xr != orow) return fail(RQ_ERR_SHAPE, "in place, both row strides are the same");
    fill_rope(*rope, a);
    a.q = static_cast<const char *>(x);
    a.out = const_cast<char *>(static_cast<const char *>(out));
    a.q_row = xr * size;
    a.out_row = orow * size;
    a.positions = positions;
    a.tokens = tokens;
    a.n_q = n_heads;
    if (flags & RQ_ROPE_BACKWARD) a.sign = -1.0f;
    run = true;
    return RQ_OK;
}

// rq_rope_append's arguments likewise.
int check_append(const rq_rope *rope, const rq_attn *attn, const rq_kv_pages *cache, const void *q, const void *k,
                 const void *v, const int32_t *starts, const int32_t *positions, int64_t tokens, const void *out,
                 RopeArgs &a, bool &run) {
    run = false;
    int st = check_rope(rope);
    if (st != RQ_OK) return st;
    AttnRows r;
    if ((st = check_attn_rows(attn, tokens, &r)) != RQ_OK) return st;
    if (rope->head_dim != attn->head_dim)
        return fail(RQ_ERR_SHAPE, "head_dim %d of the rotary descriptor, %d of the heads", rope->head_dim, attn->head_dim);
    if ((st = check_pages(cache, attn, &a.pages)) != RQ_OK) return st;
    if (!starts && tokens > cache->n_seqs) return fail(RQ_ERR_SHAPE, "more tokens than sequences, and no starts");
    if (tokens == 0 || cache->n_seqs == 0) return RQ_OK;
    if (!q || !k || !v || !out || !positions || !rope->freqs) return fail(RQ_ERR_INVALID_ARGUMENT, "null pointer");
    if (!aligned(q, 16) || !aligned(k, 16) || !aligned(v, 16) || !aligned(out, 16) || !aligned(positions, 4) ||
        !aligned(starts, 4) || !aligned(rope->freqs, 8))
        return fail(RQ_ERR_UNSUPPORTED, "pointers must be 16-byte aligned");
    if ((st = check_pages_ptr(cache)) != RQ_OK) return st;
    if (q == out && r.q != r.out) return fail(RQ_ERR_SHAPE, "in place, both row strides are the same");
    fill_rope(*rope, a);
    const int size = attn->dtype == RQ_F16 ? 2 : 4;
    a.q = static_cast<const char *>(q);
    a.k = static_cast<const char *>(k);
    a.v = static_cast<const char *>(v);
    a.out = const_cast<char *>(static_cast<const char *>(out));
    a.q_row = r.q * size;
    a.k_row = r.k * size;
    a.v_row = r.v * size;
    a.out_row = r.out * size;
    a.positions = positions;
    a.starts = starts;
    a.tokens = tokens;
    a.n_q = attn->n_heads;
    a.n_kv = attn->n_kv_heads;
    run = true;
    return RQ_OK;
}

}  // namespace
}  // namespace rq

using namespace rq;

extern "C" {

int rq_rope_frequencies(const rq_rope_config *c, double *freqs, float *magnitude) {
    if (!c || !freqs || !magnitude) return fail(RQ_ERR_INVALID_ARGUMENT, "null pointer");
    if (c->scaling < RQ_ROPE_PLAIN || c->scaling > RQ_ROPE_RAMP)
        return fail(RQ_ERR_INVALID_ARGUMENT, "unknown rotary scaling %d", c->scaling);
    if (c->rot_dim < 2 || c->rot_dim > 1024 || c->rot_dim % 2)
        return fail(RQ_ERR_SHAPE, "rot_dim %d must be even and in 2..1024", c->rot_dim);
    if (!isfinite(c->theta) || !(c->theta > 1.0)) return fail(RQ_ERR_INVALID_ARGUMENT, "theta must be finite and above 1");
    const bool scaled = c->scaling != RQ_ROPE_PLAIN, cut = c->scaling >= RQ_ROPE_BANDS;
    if (scaled && (!isfinite(c->factor) || !(c->factor >= 1.0)))
        return fail(RQ_ERR_INVALID_ARGUMENT, "factor must be finite and at least 1");
    if (cut && (!isfinite(c->trained) || !(c->trained > 0.0) || !(c->low > 0.0) || !isfinite(c->high) || !(c->high > c->low)))
        return fail(RQ_ERR_INVALID_ARGUMENT, "needs a trained context and 0 < low < high");
    const double rot = c->rot_dim, two_pi = 6.283185307179586476925;
    double theta = c->theta;
    if (c->scaling == RQ_ROPE_STRETCH) theta *= pow(c->factor, c->rot_dim > 2 ? rot / (rot - 2.0) : 1.0);
    *magnitude = c->scaling == RQ_ROPE_RAMP ? (float)(0.1 * log(c->factor) + 1.0) : 1.0f;
    // RAMP: the pairs' indexes (times 1) that make `turns` turns within the trained context
    auto index = [&](double turns) { return rot * log(c->trained / (turns * two_pi)) / (2.0 * log(c->theta)); };
    const double first = cut ? std::max(floor(index(c->high)), 0.0) : 0.0;
    const double last = cut ? std::min(ceil(index(c->low)), rot - 1.0) : 0.0;
    for (int i = 0; i < c->rot_dim / 2; ++i) {
        const double f = pow(theta, -2.0 * i / rot);
        double slow = 0.0;  // how far divided by the factor
        if (c->scaling == RQ_ROPE_LINEAR) slow = 1.0;
        if (c->scaling == RQ_ROPE_BANDS)
            slow = 1.0 - std::min(std::max((c->trained * f / two_pi - c->low) / (c->high - c->low), 0.0), 1.0);
        if (c->scaling == RQ_ROPE_RAMP) slow = std::min(std::max((i - first) / std::max(last - first, 0.001), 0.0), 1.0);
        freqs[i] = slow == 1.0 ? f / c->factor : f * (1.0 - slow + (slow > 0.0 ? slow / c->factor : 0.0));
    }
    return RQ_OK;
}

int rq_rope_rows(rq_ctx *ctx, const rq_rope *rope, const void *x, int64_t x_row, const int32_t *positions,
                 int64_t tokens, int32_t n_heads, rq_dtype dtype, void *out, int64_t out_row, unsigned flags,
                 rq_stream stream) {
    RQ_ENTER(ctx);
    RopeArgs a{};
    bool run;
    const int st = check_rows(rope, x, x_row, positions, tokens, n_heads, dtype, out, out_row, flags, a, run);
    if (st != RQ_OK || !run) return st;
    const bool inter = rope->layout == RQ_ROPE_INTERLEAVED, in_place = x == out;
    hipStream_t s = pick(ctx, stream);
    return dtype == RQ_F16 ? launch<_Float16, false>(a, inter, in_place, s) : launch<float, false>(a, inter, in_place, s);
}

int rq_rope_append(rq_ctx *ctx, const rq_rope *rope, const rq_attn *attn, const rq_kv_pages *cache, const void *q,
                   const void *k, const void *v, const int32_t *starts, const int32_t *positions, int64_t tokens,
                   void *out, rq_stream stream) {
    RQ_ENTER(ctx);
    RopeArgs a{};
    bool run;
    const int st = check_append(rope, attn, cache, q, k, v, starts, positions, tokens, out, a, run);
    if (st != RQ_OK || !run) return st;
    const bool inter = rope->layout == RQ_ROPE_INTERLEAVED, in_place = q == out;
    hipStream_t s = pick(ctx, stream);
    return attn->dtype == RQ_F16 ? launch<_Float16, true>(a, inter, in_place, s) : launch<float, true>(a, inter, in_place, s);
}

// For the tests, no part of the C ABI: the argument checks alone (attn NULL: rq_rope_rows').  Host arithmetic.
int rusty_rope_check(const rq_rope *rope, const rq_attn *attn, const rq_kv_pages *cache, const void *q, const void *k,
                     const void *v, int64_t x_row, const int32_t *starts, const int32_t *positions, int64_t tokens,
                     int32_t n_heads, int dtype, const void *out, int64_t out_row, unsigned flags) {
    RopeArgs a{};
    bool run;
    return attn ? check_append(rope, attn, cache, q, k, v, starts, positions, tokens, out, a, run)
                : check_rows(rope, q, x_row, positions, tokens, n_heads, (rq_dtype)dtype, out, out_row, flags, a, run);
}

}  // extern "C"
