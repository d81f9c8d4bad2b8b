// Attention entry points: causal attention over packed prompts
// (rq_attn_packed) and of drafted tokens over a KV cache (rq_attn_tree).
//
//   out[t, h] = sum_j p_j v[j] / sum_j p_j,  p_j = 2^(c q.k_j - m),  c = scale log2 e
//
// over the keys j token t sees, in one pass over the keys: m is a running
// maximum of c q.k, and earlier sums are rescaled when it rises.
//
// A block works on the rows of one key/value head of one sequence, a row being
// a (token, query head) pair, token-major: the n_heads / n_kv_heads query heads of
// a token share the keys, so one pass over K and V serves them all, short
// sequences and single tokens fill the matrix instructions' 32 columns, and every
// row of a block ends near the same key.  K and V pass through LDS in tiles of KT
// keys (DMA, a ring of NS tiles, one barrier per tile).  Of the block's waves, WR take
// different 32 rows and KG different 32 keys of each tile (KG partial softmaxes per
// row, joined through LDS at the end).
//
// Matrix instructions: S^T = K . Q^T (A: 32 keys from LDS, B: the wave's 32
// rows of Q, held in registers), so a row's scores lie in one lane column --
// lane l holds keys 8 (r / 4) + 4 (l / 32) + r % 4, r < 16, of row l % 32 --
// and the maximum is in-lane plus one exchange with lane l ^ 32.  Then O^T = V^T . P^T
// takes P as it stands as the B operand, V^T in the key order that gives: for
// fp16 by transposing LDS reads, for f32 one key per half-wave and instruction.
// LDS rows are swizzled by 16-byte chunks so that these reads cover the banks.
//
// Bounds and times (us): a long prompt by the matrix instructions and the exponentials, whose
// times add up on a SIMD (8192 tokens, 32/8 heads of 128, 560, 0.98 PFLOP/s; 32/4 heads of 64 321, 0.86);
// a tree over a long cache by the same, its start and the joining of its pieces (64 tokens, 32701 keys,
// 32/8 heads of 128, 59; the matrix work alone 30); short calls by the chain of latencies from the lengths to
// the first keys (one token over 513 keys 7.2, over 11 keys 5.0).
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "lds_dma.hpp"

namespace rq {
namespace {

constexpr int kMaxNodes = 64;
constexpr int kMaxPositions = 0x7fffffff - 1024;  // a sequence's positions rounded up to tiles stay below 2^31
constexpr int64_t kMaxRow = (int64_t)1 << 21;  // elements of a row stride: a tile's offsets stay below 2^31 bytes

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef _Float16 h2_t __attribute__((ext_vector_type(2)));
typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

// v of the other half of the wave (lane l ^ 32) joined to this one's.
__device__ __forceinline__ float max_halves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    const unsigned x = r[0], y = r[1];
    return fmaxf(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y));
}
__device__ __forceinline__ float add_halves(float v) {
    const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    const unsigned x = r[0], y = r[1];
    return __builtin_bit_cast(float, x) + __builtin_bit_cast(float, y);
}

// x / d for 0 <= x < 2^31 by one product: m = ceil(2^(31 + b) / d) with 2^b >= d is off by
// less than 2^b / 2^(31 + b) of 1 / d, so x m / 2^(31 + b) never reaches the next whole number.
struct Div {
    uint32_t m, sh;
    __host__ static Div by(int64_t d) {
        uint32_t b = 0;
        while (((int64_t)1 << b) < d) ++b;
        return {(uint32_t)((((uint64_t)1 << (31 + b)) + (uint64_t)d - 1) / (uint64_t)d), 31 + b};
    }
    __device__ __forceinline__ int operator()(int x) const { return (int)(((uint64_t)(uint32_t)x * m) >> sh); }
};

// Sum and maximum over the wave's 64 lanes of values >= 0.
template <typename F>
__device__ __forceinline__ int wave_join(int v, F f) {
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false));  // lanes 1, 2, 4, 8 before in the row of 16
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false));
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false));
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false));
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false));  // the row before, the half before
    v = f(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false));
    return __builtin_amdgcn_readlane(v, 63);
}
__device__ __forceinline__ int wave_sum(int v) {
    return wave_join(v, [](int a, int b) { return a + b; });
}
__device__ __forceinline__ int wave_max(int v) {
    return wave_join(v, [](int a, int b) { return max(a, b); });
}

// What the kernels read; strides in elements.
struct AttnArgs {
    const void *q, *k, *v;
    void *out;
    const int *starts, *lengths;
    const uint64_t *mask;
    int64_t q_row, out_row;
    int64_t seq_stride, head_stride;  // tree: the cache
    int k_row, v_row;                 // between a head's consecutive keys
    int n_heads, n_kv, n_seqs, capacity, max_nodes;
    int tokens;
    int ranked;   // packed: blocks in order of their work
    int wide;     // packed: row tiles per key/value head between turns of their order
    int splits;   // tree: the most pieces a sequence's keys are cut into
    // splits > 1: sums [splits][n_kv][tokens][heads of one][dim] (a block's rows side by side),
    // then (m, l) [tokens][n_heads][splits]
    float *part;
    float c;      // |scale| log2 e
    int neg;      // scale < 0: q enters negated
    Div by_kv, by_grp, by_seqs, by_rbs, by_wide;  // n_kv, n_heads / n_kv, n_seqs; tree: blocks of a head's rows; packed: wide
};

__device__ __forceinline__ int seq_start(const AttnArgs &a, int s) { return min(max(a.starts[s], 0), a.tokens); }

// The largest s < n_seqs with at(s, starts[s]) <= x (0 if there is none; at
// ascending), and its bounds; x uniform across the wave.  The 64 lanes probe at
// once: one memory round trip up to 63 sequences, one more per factor of 64.
template <typename F>
__device__ __forceinline__ int find_seq(const AttnArgs &a, int x, int *begin, int *end, F at) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = a.n_seqs;  // the answer is in lo .. lo + n - 1
    while (n > 63) {
        const int step = (n + 63) / 64, i = lo + (lane + 1) * step;
        const bool in = (lane + 1) * step < n;
        const int c = __builtin_popcountll(__builtin_amdgcn_ballot_w64(in && at(i, seq_start(a, in ? i : 0)) <= x));
        lo += c * step;
        n = min(step, n - c * step);
    }
    const int v = seq_start(a, lo + min(lane, n));
    const int c = __builtin_popcountll(__builtin_amdgcn_ballot_w64(lane > 0 && lane < n && at(lo + lane, v) <= x));
    *begin = __builtin_amdgcn_readlane(v, c);
    *end = __builtin_amdgcn_readlane(v, c + 1);
    return lo + c;
}

// Of n drafted positions, those that the i-th token of a sequence sees, as bits; word: its mask, where there is one.
__device__ __forceinline__ uint64_t tree_sees(const AttnArgs &a, uint64_t word, int i, int n) {
    const uint64_t all = n > 0 ? ~0ull >> (64 - n) : 0;
    return (a.mask ? word : ~0ull >> (63 - i)) & all;
}

// One sequence of a tree call: its tokens, and the keys cached before and with them.
struct TreeSeq {
    int s0, nodes;      // first token, tokens served
    int before, keys;   // cached positions before them; all positions there are
    __device__ __forceinline__ TreeSeq(const AttnArgs &a, int begin, int end, int length) : s0(begin) {
        nodes = min(max(end - begin, 0), a.max_nodes);
        before = min(max(length, 0), a.capacity);
        keys = before + min(nodes, a.capacity - before);
    }
    // tiles of kt keys per piece, for at most `splits` pieces
    __device__ __forceinline__ int per_piece(int kt, int splits) const {
        const int tiles = (keys + kt - 1) / kt;
        return max(1, (tiles + splits - 1) / splits);
    }
};

template <typename T, int HD, int WR, int KG, bool TREE>
struct Shape {
    static constexpr int NW = WR * KG;
    static constexpr int ROW = HD * (int)sizeof(T), CH = ROW / 16;
    static constexpr int KT = KG == 1 ? 64 : (WR == 4 ? 64 : 32) * KG;  // keys per tile
    static constexpr int TPW = KT / 32 / KG;           // 32-key pieces of it per wave
    static constexpr int TILE = KT * ROW;              // bytes of one operand's tile
    static constexpr int NS = 6 * TILE <= 49152 ? 3 : 2;
};

template <typename T, int HD, int WR, int KG, bool TREE>
__global__ __launch_bounds__(64 * WR * KG, 2) void k_attn(AttnArgs a) {
    using SH = Shape<T, HD, WR, KG, TREE>;
    constexpr bool F16 = sizeof(T) == 2;
    constexpr int NW = SH::NW, ROW = SH::ROW, CH = SH::CH, KT = SH::KT, TPW = SH::TPW, TILE = SH::TILE, NS = SH::NS;
    constexpr int BR = 32 * WR, DT = HD / 32;
    constexpr int KS = F16 ? HD / 16 : HD / 8;  // 16-byte pieces of a row per lane (both halves: 32 bytes)
    constexpr int RPU = 1024 / ROW;             // rows per DMA unit (1 KiB)
    constexpr int UW = TILE / 1024 / NW;        // units per wave and operand
    static_assert(UW >= 1 && TILE % (1024 * NW) == 0, "every wave moves whole units");
    constexpr int RING = NS * 2 * TILE;
    static_assert(KG == 1 || (KG - 1) * WR * DT * 16 * 256 <= RING, "the partial sums reuse the ring");
    __shared__ __attribute__((aligned(1024))) unsigned char lds[RING];
    __shared__ float joined[KG > 1 ? KG : 1][2][KG > 1 ? 32 * WR : 1];

    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wr = wv % WR, kg = wv / WR;
    const int col = lane & 31, hf = lane >> 5;
    const int grp = a.by_kv(a.n_heads), blk = a.by_kv(blockIdx.x), g = blockIdx.x - blk * a.n_kv;

    // the block's sequence, rows and keys
    int s0, nq, r0, nkeys, first = 0, ntiles, pieces = 1, piece = 0, before = 0;
    const char *kb, *vb;  // key 0 of this head
    if constexpr (TREE) {
        const int rbs = (a.max_nodes * grp + BR - 1) / BR, sp = a.by_rbs(blk), rb = blk - sp * rbs;
        piece = a.by_seqs(sp);
        const int s = sp - piece * a.n_seqs;
        int begin = a.starts[s], end = a.starts[s + 1], length = a.lengths[s];
        asm volatile("" : "+s"(begin), "+s"(end), "+s"(length));  // one wait for the three
        const TreeSeq q(a, min(max(begin, 0), a.tokens), min(max(end, 0), a.tokens), length);
        s0 = q.s0;
        nq = q.nodes;
        r0 = rb * BR;
        before = __builtin_amdgcn_readfirstlane(q.before);
        nkeys = q.keys;
        const int per = q.per_piece(KT, a.splits), tiles = (nkeys + KT - 1) / KT;
        pieces = max(1, (tiles + per - 1) / per);
        if (r0 >= nq * grp || piece >= pieces) return;
        first = __builtin_amdgcn_readfirstlane(piece * per);
        ntiles = min(per, tiles - piece * per);
        const int64_t at = (int64_t)s * a.seq_stride + g * a.head_stride;
        kb = static_cast<const char *>(a.k) + at * (int64_t)sizeof(T);
        vb = static_cast<const char *>(a.v) + at * (int64_t)sizeof(T);
    } else {
        int row;
        // every other run of `wide` tiles, as many as the device takes at once, the other way round:
        // a CU which got a heavy one gets a light one next
        const int run = a.by_wide(blk);
        auto turned = [&](int total) { return run & 1 ? run * a.wide + min((run + 1) * a.wide, total) - 1 - blk : blk; };
        if (a.ranked) {
            // row tiles of all sequences (at most 64) by the keys they take, the most first
            const int b0 = seq_start(a, min(lane, a.n_seqs)), b1 = seq_start(a, min(lane + 1, a.n_seqs));
            const int mine = (int)((uint32_t)(max(b1 - b0, 0) * grp + BR - 1) / BR);  // tiles of sequence `lane`
            const int total = wave_sum(mine);
            if (blk >= total) return;
            const int rank = turned(total);
            // its place in its sequence: the last that more than `rank` tiles reach; `above` tiles lie past it
            int lo = 0, hi = wave_max(mine), above = 0;
            while (hi - lo > 1) {
                const int mid = (lo + hi) / 2, c = wave_sum(max(mine - mid, 0));
                if (c > rank) {
                    lo = mid;
                } else {
                    hi = mid;
                    above = c;
                }
            }
            const uint64_t has = __builtin_amdgcn_ballot_w64(mine > lo);
            const int nth = __builtin_amdgcn_mbcnt_hi((uint32_t)(has >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)has, 0));
            const int s = __builtin_ctzll(__builtin_amdgcn_ballot_w64(mine > lo && nth == rank - above));
            s0 = __builtin_amdgcn_readlane(b0, s);
            nq = __builtin_amdgcn_readlane(b1, s) - s0;
            row = lo * BR;
        } else {
            // one sequence after another, its last tile first: sequence s has the indexes from
            // starts[s] grp / BR + s on, at least as many as it needs (tokens grp < 2^31: the grid has fewer than 2^32 threads)
            const int total = a.by_kv(gridDim.x), t = total - 1 - turned(total);
            auto tile0 = [&](int s, int begin) { return (int64_t)begin * grp / BR + s; };
            int end;
            const int s = find_seq(a, t, &s0, &end, tile0);
            nq = max(end - s0, 0);
            row = (int)(t - tile0(s, s0)) * BR;
            if (row < 0 || row >= nq * grp) return;
        }
        // rows are counted from the tile's first token on
        const int skip = a.by_grp(row);
        r0 = row - skip * grp;
        s0 += skip;
        before = skip;  // tokens of the sequence before token 0 of these
        nq -= skip;
        nkeys = before + min(nq, a.by_grp(r0 + BR - 1) + 1);
        // (per lane: where the compiler knows it uniform it keeps 16 more registers through the
        // tiles, and head_dim 128 spills: 8192 tokens 550 -> 620 us)
        asm volatile("" : "+v"(nq));
        ntiles = (nkeys + KT - 1) / KT;
        const int64_t seq = (int64_t)(s0 - skip);
        kb = static_cast<const char *>(a.k) + (seq * a.k_row + g * HD) * (int64_t)sizeof(T);
        vb = static_cast<const char *>(a.v) + (seq * a.v_row + g * HD) * (int64_t)sizeof(T);
    }
    s0 = __builtin_amdgcn_readfirstlane(s0);
    nkeys = __builtin_amdgcn_readfirstlane(nkeys);
    ntiles = __builtin_amdgcn_readfirstlane(ntiles);

    // LDS chunk c of row r holds global chunk c ^ f(r)
    auto fk = [](int r) { return F16 && HD == 64 ? (r >> 1) & 7 : r & 15; };
    auto fv = [](int r) { return F16 ? (HD == 64 ? ((r >> 1) & 1) << 2 : (r & 3) << 2) : ((r >> 2) & 1) << 3; };
    const uint32_t kst = (uint32_t)a.k_row * (uint32_t)sizeof(T), vst = (uint32_t)a.v_row * (uint32_t)sizeof(T);
    uint32_t koff[UW], voff[UW];
#pragma unroll
    for (int u = 0; u < UW; ++u) {
        const int row = (wv * UW + u) * RPU + lane / CH, c = lane % CH;
        koff[u] = (uint32_t)row * kst + (uint32_t)((c ^ fk(row)) * 16);
        voff[u] = (uint32_t)row * vst + (uint32_t)((c ^ fv(row)) * 16);
    }
    const uint32_t lds0 = lds_addr(&lds[0]);
    // tile kt of this block into its ring place; keys past the end read as zero
    auto dma = [&](int kt) {
        const int key0 = (first + kt) * KT;
        const int rows = kt < ntiles ? min(KT, nkeys - key0) : 0;
        const auto rk = make_rsrc_s(kb + (int64_t)key0 * kst, rows > 0 ? (uint32_t)(rows - 1) * kst + ROW : 0u);
        const auto rv = make_rsrc_s(vb + (int64_t)key0 * vst, rows > 0 ? (uint32_t)(rows - 1) * vst + ROW : 0u);
        const uint32_t base = lds0 + (uint32_t)(kt % NS) * (2 * TILE) + (uint32_t)(wv * UW) * 1024u;
#pragma unroll
        for (int u = 0; u < UW; ++u) {
            dma16(rk, base + (uint32_t)u * 1024u, koff[u]);
            dma16(rv, base + (uint32_t)TILE + (uint32_t)u * 1024u, voff[u]);
        }
    };
#pragma unroll
    for (int kt = 0; kt < NS - 1; ++kt) dma(kt);

    // this lane's row
    const int r = r0 + 32 * wr + col, qi = a.by_grp(r), head = g * grp + (r - qi * grp);
    const bool live = qi < nq;
    const uint64_t word = TREE && live && a.mask ? a.mask[s0 + qi] : 0;
    const uint64_t see = TREE && live ? tree_sees(a, word, qi, nkeys - before) : 0;
    // of the wave's rows: the last key any of them sees, and the first that some do not
    const int w_lo = __builtin_amdgcn_readfirstlane(a.by_grp(r0 + 32 * wr));
    const int w_hi = __builtin_amdgcn_readfirstlane(min(a.by_grp(r0 + 32 * wr + 31), nq - 1));
    const bool idle = w_lo >= nq;  // no row at all
    const int key_end = idle ? 0 : TREE ? nkeys : before + w_hi + 1;
    const int masked_from = idle ? 0 : TREE ? before : before + w_lo + 1;
    // bit j: whether this lane's row sees key key0 + j
    auto visible = [&](int key0) -> uint64_t {
        if constexpr (TREE) {
            const int d = before - key0;  // keys of these that are cached positions
            if (d >= 64) return ~0ull;
            if (d >= 0) return (see << d) | ((1ull << d) - 1);
            return d > -64 ? see >> -d : 0;
        } else {
            const int n = before + qi + 1 - key0;
            return n >= 64 ? ~0ull : n > 0 ? (1ull << n) - 1 : 0;
        }
    };

    // (after the first tiles' loads: the wait for Q is then theirs too)
    uint4 qf[KS];
    {
        const char *qp = static_cast<const char *>(a.q) + ((int64_t)(s0 + qi) * a.q_row + head * HD) * (int64_t)sizeof(T);
        const uint32_t flip = a.neg ? (F16 ? 0x80008000u : 0x80000000u) : 0u;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            uint4 v = make_uint4(0, 0, 0, 0);
            if (live) v = *reinterpret_cast<const uint4 *>(qp + 32 * s + 16 * hf);
            qf[s] = make_uint4(v.x ^ flip, v.y ^ flip, v.z ^ flip, v.w ^ flip);
        }
    }

    float mc = -__builtin_inff(), l = 0.0f;  // running maximum (scaled), this lane's share of the sum
    floatx16 o[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] = 0.0f;

    // byte offsets of this lane's reads within its 32-key pieces
    const int kp = 32 * kg * TPW;  // the wave's first key of a tile
    uint32_t ka[KS];
#pragma unroll
    for (int s = 0; s < KS; ++s) ka[s] = (uint32_t)((kp + col) * ROW + (((2 * s + hf) ^ fk(col)) * 16));
    uint32_t va[DT][2];
    if constexpr (F16) {
        // 16 lanes take a block of 4 keys x 16 dims; each gets one dim's 4 keys
        const int i16 = lane & 15;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int row = 4 * hf + i16 / 4 + 8 * e, ch = 4 * d + 2 * ((lane >> 4) & 1) + (i16 & 3) / 2;
                va[d][e] = (uint32_t)((kp + row) * ROW + ((ch ^ fv(row)) * 16) + (i16 & 1) * 8);
            }
    } else {
#pragma unroll
        for (int d = 0; d < DT; ++d)
            va[d][0] = va[d][1] = (uint32_t)((kp + 4 * hf) * ROW + (((8 * d + col / 4) ^ (hf << 3)) * 16) + (col & 3) * 4);
    }
    typedef short short4v __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) short4v lds_short4;
    typedef __attribute__((address_space(3))) const u32x4 lds_u32x4;
    typedef __attribute__((address_space(3))) const float lds_float;
    typedef __attribute__((address_space(3))) const _Float16 lds_half;

    // the first N of the wave's pieces of the tile at LDS address tb, its first key key0
    auto keys = [&](auto masked_c, auto n_c, uint32_t tb, int key0) {
        constexpr bool MASKED = decltype(masked_c)::value;
        constexpr int N = decltype(n_c)::value;
        // one piece at a time: K's, then V's, fragments all read ahead of their products,
        // which otherwise wait for one after another
        constexpr bool AHEAD = N == 1 && (TREE || KG > 1);
        floatx16 sc[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const floatx16 zero = {};
            sc[i] = zero;
            u32x4 kr[AHEAD ? KS : 1];
            if constexpr (AHEAD) {
#pragma unroll
                for (int s = 0; s < KS; ++s) kr[s] = *(lds_u32x4 *)(uintptr_t)(tb + ka[s] + (uint32_t)(i * 32 * ROW));
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                const u32x4 kf = AHEAD ? kr[s] : *(lds_u32x4 *)(uintptr_t)(tb + ka[s] + (uint32_t)(i * 32 * ROW));
                if constexpr (F16) {
                    sc[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, kf),
                                                                   __builtin_bit_cast(half8, qf[s]), sc[i], 0, 0, 0);
                } else {
                    // (whole vectors: a bit_cast of one element would read element 0)
                    const floatx4 kv = __builtin_bit_cast(floatx4, kf), qv = __builtin_bit_cast(floatx4, qf[s]);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        sc[i] = __builtin_amdgcn_mfma_f32_32x32x2f32(kv[e], qv[e], sc[i], 0, 0, 0);
                }
            }
        }
        const uint64_t sees = MASKED ? visible(key0) : 0;
        if constexpr (MASKED) {
            const uint64_t mine = sees >> (4 * hf);
            const int upto = before + qi + 1 - key0 - 4 * hf;
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    const int j = 32 * i + 8 * (e >> 2) + (e & 3);
                    sc[i][e] = (TREE ? mine >> j & 1 : j < upto) ? sc[i][e] : -__builtin_inff();
                }
        }
        float mt = sc[0][0];
#pragma unroll
        for (int i = 0; i < N; ++i)
#pragma unroll
            for (int e = 0; e < 16; ++e) mt = fmaxf(mt, sc[i][e]);
        mt = max_halves(mt) * a.c;
        // The maximum may lag by 6 (weights up to 2^6): a row's sums are then
        // rescaled a few times in all, not in most tiles.
        const bool rose = mt > mc + 6.0f;
        if (__builtin_amdgcn_ballot_w64(rose)) {
            const float alpha = rose ? __builtin_amdgcn_exp2f(mc - mt) : 1.0f;
            mc = rose ? mt : mc;
            l *= alpha;
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) o[d][e] *= alpha;
        }
        const float off = mc == -__builtin_inff() ? 0.0f : -mc;  // no key yet: every weight is 2^-inf
#pragma unroll
        for (int i = 0; i < N; ++i) {
            float t[4];
#pragma unroll
            for (int e = 0; e < 16; ++e) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i][e], a.c, off));
                sc[i][e] = p;
                t[e & 3] = e < 4 ? p : t[e & 3] + p;
            }
            l += (t[0] + t[1]) + (t[2] + t[3]);
        }
        const uint32_t vt = tb + TILE;
        if constexpr (MASKED) {
            // A value that is not finite must not meet the zero weight of a
            // row that does not see its key: such a piece is summed by element.
            float z = 0.0f;
            h2_t z2 = {(_Float16)0.0f, (_Float16)0.0f};
#pragma unroll
            for (int u = 0; u < N * 32 * ROW / 1024; ++u) {
                const u32x4 x = *(lds_u32x4 *)(uintptr_t)(vt + (uint32_t)(kp * ROW + u * 1024 + lane * 16));
                const uint32_t xw[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if constexpr (F16)
                        z2 = __builtin_elementwise_fma(__builtin_bit_cast(h2_t, xw[e]), (h2_t){(_Float16)0.0f, (_Float16)0.0f}, z2);
                    else
                        z = __builtin_fmaf(__builtin_bit_cast(float, xw[e]), 0.0f, z);
                }
            }
            if constexpr (F16) z = (float)z2.x + (float)z2.y;
            if (__builtin_amdgcn_ballot_w64(z != z)) {
                for (int kk = 0; kk < 32 * N; ++kk) {
                    float p = 0.0f;
#pragma unroll
                    for (int i = 0; i < N; ++i)
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            p = kk / 32 == i && 4 * (kk % 32 / 8) + kk % 4 == e ? sc[i][e] : p;
                    p = __shfl(p, col + 32 * (kk / 4 % 2));
                    if constexpr (F16) p = (float)(_Float16)p;
                    const bool seen = sees >> kk & 1;
#pragma unroll
                    for (int d = 0; d < DT; ++d)
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const int dim = 32 * d + 8 * (e >> 2) + 4 * hf + (e & 3), row = kp + kk;
                            const uint32_t at = vt + (uint32_t)(row * ROW) +
                                                (uint32_t)(((dim * (int)sizeof(T) / 16) ^ fv(row)) * 16) +
                                                (uint32_t)(dim * (int)sizeof(T) % 16);
                            float x;
                            if constexpr (F16) x = (float)*(lds_half *)(uintptr_t)at;
                            else x = *(lds_float *)(uintptr_t)at;
                            o[d][e] = seen ? __builtin_fmaf(p, x, o[d][e]) : o[d][e];
                        }
                }
                return;
            }
        }
        if constexpr (F16) {
            half8 pf[N][2];
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int e = 0; e < 16; ++e) pf[i][e >> 3][e & 7] = (_Float16)sc[i][e];
            auto read = [&](int d, int i, int s2) {
                lds_short4 *pa = (lds_short4 *)(uintptr_t)(vt + va[d][0]), *pb = (lds_short4 *)(uintptr_t)(vt + va[d][1]);
                const uint2 ua =
                    __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(pa + (2 * i + s2) * 16 * ROW / 8));
                const uint2 ub =
                    __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(pb + (2 * i + s2) * 16 * ROW / 8));
                return __builtin_bit_cast(half8, make_uint4(ua.x, ua.y, ub.x, ub.y));
            };
            constexpr int DR = AHEAD ? DT : 1;  // dimensions read at once
#pragma unroll
            for (int d0 = 0; d0 < DT; d0 += DR) {
                half8 vr[DR][N][2];
                if constexpr (AHEAD || TREE) {
#pragma unroll
                    for (int d = 0; d < DR; ++d)
#pragma unroll
                        for (int i = 0; i < N; ++i)
#pragma unroll
                            for (int s2 = 0; s2 < 2; ++s2) vr[d][i][s2] = read(d0 + d, i, s2);
                    if constexpr (AHEAD) __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
                for (int d = 0; d < DR; ++d)
#pragma unroll
                    for (int i = 0; i < N; ++i)
#pragma unroll
                        for (int s2 = 0; s2 < 2; ++s2)
                            o[d0 + d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
                                AHEAD || TREE ? vr[d][i][s2] : read(d0 + d, i, s2), pf[i][s2], o[d0 + d], 0, 0, 0);
            }
        } else {
            // V's values of 8 keys at a time, all read before the first is used: one by
            // one, each instruction waited for its own
#pragma unroll
            for (int i = 0; i < N; ++i)
#pragma unroll
                for (int e8 = 0; e8 < 16; e8 += 8) {
                    float x[8][DT];
#pragma unroll
                    for (int e = 0; e < 8; ++e)
#pragma unroll
                        for (int d = 0; d < DT; ++d)
                            x[e][d] = *(lds_float *)(uintptr_t)(vt + va[d][0] +
                                                                (uint32_t)((32 * i + 8 * ((e8 + e) >> 2) + (e & 3)) * ROW));
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int e = 0; e < 8; ++e)
#pragma unroll
                        for (int d = 0; d < DT; ++d)
                            o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e][d], sc[i][e8 + e], o[d], 0, 0, 0);
                }
        }
    };
    for (int kt = 0; kt < ntiles; ++kt) {
        // tile kt has landed, and every wave is done with the one whose place the next takes
        wait_vmcnt<(NS - 2) * 2 * UW>();
        __syncthreads();
        dma(kt + NS - 1);
        const int key0 = (first + kt) * KT + kp;
        const uint32_t tb = lds0 + (uint32_t)(kt % NS) * (2 * TILE);
        using All = std::integral_constant<int, TPW>;
        using One = std::integral_constant<int, 1>;
        if (key0 + 32 * TPW <= masked_from) {
            keys(std::false_type{}, All{}, tb, key0);
        } else if constexpr (TREE && TPW > 1) {
            // (few tiles: one piece at a time, in the registers that the others leave)
#pragma unroll 1
            for (int i = 0; i < TPW && key0 + 32 * i < key_end; ++i)
                keys(std::true_type{}, One{}, tb + (uint32_t)(i * 32 * ROW), key0 + 32 * i);
        }
        else if (key0 + 32 * (TPW - 1) < key_end) keys(std::true_type{}, All{}, tb, key0);
        else if (key0 < key_end) keys(std::true_type{}, One{}, tb, key0);
    }
    wait_vmcnt<0>();  // no DMA in flight past this point

    l = add_halves(l);
    if constexpr (KG > 1) {
        // the key groups' sums through the ring
        float *co = reinterpret_cast<float *>(lds);
        __syncthreads();  // every wave is done with it
        if (kg > 0) {
            if (hf == 0) {
                joined[kg][0][32 * wr + col] = mc;
                joined[kg][1][32 * wr + col] = l;
            }
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e) co[((((kg - 1) * WR + wr) * DT + d) * 16 + e) * 64 + lane] = o[d][e];
        }
        __syncthreads();
        if (kg > 0) return;
        float top = mc;
#pragma unroll
        for (int w = 1; w < KG; ++w) top = fmaxf(top, joined[w][0][32 * wr + col]);
        const float base = top == -__builtin_inff() ? 0.0f : top;
        const float w0 = __builtin_amdgcn_exp2f(mc - base);
        l *= w0;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] *= w0;
#pragma unroll
        for (int w = 1; w < KG; ++w) {
            const float ww = __builtin_amdgcn_exp2f(joined[w][0][32 * wr + col] - base);
            l = __builtin_fmaf(ww, joined[w][1][32 * wr + col], l);
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int e = 0; e < 16; ++e)
                    o[d][e] = __builtin_fmaf(ww, co[((((w - 1) * WR + wr) * DT + d) * 16 + e) * 64 + lane], o[d][e]);
        }
        mc = top;
    }
    if (TREE && pieces > 1) {
        if (!live) return;
        const int64_t slot = ((int64_t)(s0 + qi) * a.n_heads + head) * a.splits + piece;
        float *po = a.part + (((int64_t)piece * a.n_kv + g) * a.tokens * grp + (int64_t)(s0 + qi) * grp + (r - qi * grp)) * HD;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e4 = 0; e4 < 4; ++e4)
                *reinterpret_cast<float4 *>(po + 32 * d + 8 * e4 + 4 * hf) =
                    make_float4(o[d][4 * e4], o[d][4 * e4 + 1], o[d][4 * e4 + 2], o[d][4 * e4 + 3]);
        if (hf == 0)
            reinterpret_cast<float2 *>(a.part + (int64_t)a.tokens * a.n_heads * a.splits * HD)[slot] = make_float2(mc, l);
        return;
    }
    const bool none = TREE && before == 0 && see == 0;
    const float inv = none ? 0.0f : 1.0f / l;
    typedef T vec4 __attribute__((ext_vector_type(4)));
    auto four = [&](int d, int e4) {
        vec4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (T)(none ? 0.0f : o[d][4 * e4 + e] * inv);
        return v;
    };
    if constexpr (KG > 1) {
        // few rows: as they lie
        if (!live) return;
        T *op = static_cast<T *>(a.out) + (int64_t)(s0 + qi) * a.out_row + head * HD;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e4 = 0; e4 < 4; ++e4) *reinterpret_cast<vec4 *>(op + 32 * d + 8 * e4 + 4 * hf) = four(d, e4);
    } else {
        // Through the ring: whole rows side by side instead of four values of each of 32
        // (32 prompts of 100 tokens, 32/8 heads of 128, 27.4 -> 25.3 us).
        __syncthreads();  // every wave is done with the ring
        unsigned char *ol = lds + wr * 32 * ROW;
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
            for (int e4 = 0; e4 < 4; ++e4) {
                const int at = (32 * d + 8 * e4 + 4 * hf) * (int)sizeof(T);  // chunk c of row r at c ^ (r % 8)
                *reinterpret_cast<vec4 *>(ol + col * ROW + (((at / 16) ^ (col & 7)) * 16) + at % 16) = four(d, e4);
            }
        wait_lgkm0();  // (also keeps the reads below behind)
        constexpr int RPI = 64 / CH;  // rows per store
#pragma unroll
        for (int i = 0; i < 32 / RPI; ++i) {
            const int ro = i * RPI + lane / CH, c = lane % CH, rr = r0 + 32 * wr + ro, q2 = a.by_grp(rr);
            if (q2 >= nq) continue;
            const uint4 v = *reinterpret_cast<const uint4 *>(ol + ro * ROW + (c ^ (ro & 7)) * 16);
            T *op = static_cast<T *>(a.out) + (int64_t)(s0 + q2) * a.out_row + (g * grp + (rr - q2 * grp)) * HD;
            *reinterpret_cast<uint4 *>(reinterpret_cast<unsigned char *>(op) + c * 16) = v;
        }
    }
}

// Joins the pieces of rows whose keys were cut: one wave per (token, head).
// Such a sequence has cached positions, which every row sees: drafted keys alone are one tile.
template <typename T, int HD, int KT>
__global__ __launch_bounds__(256) void k_attn_join(AttnArgs a) {
    static_assert(KT >= kMaxNodes, "a cut sequence has cached positions");
    constexpr int L = HD / 4, G = 64 / L, U = 8;  // pieces added at once, 16 bytes a lane; read ahead of use
    const int64_t row = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (row >= (int64_t)a.tokens * a.n_heads) return;
    const int t = (int)(row / a.n_heads), head = (int)(row - (int64_t)t * a.n_heads), lane = threadIdx.x & 63;
    const int grp = a.by_kv(a.n_heads), g = a.by_grp(head), gi = lane / L, at = 4 * (lane % L);
    const int64_t step = (int64_t)a.tokens * a.n_heads * HD;  // between pieces
    const float *po = a.part + (((int64_t)g * a.tokens + t) * grp + head - g * grp) * HD + at;
    const float2 *ml = reinterpret_cast<const float2 *>(a.part + (int64_t)a.tokens * a.n_heads * a.splits * HD) + row * a.splits;
    // lane p has piece p's weight (at most 64 pieces).  It and the first pieces' sums are
    // read before it is known how many there are; those past the last go unused.
    const float2 raw = ml[min(lane, a.splits - 1)];
    float4 v[U];
#pragma unroll
    for (int u = 0; u < U; ++u) v[u] = *reinterpret_cast<const float4 *>(po + min(gi + u * G, a.splits - 1) * step);
    int begin, end;
    const int s = find_seq(a, t, &begin, &end, [](int, int at) { return at; });
    const TreeSeq q(a, begin, end, a.lengths[s]);
    const int i = t - q.s0;
    if (i < 0 || i >= q.nodes) return;
    const int per = q.per_piece(KT, a.splits), tiles = (q.keys + KT - 1) / KT;
    const int pieces = (tiles + per - 1) / per;
    if (pieces <= 1) return;  // written by the block that had them all
    const float2 mine = lane < pieces ? raw : make_float2(-__builtin_inff(), 0.0f);
    float top = mine.x;
#pragma unroll
    for (int w = 32; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor(top, w));
    const float base = top == -__builtin_inff() ? 0.0f : top;
    const float wt = __builtin_amdgcn_exp2f(mine.x - base);
    float l = wt * mine.y, o[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int w = 32; w > 0; w >>= 1) l += __shfl_xor(l, w);
    for (int p0 = 0; p0 < pieces; p0 += U * G) {
        if (p0 > 0) {
#pragma unroll
            for (int u = 0; u < U; ++u)
                v[u] = *reinterpret_cast<const float4 *>(po + min(p0 + gi + u * G, pieces - 1) * step);
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int p = p0 + gi + u * G;
            const bool in = p < pieces;
            const float w = __shfl(wt, in ? p : 0);
            if (in) {
                o[0] = __builtin_fmaf(w, v[u].x, o[0]);
                o[1] = __builtin_fmaf(w, v[u].y, o[1]);
                o[2] = __builtin_fmaf(w, v[u].z, o[2]);
                o[3] = __builtin_fmaf(w, v[u].w, o[3]);
            }
        }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int w = 32; w >= L; w >>= 1) o[e] += __shfl_xor(o[e], w);
    if (gi != 0) return;
    typedef T vec4 __attribute__((ext_vector_type(4)));
    vec4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (T)(o[e] / l);
    *reinterpret_cast<vec4 *>(static_cast<T *>(a.out) + (int64_t)t * a.out_row + head * HD + at) = y;
}

// Launches k_attn<T, HD, WR, KG, TREE> with BR = 32 WR rows per block.
template <typename T, int HD, int WR, int KG, bool TREE>
int launch(AttnArgs a, hipStream_t s) {
    using SH = Shape<T, HD, WR, KG, TREE>;
    const int64_t grp = a.n_heads / a.n_kv, br = 32 * WR;
    a.by_kv = Div::by(a.n_kv);
    a.by_grp = Div::by(grp);
    a.by_seqs = Div::by(a.n_seqs);
    a.by_wide = Div::by(TREE ? 1 : a.wide);
    a.by_rbs = Div::by(TREE ? cdiv(a.max_nodes * grp, br) : 1);
    const int64_t tiles = TREE ? cdiv(a.max_nodes * grp, br) * a.n_seqs * a.splits : (int64_t)a.tokens * grp / br + a.n_seqs;
    if (!grid_ok(tiles * a.n_kv, 64 * SH::NW)) return fail(RQ_ERR_SHAPE, "too many rows for one call");
    hipLaunchKernelGGL((k_attn<T, HD, WR, KG, TREE>), dim3((unsigned)(tiles * a.n_kv)), dim3(64 * SH::NW), 0, s, a);
    RQ_LAUNCH_CHECK();
    if (TREE && a.splits > 1) {
        const int64_t blocks = cdiv((int64_t)a.tokens * a.n_heads, 4);
        if (!grid_ok(blocks, 256)) return fail(RQ_ERR_SHAPE, "too many rows for one call");
        hipLaunchKernelGGL((k_attn_join<T, HD, SH::KT>), dim3((unsigned)blocks), dim3(256), 0, s, a);
        RQ_LAUNCH_CHECK();
    }
    return RQ_OK;
}

// Rows per block: 64 where blocks of 128 would leave CUs without work, or are the tiles of one long prompt,
// in f32, whose blocks take longer, without two blocks (us, 128 rows / 64: one prompt of 300
// tokens, 32/4 heads of 64, 8.0 / 7.2, of 1200 21.8 / 18.2, of 2048 36.4 / 33.8, of 3000 57.8 / 60.9, three
// of 700, 800 and 500 18.3 / 20.5, one of 8192 with 32/8 heads of 128 557 / 641; f32, three of 417, 1000
// and 83 87 / 59, one of 2048 158 / 166).
// Blocks are ranked by their work where some have to wait for others and the sequences
// fit a wave's lanes (9 prompts of 1 to 1047 tokens, 32/4 heads of 64, in the order of the tokens
// 31.4, ranked 28 when this was chosen, 26 to 27 now; in one round of blocks the search only costs, 5 prompts of 1 to 64 4.9 / 5.2).
// Every other run of them is turned round in f32 only (one prompt of 2048 158, in order 206; fp16 560 / 545
// for 8192 tokens).
template <typename T, int HD>
int launch_packed(AttnArgs a, int cus, hipStream_t s) {
    constexpr bool F16 = sizeof(T) == 2;
    const int64_t blocks = cdiv((int64_t)a.tokens * a.n_heads, 128);
    const bool half = blocks < (F16 ? 1 : 2) * cus || (F16 && a.n_seqs == 1 && blocks <= 2 * cus);
    a.wide = F16 ? 1 << 30 : std::max(1, cus / a.n_kv);
    a.ranked = a.n_seqs > 1 && a.n_seqs <= 64 && (half ? 2 : 1) * blocks > cus;
    return half ? launch<T, HD, 2, 2, false>(a, s) : launch<T, HD, 4, 1, false>(a, s);
}

// How a tree call is cut: blocks of 32 wr rows and kg groups of keys, the keys of a
// sequence into at most `splits` pieces, for about kCus blocks at work.  Joining pieces
// costs a launch and the sums' way to memory and back, so keys are cut only as
// long as there are too few blocks without (us; rows: of a key/value head):
//   rows <= 32, tiles of 128 keys: one token, 513 keys, 7.9 whole, 8.9 in 4 pieces.
//   enough blocks of 128 rows: whole; 16 trees of 64 over 1500 keys, 32/8 heads of 128, 4x2 41.5,
//     2x4 55.5; 32 of them 4x1 72, 4x2 83.
//   enough of 64 rows, or half of that and a short cache: whole, 2x4; 8 of these trees 29.5, 4x2 in 2 pieces 36.9; 4 of them 25.6, 26.2 in 4.
//   few: 64 rows, 2x2, a long axis 128 rows, 4x2, for half the bytes of sums; 2 trees of 32
//     2x2 in 8 13.6, 4x2 in 16 17.4; one of 64 over 32701 keys 4x2 in 16 55, 2x2 in 16 62, 2x4 in 8 62.
//   f32, whose blocks are matrix-bound: 4x1 where there are enough, else 2x2 (4 sequences of up to 1501 keys
//     2x2 in 8 17.0, 4x1 in 16 18.6).
constexpr int64_t kCus = 256;
struct TreeShape {
    int wr, kg, splits;
};
TreeShape tree_shape(int64_t n_seqs, int64_t n_kv, int64_t rows, int64_t capacity, bool f16) {
    const int64_t heads = std::max<int64_t>(n_seqs * n_kv, 1), t64 = cdiv(capacity, 64), t128 = cdiv(capacity, 128);
    auto cut = [](int64_t blocks, int64_t tiles) {
        return (int)std::max<int64_t>(1, std::min<int64_t>({kCus / blocks, tiles, 64}));
    };
    if (rows <= 32) {
        if (f16) return {1, 4, t128 <= 5 ? 1 : cut(heads, t128)};
        return {1, 2, cut(heads, t64)};
    }
    const int64_t r64 = heads * cdiv(rows, 64), r128 = heads * cdiv(rows, 128);
    if (!f16) {
        if (rows > 64 && r128 >= kCus) return {4, 1, 1};
        return {2, 2, cut(r64, t64)};
    }
    if (rows > 64 && r128 >= kCus) return {4, r128 >= 2 * kCus ? 1 : 2, 1};
    if (r64 >= 2 * kCus) return {2, 2, 1};
    if (r64 >= kCus || (2 * r64 >= kCus && t64 <= 40)) return {2, 4, 1};
    const int few = t64 <= 5 ? 1 : cut(r64, cdiv(t64, 2));
    if (rows <= 64 || t64 < 8 * few) return {2, 2, few};
    return {4, 2, cut(r128, t128)};
}

template <typename T, int HD>
int launch_tree(const AttnArgs &a, hipStream_t s) {
    constexpr bool F16 = sizeof(T) == 2;
    const TreeShape sh = tree_shape(a.n_seqs, a.n_kv, (int64_t)a.max_nodes * (a.n_heads / a.n_kv), a.capacity, F16);
    if (sh.wr == 2) {
        if constexpr (F16)
            if (sh.kg == 4) return launch<T, HD, 2, 4, true>(a, s);
        return launch<T, HD, 2, 2, true>(a, s);
    }
    if (sh.wr == 4) {
        if constexpr (F16)
            if (sh.kg == 2) return launch<T, HD, 4, 2, true>(a, s);
        return launch<T, HD, 4, 1, true>(a, s);
    }
    return launch<T, HD, 1, F16 ? 4 : 2, true>(a, s);
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
    const int64_t unit = at->dtype == RQ_F16 ? 8 : 4;
    const int64_t qr = at->q_row ? at->q_row : qw, kr = at->k_row ? at->k_row : kw, vr = at->v_row ? at->v_row : kw,
                  orow = at->out_row ? at->out_row : qw;
    if (qr < qw || orow < qw || kr < kw || vr < kw || qr > kMaxRow || orow > kMaxRow || kr > kMaxRow || vr > kMaxRow)
        return fail(RQ_ERR_SHAPE, "row strides must hold a row and be at most 2^21 elements");
    if (qr % unit || orow % unit || kr % unit || vr % unit)
        return fail(RQ_ERR_UNSUPPORTED, "row strides must be multiples of 16 bytes");
    a.q_row = qr;
    a.out_row = orow;
    a.k_row = (int)kr;
    a.v_row = (int)vr;
    a.n_heads = at->n_heads;
    a.n_kv = at->n_kv_heads;
    a.tokens = (int)tokens;
    const float scale = at->scale != 0.0f ? at->scale : 1.0f / sqrtf((float)at->head_dim);
    a.neg = scale < 0.0f;
    // (not below the normal numbers: a hidden key's -inf times c stays -inf)
    a.c = (float)std::min(std::max(fabs((double)scale) * 1.4426950408889634, 1.2e-38), 3.4e38);
    a.splits = 1;
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
    if (cache->capacity > kMaxPositions) return fail(RQ_ERR_SHAPE, "capacity %d above %d", cache->capacity, kMaxPositions);
    const int64_t hd = attn->head_dim, unit = attn->dtype == RQ_F16 ? 8 : 4, most = (int64_t)1 << 40;
    a.seq_stride = cache->seq_stride;
    a.head_stride = cache->head_stride;
    int64_t pos = cache->pos_stride;
    if (a.seq_stride == 0 && a.head_stride == 0 && pos == 0) {
        pos = hd;
        a.head_stride = hd * cache->capacity;
        a.seq_stride = a.head_stride * a.n_kv;
    }
    // (a stride that is never taken, of one head or one sequence, may be 0)
    if (a.head_stride < 0 || a.seq_stride < 0 || pos > kMaxRow || pos < 0 || a.head_stride > most ||
        a.seq_stride > most ||
        (cache->capacity > 0 && (pos < hd || (a.n_kv > 1 && a.head_stride < hd) ||
                                 (cache->n_seqs > 1 && a.seq_stride < hd))))
        return fail(RQ_ERR_SHAPE, "cache strides shorter than a row or out of range");
    if (pos % unit || a.head_stride % unit || a.seq_stride % unit)
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
    a.k_row = a.v_row = (int)pos;
    a.splits = tree_shape(cache->n_seqs, a.n_kv, (int64_t)max_nodes * (a.n_heads / a.n_kv), cache->capacity,
                          attn->dtype == RQ_F16)
                   .splits;
    a.part = static_cast<float *>(workspace);
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
    hipStream_t s = pick(ctx, stream);
    const int cus = ctx->num_cus;
    if (attn->dtype == RQ_F16)
        return attn->head_dim == 64 ? launch_packed<_Float16, 64>(a, cus, s) : launch_packed<_Float16, 128>(a, cus, s);
    return attn->head_dim == 64 ? launch_packed<float, 64>(a, cus, s) : launch_packed<float, 128>(a, cus, s);
}

size_t rq_attn_tree_workspace(const rq_attn *attn, int32_t n_seqs, int64_t tokens, int32_t max_nodes,
                              int32_t capacity) {
    AttnArgs a{};
    if (n_seqs < 1 || tokens < 1 || max_nodes < 1 || max_nodes > kMaxNodes || capacity < 0 || capacity > kMaxPositions ||
        check_attn(attn, tokens, a) != RQ_OK)
        return 0;
    const int splits = tree_shape(n_seqs, a.n_kv, (int64_t)max_nodes * (a.n_heads / a.n_kv), capacity,
                                  attn->dtype == RQ_F16)
                           .splits;
    const size_t rows = (size_t)tokens * (size_t)a.n_heads * (size_t)splits;
    return splits > 1 ? (rows * ((size_t)attn->head_dim * 4 + 8) + 15) / 16 * 16 : 0;
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
    hipStream_t s = pick(ctx, stream);
    if (attn->dtype == RQ_F16)
        return attn->head_dim == 64 ? launch_tree<_Float16, 64>(a, s) : launch_tree<_Float16, 128>(a, s);
    return attn->head_dim == 64 ? launch_tree<float, 64>(a, s) : launch_tree<float, 128>(a, s);
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
