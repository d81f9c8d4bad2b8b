// Attention of one new token per sequence over a paged KV cache (rq_attn_paged).
//
//   out[s, h] = sum_j p_j v[j] / sum_j p_j,  p_j = 2^(c q.k_j - m),  c = scale log2 e
//
// in one pass over the keys with a running maximum m.  K and V are read once, so
// the bound is their way from memory; the matrix instructions only have to keep up.  For the products with fp16 V
// the weights p are two fp16 terms (off by 2^-22 of each: 2.0e-4 rms of the output, its own rounding); m, sums and
// accumulators are f32.
//
// The query heads of a key/value head are the 16 columns of a matrix
// instruction (more heads: more blocks), so one pass serves them all:
// S^T = K . Q^T, then O^T = V^T . P^T takes P as it stands in the lanes, V^T in the
// key order that gives -- for fp16 by transposing LDS reads, for f32 one
// key per quarter wave and instruction.
//
// Work is cut by its amount, not by sequence: the keys of all sequences in
// units of KT (a sequence has at least one), laid one behind another, are dealt
// out in equal runs to as many blocks as the device holds at once, so a batch of one
// long and many short sequences fills it.  The lengths are on the device, so
// every block finds its run from them (a wave scans them).  A block deals the parts
// of its run, one sequence each, to its eight waves, which join through LDS; a
// sequence that several blocks have parts of is joined by the one that arrives
// last (the context's counters, on its own stream), or by a launch of its own.
//
// Each wave streams its units through a place of its own in LDS (DMA, no block
// barrier needed), K's next unit under way as soon as K has been read, V's as V
// has.  The pages' entries lie in a wave's lanes, 64 at a time; the rows of a DMA
// instruction share a page and their address is formed on the scalar unit, but for pages
// smaller than that.
//
// Times (us; the bytes at the rate of a plain read of as much, 6.9 TB/s): six sequences
// of up to 32701 keys, 32/8 heads of 128, 68 (55); f32, seven of up to 3001, 16/16 heads of 128, 26
// (16); 48 chats of 37 to 2047 keys, 32/4 heads of 64, 12.5 (3.6); one of 513 7.5.  What is left is
// latency: about 1 us each for the launch, the lengths, a page's entry, the first keys, and 3 for a join (the
// stores' acknowledgement, the counter, the pieces); that blocks of one size are not done at one time (the
// first of six long sequences' at 50 us, the last at 61); and that short batches are not dealt evenly (the 48 chats' 765
// units to 61 of 128 runs, 3 to 30 each).  Loads that leave the caches alone (nt) took 10 % off the
// long calls, one block of eight waves per CU over two of four 2 %, waves in step (s_barrier) 3 %.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "lds_dma.hpp"
#include "paged.hpp"

namespace rq {
namespace {

typedef _Float16 half8 __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));

constexpr int64_t kCus = 256;
constexpr int kMaxSeqs = 65536;  // (every block scans the lengths)
constexpr int kCounterStride = 32;  // of the context's arrival counters, a line each

struct PagedArgs {
    const char *q;
    char *out;
    const int *lengths;
    int64_t q_row, out_row;  // bytes
    Pages pages;
    int n_heads, n_kv, grp, rbs;  // grp: query heads of a key/value head, in rbs blocks of 16
    int runs;                     // blocks that the units are dealt to
    float *part;                  // sums [2 runs][n_heads][dim], then (m, l) [2 runs][n_heads]
    int *counters;                // a cut sequence's arrived pieces, zero between launches; null: k_paged_join joins
    float c;                      // |scale| log2 e
    int neg;                      // scale < 0
    Div by_runs;
};

constexpr int NW = 8;  // waves per block
constexpr int TH = 64 * NW;
// Blocks per CU that the rings (8 or 16 KiB a wave) leave room for.
constexpr int blocks_per_cu(int hd) { return hd == 64 ? 2 : 1; }

template <typename T, int HD>
struct PShape {
    static constexpr bool F16 = sizeof(T) == 2;
    static constexpr int KT = F16 ? 32 : 16;          // keys per unit
    static constexpr int ROW = HD * (int)sizeof(T), CH = ROW / 16;
    static constexpr int TILE = KT * ROW;             // bytes of K or V of a unit
    static constexpr int RPU = 1024 / ROW, UN = TILE / 1024;  // rows per DMA instruction, instructions
    static constexpr int RING = 2 * TILE;             // of a wave
    static constexpr int L = HD / 4;                  // lanes of a row of sums
    static constexpr int PAD = HD + 4;                // floats between rows of the joined sums
    static_assert(16 * PAD * 4 <= RING, "the partial sums reuse the ring");
};

// v of lanes l, l ^ 16, l ^ 32, l ^ 48 joined.
template <typename F>
__device__ __forceinline__ float join4(float v, F f) {
    const auto a = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    const unsigned a0 = a[0], a1 = a[1];
    v = f(__builtin_bit_cast(float, a0), __builtin_bit_cast(float, a1));
    const auto b = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
    const unsigned b0 = b[0], b1 = b[1];
    return f(__builtin_bit_cast(float, b0), __builtin_bit_cast(float, b1));
}

__device__ __forceinline__ int clamped(const PagedArgs &a, int s) { return min(max(a.lengths[s], 0), a.pages.capacity()); }
template <int KT>
__device__ __forceinline__ int units_of(int length) {
    return max(1, (int)(((unsigned)length + KT - 1) / KT));
}

__device__ __forceinline__ int scan_add(int v) {  // inclusive, over the wave
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xF, 0xF, false);  // lanes 1, 2, 4, 8 before in the row of 16
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xF, 0xF, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xA, 0xF, false);  // the row before, the half before
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xC, 0xF, false);
    return v;
}

// A run's units: an equal share, at least 12; and a sequence of up to so many units is not cut, the run
// that it begins in has all of it.  Shorter runs and more cuts cost joining, longer ones the waves' turns (us, weights in one
// term, 48 chats of 37 to 2047 keys, 32/4 heads of 64 / one sequence of 513: at least 8, all cut 12.9 / 7.9, up to 16
// whole 12.6 / 7.9; 12, up to 24 whole 12.5 / 7.3; 24, up to 24 whole 14.2 / 7.1).
__device__ __forceinline__ int run_length(const PagedArgs &a, int total) { return max(12, a.by_runs(total + a.runs - 1)); }
__device__ __forceinline__ int whole_units(int len) { return min(2 * len, 24); }

// Where a run lies: the units of all sequences, of a run, its own x0 .. x1 - 1, and 64 (`held`) sequences
// from `base` on, lane l's units begin .. end - 1 and its length; the run's first unit is among them.
// Whole wave, `run` uniform.  Up to 64 sequences take one trip for the lengths, one more per factor of 64.
template <typename T, int HD>
struct Where {
    static constexpr int KT = PShape<T, HD>::KT;
    int total, len, x0, x1;
    int base, held, length, begin, end;
    bool none;  // the run is past all units
    __device__ __forceinline__ Where(const PagedArgs &a, int run) {
        const int lane = threadIdx.x & 63;
        int lo = 0, n = a.pages.n_seqs, t0 = 0;  // in sequences lo .. lo + n - 1, whose units begin at t0
        for (bool first = true;; first = false) {
            const int m = (n + 63) / 64;  // sequences of a lane
            int u = 0;
            length = 0;
            for (int j = 0; j < m; ++j) {
                const int i = lane * m + j;
                if (i < n) {
                    length = clamped(a, lo + i);
                    u += units_of<KT>(length);
                }
            }
            const int upto = scan_add(u);
            if (first) {
                total = __builtin_amdgcn_readlane(upto, 63);
                len = run_length(a, total);
                const int64_t x = (int64_t)run * len;
                none = x >= total;
                if (none) return;
                x0 = (int)x;
                x1 = x0 + min(len, total - x0);
            }
            begin = t0 + upto - u;
            end = t0 + upto;
            if (m == 1) break;
            const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(end > x0) | 1ull << 63);
            t0 = __builtin_amdgcn_readlane(begin, l);
            lo += l * m;
            n = min(m, n - l * m);
        }
        base = lo;
        held = n;
    }
    // The 64 sequences from the one whose units begin at x on, the next after those held.
    __device__ __forceinline__ void next(const PagedArgs &a, int x) {
        const int lane = threadIdx.x & 63;
        base += held;
        held = min(64, a.pages.n_seqs - base);
        length = lane < held ? clamped(a, base + lane) : 0;
        const int u = lane < held ? units_of<KT>(length) : 0;
        end = x + scan_add(u);
        begin = end - u;
    }
};

// Device-coherent stores and loads (sc1): the blocks of a sequence may sit on different XCDs.
__device__ __forceinline__ void store_part(__amdgpu_buffer_rsrc_t r, uint32_t at, floatx4 v) {
    __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u32x4, v), r, at, 0, 16);
}

// Pieces of one row joined: their maximum, sum, and 4 dims of their sums.
struct Joined {
    float top = -__builtin_inff(), l = 0.0f;
    floatx4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    // The maximum rises to t: returns what new pieces' maxima are taken relative to.
    __device__ __forceinline__ float rise(float t) {
        t = fmaxf(top, t);
        const float base = t == -__builtin_inff() ? 0.0f : t, w = __builtin_amdgcn_exp2f(top - base);
        top = t;
        l *= w;
        o *= w;
        return base;
    }
    __device__ __forceinline__ void add(float m, float wl, floatx4 v, float base) {
        const float w = __builtin_amdgcn_exp2f(m - base);
        l = __builtin_fmaf(w, wl, l);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(w, v[e], o[e]);
    }
    // Pieces first, first + step, ... < pieces of a sequence whose first run is b0 (that run's last part: slot
    // 2 b0 + 1; then the first part of each), head `head`, dims `at` ..; HD of them in a row.
    template <int HD>
    __device__ __forceinline__ void read(const PagedArgs &a, __amdgpu_buffer_rsrc_t r, int b0, int pieces, int head, int at,
                                         int first, int step) {
        constexpr int U = 4;  // pieces read at once
        const uint32_t mls = (uint32_t)(2 * a.runs * a.n_heads) * (HD * 4);
#pragma unroll 1
        for (int p0 = first; p0 < pieces; p0 += U * step) {
            floatx4 v[U];
            float2 ml[U];
            float t = -__builtin_inff();
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int p = min(p0 + u * step, pieces - 1), slot = 2 * (b0 + p) + (p == 0 ? 1 : 0);
                const uint32_t row = (uint32_t)(slot * a.n_heads + head);
                v[u] = __builtin_bit_cast(floatx4, __builtin_amdgcn_raw_buffer_load_b128(r, row * (HD * 4) + at * 4, 0, 16));
                ml[u] = __builtin_bit_cast(float2, __builtin_amdgcn_raw_buffer_load_b64(r, mls + row * 8, 0, 16));
            }
#pragma unroll
            for (int u = 0; u < U; ++u) t = fmaxf(t, ml[u].x);  // (one read twice does not tell)
            const float base = rise(t);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (p0 + u * step < pieces) add(ml[u].x, ml[u].y, v[u], base);
        }
    }
};

__device__ __forceinline__ __amdgpu_buffer_rsrc_t part_rsrc(const PagedArgs &a, int hd) {
    return make_rsrc(a.part, (uint32_t)(2 * a.runs * a.n_heads) * (uint32_t)(hd * 4 + 8));
}

template <typename T>
__device__ __forceinline__ void write_out(const PagedArgs &a, int s, int64_t at, float top, float l, floatx4 o) {
    typedef T vec4 __attribute__((ext_vector_type(4)));
    vec4 y;
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = (T)(top == -__builtin_inff() ? 0.0f : o[i] / l);
    *reinterpret_cast<vec4 *>(a.out + s * a.out_row + at * (int)sizeof(T)) = y;
}

// fp16: weights enter the products with V at 2^8 of their place below the maximum (2^14 at most, as it may lag by 2^6) and
// as two terms, hi = fp16(p) and fp16(p - hi): off by 2^-22 of p or, near fp16's smallest, 2^-33 of the largest
// weight, so a light key beside a heavy one keeps its share.  The terms' sums stay apart: the second terms, 0 or
// below, make NaN of an infinite V, or the other infinity; the first ones have the infinity, and the others' sum is kept finite.
//
// Block (key/value head, 16 of its query heads, run).  WIDE: the rows of a DMA instruction lie in one page.
template <typename T, int HD, bool WIDE>
__global__ __launch_bounds__(TH, NW * blocks_per_cu(HD) / 4) void k_attn_paged(PagedArgs a) {
    using SH = PShape<T, HD>;
    constexpr bool F16 = SH::F16;
    constexpr int KT = SH::KT, ROW = SH::ROW, CH = SH::CH, TILE = SH::TILE, RPU = SH::RPU, UN = SH::UN, L = SH::L;
    constexpr int DT = HD / 16, KS = F16 ? HD / 32 : HD / 16;  // 16-dim tiles; 16-byte pieces of a row per lane
    constexpr float UP = F16 ? 256.0f : 1.0f;
    __shared__ __attribute__((aligned(1024))) unsigned char lds[NW * SH::RING];
    __shared__ float joined[2][NW][16];
    __shared__ int last[2];

    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, qt = lane >> 4;
    const int g = blockIdx.x, rb = blockIdx.y, run = blockIdx.z;
    Where<T, HD> where(a, run);
    if (where.none) return;
    const int x0 = where.x0, x1 = where.x1, len = where.len;

    const int rows = min(16, a.grp - 16 * rb), head0 = g * a.grp + 16 * rb;  // of this block
    const char *kb = a.pages.k + g * a.pages.head_stride, *vb = a.pages.v + g * a.pages.head_stride;
    const int page_mask = (1 << a.pages.shift) - 1;

    // LDS chunk c of row r holds global chunk c ^ f(r): reads of one chunk of 16 rows, and of 4 x 32 bytes, cover the banks
    auto fk = [](int r) { return F16 && HD == 64 ? (r >> 1) & 7 : r & 15; };
    auto fv = [](int r) {
        if (!F16) return 0;
        return HD == 64 ? (((r >> 1) & 1) << 2) ^ (((r >> 2) & 1) << 1) : ((r & 3) << 2) ^ (((r >> 2) & 1) << 1);
    };
    // this lane's 16 bytes within its row of each DMA instruction (WIDE: within its rows)
    uint32_t koff[UN], voff[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
        const int row = u * RPU + lane / CH, c = lane % CH;
        const uint32_t at = WIDE ? (uint32_t)(lane / CH) * (uint32_t)a.pages.pos_stride : 0u;
        koff[u] = at + (uint32_t)((c ^ fk(row)) * 16);
        voff[u] = at + (uint32_t)((c ^ fv(row)) * 16);
    }
    const uint32_t lds0 = lds_addr(&lds[0]) + (uint32_t)(wv * SH::RING);
    uint32_t ka[KS];
#pragma unroll
    for (int j = 0; j < KS; ++j) ka[j] = (uint32_t)(col * ROW + (((4 * j + qt) ^ fk(col)) * 16));
    uint32_t va[DT];
    if constexpr (F16) {
        // 16 lanes take a block of 4 keys x 16 dims; each gets one dim's 4 keys
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            const int row = 4 * qt + col / 4, ch = 2 * d + (col & 3) / 2;
            va[d] = (uint32_t)(row * ROW + ((ch ^ fv(row)) * 16) + (col & 1) * 8);
        }
    }
    typedef short short4v __attribute__((ext_vector_type(4)));
    typedef __attribute__((address_space(3))) short4v lds_short4;
    typedef __attribute__((address_space(3))) u32x4 lds_u32x4;

    // Sequences that other blocks have parts of, too: at most the first and the last of the run.
    int cuts = 0, cut_s[2] = {0, 0}, cut_begin[2] = {0, 0}, cut_end[2] = {1, 1};

    const int whole = whole_units(len);
    for (int x = x0; x < x1;) {
        const int held_end = __builtin_amdgcn_readlane(where.end, 63);
        if (x >= held_end) where.next(a, held_end);
        // This round's parts: lane l's of its sequence, units from .. from + mine - 1 of the flat order, to waves
        // until - need .. until - 1, per units each; as many parts as find waves, with per up to twice an equal share.
        const bool entire = where.end - where.begin <= whole;
        const int from = max(where.begin, x);
        const int mine = max((entire ? (where.begin >= x0 && where.begin < x1 ? where.end : 0) : min(where.end, x1)) - from, 0);
        const int share = (__builtin_amdgcn_readlane(scan_add(mine), 63) + NW - 1) / NW;
        if (share == 0) {  // (what is held began in another run)
            x = __builtin_amdgcn_readlane(where.end, 63);
            continue;
        }
        int per = share, need = 0, until = 0;
#pragma unroll
        for (int t = 0; t < 2; ++t) {
            need = 0;  // mine / per rounded up, as far as it tells
#pragma unroll
            for (int k = 0; k <= NW; ++k) need += (uint32_t)mine > (uint32_t)k * (uint32_t)per ? 1 : 0;
            until = scan_add(need);
            if (t == 1 || __builtin_amdgcn_readlane(until, 63) <= NW) break;
            per *= 2;
        }
        const uint64_t dealt = __builtin_amdgcn_ballot_w64(mine > 0 && until <= NW);  // a run of lanes, not empty
        const int l0 = __builtin_ctzll(dealt), l1 = 63 - __builtin_clzll(dealt);
        x = __builtin_amdgcn_readlane(from + mine, l1);
        // this wave's (the last waves may have none)
        const uint64_t past = __builtin_amdgcn_ballot_w64(until > wv) & dealt;
        const int pl = past ? __builtin_ctzll(past) : l0;
        const int ms = where.base + pl, length = __builtin_amdgcn_readlane(where.length, pl);
        const int waves = __builtin_amdgcn_readlane(need, pl), wave0 = __builtin_amdgcn_readlane(until, pl) - waves;
        const int sb = __builtin_amdgcn_readlane(where.begin, pl), se = __builtin_amdgcn_readlane(where.end, pl);
        const int pf = __builtin_amdgcn_readlane(from, pl), pm = __builtin_amdgcn_readlane(mine, pl);
        const int w0 = pf - sb + (wv - wave0) * per;  // its first unit within the sequence
        const int n = past && length > 0 ? min(per, pm - (wv - wave0) * per) : 0;

        // the pages' entries, lane l's of page p0 + l, and the queries: one trip
        int p0 = (w0 * KT) >> a.pages.shift;
        int entry = a.pages.page(ms, p0 + lane);
        u32x4 qf[KS];
        {
            const char *qp = a.q + ms * a.q_row + (int64_t)(head0 + min(col, rows - 1)) * ROW;
            const uint32_t flip = a.neg ? (F16 ? 0x80008000u : 0x80000000u) : 0u;
#pragma unroll
            for (int j = 0; j < KS; ++j) {
                qf[j] = *reinterpret_cast<const u32x4 *>(qp + 64 * j + 16 * qt);
                qf[j] ^= flip;
                asm volatile("" : "+v"(qf[j]));  // (waited for here: later the wait would be for the DMA, too)
            }
        }
        asm volatile("" : "+v"(entry));

        // The offsets of unit w0 + i's rows, and which of its keys are seen, as bits; keys that lie in
        // no page read another row's bytes.
        int64_t rowat[UN];
        uint32_t bits = 0;
        int64_t pageat = (int64_t)max(entry, 0) * a.pages.page_stride;
        auto locate = [&](int i) {
            const int key0 = (w0 + i) * KT;
            if (((key0 + KT - 1) >> a.pages.shift) - p0 > 63) {
                p0 = key0 >> a.pages.shift;
                entry = a.pages.page(ms, p0 + lane);
                asm volatile("" : "+v"(entry));
                pageat = (int64_t)max(entry, 0) * a.pages.page_stride;
            }
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                if constexpr (WIDE) {
                    const int key = key0 + u * RPU, p = (key >> a.pages.shift) - p0;
                    const uint64_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)pageat, p);
                    const uint64_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(pageat >> 32), p);
                    rowat[u] = (int64_t)((hi << 32 | lo) + (uint64_t)((uint32_t)(key & page_mask) * (uint32_t)a.pages.pos_stride));
                } else {
                    const int key = key0 + u * RPU + lane / CH;
                    const int e = max(__shfl(entry, (key >> a.pages.shift) - p0), 0);
                    rowat[u] = e * a.pages.page_stride + (int64_t)(key & page_mask) * a.pages.pos_stride;
                }
            }
            const int key = key0 + (lane & (KT - 1));
            const int e = __shfl(entry, (key >> a.pages.shift) - p0);
            bits = (uint32_t)__builtin_amdgcn_ballot_w64(lane < KT && key < length && e >= 0);
        };
        auto dma = [&](const char *from, const uint32_t *off, uint32_t to) {
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                if constexpr (WIDE) dma16_from((uint64_t)from + (uint64_t)rowat[u], off[u], to + (uint32_t)u * 1024u);
                else dma16_at(from + rowat[u] + off[u], to + (uint32_t)u * 1024u);
            }
        };
        const uint32_t kt = lds0, vt = lds0 + (uint32_t)TILE;
        if (n > 0) {
            locate(0);
            dma(kb, koff, kt);
            dma(vb, voff, vt);
        }

        float mc = -__builtin_inff(), l = 0.0f;  // running maximum (scaled), this lane's share of the sum
        floatx4 o[DT], ol[F16 ? DT : 1];
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] = ol[F16 ? d : 0] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        bool any = false, far = false;

        for (int i = 0; i < per; ++i) {
            if (i > 0) __builtin_amdgcn_s_barrier();  // (for an even pace: older waves' loads go first)
            if (i >= n) continue;
            constexpr uint32_t ALL = KT == 32 ? 0xffffffffu : 0xffffu;
            constexpr int NT = KT / 16;
            const uint32_t sees = bits;
            any = any || sees != 0;
            wait_vmcnt<UN>();  // K has landed, V may not have
            floatx4 sc[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                sc[t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < KS; ++j) {
                    const u32x4 kf = *(lds_u32x4 *)(uintptr_t)(kt + ka[j] + (uint32_t)(16 * t * ROW));
                    if constexpr (F16) {
                        sc[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, kf),
                                                                       __builtin_bit_cast(half8, qf[j]), sc[t], 0, 0, 0);
                    } else {
                        const floatx4 kv = __builtin_bit_cast(floatx4, kf), qv = __builtin_bit_cast(floatx4, qf[j]);
#pragma unroll
                        for (int e = 0; e < 4; ++e) sc[t] = __builtin_amdgcn_mfma_f32_16x16x4f32(kv[e], qv[e], sc[t], 0, 0, 0);
                    }
                }
            }
            wait_lgkm0();  // K has been read: the next unit's may take its place
            if (i + 1 < n) {
                locate(i + 1);
                dma(kb, koff, kt);
            }
            if (sees != ALL) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        sc[t][e] = sees >> (16 * t + 4 * qt + e) & 1 ? sc[t][e] : -__builtin_inff();
            }
            float mt = sc[0][0];
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) mt = fmaxf(mt, sc[t][e]);
            mt = join4(mt, [](float x, float y) { return fmaxf(x, y); }) * a.c;
            // The maximum may lag by 6 (weights up to 2^6): sums are then rescaled a few times in all.
            const bool rose = mt > mc + 6.0f;
            if (__builtin_amdgcn_ballot_w64(rose)) {
                const float alpha = rose ? __builtin_amdgcn_exp2f(mc - mt) : 1.0f;
                mc = rose ? mt : mc;
                // An fma takes the product unrounded where mc was rounded: past 2^22, where that tells, it is rounded first.
                far = __builtin_amdgcn_ballot_w64(fabsf(mc) > 4194304.0f && mc != -__builtin_inff()) != 0;
                l *= alpha;
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    o[d] *= alpha;
                    if constexpr (F16) ol[d] *= alpha;
                }
            }
            const float off = mc == -__builtin_inff() ? 0.0f : -mc;  // no key yet: every weight is 2^-inf
            if (__builtin_expect(far, false)) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float x = sc[t][e] * a.c;
                        asm volatile("" : "+v"(x));  // (kept here: moved across, it takes 12 registers)
                        sc[t][e] = x;
                    }
            }
            const float c = far ? 1.0f : a.c;
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sc[t][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][e], c, off));
                    l += sc[t][e];
                }
            if (i + 1 < n) wait_vmcnt<UN>();
            else wait_vmcnt<0>();
            if (sees != ALL) {
                // V's rows of keys that are not seen: zeros, whatever the bytes were
#pragma unroll
                for (int u = 0; u < UN; ++u)
                    if (!(sees >> (u * RPU + lane / CH) & 1))
                        *(lds_u32x4 *)(uintptr_t)(vt + (uint32_t)(u * 1024 + lane * 16)) = u32x4{0, 0, 0, 0};
                wait_lgkm0();
            }
            if constexpr (F16) {
                half8 pf, pl;
#pragma unroll
                for (int e = 0; e < 8; ++e) pf[e] = (_Float16)(sc[e / 4][e % 4] * UP);
                asm("" : "+v"(pf));  // (formed once: otherwise each is formed for the second term again)
#pragma unroll
                for (int e = 0; e < 8; ++e) pl[e] = (_Float16)__builtin_fmaf(sc[e / 4][e % 4], UP, -(float)pf[e]);
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    lds_short4 *p = (lds_short4 *)(uintptr_t)(vt + va[d]);
                    const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(p));
                    const uint2 y = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(p + 16 * ROW / 8));
                    const half8 vf = __builtin_bit_cast(half8, make_uint4(x.x, x.y, y.x, y.y));
                    o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pf, o[d], 0, 0, 0);
                    ol[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, pl, ol[d], 0, 0, 0);
                }
            } else {
                // instruction (e, h, i): key 4 qt + e, dims 64 h + 4 col + i
#pragma unroll
                for (int e = 0; e < 4; ++e)
#pragma unroll
                    for (int h = 0; h < HD / 64; ++h) {
                        const floatx4 x = __builtin_bit_cast(
                            floatx4, *(lds_u32x4 *)(uintptr_t)(vt + (uint32_t)((4 * qt + e) * ROW + h * 256 + col * 16)));
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            o[4 * h + i] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[i], sc[0][e], o[4 * h + i], 0, 0, 0);
                    }
            }
            wait_lgkm0();  // V has been read
            if (i + 1 < n) dma(vb, voff, vt);
        }
        l = join4(l, [](float x, float y) { return x + y; });
        if constexpr (F16) {
#pragma unroll
            for (int d = 0; d < DT; ++d)
#pragma unroll
                for (int e = 0; e < 4; ++e) o[d][e] = (o[d][e] + __builtin_amdgcn_fmed3f(ol[d][e], -3e38f, 3e38f)) * (1.0f / UP);
        }
        // -inf as the maximum means no key at all: keys whose scores are all -inf give NaN, as 0 / 0
        if (any && mc == -__builtin_inff()) mc = -3.0e38f;

        // the waves' sums through their rings
        __syncthreads();
        float *put = reinterpret_cast<float *>(lds + wv * SH::RING) + col * SH::PAD;
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            if constexpr (F16) {
                *reinterpret_cast<floatx4 *>(put + 16 * d + 4 * qt) = o[d];
            } else {
                // row r of instruction (h, i): dim 64 h + 4 (4 qt + r) + i
#pragma unroll
                for (int r = 0; r < 4; ++r) put[64 * (d / 4) + 16 * qt + 4 * r + d % 4] = o[d][r];
            }
        }
        if (qt == 0) {
            joined[0][wv][col] = mc;
            joined[1][wv][col] = l;
        }
        __syncthreads();
        const auto rp = part_rsrc(a, HD);
        const bool cut = se - sb > whole && (sb < x0 || se > x1);
        const int slot = 2 * run + (sb < x0 ? 0 : 1);
        // the part's waves join it
        for (int e = past ? (wv - wave0) * 64 + lane : rows * L; e < rows * L; e += waves * 64) {
            const int row = e / L, at = 4 * (e % L);
            float t = -__builtin_inff();
            for (int w = wave0; w < wave0 + waves; ++w) t = fmaxf(t, joined[0][w][row]);
            Joined j;
            const float base = j.rise(t);
            for (int w = wave0; w < wave0 + waves; ++w)
                j.add(joined[0][w][row], joined[1][w][row],
                      *reinterpret_cast<const floatx4 *>(reinterpret_cast<const float *>(lds + w * SH::RING) + row * SH::PAD + at), base);
            if (!cut) {
                write_out<T>(a, ms, (int64_t)(head0 + row) * HD + at, j.top, j.l, j.o);
                continue;
            }
            const uint32_t r = (uint32_t)(slot * a.n_heads + head0 + row);
            store_part(rp, r * (HD * 4) + at * 4, j.o);
            if (at == 0) {
                typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
                __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u32x2, make_float2(j.top, j.l)), rp,
                                                      (uint32_t)(2 * a.runs * a.n_heads) * (HD * 4) + r * 8, 0, 16);
            }
        }
        // its cut sequences: one that began before the run, one that goes on behind it
        const int fb = __builtin_amdgcn_readlane(where.begin, l0), fe = __builtin_amdgcn_readlane(where.end, l0);
        const int lb = __builtin_amdgcn_readlane(where.begin, l1), le = __builtin_amdgcn_readlane(where.end, l1);
        if (fe - fb > whole && fb < x0) {
            cut_s[0] = where.base + l0;
            cut_begin[0] = fb;
            cut_end[0] = fe;
            cuts = 1;
        }
        if (le - lb > whole && le > x1 && lb >= x0) {
            const int i = cuts++;  // (selects: an index that is not known would put the arrays in memory)
            cut_s[0] = i == 0 ? where.base + l1 : cut_s[0];
            cut_begin[0] = i == 0 ? lb : cut_begin[0];
            cut_end[0] = i == 0 ? le : cut_end[0];
            cut_s[1] = where.base + l1;
            cut_begin[1] = lb;
            cut_end[1] = le;
        }
        __syncthreads();  // the rings are free again
    }
    if (!cuts || !a.counters) return;

    // The block that arrives last joins a sequence's pieces, in their order.  Stores and loads are
    // device-coherent (sc1), a store's acknowledgement says that it is visible, and the barrier that all of
    // the block's are, before the relaxed atomic counts them; the loads follow its result.  No block waits for another.
    wait_vmcnt<0>();
    __syncthreads();
    auto mine_of = [&](int i, int &seq, int &b0, int &pieces) {
        const int begin = i ? cut_begin[1] : cut_begin[0], end = i ? cut_end[1] : cut_end[0];
        seq = i ? cut_s[1] : cut_s[0];
        b0 = begin / len;
        pieces = (end - 1) / len - b0 + 1;
        return a.counters + (((int64_t)b0 * a.n_kv + g) * a.rbs + rb) * kCounterStride;
    };
    if ((int)threadIdx.x < cuts) {
        int seq, b0, pieces;
        int *counter = mine_of(threadIdx.x, seq, b0, pieces);
        const bool all = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == pieces - 1;
        last[threadIdx.x] = all;
        if (all) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
#pragma unroll 1
    for (int i = 0; i < cuts; ++i) {
        if (!last[i]) continue;
        int seq, b0, pieces;
        mine_of(i, seq, b0, pieces);
        // threads: 4 dims of a row each, and as many pieces side by side as that leaves room for
        const int lr = rows > 8 ? 4 : rows > 4 ? 3 : rows > 2 ? 2 : rows > 1 ? 1 : 0;
        const int sub = threadIdx.x / L, row = sub & ((1 << lr) - 1), gi = sub >> lr, groups = (TH / L) >> lr, at = 4 * (threadIdx.x % L);
        Joined j;
        if (row < rows) j.read<HD>(a, part_rsrc(a, HD), b0, pieces, head0 + row, at, gi, groups);
        float *x = reinterpret_cast<float *>(lds) + threadIdx.x * 8;
        __syncthreads();  // the last sequence's have been read
        *reinterpret_cast<floatx4 *>(x) = j.o;
        x[4] = j.top;
        x[5] = j.l;
        __syncthreads();
        if (gi != 0 || row >= rows) continue;
        const int used = min(groups, pieces);
        float t = -__builtin_inff();
        for (int k = 1; k < used; ++k) t = fmaxf(t, x[k * (8 * L << lr) + 4]);
        const float base = j.rise(t);
        for (int k = 1; k < used; ++k) {
            const float *y = x + k * (8 * L << lr);
            j.add(y[4], y[5], *reinterpret_cast<const floatx4 *>(y), base);
        }
        write_out<T>(a, seq, (int64_t)(head0 + row) * HD + at, j.top, j.l, j.o);
    }
}

// The same in a launch of its own, where the context's counters may not be used: block (four heads, run b + 1) joins
// the sequence that is cut where that run begins, if it is not cut before.  One wave per head.
template <typename T, int HD>
__global__ __launch_bounds__(256) void k_paged_join(PagedArgs a) {
    constexpr int L = HD / 4, G = 64 / L;  // lanes of a piece, pieces side by side
    const int head = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), b = blockIdx.y, lane = threadIdx.x & 63;
    if (head >= a.n_heads) return;
    const Where<T, HD> where(a, b + 1);
    if (where.none) return;
    const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(where.end > where.x0) | 1ull << 63);
    const int begin = __builtin_amdgcn_readlane(where.begin, l), end = __builtin_amdgcn_readlane(where.end, l);
    if (begin >= where.x0 || begin / where.len != b || end - begin <= whole_units(where.len)) return;
    const int pieces = (end - 1) / where.len - b + 1;
    const int gi = lane / L, at = 4 * (lane % L);
    Joined j;
    j.read<HD>(a, part_rsrc(a, HD), b, pieces, head, at, gi, G);
#pragma unroll
    for (int w = 32; w >= L; w >>= 1) {
        floatx4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = __shfl_xor(j.o[e], w);
        const float m = __shfl_xor(j.top, w), l = __shfl_xor(j.l, w);
        j.add(m, l, o, j.rise(m));
    }
    if (gi == 0) write_out<T>(a, where.base + l, (int64_t)head * HD + at, j.top, j.l, j.o);
}

// Blocks that the units are dealt to, per key/value head and 16 rows: as many as the device holds at once.
int paged_runs(int n_heads, int n_kv, int head_dim) {
    return (int)std::max<int64_t>(1, blocks_per_cu(head_dim) * kCus / (n_kv * cdiv(n_heads / n_kv, 16)));
}

template <typename T, int HD>
int launch(PagedArgs a, hipStream_t s) {
    using SH = PShape<T, HD>;
    // (n_kv and n_heads are at most 65536, rbs 4096, runs 512)
    a.by_runs = Div::by(a.runs);
    const dim3 grid((unsigned)a.n_kv, (unsigned)a.rbs, (unsigned)a.runs);
    // (offsets within a page and within the rows of a DMA instruction in 32 bits)
    const int64_t page = (int64_t)1 << a.pages.shift;
    if (page >= SH::RPU && page * a.pages.pos_stride < ((int64_t)1 << 31))
        hipLaunchKernelGGL((k_attn_paged<T, HD, true>), grid, dim3(TH), 0, s, a);
    else
        hipLaunchKernelGGL((k_attn_paged<T, HD, false>), grid, dim3(TH), 0, s, a);
    RQ_LAUNCH_CHECK();
    if (a.runs > 1 && !a.counters) {
        hipLaunchKernelGGL((k_paged_join<T, HD>), dim3((unsigned)cdiv(a.n_heads, 4), (unsigned)a.runs - 1), dim3(256), 0, s, a);
        RQ_LAUNCH_CHECK();
    }
    return RQ_OK;
}

// rq_attn_paged's arguments; a is complete where there is work (*run).
int check_paged(const rq_attn *attn, const rq_kv_pages *cache, const void *q, const int32_t *lengths, void *out,
                void *workspace, size_t workspace_bytes, PagedArgs &a, bool &run) {
    run = false;
    AttnRows r;
    int st = check_attn_rows(attn, 0, &r);
    if (st != RQ_OK) return st;
    if ((st = check_pages(cache, attn, &a.pages)) != RQ_OK) return st;
    if (cache->n_seqs == 0) return RQ_OK;
    if (cache->n_seqs > kMaxSeqs) return fail(RQ_ERR_SHAPE, "more than %d sequences in one call", kMaxSeqs);
    if (!q || !lengths || !out) return fail(RQ_ERR_INVALID_ARGUMENT, "null pointer");
    if (!aligned(q, 16) || !aligned(out, 16) || !aligned(lengths, 4))
        return fail(RQ_ERR_UNSUPPORTED, "pointers must be 16-byte aligned");
    if ((st = check_pages_ptr(cache)) != RQ_OK) return st;
    const size_t need = rq_attn_paged_workspace(attn, cache);
    if (need > 0 && (!workspace || workspace_bytes < need))
        return fail(RQ_ERR_INVALID_ARGUMENT, "workspace of %zu bytes, %zu needed", workspace_bytes, need);
    if (need > 0 && !aligned(workspace, 16)) return fail(RQ_ERR_UNSUPPORTED, "workspace must be 16-byte aligned");
    if (cache->n_pages == 0) a.pages.max_pages = 0;  // nothing is cached: no row to read in place of one past the end
    const int64_t size = attn->dtype == RQ_F16 ? 2 : 4;
    a.q = static_cast<const char *>(q);
    a.out = static_cast<char *>(out);
    a.lengths = lengths;
    a.q_row = r.q * size;
    a.out_row = r.out * size;
    a.n_heads = attn->n_heads;
    a.n_kv = attn->n_kv_heads;
    a.grp = a.n_heads / a.n_kv;
    a.rbs = (int)cdiv(a.grp, 16);
    a.runs = paged_runs(a.n_heads, a.n_kv, attn->head_dim);
    a.part = static_cast<float *>(workspace);
    a.c = r.c;
    a.neg = r.neg;
    run = true;
    return RQ_OK;
}

}  // namespace

int check_pages(const rq_kv_pages *c, const rq_attn *at, Pages *out) {
    if (!c) return fail(RQ_ERR_INVALID_ARGUMENT, "null cache");
    if (c->n_seqs < 0 || c->max_pages < 0 || c->n_pages < 0) return fail(RQ_ERR_SHAPE, "negative cache size");
    if (c->page_size < 1 || c->page_size > 65536 || (c->page_size & (c->page_size - 1)))
        return fail(RQ_ERR_UNSUPPORTED, "page_size %d is no power of two up to 65536", c->page_size);
    const int64_t capacity = (int64_t)c->max_pages * c->page_size;
    if (capacity > kMaxPagedPositions) return fail(RQ_ERR_SHAPE, "capacity above %d", kMaxPagedPositions);
    if (c->n_seqs > 0 && (capacity > ((int64_t)1 << 34) / c->n_seqs || c->n_seqs > (1 << 29)))
        return fail(RQ_ERR_SHAPE, "n_seqs times the capacity above 2^34 positions");
    const int64_t hd = at->head_dim, unit = at->dtype == RQ_F16 ? 8 : 4, size = 16 / unit;
    int64_t page = c->page_stride, head = c->head_stride, pos = c->pos_stride;
    if (page == 0 && head == 0 && pos == 0) {
        pos = hd;
        head = hd * c->page_size;
        page = head * at->n_kv_heads;
    }
    // (a stride that is never taken, of one page, head or position, may be 0)
    if (page < 0 || head < 0 || pos < 0 || page > kMaxPageStride || head > kMaxPageStride || pos > kMaxPageStride ||
        (c->page_size > 1 && pos < hd) || (at->n_kv_heads > 1 && head < hd) || (c->n_pages > 1 && page < hd))
        return fail(RQ_ERR_SHAPE, "cache strides shorter than a row or out of range");
    if (page % unit || head % unit || pos % unit)
        return fail(RQ_ERR_UNSUPPORTED, "cache strides must be multiples of 16 bytes");
    int64_t bytes;
    if (!mul_ok(c->n_pages, page * size, &bytes)) return fail(RQ_ERR_SHAPE, "the pool's size overflows");
    const int64_t row = c->table_row ? c->table_row : c->max_pages;
    if (row < c->max_pages || row > 0x7fffffff) return fail(RQ_ERR_SHAPE, "table_row must hold max_pages entries");
    out->k = static_cast<char *>(c->k);
    out->v = static_cast<char *>(c->v);
    out->table = c->table;
    out->table_row = row;
    out->page_stride = page * size;
    out->head_stride = head * size;
    out->pos_stride = pos * size;
    out->n_seqs = c->n_seqs;
    out->max_pages = c->max_pages;
    out->n_pages = c->n_pages;
    out->shift = __builtin_ctz((unsigned)c->page_size);
    return RQ_OK;
}

int check_pages_ptr(const rq_kv_pages *c) {
    if ((c->max_pages > 0 && !c->table) || (c->n_pages > 0 && (!c->k || !c->v)))
        return fail(RQ_ERR_INVALID_ARGUMENT, "null cache pointer");
    if (!aligned(c->k, 16) || !aligned(c->v, 16) || !aligned(c->table, 4))
        return fail(RQ_ERR_UNSUPPORTED, "cache pointers must be 16-byte aligned");
    return RQ_OK;
}

}  // namespace rq

using namespace rq;

extern "C" {

size_t rq_attn_paged_workspace(const rq_attn *attn, const rq_kv_pages *cache) {
    AttnRows r;
    Pages p;
    if (check_attn_rows(attn, 0, &r) != RQ_OK || check_pages(cache, attn, &p) != RQ_OK || cache->n_seqs == 0) return 0;
    const int runs = paged_runs(attn->n_heads, attn->n_kv_heads, attn->head_dim);
    const size_t rows = (size_t)2 * runs * attn->n_heads;
    return runs > 1 ? rows * ((size_t)attn->head_dim * 4 + 8) : 0;
}

int rq_attn_paged(rq_ctx *ctx, const rq_attn *attn, const rq_kv_pages *cache, const void *q, const int32_t *lengths,
                  void *out, void *workspace, size_t workspace_bytes, rq_stream stream) {
    RQ_ENTER(ctx);
    PagedArgs a{};
    bool run;
    const int st = check_paged(attn, cache, q, lengths, out, workspace, workspace_bytes, a, run);
    if (st != RQ_OK || !run) return st;
    hipStream_t s = pick(ctx, stream);
    const GemmWorkspace ws = gemm_workspace(ctx, s);
    if (ws.counters && a.runs * a.n_kv * a.rbs <= ws.n_counters) a.counters = ws.counters;
    if (attn->dtype == RQ_F16) return attn->head_dim == 64 ? launch<_Float16, 64>(a, s) : launch<_Float16, 128>(a, s);
    return attn->head_dim == 64 ? launch<float, 64>(a, s) : launch<float, 128>(a, s);
}

// For the tests, no part of the C ABI: the argument checks alone, and where the kernels find a position
// (table read on the host).  Host arithmetic.
int rusty_paged_check(const rq_attn *attn, const rq_kv_pages *cache, const void *q, const int32_t *lengths, void *out,
                      void *workspace, size_t workspace_bytes) {
    PagedArgs a{};
    bool run;
    return check_paged(attn, cache, q, lengths, out, workspace, workspace_bytes, a, run);
}
int64_t rusty_paged_at(const rq_attn *attn, const rq_kv_pages *cache, int s, int p) {
    Pages pages;
    if (check_pages(cache, attn, &pages) != RQ_OK) return -2;
    return pages.at(s, p);
}

}  // extern "C"
