// Attention of one new token per sequence over a paged KV cache (rq_attn_paged).
//
//   out[s, h] = sum_j p_j v[j] / sum_j p_j,  p_j = 2^(c q.k_j - m),  c = scale log2 e
//
// in one pass over the keys with a running maximum m.  K and V are read once, so
// the bound is their way from memory; the matrix instructions only have to keep up.
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
// every block finds its run from them (a wave sums them).  A block
// takes the parts of its run, one sequence each, in turn; its four waves
// take quarters of a part and join through LDS; a sequence that ends in another
// block than it began leaves partial sums that k_paged_join joins.
//
// Each wave streams its keys through a ring of its own in LDS (DMA, two units,
// no block barrier): the pages' entries lie in its lanes, 64 at a time, and each lane
// forms the address of its own 16 bytes, so pages may be of any size and order.
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

constexpr int NW = 4;         // waves per block
constexpr int NS = 2;         // units of a wave's ring
constexpr int64_t kCus = 256;
constexpr int kMinRun = NW;   // units: one per wave

struct PagedArgs {
    const char *q;
    char *out;
    const int *lengths;
    int64_t q_row, out_row;  // bytes
    Pages pages;
    int n_heads, n_kv, grp, rbs;  // grp: query heads of a key/value head, in rbs blocks of 16
    int runs;                     // blocks that the units are dealt to
    float *part;                  // sums [2 runs][n_kv][grp][dim], then (m, l) [2 runs][n_kv][grp]
    float c;                      // |scale| log2 e
    int neg;                      // scale < 0
};

template <typename T, int HD>
struct PShape {
    static constexpr bool F16 = sizeof(T) == 2;
    static constexpr int KT = F16 ? 32 : 16;          // keys per unit
    static constexpr int ROW = HD * (int)sizeof(T), CH = ROW / 16;
    static constexpr int TILE = KT * ROW;             // bytes of K or V of a unit
    static constexpr int RPU = 1024 / ROW, UN = TILE / 1024;  // rows per DMA instruction, instructions
    static constexpr int RING = NS * 2 * TILE;        // of a wave
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

// DMA of 16 bytes per lane from 64-bit addresses: LDS[lds_addr + 16 * lane] = *p (see dma16).
__device__ __forceinline__ void dma16_at(const char *p, uint32_t lds_addr) {
    const uint32_t l = __builtin_amdgcn_readfirstlane(lds_addr);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(l), "v"(p) : "memory", "m0");
}

__device__ __forceinline__ int clamped(const PagedArgs &a, int s) { return min(max(a.lengths[s], 0), a.pages.capacity()); }
template <int KT>
__device__ __forceinline__ int units_of(int length) {
    return max(1, (int)(((unsigned)length + KT - 1) / KT));
}

__device__ __forceinline__ int scan_add(int v) {  // inclusive, over the wave
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int w = 1; w < 64; w <<= 1) {
        const int o = __shfl_up(v, w);
        v += lane >= w ? o : 0;
    }
    return v;
}

// Units of all sequences, and of those before sequence `upto`.
template <int KT>
__device__ __forceinline__ int total_units(const PagedArgs &a, int upto, int *before) {
    const int lane = threadIdx.x & 63;
    int all = 0, some = 0;
    for (int s = lane; s < a.pages.n_seqs; s += 64) {
        const int u = units_of<KT>(clamped(a, s));
        all += u;
        some += s < upto ? u : 0;
    }
#pragma unroll
    for (int w = 32; w > 0; w >>= 1) {
        all += __shfl_xor(all, w);
        some += __shfl_xor(some, w);
    }
    *before = __builtin_amdgcn_readfirstlane(some);
    return __builtin_amdgcn_readfirstlane(all);
}

// The sequence that unit x (below the total) belongs to, and its first unit.  Whole wave, x uniform.
template <int KT>
__device__ __forceinline__ int find_unit(const PagedArgs &a, int x, int *first) {
    const int lane = threadIdx.x & 63;
    int lo = 0, n = a.pages.n_seqs, t0 = 0;  // in sequences lo .. lo + n - 1, whose units begin at t0
    for (;;) {
        const int m = (n + 63) / 64;  // sequences of a lane
        int u = 0;
        for (int j = 0; j < m; ++j) {
            const int i = lane * m + j;
            if (i < n) u += units_of<KT>(clamped(a, lo + i));
        }
        const int upto = scan_add(u);
        const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(t0 + upto > x) | 1ull << 63);
        t0 += __builtin_amdgcn_readlane(upto - u, l);
        lo += l * m;
        n = min(m, n - l * m);
        if (m == 1) break;
    }
    *first = t0;
    return lo;
}

__device__ __forceinline__ int run_length(const PagedArgs &a, int total) { return max(kMinRun, (total + a.runs - 1) / a.runs); }

template <typename T, int HD>
__global__ __launch_bounds__(64 * NW, 1) void k_attn_paged(PagedArgs a) {
    using SH = PShape<T, HD>;
    constexpr bool F16 = SH::F16;
    constexpr int KT = SH::KT, ROW = SH::ROW, CH = SH::CH, TILE = SH::TILE, RPU = SH::RPU, UN = SH::UN;
    constexpr int DT = HD / 16, KS = F16 ? HD / 32 : HD / 16;  // 16-dim tiles; 16-byte pieces of a row per lane
    __shared__ __attribute__((aligned(1024))) unsigned char lds[NW * SH::RING];
    __shared__ float joined[2][NW][16];

    const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, qt = lane >> 4;
    const int per_run = a.n_kv * a.rbs;
    const int run = blockIdx.x / per_run, rest = blockIdx.x - run * per_run, g = rest / a.rbs, rb = rest - g * a.rbs;
    int dummy;
    const int total = total_units<KT>(a, 0, &dummy), len = run_length(a, total);
    const int64_t x0l = (int64_t)run * len;
    if (x0l >= total) return;
    const int x0 = (int)x0l, x1 = (int)min(x0l + len, (int64_t)total);
    int t0, s = __builtin_amdgcn_readfirstlane(find_unit<KT>(a, x0, &t0));
    t0 = __builtin_amdgcn_readfirstlane(t0);

    const int rows = min(16, a.grp - 16 * rb), head0 = g * a.grp + 16 * rb;  // of this block
    const char *kb = a.pages.k + g * a.pages.head_stride, *vb = a.pages.v + g * a.pages.head_stride;
    const int page_mask = (1 << a.pages.shift) - 1;

    // LDS chunk c of row r holds global chunk c ^ f(r): reads of one chunk of 16 rows, and of 4 x 32 bytes, cover the banks
    auto fk = [](int r) { return F16 && HD == 64 ? (r >> 1) & 7 : r & 15; };
    auto fv = [](int r) {
        if (!F16) return 0;
        return HD == 64 ? (((r >> 1) & 1) << 2) ^ (((r >> 2) & 1) << 1) : ((r & 3) << 2) ^ (((r >> 2) & 1) << 1);
    };
    int koff[UN], voff[UN];  // this lane's 16 bytes within its row of each DMA instruction
#pragma unroll
    for (int u = 0; u < UN; ++u) {
        const int row = u * RPU + lane / CH, c = lane % CH;
        koff[u] = (c ^ fk(row)) * 16;
        voff[u] = (c ^ fv(row)) * 16;
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

    while (t0 < x1) {
        const int length = __builtin_amdgcn_readfirstlane(clamped(a, s)), units = units_of<KT>(length);
        // this part: units ua .. ub - 1 of the sequence, and of them this wave's
        const int ua = max(x0 - t0, 0), ub = min(x1 - t0, units);
        const int per = (ub - ua + NW - 1) / NW;
        const int w0 = min(ua + wv * per, ub), n = length > 0 ? min(w0 + per, ub) - w0 : 0;

        // the pages' entries, lane l's of page p0 + l, and the queries: one trip
        int p0 = (w0 * KT) >> a.pages.shift;
        int entry = a.pages.page(s, p0 + lane);
        u32x4 qf[KS];
        {
            const char *qp = a.q + s * a.q_row + (int64_t)(head0 + min(col, rows - 1)) * ROW;
            const uint32_t flip = a.neg ? (F16 ? 0x80008000u : 0x80000000u) : 0u;
#pragma unroll
            for (int j = 0; j < KS; ++j) {
                qf[j] = *reinterpret_cast<const u32x4 *>(qp + 64 * j + 16 * qt);
                qf[j] ^= flip;
                asm volatile("" : "+v"(qf[j]));  // (waited for here: later the wait would be for the DMA, too)
            }
        }
        asm volatile("" : "+v"(entry));

        // unit w0 + i into its place; keys that lie in no page read another row's bytes
        auto dma = [&](int i) {
            const int key0 = (w0 + i) * KT;
            if (((key0 + KT - 1) >> a.pages.shift) - p0 > 63) {
                p0 = key0 >> a.pages.shift;
                entry = a.pages.page(s, p0 + lane);
                asm volatile("" : "+v"(entry));
            }
            const uint32_t base = lds0 + (uint32_t)(i % NS) * (2 * TILE);
#pragma unroll
            for (int u = 0; u < UN; ++u) {
                const int key = key0 + u * RPU + lane / CH;
                const int e = max(__shfl(entry, (key >> a.pages.shift) - p0), 0);
                const int64_t at = e * a.pages.page_stride + (int64_t)(key & page_mask) * a.pages.pos_stride;
                dma16_at(kb + at + koff[u], base + (uint32_t)u * 1024u);
                dma16_at(vb + at + voff[u], base + (uint32_t)TILE + (uint32_t)u * 1024u);
            }
        };
        // which keys of unit w0 + i are seen, as bits (after its dma: the entries are those of its pages)
        auto seen = [&](int i) -> uint32_t {
            const int key = (w0 + i) * KT + (lane & (KT - 1));
            const int e = __shfl(entry, (key >> a.pages.shift) - p0);
            return (uint32_t)__builtin_amdgcn_ballot_w64(lane < KT && key < length && e >= 0);
        };
        uint32_t sees[NS];
#pragma unroll
        for (int i = 0; i < NS; ++i) {
            sees[i] = 0;
            if (i < n) {
                dma(i);
                sees[i] = seen(i);
            }
        }

        float mc = -__builtin_inff(), l = 0.0f;  // running maximum (scaled), this lane's share of the sum
        floatx4 o[DT];
#pragma unroll
        for (int d = 0; d < DT; ++d) o[d] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
        bool any = false;

        auto unit = [&](uint32_t tb, uint32_t bits) {
            constexpr uint32_t ALL = KT == 32 ? 0xffffffffu : 0xffffu;
            constexpr int NT = KT / 16;
            any = any || bits != 0;
            if (bits != ALL) {
                // V's rows of keys that are not seen: zeros, whatever the bytes were
#pragma unroll
                for (int u = 0; u < UN; ++u)
                    if (!(bits >> (u * RPU + lane / CH) & 1))
                        *(lds_u32x4 *)(uintptr_t)(tb + TILE + (uint32_t)(u * 1024 + lane * 16)) = u32x4{0, 0, 0, 0};
                wait_lgkm0();
            }
            floatx4 sc[NT];
#pragma unroll
            for (int t = 0; t < NT; ++t) {
                sc[t] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int j = 0; j < KS; ++j) {
                    const u32x4 kf = *(lds_u32x4 *)(uintptr_t)(tb + ka[j] + (uint32_t)(16 * t * ROW));
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
            if (bits != ALL) {
#pragma unroll
                for (int t = 0; t < NT; ++t)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        sc[t][e] = bits >> (16 * t + 4 * qt + e) & 1 ? sc[t][e] : -__builtin_inff();
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
                l *= alpha;
#pragma unroll
                for (int d = 0; d < DT; ++d) o[d] *= alpha;
            }
            const float off = mc == -__builtin_inff() ? 0.0f : -mc;  // no key yet: every weight is 2^-inf
#pragma unroll
            for (int t = 0; t < NT; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    sc[t][e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[t][e], a.c, off));
                    l += sc[t][e];
                }
            const uint32_t vt = tb + TILE;
            if constexpr (F16) {
                half8 pf;
#pragma unroll
                for (int e = 0; e < 8; ++e) pf[e] = (_Float16)sc[e / 4][e % 4];
#pragma unroll
                for (int d = 0; d < DT; ++d) {
                    lds_short4 *p = (lds_short4 *)(uintptr_t)(vt + va[d]);
                    const uint2 x = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(p));
                    const uint2 y = __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(p + 16 * ROW / 8));
                    o[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8, make_uint4(x.x, x.y, y.x, y.y)), pf,
                                                                  o[d], 0, 0, 0);
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
        };
        for (int i = 0; i < n; ++i) {
            if (i + 1 < n) wait_vmcnt<2 * UN>();
            else wait_vmcnt<0>();
            const uint32_t bits = sees[0];
            sees[0] = sees[1];
            unit(lds0 + (uint32_t)(i % NS) * (2 * TILE), bits);
            wait_lgkm0();  // (the unit has been read)
            if (i + NS < n) {
                dma(i + NS);
                sees[1] = seen(i + NS);
            }
        }
        l = join4(l, [](float x, float y) { return x + y; });
        // -inf as the maximum means no key at all: keys whose scores are all -inf give NaN, as 0 / 0
        if (any && mc == -__builtin_inff()) mc = -3.0e38f;

        // the waves' sums through their rings
        __syncthreads();
        float *mine = reinterpret_cast<float *>(lds + wv * SH::RING) + col * SH::PAD;
#pragma unroll
        for (int d = 0; d < DT; ++d) {
            if constexpr (F16) {
                *reinterpret_cast<floatx4 *>(mine + 16 * d + 4 * qt) = o[d];
            } else {
                // row r of instruction (h, i): dim 64 h + 4 (4 qt + r) + i
#pragma unroll
                for (int r = 0; r < 4; ++r) mine[64 * (d / 4) + 16 * qt + 4 * r + d % 4] = o[d][r];
            }
        }
        if (qt == 0) {
            joined[0][wv][col] = mc;
            joined[1][wv][col] = l;
        }
        __syncthreads();
        const bool cut = t0 < x0 || t0 + units > x1;
        const int slot = 2 * run + (t0 < x0 ? 0 : 1);
        for (int e = threadIdx.x; e < rows * (HD / 4); e += 64 * NW) {
            const int row = e / (HD / 4), at = 4 * (e % (HD / 4));
            float top = joined[0][0][row];
#pragma unroll
            for (int w = 1; w < NW; ++w) top = fmaxf(top, joined[0][w][row]);
            const float base = top == -__builtin_inff() ? 0.0f : top;
            float sum = 0.0f;
            floatx4 v = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < NW; ++w) {
                const float wt = __builtin_amdgcn_exp2f(joined[0][w][row] - base);
                const floatx4 x = *reinterpret_cast<const floatx4 *>(reinterpret_cast<const float *>(lds + w * SH::RING) + row * SH::PAD + at);
                sum = __builtin_fmaf(wt, joined[1][w][row], sum);
#pragma unroll
                for (int i = 0; i < 4; ++i) v[i] = __builtin_fmaf(wt, x[i], v[i]);
            }
            if (cut) {
                const int64_t r = ((int64_t)slot * a.n_kv + g) * a.grp + 16 * rb + row;
                *reinterpret_cast<floatx4 *>(a.part + r * HD + at) = v;
                if (at == 0)
                    reinterpret_cast<float2 *>(a.part + (int64_t)2 * a.runs * a.n_kv * a.grp * HD)[r] = make_float2(top, sum);
            } else {
                typedef T vec4 __attribute__((ext_vector_type(4)));
                vec4 y;
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = (T)(top == -__builtin_inff() ? 0.0f : v[i] / sum);
                *reinterpret_cast<vec4 *>(a.out + s * a.out_row + ((int64_t)(head0 + row) * HD + at) * (int)sizeof(T)) = y;
            }
        }
        __syncthreads();  // the ring is free again
        t0 += units;
        ++s;
    }
}

// Joins the pieces of sequences that more than one block had: one wave per (sequence, head).
template <typename T, int HD>
__global__ __launch_bounds__(256) void k_paged_join(PagedArgs a) {
    constexpr int KT = PShape<T, HD>::KT, L = HD / 4, G = 64 / L;  // lanes of a piece, pieces side by side
    const int64_t row = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (row >= (int64_t)a.pages.n_seqs * a.n_heads) return;
    const int s = (int)(row / a.n_heads), head = (int)(row - (int64_t)s * a.n_heads), lane = threadIdx.x & 63;
    int t0;
    const int total = total_units<KT>(a, s, &t0), len = run_length(a, total);
    const int t1 = t0 + units_of<KT>(clamped(a, s));
    const int b0 = t0 / len, pieces = (t1 - 1) / len - b0 + 1;
    if (pieces <= 1) return;  // written by the block that had them all
    const int gi = lane / L, at = 4 * (lane % L);
    // piece p's row: the part that a run begins with, but for the first, unless the run begins with the sequence
    auto place = [&](int p) { return (int64_t)(2 * (b0 + p) + (p == 0 ? 1 : 0)) * a.n_heads + head; };
    const float2 *ml = reinterpret_cast<const float2 *>(a.part + (int64_t)2 * a.runs * a.n_heads * HD);
    float top = -__builtin_inff();
    for (int p = lane; p < pieces; p += 64) top = fmaxf(top, ml[place(p)].x);
#pragma unroll
    for (int w = 32; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor(top, w));
    const float base = top == -__builtin_inff() ? 0.0f : top;
    float l = 0.0f;
    floatx4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int p = gi; p < pieces; p += G) {
        const float2 m = ml[place(p)];
        const floatx4 v = *reinterpret_cast<const floatx4 *>(a.part + place(p) * HD + at);
        const float w = __builtin_amdgcn_exp2f(m.x - base);
        l = __builtin_fmaf(w, m.y, l);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = __builtin_fmaf(w, v[e], o[e]);
    }
#pragma unroll
    for (int w = 32; w >= L; w >>= 1) {
        l += __shfl_xor(l, w);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], w);
    }
    if (gi != 0) return;
    typedef T vec4 __attribute__((ext_vector_type(4)));
    vec4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) y[e] = (T)(top == -__builtin_inff() ? 0.0f : o[e] / l);
    *reinterpret_cast<vec4 *>(a.out + s * a.out_row + ((int64_t)head * HD + at) * (int)sizeof(T)) = y;
}

// Blocks that the units are dealt to, per key/value head and 16 rows: as many as the device holds at once.
int paged_runs(int n_heads, int n_kv, int head_dim) {
    const int64_t rbs = cdiv(n_heads / n_kv, 16), blocks = kCus * (head_dim == 64 ? 2 : 1);
    return (int)std::max<int64_t>(1, blocks / (n_kv * rbs));
}

template <typename T, int HD>
int launch(PagedArgs a, hipStream_t s) {
    const int64_t blocks = (int64_t)a.runs * a.n_kv * a.rbs, rows = cdiv((int64_t)a.pages.n_seqs * a.n_heads, 4);
    if (!grid_ok(blocks, 64 * NW) || !grid_ok(rows, 256)) return fail(RQ_ERR_SHAPE, "too many rows for one call");
    hipLaunchKernelGGL((k_attn_paged<T, HD>), dim3((unsigned)blocks), dim3(64 * NW), 0, s, a);
    RQ_LAUNCH_CHECK();
    if (a.runs > 1) {
        hipLaunchKernelGGL((k_paged_join<T, HD>), dim3((unsigned)rows), dim3(256), 0, s, a);
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
