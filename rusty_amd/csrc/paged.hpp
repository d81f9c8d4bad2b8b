// A paged KV cache as the kernels see it, shared by the kernels that fill it
// (rope.hip) and read it (attn_paged.hip).
#pragma once

#include "common.hpp"

namespace rq {

constexpr int kMaxPagedPositions = 0x7fffffff - 1024;  // positions rounded up to tiles stay below 2^31
constexpr int64_t kMaxPageStride = (int64_t)1 << 40;   // elements

// Position p of sequence s and key/value head g lies at byte
// page * page_stride + g * head_stride + (p % page_size) * pos_stride of k and v,
// page = table[s * table_row + p / page_size].
struct Pages {
    char *k, *v;
    const int *table;
    int64_t table_row;                             // entries
    int64_t page_stride, head_stride, pos_stride;  // bytes
    int n_seqs, max_pages, n_pages;
    int shift;  // page_size = 2^shift

    // The table's entry for page i of sequence s: -1 where it names none of the pool's pages.
    __host__ __device__ __forceinline__ int page(int s, int i) const {
        if (i < 0 || i >= max_pages) return -1;
        const int e = table[(int64_t)s * table_row + i];
        return (uint32_t)e < (uint32_t)n_pages ? e : -1;
    }
    // Byte offset of position p (head 0), -1 if it lies in no page.
    __host__ __device__ __forceinline__ int64_t at(int s, int p) const {
        const int e = p < 0 ? -1 : page(s, p >> shift);
        return e < 0 ? -1 : e * page_stride + (int64_t)(p & ((1 << shift) - 1)) * pos_stride;
    }
    __host__ __device__ __forceinline__ int capacity() const { return max_pages << shift; }
};

// Checks a cache's sizes and strides against the attention descriptor's heads and fills *out (pointers: check_pages_ptr).
int check_pages(const rq_kv_pages *c, const rq_attn *at, Pages *out);
// Its pointers, where there is anything to read or write.
int check_pages_ptr(const rq_kv_pages *c);

}  // namespace rq
