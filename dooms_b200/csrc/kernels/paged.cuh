#pragma once
// A key / value cache in pages, as the kernels see it: pools of f16 [n_pages][page_size][n_kv][D] and a table of page ids per sequence. Every id, sequence and
// position that a kernel takes from device memory is checked before an address is made of it; what fails is skipped and reported through the error word.
#include <cuda_fp16.h>

#include "kernels.h"

namespace dooms {
namespace cuda {

struct PagedView {
    __half * k, * v;
    const int32_t * table;        // [n_sequences][max_pages]
    int n_pages, page_shift, n_sequences, max_pages, n_kv;
    int * error;

    __device__ __forceinline__ void fail() const { if (error) *reinterpret_cast<volatile int *>(error) = kErrorPaged; }
    // Positions a sequence can have: its pages, kept inside 32 bits.
    __device__ __forceinline__ int capacity() const { return int(min(int64_t(max_pages) << page_shift, int64_t(0x7fffff00))); }
    // The pool's row (of n_kv * D values) of position `at` of sequence `seq`, both in range; -1: the page is not one.
    __device__ __forceinline__ int64_t row(int seq, int at) const {
        const int page = __ldg(table + int64_t(seq) * max_pages + (at >> page_shift));
        if (uint32_t(page) >= uint32_t(n_pages)) return -1;
        return (int64_t(page) << page_shift) + (at & ((1 << page_shift) - 1));
    }
};

inline PagedView paged_view(const PagedCache & c, int * error) {
    int shift = 0;
    while ((1 << shift) < c.page_size) shift++;
    return {static_cast<__half *>(c.keys), static_cast<__half *>(c.values), c.page_table, c.n_pages, shift, c.n_sequences, c.max_pages, c.n_head_kv, error};
}

}  // namespace cuda
}  // namespace dooms
