#pragma once
// A key / value cache in pages, as the kernels see it: pools of f16 [n_pages][page_size][n_kv][D] and a table of page ids per sequence. Every id, sequence and
// position that a kernel takes from device memory is checked before an address is made of it; what fails is skipped and reported through the error words.
#include <cuda_fp16.h>

#include <atomic>
#include <chrono>

#include "arrivals.h"
#include "kernels.h"

namespace dooms {
namespace cuda {

struct PagedView {
    __half * k, * v;
    const int32_t * table;        // [n_sequences][max_pages]
    int n_pages, page_shift, n_sequences, max_pages, n_kv;
    int * error;                  // kErrorWords of them

    __device__ __forceinline__ void fail() const { reinterpret_cast<volatile int *>(error)[1] = kErrorPaged; }
    __device__ __forceinline__ void gave_up() const { reinterpret_cast<volatile int *>(error)[2] = kErrorPagedWait; }
    // Positions a sequence can have: its pages, kept inside 32 bits.
    __device__ __forceinline__ int capacity() const { return int(min(int64_t(max_pages) << page_shift, int64_t(0x7fffff00))); }
    // The pool's row (of n_kv * D values) of position `at` of sequence `seq`, both in range; -1: the page is not one.
    __device__ __forceinline__ int64_t row(int seq, int at) const {
        const int page = __ldg(table + int64_t(seq) * max_pages + (at >> page_shift));
        if (uint32_t(page) >= uint32_t(n_pages)) return -1;
        return (int64_t(page) << page_shift) + (at & ((1 << page_shift) - 1));
    }
};

// a / b for a >= 0, b > 0: in 32 bits where they fit (a 64-bit division is some hundred cycles, and stands in front of everything else a block does).
__device__ __forceinline__ int64_t quotient(int64_t a, int64_t b) {
    return ((a | b) >> 32) == 0 ? int64_t(uint32_t(a) / uint32_t(b)) : a / b;
}
// Where the b-th of n equal parts of `total` begins.
__device__ __forceinline__ int64_t part_of(int64_t total, int64_t each, int b, int n) { return each * b + int64_t(uint64_t(total - each * n) * uint32_t(b) / uint32_t(n)); }

// A call's own number for its arrival counters (arrivals.h).
inline unsigned long long paged_call() {
    static std::atomic<unsigned long long> calls{(unsigned long long)(std::chrono::steady_clock::now().time_since_epoch().count()) * 0x9E3779B97F4A7C15ull >> 20};
    unsigned long long c;
    do c = calls.fetch_add(1, std::memory_order_relaxed) % kArrivalsCalls; while (c == 0 || c == kArrivalsCalls - 1);
    return c;
}
struct ArrivalsInMemory {
    Arrivals * at;
    __device__ __forceinline__ Arrivals load() const { return *reinterpret_cast<volatile Arrivals *>(at); }
    __device__ __forceinline__ Arrivals swap(Arrivals was, Arrivals to) const { return atomicCAS(at, was, to); }
    __device__ __forceinline__ Arrivals add(Arrivals n) const { return atomicAdd(at, n); }
    __device__ __forceinline__ void store(Arrivals to) const { *reinterpret_cast<volatile Arrivals *>(at) = to; }
};
// One thread, behind a barrier of those whose stores it stands for and a __threadfence of each: whether it is the last of `count` to arrive, and none of them failed.
__device__ __forceinline__ bool paged_counter_arrive(Arrivals * counter, unsigned long long call, int count, bool failed) {
    return arrive(ArrivalsInMemory{counter}, call, count, failed) == Arrival::kLast;
}
// One thread of the first of two blocks that share a counter: 1: the other has left its part, and this one has arrived behind it; -1: it came, but failed; 0: it is not there
// yet, and this one has not arrived. The other block may not run before this one's SM is free (beside a long kernel of another stream, say), so the wait is short: about
// a millisecond; usually the other came long before.
__device__ __forceinline__ int paged_counter_wait(Arrivals * counter, unsigned long long call, bool failed) {
    const ArrivalsInMemory memory{counter};
    const auto there = [&] { const Arrivals a = memory.load(); return arrivals_call(a) == call && arrivals_count(a) == 1; };
    bool came = there();
    for (int polls = 0; !came && polls < 2048; polls++) came = there();
    return !came ? 0 : paged_counter_arrive(counter, call, 2, failed) ? 1 : -1;
}

inline PagedView paged_view(const PagedCache & c, int * error) {
    int shift = 0;
    while ((1 << shift) < c.page_size) shift++;
    return {static_cast<__half *>(c.keys), static_cast<__half *>(c.values), c.page_table, c.n_pages, shift, c.n_sequences, c.max_pages, c.n_head_kv, error};
}

}  // namespace cuda
}  // namespace dooms
