#pragma once
// Arrival counters in scratch memory whose contents at the start do not matter: which of the blocks that share a piece of work is the last to leave its part.
//
// A counter is (a call's own number, 44 bits, not zero) << 20 | blocks that failed << 10 | blocks that have arrived, failed ones too. Whoever arrives first finds another
// call's number, or anything else, and replaces it. Every block of a launch arrives exactly once at each counter that is its, whatever happened to it before, and the
// last one leaves zero: so when a launch is over no counter has its number, and a replay of it in a graph, whose number is the same, finds no count of an earlier one.
// That holds for a launch in which a bounded wait ran out as well. No block needs another one to run beside it.
#include <cstdint>

#ifdef __CUDACC__
#define DOOMS_BOTH __host__ __device__ __forceinline__
#else
#define DOOMS_BOTH inline
#endif

namespace dooms {
namespace cuda {

using Arrivals = unsigned long long;
constexpr int kArrivalsMost = 1023;      // blocks that can share a counter
constexpr Arrivals kArrivalsCalls = Arrivals(1) << 44;

DOOMS_BOTH constexpr Arrivals arrival_of(bool failed) { return failed ? 1ull << 10 | 1ull : 1ull; }
DOOMS_BOTH constexpr Arrivals arrivals_call(Arrivals a) { return a >> 20; }
DOOMS_BOTH constexpr int arrivals_count(Arrivals a) { return int(a & 1023u); }
DOOMS_BOTH constexpr bool arrivals_failed(Arrivals a) { return (a >> 10 & 1023u) != 0; }

enum class Arrival { kNotLast, kLast, kLastAfterFailure };

// One arrival of `count`. M: the memory's load, compare-and-swap and add (both give back what was there), and store.
#ifdef __CUDACC__
#pragma nv_exec_check_disable
#endif
template <class M>
DOOMS_BOTH Arrival arrive(M memory, Arrivals call, int count, bool failed) {
    const Arrivals mine = arrival_of(failed), first = call << 20 | mine;
    Arrivals now, was = memory.load();
    // (what changes it under this call's hands is another arrival of the same launch, so a swap that fails finds the call's number)
    if (arrivals_call(was) != call && memory.swap(was, first) == was) now = first;
    else now = memory.add(mine) + mine;
    if (arrivals_count(now) != count) return Arrival::kNotLast;
    memory.store(0);
    return arrivals_failed(now) ? Arrival::kLastAfterFailure : Arrival::kLast;
}

}  // namespace cuda
}  // namespace dooms
