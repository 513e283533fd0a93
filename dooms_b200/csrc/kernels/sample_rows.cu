// One token per row of logits from given random numbers: top-k, then top-p and min-p on the probabilities at temperature 1, then the temperature, then the draw (the
// order of the host sampler's chain). In the order (logit descending, index ascending), with the row's largest logit m and g = m - l:
//   kept by top-k: the first k;  by top-p: while what is in front of a token holds less than top_p of the mass e^-g of what top-k kept;  by min-p: e^-g >= min_p;
//   the token: the first whose cumulative weight e^(-g / T) exceeds u times the kept tokens' total.
//
// A row belongs to one block, or to a cluster of up to eight that share it. The first pass finds the maximum and a bound (see there): for a top-k one that the k largest
// lie above, where a total of everything is needed one that a tenth of the row does; later passes read the row from L2. A cut ("the first element at which a
// cumulative weight reaches a goal") is found by a histogram over all blocks of the cluster, of 1/24 nat per bin, then by sorting the few elements of the bin where
// the goal falls. Histograms are of lists wherever there is one to make (what is above the bound or a min-p's limit, a step below the bound, or in front of a goal):
// an element costs a histogram some hundred instructions, a list two votes, and the sum of the weights that are in no list some fifty. Where at most kList
// elements are left to look at, they are sorted and everything else is decided among them. A bin of more than kList elements is divided again by the bits of the
// logits, down to a single value, whose elements are counted out in the order of their indices.
// Bound by instructions where a total is needed (256 rows of 128256 normal logits at temperature 0.9, B200: 200 us at no filter, 346 at a nucleus of 0.9), else by latencies
// and memory (top-k 40: 57 us, the largest alone: 31 us, of the 20 that reading the 131 MB takes); a mix of all that 195.
// Rows that do not begin on 16 bytes are read a logit at a time, and of a warp's lanes one in four has a sample then, so that the list that a total begins with is mostly given
// up for the histogram of the row: up to twice as long (128 rows of 151643 / 151644, no filter 278 / 145 us, nucleus 443 / 221, top-k 40 101 / 52, largest 50 / 22).
// Weights are 64-bit integers, e^-x 2^45 rounded (x and the exponential in 64-bit floating point): sums do not depend on the order of the atomics, and the blocks of
// a cluster, which all work out every cut for themselves, agree on it. 2^18 logits of the largest weight still fit. What is rounded off is 2^-46 of
// the row's largest weight per token.
#include <math_constants.h>

#include <algorithm>
#include <cmath>

#include "kernels.h"
#include "launch.cuh"
#include "ptx.cuh"

namespace dooms {
namespace cuda {

using namespace dooms::dev;

namespace {

constexpr int kThreads = 512, kBins = 256, kList = 512, kMostBlocks = 8;
constexpr int kMostLogits = 1 << 18;
constexpr float kBinsPerNat = 24.f, kFarBinsPerNat = 8.f;
constexpr int kFar = 240;              // the bin of everything from 10 nats below the largest logit on
constexpr int kPowers = 256;
constexpr int kNearMost = 8192, kPerWarp = kNearMost / (kThreads / 32);      // logits a block lists, and each of its warps
constexpr int kSamples = 8;            // logits per thread that say how far down a list goes
constexpr int kTurns = 4;              // passes that weigh steps before it is a histogram's: ten nats, at temperature 1, below the list
static_assert(kList == kThreads && kBins <= kThreads, "one list element and at most one bin per thread");

struct SampleArgs {
    const float * logits;
    int64_t stride;
    int n, slice;
    int sample_every, sample_rank;      // of a thread's groups of four logits one in so many (a power of two) is sampled; m (see the kernel)
    const float * temperature, * top_p, * min_p, * uniform;
    const int32_t * top_k;
    int32_t * tokens;
    float * probability;
    int rows_of;
};
enum { kAllRows, kBoundedRows, kOpenRows };

struct Shared {
    uint32_t count[kBins], low[kBins], high[kBins];      // this block's histogram: elements, and their weights in two words
    double power[kPowers];                               // 2^(-i / kPowers)
    unsigned long long local[kList];                     // this block's elements of the list
    unsigned long long all[kList], sorted[kList];
    unsigned long long warp_sum[kThreads / 32];
    float near_value[kNearMost];
    int near_at[kNearMost];                              // where in the share
    uint32_t n_near;                                     // all of them; kNearMost + 1 where a warp's did not fit
    int warp_near[kThreads / 32];
    unsigned long long rest[3];                          // weights of what is not listed
    uint32_t n_local, lo_key, hi_key, index, ties;
    float top, bound;
    // what a step leaves for all threads
    int bin;
    uint32_t in_bin, up_to;
    unsigned long long before, total;
};

__device__ __forceinline__ uint32_t key_of(float x) { const uint32_t b = __float_as_uint(x + 0.f);      // (one zero)
    return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u); }
__device__ __forceinline__ float value_of(uint32_t k) { return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xffffffffu)); }
__device__ __forceinline__ uint32_t map_to(uint32_t addr, uint32_t rank) {
    uint32_t at;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at) : "r"(addr), "r"(rank));
    return at;
}
__device__ __forceinline__ uint32_t ld_remote(const uint32_t * p, uint32_t rank) {
    uint32_t v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(map_to(smem_u32(p), rank)) : "memory");
    return v;
}
__device__ __forceinline__ unsigned long long ld_remote(const unsigned long long * p, uint32_t rank) {
    unsigned long long v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(map_to(smem_u32(p), rank)) : "memory");
    return v;
}

// A word of every block of the cluster, reduced: one lane per block.
template <class F>
__device__ __forceinline__ uint32_t of_blocks(const uint32_t * p, uint32_t blocks, uint32_t other, F reduce) {
    const uint32_t lane = threadIdx.x % 32;
    return reduce(lane < blocks ? ld_remote(p, lane) : other);
}
__device__ __forceinline__ uint32_t least_of_blocks(const uint32_t * p, uint32_t blocks) {
    return of_blocks(p, blocks, 0xffffffffu, [](uint32_t v) { return __reduce_min_sync(0xffffffffu, v); });
}
__device__ __forceinline__ uint32_t most_of_blocks(const uint32_t * p, uint32_t blocks) {
    return of_blocks(p, blocks, 0u, [](uint32_t v) { return __reduce_max_sync(0xffffffffu, v); });
}

struct Row {
    const float * share;          // this block's logits
    int first, n_share;           // their first index, and how many
    bool wide;                    // whether they begin on 16 bytes
    const float * x;              // those at work: the share (at: nullptr), or the list
    const int * at;
    int here;
    uint32_t rank, blocks;
    Shared & s;
    float top;
    double top64;
    // what is kept so far: logits of at least `least`, and in front of or at (cut, cut_index)
    float least = -INFINITY, cut = -INFINITY;
    uint32_t cut_index = 0;
    bool histogram_used = false, list_used = false;      // whether other blocks may be reading this block's

    __device__ __forceinline__ uint32_t index(int i) const { return uint32_t(first + (at ? at[i] : i)); }
    __device__ __forceinline__ bool kept(float v, int i) const { return v >= least && (v > cut || (v == cut && index(i) <= cut_index && v > -CUDART_INF_F)); }
    __device__ __forceinline__ double gap(float v) const { return v == top ? 0.0 : top64 - double(v); }
    __device__ __forceinline__ int bin(float v) const { return v == top ? 0 : int(fminf((top - v) * kBinsPerNat, float(kFar))); }
    __device__ __forceinline__ int far_bin(float v) const { return int(fminf(fmaxf((top - v) - float(kFar) / kBinsPerNat, 0.f) * kFarBinsPerNat, float(kBins - 1))); }
    // per: log2(e) / T; the weight 2^(45 - gap * per), rounded. 2^-y = 2^-n 2^(-i / 256) 2^-r with y = n + i / 256 + r: a table and the exponential's series to the
    // third power (|r| <= 1/512: what is left out is 1.4e-13 of it)
    __device__ __forceinline__ unsigned long long weight(float v, double per) const { return weight_of(gap(v) * per); }
    __device__ __forceinline__ unsigned long long weight_of(double y) const {
        constexpr double kMagic = 6755399441055744.0, kLn2 = 0.69314718055994530942;      // 1.5 2^52: what is added to it is rounded to a whole number in its low bits
        const bool some = y < 46.0;      // (not so for a NaN either)
        const double at = fma(y, double(kPowers), kMagic);
        const uint32_t k = some ? uint32_t(__double2loint(at)) : 0u;
        const double r = fma(at - kMagic, -1.0 / kPowers, y);
        const double e = fma(fma(fma(r, -kLn2 * kLn2 * kLn2 / 6.0, kLn2 * kLn2 / 2.0), r, -kLn2), r, 1.0) * s.power[k % kPowers];
        const double scaled = fma(e, __hiloint2double(int((1023u + 45u - k / kPowers) << 20), 0), 4503599627370496.0);      // + 2^52
        return some ? (unsigned long long)(__double_as_longlong(scaled)) & 0xfffffffffffffull : 0ull;
    }
};

// f(value, place) for this thread's logits at work: of the share four at a time, with kAhead loads in flight; of a list, what the thread's warp has of it. All lanes
// of a warp make the same calls: what is not there is a NaN, which is larger than nothing, equal to nothing and weighs nothing.
template <int kAhead, class F>
__device__ __forceinline__ void each(const Row & r, F f) {
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const float none = __int_as_float(0x7fffffff);
    if (r.at || !r.wide) {
        const int step = r.at ? 32 : kThreads, begin = r.at ? warp * kPerWarp : warp * 32, end = r.at ? begin + r.here : r.here;
        #pragma unroll 2
        for (int i = begin; i < end; i += step) f(i + lane < end ? r.x[i + lane] : none, i + lane);
        return;
    }
    const int quads = r.here / 4;
    const float4 * x4 = reinterpret_cast<const float4 *>(r.x);
    auto four = [&](float4 v, int i) { f(v.x, 4 * i); f(v.y, 4 * i + 1); f(v.z, 4 * i + 2); f(v.w, 4 * i + 3); };
    int i = warp * 32;
    for (; i + (kAhead - 1) * kThreads + 31 < quads; i += kAhead * kThreads) {
        float4 v[kAhead];
        #pragma unroll
        for (int j = 0; j < kAhead; j++) v[j] = __ldg(x4 + i + lane + j * kThreads);
        #pragma unroll
        for (int j = 0; j < kAhead; j++) four(v[j], i + lane + j * kThreads);
    }
    for (; i < quads; i += kThreads) four(i + lane < quads ? __ldg(x4 + i + lane) : make_float4(none, none, none, none), i + lane);
    if (warp == 0 && 4 * quads < r.here) f(4 * quads + lane < r.here ? r.x[4 * quads + lane] : none, 4 * quads + lane);
}

// The same four at a time: f(values, place of the first).
template <int kAhead, class F>
__device__ __forceinline__ void each_four(const Row & r, F f) {
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const float none = __int_as_float(0x7fffffff);
    if (!r.wide) {
        for (int i = warp * 32; i < r.here; i += kThreads) {
            const float v[4] = {i + lane < r.here ? r.x[i + lane] : none, none, none, none};
            f(v, i + lane);
        }
        return;
    }
    const int quads = (r.here + 3) / 4;
    const float4 * x4 = reinterpret_cast<const float4 *>(r.x);
    for (int i = warp * 32; i < quads; i += kAhead * kThreads) {
        float v[kAhead][4];
        #pragma unroll
        for (int j = 0; j < kAhead; j++) {
            const int q = i + lane + j * kThreads;
            if (4 * q + 3 < r.here) {
                const float4 w = __ldg(x4 + q);
                v[j][0] = w.x; v[j][1] = w.y; v[j][2] = w.z; v[j][3] = w.w;
            } else {
                #pragma unroll
                for (int k = 0; k < 4; k++) v[j][k] = 4 * q + k < r.here ? r.x[4 * q + k] : none;
            }
        }
        #pragma unroll
        for (int j = 0; j < kAhead; j++) f(v[j], 4 * (i + lane + j * kThreads));
    }
}

// Inclusive sums over the block of a value per thread; *total: of all.
__device__ __forceinline__ unsigned long long scan(unsigned long long v, unsigned long long * warp_sum, unsigned long long * total) {
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    #pragma unroll
    for (int d = 1; d < 32; d <<= 1) { const unsigned long long o = __shfl_up_sync(0xffffffffu, v, d); if (lane >= d) v += o; }
    __syncthreads();
    if (lane == 31) warp_sum[warp] = v;
    __syncthreads();
    unsigned long long w = lane < kThreads / 32 ? warp_sum[lane] : 0;
    #pragma unroll
    for (int d = 1; d < kThreads / 32; d <<= 1) { const unsigned long long o = __shfl_up_sync(0xffffffffu, w, d); if (lane >= d) w += o; }
    *total = __shfl_sync(0xffffffffu, w, kThreads / 32 - 1);
    const unsigned long long ahead = __shfl_sync(0xffffffffu, w, max(0, warp - 1));
    return warp ? v + ahead : v;
}

// One element per thread of what the blocks of the cluster have together, `count` of them in each: thread t's is element *at of block *from, if t is less than the
// number that comes back.
__device__ __forceinline__ uint32_t deal(const uint32_t * count, uint32_t blocks, uint32_t * from, uint32_t * at) {
    const uint32_t lane = threadIdx.x % 32;
    uint32_t upto = lane < blocks ? ld_remote(count, lane) : 0u;
    #pragma unroll
    for (int d = 1; d < kMostBlocks; d <<= 1) { const uint32_t o = __shfl_up_sync(0xffffffffu, upto, d); if (lane >= uint32_t(d)) upto += o; }
    *from = 0;
    *at = threadIdx.x;
    #pragma unroll
    for (uint32_t b = 0; b < kMostBlocks - 1; b++) {
        const uint32_t end = __shfl_sync(0xffffffffu, upto, b);
        if (threadIdx.x >= end) { *from = b + 1; *at = threadIdx.x - end; }
    }
    return __shfl_sync(0xffffffffu, upto, kMostBlocks - 1);
}

// The threads' elements (the first n threads have one), largest first, into s.sorted.
__device__ __forceinline__ void sort_list(Shared & s, int n, unsigned long long mine) {
    if (int(threadIdx.x) < n) s.all[threadIdx.x] = mine;
    __syncthreads();
    if (int(threadIdx.x) < n) {
        int ahead = 0;
        #pragma unroll 8
        for (int j = 0; j < n; j++) ahead += s.all[j] > mine;
        s.sorted[ahead] = mine;
    }
    __syncthreads();
}

// All blocks' elements for which take(value, i) holds (at most kList of them over the cluster), sorted, into s.sorted; returns their number.
template <class Take>
__device__ int gather(Row & r, Take take) {
    Shared & s = r.s;
    if (r.list_used) cluster_barrier();      // (others may still read the last one)
    r.list_used = true;
    if (threadIdx.x == 0) s.n_local = 0;
    __syncthreads();
    each<4>(r, [&](float v, int i) {
        if (take(v, i)) {
            const uint32_t n = atomicAdd(&s.n_local, 1u);
            if (n < kList) s.local[n] = (unsigned long long)key_of(v) << 32 | (0xffffffffu - r.index(i));
        }
    });
    cluster_barrier();
    uint32_t from, at;
    const uint32_t n = deal(&s.n_local, r.blocks, &from, &at);
    const unsigned long long mine = threadIdx.x < n ? ld_remote(&s.local[at], from) : 0ull;
    sort_list(s, int(n), mine);
    return int(n);
}

// Where the cumulative weight over the sorted list's first n elements, on top of `before`, reaches goal(total): the element's place (n: nowhere). by_count: one each.
template <class Goal>
__device__ int place_in_list(Row & r, int n, bool by_count, double per, unsigned long long before, Goal goal, unsigned long long * total) {
    Shared & s = r.s;
    const int i = threadIdx.x;
    const unsigned long long own = i < n ? (by_count ? 1ull : r.weight(value_of(uint32_t(s.sorted[i] >> 32)), per)) : 0ull;
    unsigned long long all;
    const unsigned long long upto = before + scan(own, s.warp_sum, &all);
    if (i == 0) s.bin = n;
    __syncthreads();
    *total = before + all;
    const unsigned long long g = goal(before + all);
    if (i < n && upto >= g && upto - own < g) s.bin = i;
    __syncthreads();
    return s.bin;      // (written again only behind a barrier)
}

// A histogram over the kept elements that in(v) takes, by bin_of(v); leaves in s the first bin where the cumulative weight on top of `before` reaches
// goal(total), what is in front of it, and how many elements it holds, and it and the bins in front. s.bin = kBins: the goal is not reached.
// kSumFar: bin kFar is added up in registers (an atomic per element of the many that lie there would be the longest part of the whole row).
// beyond: weights that are in none of the bins and behind all of them.
template <bool kSumFar, class In, class BinOf, class Goal>
__device__ void histogram(Row & r, bool by_count, double per, unsigned long long before, unsigned long long beyond, In in, BinOf bin_of, Goal goal) {
    Shared & s = r.s;
    if (r.histogram_used) cluster_barrier();      // (others may still read the last one)
    r.histogram_used = true;
    if (threadIdx.x < kBins) s.count[threadIdx.x] = s.low[threadIdx.x] = s.high[threadIdx.x] = 0;
    __syncthreads();
    auto add = [&](int b, uint32_t elements, unsigned long long w) {
        atomicAdd(&s.count[b], elements);
        if (!by_count) {      // two words: the low one's overflow is carried into the high one
            const uint32_t low = uint32_t(w), was = atomicAdd(&s.low[b], low), high = uint32_t(w >> 32) + (was + low < was ? 1u : 0u);
            if (high) atomicAdd(&s.high[b], high);
        }
    };
    uint32_t far = 0;
    unsigned long long far_weight = 0;
    each<2>(r, [&](float v, int i) {
        if (!r.kept(v, i) || !in(v)) return;
        const int b = bin_of(v);
        const unsigned long long w = by_count ? 0ull : r.weight(v, per);
        if (kSumFar && b == kFar && !r.at) { far++; far_weight += w; }
        else add(b, 1u, w);
    });
    if (kSumFar) {
        #pragma unroll
        for (int d = 16; d; d >>= 1) far_weight += __shfl_xor_sync(0xffffffffu, far_weight, d);
        far = __reduce_add_sync(0xffffffffu, far);
        if (threadIdx.x % 32 == 0 && far) add(kFar, far, far_weight);
    }
    cluster_barrier();
    unsigned long long m = 0;
    uint32_t c = 0;
    if (threadIdx.x < kBins) {
        const int b = threadIdx.x;
        #pragma unroll 8
        for (uint32_t blk = 0; blk < r.blocks; blk++) {
            c += ld_remote(&s.count[b], blk);
            if (!by_count) m += ((unsigned long long)ld_remote(&s.high[b], blk) << 32) + ld_remote(&s.low[b], blk);
        }
        if (by_count) m = c;
    }
    unsigned long long total, elements = 0;
    const unsigned long long upto = before + scan(m, s.warp_sum, &total);
    total += before + beyond;
    if (threadIdx.x == 0) { s.total = total; s.bin = kBins; }
    const unsigned long long up_to = by_count ? upto - before : scan(c, s.warp_sum, &elements);
    __syncthreads();
    const unsigned long long g = goal(total);
    if (upto >= g && upto - m < g) {
        s.bin = threadIdx.x;
        s.before = upto - m;
        s.in_bin = c;
        s.up_to = uint32_t(up_to);
    }
    __syncthreads();
}

// The element at which the cumulative weight over what is kept, past the histogram that is in s, reaches the goal: as its (value, index). The goal is reached in the
// histogram's bin s.bin, whose elements in_bin takes.
template <class InBin>
__device__ void resolve(Row & r, bool by_count, double per, unsigned long long goal, InBin in_bin, float * value, uint32_t * index) {
    Shared & s = r.s;
    unsigned long long before = s.before;
    uint32_t count = s.in_bin, lo = 0, hi = 0xffffffffu;
    auto in = [&](float v) { const uint32_t k = key_of(v); return k >= lo && k <= hi && in_bin(v); };
    while (count > kList) {
        cluster_barrier();
        if (threadIdx.x == 0) { s.lo_key = 0xffffffffu; s.hi_key = 0; }
        __syncthreads();
        uint32_t l = 0xffffffffu, h = 0;
        each<2>(r, [&](float v, int i) { if (r.kept(v, i) && in(v)) { l = min(l, key_of(v)); h = max(h, key_of(v)); } });
        l = __reduce_min_sync(0xffffffffu, l);
        h = __reduce_max_sync(0xffffffffu, h);
        if (threadIdx.x % 32 == 0) { atomicMin(&s.lo_key, l); atomicMax(&s.hi_key, h); }
        cluster_barrier();
        lo = least_of_blocks(&s.lo_key, r.blocks);
        hi = most_of_blocks(&s.hi_key, r.blocks);
        if (lo == hi) {      // one value: the goal falls on its m-th element in the order of the indices
            const unsigned long long w = by_count ? 1ull : r.weight(value_of(lo), per), m = (goal - before + w - 1) / w;
            r.x = r.share; r.at = nullptr; r.here = r.n_share;      // (in order, as a list is not; the value says which bin)
            uint32_t mine = 0;
            each<2>(r, [&](float v, int i) { mine += r.kept(v, i) && key_of(v) == lo; });
            if (threadIdx.x == 0) { s.ties = 0; s.index = 0xffffffffu; }
            __syncthreads();
            mine = __reduce_add_sync(0xffffffffu, mine);
            if (threadIdx.x % 32 == 0) atomicAdd(&s.ties, mine);
            cluster_barrier();
            unsigned long long seen = 0;
            for (uint32_t b = 0; b < r.rank; b++) seen += ld_remote(&s.ties, b);
            if (seen < m && m <= seen + s.ties) {
                for (int base = 0; base < r.here; base += kThreads) {
                    const int i = base + threadIdx.x;
                    const bool is = i < r.here && r.kept(r.x[i], i) && key_of(r.x[i]) == lo;
                    unsigned long long here;
                    const unsigned long long at = seen + scan(is, s.warp_sum, &here);
                    if (is && at == m) s.index = uint32_t(r.first + i);
                    seen += here;
                    if (seen >= m) break;
                }
            }
            cluster_barrier();
            *value = value_of(lo);
            *index = least_of_blocks(&s.index, r.blocks);
            return;
        }
        const int shift = max(0, 32 - __clz(hi - lo) - 8);
        const uint32_t top = hi;
        histogram<false>(r, by_count, per, before, 0, in, [&](float v) { return int((top - key_of(v)) >> shift); }, [&](unsigned long long) { return goal; });
        before = s.before;
        count = s.in_bin;
        hi = top - (uint32_t(s.bin) << shift);
        lo = max(lo, hi - min(hi, (1u << shift) - 1u));
    }
    const int n = gather(r, [&](float v, int i) { return r.kept(v, i) && in(v); });
    unsigned long long total;
    const int at = place_in_list(r, n, by_count, per, before, [&](unsigned long long) { return goal; }, &total);
    const unsigned long long e = s.sorted[min(at, max(n - 1, 0))];
    *value = value_of(uint32_t(e >> 32));
    *index = 0xffffffffu - uint32_t(e);
}

__global__ void __launch_bounds__(kThreads, 2) k_sample_rows(const SampleArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    Shared & s = *reinterpret_cast<Shared *>(smem);
    // With two launches the second may start as soon as the first's blocks have, which is when what both read is there; it waits for the first at its end. What follows the
    // call in the stream is the caller's (and may be a programmatic dependent that does not wait before it reads): it is released by the last launch's finishing alone.
    if (a.rows_of != kOpenRows) pdl_wait();
    if (a.rows_of == kBoundedRows) pdl_trigger();
    uint32_t rank, blocks;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(blocks));
    const int row = int(blockIdx.x / blocks), warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int first = int(rank) * a.slice, here = max(0, min(a.slice, a.n - first));
    const float * from = a.logits + int64_t(row) * a.stride + first;
    const bool wide = (reinterpret_cast<uintptr_t>(from) & 15u) == 0;
    const float t = a.temperature ? a.temperature[row] : 1.f, top_p = a.top_p ? a.top_p[row] : 1.f, min_p = a.min_p ? a.min_p[row] : 0.f, uniform = a.uniform[row];
    const int k = a.top_k ? a.top_k[row] : 0;
    // (a min-p above 1 is reached by no token: the first alone is kept, as of a temperature of 0)
    const bool greedy = !(t > 0.f) || min_p > 1.f, by_k = k > 0 && k < a.n, by_p = top_p < 1.f, by_m = min_p > 0.f;
    // open: a total of everything is needed. sampled: what is listed there, and for a top-k of more than there are threads, is what lies above the least of the warps' m-th
    // largest of the threads' largest of kSamples logits each: a share of the row that does not depend on what its logits are like.
    const bool open = !greedy && !by_k && (by_p || !by_m), sampled = open || (!greedy && by_k && k > kThreads), bounded = !greedy && (open || by_k);
    // (rows of the other launch: their clusters leave at once)
    if (a.rows_of != kAllRows && open != (a.rows_of == kOpenRows)) { if (a.rows_of == kOpenRows) pdl_wait(); return; }
    if (threadIdx.x < kPowers) s.power[threadIdx.x] = exp2(double(threadIdx.x) * (-1.0 / kPowers));
    if (threadIdx.x == 0) { s.n_near = 0; s.index = 0xffffffffu; }

    // ---- the first pass: every thread's largest logit, and with them the row's ----
    Row r{from, first, here, wide, from, nullptr, here, rank, blocks, s, 0.f, 0.0};
    float mine = -CUDART_INF_F, sample = -CUDART_INF_F;
    uint32_t mine_at = 0xffffffffu;
    if (greedy) each<8>(r, [&](float v, int i) { if (v > mine) { mine = v; mine_at = uint32_t(first + i); } });      // (a NaN loses, and the first of equal ones wins)
    else if (!sampled) each<8>(r, [&](float v, int) { mine = fmaxf(mine, v); });
    else each<8>(r, [&](float v, int i) {
        mine = fmaxf(mine, v);
        if (i % 4 == 0 && (i / (4 * kThreads) & (a.sample_every - 1)) == 0) sample = fmaxf(sample, v);
    });
    float top = mine;
    #pragma unroll
    for (int m = 16; m; m >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
    // A bound for a top-k: if every warp has m = k / 16 (rounded up) threads with a logit of at least b, the row has k of them. b: the least of the warps' m-th largest.
    float bound = -CUDART_INF_F;
    if (bounded) {
        float v = sampled ? sample : mine;      // sorted over the lanes, largest first
        #pragma unroll
        for (int size = 2; size <= 32; size *= 2) {
            #pragma unroll
            for (int d = size / 2; d; d /= 2) {
                const float o = __shfl_xor_sync(0xffffffffu, v, d);
                const bool larger_first = ((lane & size & 31) == 0) == ((lane & d) == 0);
                v = larger_first ? fmaxf(v, o) : fminf(v, o);
            }
        }
        bound = __shfl_sync(0xffffffffu, v, sampled ? a.sample_rank - 1 : (k + kThreads / 32 - 1) / (kThreads / 32) - 1);
    }
    float2 * const tops = reinterpret_cast<float2 *>(s.warp_sum);
    if (lane == 0) tops[warp] = make_float2(top, bound);
    __syncthreads();
    if (warp == 0) {
        const float2 v = tops[lane % (kThreads / 32)];
        top = v.x;
        bound = v.y;
        #pragma unroll
        for (int m = kThreads / 64; m; m >>= 1) { top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m)); bound = fminf(bound, __shfl_xor_sync(0xffffffffu, bound, m)); }
        if (lane == 0) { s.top = top; s.bound = bound; }
    }
    cluster_barrier();
    top = lane < int(blocks) ? ld_cluster(smem_u32(&s.top), lane) : -CUDART_INF_F;
    bound = lane < int(blocks) ? ld_cluster(smem_u32(&s.bound), lane) : -CUDART_INF_F;      // (each block's holds for the row)
    #pragma unroll
    for (int m = kMostBlocks / 2; m; m >>= 1) { top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m)); bound = fmaxf(bound, __shfl_xor_sync(0xffffffffu, bound, m)); }
    top = __shfl_sync(0xffffffffu, top, 0);
    bound = __shfl_sync(0xffffffffu, bound, 0);
    r.top = top;
    r.top64 = double(top);

    uint32_t token = 0;
    double chance = 1.0;
    if (!(top > -CUDART_INF_F) || greedy) {
        // the lowest index of the largest logit; a row with nothing above the lowest: the first that is a number, with nothing to draw
        uint32_t found = mine == top ? mine_at : 0xffffffffu;
        if (!(top > -CUDART_INF_F)) { found = 0xffffffffu; each<8>(r, [&](float v, int i) { if (v == v) found = min(found, uint32_t(first + i)); }); }
        found = __reduce_min_sync(0xffffffffu, found);
        if (lane == 0) atomicMin(&s.index, found);
        cluster_barrier();
        token = least_of_blocks(&s.index, blocks);
        if (token == 0xffffffffu) token = 0;
        chance = top > -CUDART_INF_F ? 1.0 : 0.0;
    } else {
        constexpr double kLog2e = 1.4426950408889634074;
        const double per_t = kLog2e / double(t);
        // min-p as the least logit kept: the smallest float whose gap is within -log(min_p)
        float least = -CUDART_INF_F;
        if (top == CUDART_INF_F) {
            least = top;      // an infinity takes all
        } else if (by_m) {
            const double limit = min_p == 1.f ? 0.0 : -log(double(min_p));
            least = __double2float_ru(double(top) - limit);
            while (r.gap(least) > limit) least = nextafterf(least, CUDART_INF_F);
        }
        auto p_goal = [&](unsigned long long total) { return max(1ull, min(total, (unsigned long long)(ceil(double(top_p) * double(total))))); };
        auto u_goal = [&](unsigned long long total) {
            const double u = double(uniform) * double(total);
            return u > 0.0 ? min(total, (unsigned long long)u + 1ull) : 1ull;
        };
        // The list: every warp appends to a piece of its own, so that no counter is shared.
        int listed_here = 0;
        auto append = [&](bool take, float v, int i) {
            const uint32_t m = __ballot_sync(0xffffffffu, take);
            if (m) {
                const int at = listed_here + __popc(m & ((1u << lane) - 1u));
                if (take && at < kPerWarp) { s.near_value[warp * kPerWarp + at] = v; s.near_at[warp * kPerWarp + at] = i; }
                listed_here += __popc(m);
            }
        };
        bool lists_made = false;
        auto list_begin = [&] {
            if (lists_made) cluster_barrier();      // (others may still read the last one's number)
            lists_made = true;
            __syncthreads();
            if (threadIdx.x == 0) s.n_near = 0;
            __syncthreads();
            listed_here = 0;
        };
        auto list_end = [&] {
            if (lane == 0) atomicAdd(&s.n_near, listed_here > kPerWarp ? uint32_t(kNearMost + 1) : uint32_t(listed_here));
            listed_here = min(listed_here, kPerWarp);
        };
        auto use_list = [&] { r.x = s.near_value; r.at = s.near_at; r.here = listed_here; };

        auto sorted_up_to = [&](int to) { return gather(r, [&](float v, int i) { return r.kept(v, i) && r.bin(v) <= to; }); };
        bool listed = false;
        int n = 0;
        unsigned long long total_p = 0;
        float cut;
        uint32_t index;
        auto use_share = [&] { r.x = r.share; r.at = nullptr; r.here = r.n_share; };
        auto fits = [&] { return most_of_blocks(&s.n_near, blocks) <= kNearMost; };

        // ---- a top-k's bound, or a min-p alone, says at once what to look at ----
        const bool alone = least > -CUDART_INF_F && !by_k && !by_p;
        const float near = alone ? least : fmaxf(bound, -3.402823466e38f);
        if (alone || by_k) {
            list_begin();
            each<4>(r, [&](float v, int i) { append(v >= near, v, i); });
            list_end();
            cluster_barrier();
            const uint32_t n_near = of_blocks(&s.n_near, blocks, 0u, [](uint32_t v) { return __reduce_add_sync(0xffffffffu, v); });
            if (fits() && (!sampled || n_near >= uint32_t(k))) use_list();      // (sampled: a top-k's, and not sure to hold it)
            if (n_near <= kList && !sampled) {
                n = gather(r, [](float v, int) { return v == v; });
                listed = true;
            }
        }

        // A cut over what is kept. Of a list: the histogram. Of the share, by count: the histogram, its far bin divided if the goal falls there; what is in front of the goal
        // becomes the list where it fits. Of the share, by weight: one pass without a branch adds up the weights below three steps down from the bound and lists what
        // is above it; if the goal is in front of the end of one of the steps, that step is listed; if it is further down, the next three steps are weighed; where that ends
        // (or the first list does not fit), the histogram of the share. (With that histogram for everything below the first steps a single row that drew from there kept
        // 256 rows of a mix waiting: 246 us against 203.) Then the element.
        int where = 0;      // what the histogram was of: 0 bins from the largest logit down, 1 the far bin's, 2 a step's
        float step_top = 0.f, step_scale = 0.f, step_end = 0.f;
        auto step_bin = [&](float v) { return int(fminf((step_top - v) * step_scale, float(kBins - 1))); };
        auto every = [](float) { return true; };
        auto from_top = [&](float v) { return r.bin(v); };
        auto divide = [&](bool by_count, double per, auto goal) {
            where = 0;
            if (!r.at && !by_count) {
                const float nat = float(kLog2e / per);
                unsigned long long all = 0, g = 0, below = 0;       // below: the weights below `from`
                float from = near;
                for (int turn = 0; turn < kTurns; turn++) {
                    // the weights below three ends; in the first turn what is above the first is listed
                    const float width = turn ? 0.9f * nat : 0.8f * nat, end[3] = {turn ? from - width : from, turn ? from - 2.f * width : from - width, turn ? from - 3.f * width : from - 2.f * width};
                    unsigned long long rest[3] = {0, 0, 0};
                    list_begin();
                    if (threadIdx.x < 3) s.rest[threadIdx.x] = 0;
                    each_four<2>(r, [&](const float (&v)[4], int i) {
                        bool kept[4];
                        unsigned long long w[4];
                        #pragma unroll
                        for (int j = 0; j < 4; j++) {
                            kept[j] = r.kept(v[j], i + j);
                            w[j] = r.weight_of(kept[j] ? (r.top64 - double(v[j])) * per : 64.0);
                        }
                        #pragma unroll
                        for (int j = 0; j < 4; j++) {
                            #pragma unroll
                            for (int e = 0; e < 3; e++) rest[e] += v[j] < end[e] ? w[j] : 0ull;
                        }
                        if (turn == 0) {
                            #pragma unroll
                            for (int j = 0; j < 4; j++) append(kept[j] && v[j] >= near, v[j], i + j);
                        }
                    });
                    __syncthreads();
                    #pragma unroll
                    for (int e = 0; e < 3; e++) {
                        #pragma unroll
                        for (int d = 16; d; d >>= 1) rest[e] += __shfl_xor_sync(0xffffffffu, rest[e], d);
                        if (lane == 0) atomicAdd(&s.rest[e], rest[e]);
                    }
                    list_end();
                    cluster_barrier();
                    #pragma unroll
                    for (int e = 0; e < 3; e++) {
                        rest[e] = lane < int(blocks) ? ld_remote(&s.rest[e], lane) : 0ull;
                        #pragma unroll
                        for (int d = kMostBlocks / 2; d; d >>= 1) rest[e] += __shfl_xor_sync(0xffffffffu, rest[e], d);
                        rest[e] = __shfl_sync(0xffffffffu, rest[e], 0);
                    }
                    if (turn == 0) {
                        if (!fits()) break;
                        use_list();
                        histogram<false>(r, false, per, 0, rest[0], every, from_top, goal);
                        if (s.bin < kBins) return;
                        all = s.total;
                        g = goal(all);
                        use_share();
                        below = rest[0];
                    }
                    // the step, from `from` down to an end, that the goal falls in
                    unsigned long long below_end = below;
                    step_end = from;
                    bool found = false;
                    #pragma unroll
                    for (int e = 0; e < 3; e++) {
                        if (!found) {
                            below = below_end;
                            from = step_end;
                            step_end = end[e];
                            below_end = rest[e];
                            found = g <= all - below_end;
                        }
                    }
                    if (found) {
                        where = 2;
                        step_top = from;
                        step_scale = float(kBins) / (step_top - step_end);
                        list_begin();
                        each<4>(r, [&](float v, int i) { append(v < step_top && v >= step_end && r.kept(v, i), v, i); });
                        list_end();
                        cluster_barrier();
                        if (fits()) use_list();
                        histogram<false>(r, false, per, all - below, below_end, [&](float v) { return v < step_top && v >= step_end; }, step_bin, goal);
                        return;
                    }
                    from = step_end;
                    below = below_end;
                }
            }
            if (r.at) {
                histogram<false>(r, by_count, per, 0, 0, every, from_top, goal);
                return;
            }
            histogram<true>(r, by_count, per, 0, 0, every, from_top, goal);
            if (s.bin == kFar) {
                where = 1;
                histogram<false>(r, by_count, per, s.before, 0, [&](float v) { return r.bin(v) == kFar; }, [&](float v) { return r.far_bin(v); }, goal);
            } else if (s.bin < kBins && s.up_to > kList && s.up_to <= kNearMost) {
                const int to = s.bin;
                list_begin();
                each<4>(r, [&](float v, int i) { append(r.kept(v, i) && r.bin(v) <= to, v, i); });
                list_end();
                cluster_barrier();
                if (fits()) use_list();
            }
        };
        auto element = [&](bool by_count, double per, unsigned long long goal, float * value, uint32_t * index) {
            const int bin = s.bin, w = where;
            resolve(r, by_count, per, goal, [&](float v) {
                return w == 0 ? r.bin(v) == bin : w == 1 ? r.bin(v) == kFar && r.far_bin(v) == bin : v < step_top && v >= step_end && step_bin(v) == bin;
            }, value, index);
            if (w != 0) use_share();      // (a step's list is not all that is kept)
        };
        if (by_k && !listed) {
            divide(true, 0.0, [&](unsigned long long) { return (unsigned long long)k; });
            if (s.bin < kBins) {
                listed = where == 0 && s.up_to <= kList;
                if (listed) n = sorted_up_to(s.bin);
                else { element(true, 0.0, (unsigned long long)k, &cut, &index); r.cut = cut; r.cut_index = index; }
            }
        }
        if (by_p && !listed) {
            divide(false, kLog2e, p_goal);
            total_p = s.total;
            listed = where == 0 && s.up_to <= kList;
            if (listed) n = sorted_up_to(s.bin);
            else { element(false, kLog2e, p_goal(total_p), &cut, &index); r.cut = cut; r.cut_index = index; }
        }
        if (listed) {
            if (by_k) n = min(n, k);
            unsigned long long total;
            if (by_p) {
                const unsigned long long given = total_p;
                const int at = place_in_list(r, n, false, kLog2e, 0, [&](unsigned long long sum) { return p_goal(given ? given : sum); }, &total);
                n = min(n, at + 1);
            }
            n = max(1, min(n, __syncthreads_count(int(threadIdx.x) < n && value_of(uint32_t(s.sorted[threadIdx.x] >> 32)) >= least)));
            const int at = min(place_in_list(r, n, false, per_t, 0, u_goal, &total), n - 1);
            const unsigned long long e = s.sorted[at];
            token = 0xffffffffu - uint32_t(e);
            chance = double(r.weight(value_of(uint32_t(e >> 32)), per_t)) / double(total);
        } else {
            r.least = least;
            divide(false, per_t, u_goal);
            const unsigned long long total = s.total;
            element(false, per_t, u_goal(total), &cut, &token);
            chance = double(r.weight(cut, per_t)) / double(total);
        }
    }
    if (rank == 0 && threadIdx.x == 0) {
        a.tokens[row] = int32_t(token);
        if (a.probability) a.probability[row] = float(chance);
    }
    cluster_barrier();      // no block leaves while another reads its shared memory
    if (a.rows_of == kOpenRows) pdl_wait();      // the first launch's rows are done when this one is
}

}  // namespace

int sample_rows_most() { return kMostLogits; }

cudaError_t launch_sample_rows(const float * logits, int64_t stride, int rows, int n, const float * temperature, const int32_t * top_k, const float * top_p, const float * min_p,
                               const float * uniform, int32_t * tokens, float * probability, cudaStream_t stream) {
    if (n < 1 || n > kMostLogits) return cudaErrorInvalidValue;
    constexpr int bytes = int(sizeof(Shared));
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_dynamic_smem(k_sample_rows, bytes, done);
    if (e != cudaSuccess) return e;
    // As many blocks per row, each of at least 2048 logits, as make up to `most` in all: a cluster costs a row its barriers, but a block alone leaves a row that needs a total
    // of everything to itself.
    auto blocks_for = [&](int64_t most) {
        int blocks = 1;
        while (blocks < kMostBlocks && n > blocks * 2048 && int64_t(rows) * blocks * 2 <= most) blocks *= 2;
        return blocks;
    };
    auto go = [&](int rows_of, int blocks) {
        const int slice = ((n + blocks - 1) / blocks + 3) & ~3;      // (whole 16 bytes, so that every block's share begins as the row does)
        const double groups = slice / 4.0 / kThreads, share = std::min(0.1, 0.5 * kNearMost / slice);
        int every = 1;
        while (every * 2 * kSamples <= groups) every *= 2;
        const int samples = std::max(1, int(groups / every)), rank = std::clamp(int(32.0 * (1.0 - std::pow(1.0 - share, samples))), 1, 32);
        const SampleArgs a{logits, stride, n, slice, every, rank, temperature, top_p, min_p, uniform, top_k, tokens, probability, rows_of};
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(unsigned(rows) * unsigned(blocks));
        cfg.blockDim = dim3(kThreads);
        cfg.dynamicSmemBytes = size_t(bytes);
        cfg.stream = stream;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = unsigned(blocks);
        attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = 1;
        cfg.attrs = attr;
        cfg.numAttrs = pdl_enabled() ? 2 : 1;
        return cudaLaunchKernelEx(&cfg, k_sample_rows, a);
    };
    const int all = blocks_for(4 * sm_count()), open = std::max(all, std::min(blocks_for(INT64_MAX), 4));
    if (all == open) return go(kAllRows, all);
    // Too many rows for four blocks each: those that a bound leaves little of get fewer, the others four, in two launches that overlap. Rows x logits, mix of filters /
    // nucleus alone, with eight blocks for the open rows against four, in us: 256 x 32000 139 / 322 against 98 / 147, 256 x 128256 232 / 506 against 206 / 304,
    // 128 x 151936 (four fit all rows, one launch) 151 / 275 against 128 / 203. Four for all 256 rows: 95 for top-k 40 alone, two: 59.
    e = go(kBoundedRows, all);
    return e == cudaSuccess ? go(kOpenRows, open) : e;
}

}  // namespace cuda
}  // namespace dooms
