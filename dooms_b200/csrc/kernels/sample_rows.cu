// One token per row of logits from given random numbers: top-k, then top-p and min-p on the probabilities at temperature 1, then the temperature, then the draw (the
// order of the host sampler's chain). In the order (logit descending, index ascending), with the row's largest logit m and g = m - l:
//   kept by top-k: the first k;  by top-p: while what is in front of a token holds less than top_p of the mass e^-g of what top-k kept;  by min-p: e^-g >= min_p;
//   the token: the first whose cumulative weight e^(-g / T) exceeds u times the kept tokens' total.
//
// A row belongs to a cluster of up to eight blocks; each holds its share of the logits in shared memory, so that they are read once. No sort of the row: a cut
// ("the first element at which a cumulative weight reaches a goal") is found by a histogram of 1/8 nat per bin over all blocks of the cluster, then by sorting
// the few elements of the bin where the goal falls (or of all bins up to there, where they are few: then everything else is decided in that list too). A bin of
// more than kList elements (flat logits, or many equal ones) is divided again by the bits of the logits, down to a single value, whose elements are then
// counted out in the order of their indices.
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
constexpr int kMostSlice = 32768;      // logits per block
constexpr float kBinsPerNat = 8.f;
constexpr int kNearBins = 48;          // a short top-k is looked for among the logits less than 6 below the largest first
constexpr double kNoLimit = 1e300;     // (gaps are below 2^129, or infinite)
static_assert(kList == kThreads && kBins <= kThreads, "one list element and at most one bin per thread");

struct SampleArgs {
    const float * logits;
    int64_t stride;
    int n, slice;
    const float * temperature, * top_p, * min_p, * uniform;
    const int32_t * top_k;
    int32_t * tokens;
    float * probability;
};

struct Shared {
    uint32_t count[kBins], low[kBins], high[kBins];      // this block's histogram: elements, and their weights in two words
    double power[64];                                    // 2^(-i / 64)
    unsigned long long local[kList];                     // this block's elements of the list
    unsigned long long all[kList], sorted[kList];
    unsigned long long warp_sum[kThreads / 32];
    uint32_t n_local, lo_key, hi_key, index, ties;
    float top;
    // what a step leaves for all threads
    int bin;
    uint32_t in_bin, up_to;
    unsigned long long before, total;
};

__device__ __forceinline__ uint32_t key_of(float x) { const uint32_t b = __float_as_uint(x); return b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u); }
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

struct Row {
    const float * x;              // this block's logits in shared memory
    int first, here;              // their first index, and how many
    uint32_t rank, blocks;
    Shared & s;
    float top;
    double top64;
    // what is kept so far: logits of at least `least`, and in front of or at (cut, cut_index)
    float least = -INFINITY, cut = -INFINITY;
    uint32_t cut_index = 0;
    bool histogram_used = false, list_used = false;      // whether other blocks may be reading this block's

    __device__ __forceinline__ bool kept(float v, int i) const { return v >= least && (v > cut || (v == cut && uint32_t(first + i) <= cut_index && v > -CUDART_INF_F)); }
    __device__ __forceinline__ double gap(float v) const { return v == top ? 0.0 : top64 - double(v); }
    __device__ __forceinline__ int bin(float v) const { return v == top ? 0 : int(fminf((top - v) * kBinsPerNat, float(kBins - 1))); }
    // per: log2(e) / T; the weight 2^(45 - gap * per), rounded. 2^-y = 2^-n 2^(-i / 64) 2^-r with y = n + i / 64 + r: a table and the exponential's series to the
    // fourth power (|r| <= 1/128: what is left out is 4e-14 of it)
    __device__ __forceinline__ unsigned long long weight(float v, double per) const {
        const double y = gap(v) * per;
        if (!(y < 46.0)) return 0ull;
        constexpr double kMagic = 6755399441055744.0, kLn2 = 0.69314718055994530942;      // 1.5 2^52: what is added to it is rounded to a whole number in its low bits
        const double at = fma(y, 64.0, kMagic);
        const uint32_t k = uint32_t(__double2loint(at));
        const double r = fma(at - kMagic, -1.0 / 64.0, y) * -kLn2;
        const double e = fma(fma(fma(fma(r, 1.0 / 24.0, 1.0 / 6.0), r, 0.5), r, 1.0), r, 1.0) * s.power[k & 63u];
        const double scaled = fma(e, __hiloint2double(int((1023u + 45u - (k >> 6)) << 20), 0), 4503599627370496.0);      // + 2^52
        return (unsigned long long)(__double_as_longlong(scaled)) & 0xfffffffffffffull;
    }
};

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

// All blocks' elements for which take(value, i) holds (at most kList of them over the cluster), sorted, into s.sorted; returns their number.
template <class Take>
__device__ int gather(Row & r, Take take) {
    Shared & s = r.s;
    if (r.list_used) cluster_barrier();      // (others may still read the last one)
    r.list_used = true;
    if (threadIdx.x == 0) s.n_local = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < r.here; i += kThreads) {
        const float v = r.x[i];
        if (take(v, i)) s.local[atomicAdd(&s.n_local, 1u)] = (unsigned long long)key_of(v) << 32 | (0xffffffffu - uint32_t(r.first + i));
    }
    cluster_barrier();
    // one element per thread: where it is, from the blocks' counts
    uint32_t n = 0, from = 0, at = 0;
    for (uint32_t b = 0; b < r.blocks; b++) {
        const uint32_t m = ld_remote(&s.n_local, b);
        if (threadIdx.x >= n && threadIdx.x < n + m) { from = b; at = threadIdx.x - n; }
        n += m;
    }
    unsigned long long mine = 0;
    if (threadIdx.x < n) s.all[threadIdx.x] = mine = ld_remote(&s.local[at], from);
    __syncthreads();
    if (threadIdx.x < n) {
        uint32_t ahead = 0;
        #pragma unroll 8
        for (uint32_t j = 0; j < n; j++) ahead += s.all[j] > mine;
        s.sorted[ahead] = mine;
    }
    __syncthreads();
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
template <class In, class BinOf, class Goal>
__device__ void histogram(Row & r, bool by_count, double per, unsigned long long before, In in, BinOf bin_of, Goal goal) {
    Shared & s = r.s;
    if (r.histogram_used) cluster_barrier();      // (others may still read the last one)
    r.histogram_used = true;
    if (threadIdx.x < kBins) s.count[threadIdx.x] = s.low[threadIdx.x] = s.high[threadIdx.x] = 0;
    __syncthreads();
    #pragma unroll 2
    for (int i = threadIdx.x; i < r.here; i += kThreads) {
        const float v = r.x[i];
        if (!r.kept(v, i) || !in(v)) continue;
        const int b = bin_of(v);
        atomicAdd(&s.count[b], 1u);
        if (!by_count) {      // two words: the low one's overflow is carried into the high one
            const unsigned long long w = r.weight(v, per);
            const uint32_t low = uint32_t(w), was = atomicAdd(&s.low[b], low), high = uint32_t(w >> 32) + (was + low < was ? 1u : 0u);
            if (high) atomicAdd(&s.high[b], high);
        }
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
    total += before;
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

// The element at which the cumulative weight over what is kept, past the histogram that is in s, reaches the goal: as its (value, index). The goal is reached.
__device__ void resolve(Row & r, bool by_count, double per, unsigned long long goal, float * value, uint32_t * index) {
    Shared & s = r.s;
    const int bin = s.bin;
    unsigned long long before = s.before;
    uint32_t count = s.in_bin, lo = 0, hi = 0xffffffffu;
    auto in = [&](float v) { const uint32_t k = key_of(v); return r.bin(v) == bin && k >= lo && k <= hi; };
    while (count > kList) {
        cluster_barrier();
        if (threadIdx.x == 0) { s.lo_key = 0xffffffffu; s.hi_key = 0; }
        __syncthreads();
        uint32_t l = 0xffffffffu, h = 0;
        for (int i = threadIdx.x; i < r.here; i += kThreads) {
            const float v = r.x[i];
            if (r.kept(v, i) && in(v)) { l = min(l, key_of(v)); h = max(h, key_of(v)); }
        }
        l = __reduce_min_sync(0xffffffffu, l);
        h = __reduce_max_sync(0xffffffffu, h);
        if (threadIdx.x % 32 == 0) { atomicMin(&s.lo_key, l); atomicMax(&s.hi_key, h); }
        cluster_barrier();
        lo = 0xffffffffu;
        hi = 0;
        for (uint32_t b = 0; b < r.blocks; b++) { lo = min(lo, ld_remote(&s.lo_key, b)); hi = max(hi, ld_remote(&s.hi_key, b)); }
        if (lo == hi) {      // one value: the goal falls on its m-th element in the order of the indices
            const unsigned long long w = by_count ? 1ull : r.weight(value_of(lo), per), m = (goal - before + w - 1) / w;
            uint32_t mine = 0;
            for (int i = threadIdx.x; i < r.here; i += kThreads) mine += r.kept(r.x[i], i) && key_of(r.x[i]) == lo;
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
            uint32_t found = 0xffffffffu;
            for (uint32_t b = 0; b < r.blocks; b++) found = min(found, ld_remote(&s.index, b));
            *value = value_of(lo);
            *index = found;
            return;
        }
        const int shift = max(0, 32 - __clz(hi - lo) - 8);
        const uint32_t top = hi;
        histogram(r, by_count, per, before, in, [&](float v) { return int((top - key_of(v)) >> shift); }, [&](unsigned long long) { return goal; });
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
    float * const x = reinterpret_cast<float *>(smem + (sizeof(Shared) + 15) / 16 * 16);
    uint32_t rank, blocks;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(blocks));
    const int row = int(blockIdx.x / blocks);
    const float * logits = a.logits + int64_t(row) * a.stride;
    const int first = int(rank) * a.slice, here = max(0, min(a.slice, a.n - first));
    const float * from = logits + first;
    // the share of the row into shared memory, 16 bytes at a time where it begins on such a boundary
    const bool wide = (reinterpret_cast<uintptr_t>(from) & 15u) == 0;
    const int quads = wide ? here / 4 : 0;
    for (int i = threadIdx.x; i < quads; i += kThreads) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(x + 4 * i)), "l"(from + 4 * i) : "memory");
    for (int i = 4 * quads + threadIdx.x; i < here; i += kThreads) asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(smem_u32(x + i)), "l"(from + i) : "memory");
    if (threadIdx.x < 64) s.power[threadIdx.x] = exp2(double(threadIdx.x) * (-1.0 / 64.0));
    const float t = a.temperature ? a.temperature[row] : 1.f, top_p = a.top_p ? a.top_p[row] : 1.f, min_p = a.min_p ? a.min_p[row] : 0.f, uniform = a.uniform[row];
    const int k = a.top_k ? a.top_k[row] : 0;
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();
    float top = -CUDART_INF_F;
    #pragma unroll 4
    for (int i = threadIdx.x; i < here; i += kThreads) {
        float v = x[i] + 0.f;                           // (one zero)
        v = v == v ? v : -CUDART_INF_F;                 // a NaN never wins
        x[i] = v;
        top = fmaxf(top, v);
    }
    #pragma unroll
    for (int m = 16; m; m >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
    float * const tops = reinterpret_cast<float *>(s.warp_sum);
    if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = top;
    __syncthreads();
    if (threadIdx.x == 0) { for (int w = 1; w < kThreads / 32; w++) top = fmaxf(top, tops[w]); s.top = top; s.index = 0xffffffffu; }
    cluster_barrier();
    for (uint32_t b = 0; b < blocks; b++) top = fmaxf(top, ld_cluster(smem_u32(&s.top), b));

    Row r{x, first, here, rank, blocks, s, top, double(top)};
    uint32_t token = 0;
    double chance = 1.0;
    if (!(top > -CUDART_INF_F) || !(t > 0.f)) {
        // the lowest index of the largest logit; a row with nothing above the lowest: the first that is a number, with nothing to draw
        uint32_t found = 0xffffffffu;
        if (top > -CUDART_INF_F) { for (int i = threadIdx.x; i < here; i += kThreads) if (x[i] == top) { found = uint32_t(first + i); break; } }
        else { for (int i = threadIdx.x; i < here; i += kThreads) { const float v = from[i]; if (v == v) { found = uint32_t(first + i); break; } } }
        found = __reduce_min_sync(0xffffffffu, found);
        if (threadIdx.x % 32 == 0) atomicMin(&s.index, found);
        cluster_barrier();
        token = 0xffffffffu;
        for (uint32_t b = 0; b < blocks; b++) token = min(token, ld_remote(&s.index, b));
        if (token == 0xffffffffu) token = 0;
        chance = top > -CUDART_INF_F ? 1.0 : 0.0;
    } else {
        constexpr double kLog2e = 1.4426950408889634074;
        const double per_t = kLog2e / double(t);
        const bool by_k = k > 0 && k < a.n, by_p = top_p < 1.f;
        // min-p as the least logit kept: the smallest float whose gap is within the limit
        const double limit = min_p > 0.f ? (min_p >= 1.f ? 0.0 : -log(double(min_p))) : kNoLimit;
        float least = -CUDART_INF_F;
        if (top == CUDART_INF_F) {
            least = top;      // an infinity takes all
        } else if (limit < kNoLimit) {
            least = __double2float_ru(double(top) - limit);
            while (r.gap(least) > limit) least = nextafterf(least, CUDART_INF_F);
        }
        auto p_goal = [&](unsigned long long total) { return max(1ull, min(total, (unsigned long long)(ceil(double(top_p) * double(total))))); };
        auto u_goal = [&](unsigned long long total) {
            const double u = double(uniform) * double(total);
            return u > 0.0 ? min(total, (unsigned long long)u + 1ull) : 1ull;
        };
        auto any = [](float) { return true; };
        auto by_gap = [&](float v) { return r.bin(v); };
        bool listed = false;
        unsigned long long total_p = 0;
        float cut;
        uint32_t index;
        if (by_k) {
            auto k_goal = [&](unsigned long long) { return (unsigned long long)k; };
            histogram(r, true, 0.0, 0, [&](float v) { return r.bin(v) < kNearBins; }, by_gap, k_goal);
            if (s.bin == kBins) histogram(r, true, 0.0, 0, any, by_gap, k_goal);
            if (s.bin < kBins) {
                listed = s.up_to <= kList;
                if (!listed) { resolve(r, true, 0.0, (unsigned long long)k, &cut, &index); r.cut = cut; r.cut_index = index; }
            }
        }
        if (by_p && !listed) {
            histogram(r, false, kLog2e, 0, any, by_gap, p_goal);
            total_p = s.total;
            listed = s.up_to <= kList;
            if (!listed) { resolve(r, false, kLog2e, p_goal(total_p), &cut, &index); r.cut = cut; r.cut_index = index; }
        }
        if (listed) {
            const int to = s.bin;
            int n = gather(r, [&](float v, int i) { return r.kept(v, i) && r.bin(v) <= to; });
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
            histogram(r, false, per_t, 0, any, by_gap, u_goal);
            const unsigned long long total = s.total;
            resolve(r, false, per_t, u_goal(total), &cut, &token);
            chance = double(r.weight(cut, per_t)) / double(total);
        }
    }
    if (rank == 0 && threadIdx.x == 0) {
        a.tokens[row] = int32_t(token);
        if (a.probability) a.probability[row] = float(chance);
    }
    cluster_barrier();      // no block leaves while another reads its shared memory
}

}  // namespace

int sample_rows_most() { return kMostBlocks * kMostSlice; }

cudaError_t launch_sample_rows(const float * logits, int64_t stride, int rows, int n, const float * temperature, const int32_t * top_k, const float * top_p, const float * min_p,
                               const float * uniform, int32_t * tokens, float * probability, cudaStream_t stream) {
    // as many blocks per row as leave each at least 2048 logits
    int blocks = 1;
    while (blocks < kMostBlocks && n > blocks * 2048) blocks *= 2;
    const int slice = ((n + blocks - 1) / blocks + 3) & ~3;      // (whole 16 bytes, so that every block's share begins as the row does)
    if (n < 1 || slice > kMostSlice) return cudaErrorInvalidValue;
    const int bytes = int(sizeof(Shared)) + 16 + slice * 4;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_dynamic_smem(k_sample_rows, int(sizeof(Shared)) + 16 + kMostSlice * 4, done);
    if (e != cudaSuccess) return e;
    const SampleArgs a{logits, stride, n, slice, temperature, top_p, min_p, uniform, top_k, tokens, probability};
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(unsigned(rows) * unsigned(blocks));
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = size_t(bytes);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = unsigned(blocks);
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, k_sample_rows, a);
}

}  // namespace cuda
}  // namespace dooms
