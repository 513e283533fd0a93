// One token per row of logits from given random numbers: top-k, then top-p and min-p on the probabilities at temperature 1, then the temperature, then the draw (the
// order of the host sampler's chain). In the order (logit descending, index ascending), with the row's largest logit m and g = m - l:
//   kept by top-k: the first k;  by top-p: while what is in front of a token holds less than top_p of the mass e^-g of what top-k kept;  by min-p: e^-g >= min_p;
//   the token: the first whose cumulative weight e^(-g / T) exceeds u times the kept tokens' total.
//
// A row belongs to a cluster of up to eight blocks; each holds its share of the logits in shared memory, so that they are read once. No sort of the row: a cut
// ("the first element at which a cumulative weight reaches a goal") is found by a histogram of 1/32 nat per bin over all blocks of the cluster, then by sorting
// the few elements of the bin where the goal falls (or of all bins up to there, where they are few: then everything else is decided in that list too). A bin of
// more than kList elements (flat logits, or many equal ones) is divided again by the bits of the logits, down to a single value, whose elements are then
// counted out in the order of their indices.
// Weights are 64-bit integers, e^-x 2^45 rounded (x and the exponential in 64-bit floating point): sums do not depend on the order of the atomics, and the blocks of
// a cluster, which all work out every cut for themselves, agree on it. 2^18 logits of the largest weight still fit. What is rounded off is 2^-46 of
// the row's largest weight per token.
#include <math_constants.h>

#include <algorithm>

#include "kernels.h"
#include "launch.cuh"
#include "ptx.cuh"

namespace dooms {
namespace cuda {

using namespace dooms::dev;

namespace {

constexpr int kThreads = 512, kBins = 1024, kList = 1024, kMostBlocks = 8;
constexpr int kMostSlice = 32768;      // logits per block
constexpr float kBinsPerNat = 32.f;
constexpr double kNoLimit = 1e300;     // (gaps are below 2^129, or infinite)
static_assert(kBins == 2 * kThreads && kList == 2 * kThreads, "two bins and two list elements per thread");

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
    unsigned long long mass[kBins];        // this block's histogram
    uint32_t count[kBins];
    unsigned long long local[kList];       // this block's elements of the list
    unsigned long long all[kList], sorted[kList];
    unsigned long long warp_sum[2][kThreads / 32];
    uint32_t n_local, lo_key, hi_key, index, ties;
    float top;
    // what a step leaves for all threads
    int bin, list_to;
    uint32_t in_bin;
    unsigned long long before, total, total_count;
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
    // what is kept so far: elements in front of or at (key, index), and with a gap of at most `limit`
    uint32_t cut_key = 0, cut_index = 0xffffffffu;
    double limit = kNoLimit;

    __device__ bool kept(float v, int i) const {
        if (!(v > -CUDART_INF_F)) return false;
        const uint32_t k = key_of(v);
        return (k > cut_key || (k == cut_key && uint32_t(first + i) <= cut_index)) && gap(v) <= limit && gap(v) < kNoLimit;
    }
    __device__ double gap(float v) const { return v == top ? 0.0 : double(top) - double(v); }
    __device__ int bin(float v) const { return v == top ? 0 : int(fminf((top - v) * kBinsPerNat, float(kBins - 1))); }
    // kind < 0: one per element; otherwise e^(-gap * kind)
    __device__ unsigned long long weight(float v, double kind) const { return kind < 0 ? 1ull : (unsigned long long)(rint(exp(-gap(v) * kind) * 35184372088832.0)); }
};

// Inclusive sums over the block of two values per thread (its elements 2 tid and 2 tid + 1 of kBins or kList).
__device__ void scan_pairs(unsigned long long (&v)[2], unsigned long long * warp_sum) {
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    unsigned long long t = v[0] + v[1];
    for (int d = 1; d < 32; d <<= 1) { const unsigned long long o = __shfl_up_sync(0xffffffffu, t, d); if (lane >= d) t += o; }
    __syncthreads();
    if (lane == 31) warp_sum[warp] = t;
    __syncthreads();
    if (warp == 0) {
        unsigned long long w = lane < kThreads / 32 ? warp_sum[lane] : 0;
        for (int d = 1; d < 32; d <<= 1) { const unsigned long long o = __shfl_up_sync(0xffffffffu, w, d); if (lane >= d) w += o; }
        if (lane < kThreads / 32) warp_sum[lane] = w;
    }
    __syncthreads();
    if (warp > 0) t += warp_sum[warp - 1];
    v[0] = t - v[1];
    v[1] = t;
}

// All blocks' elements for which take(value, i) holds (at most kList of them over the cluster), sorted, into s.sorted; returns their number.
template <class Take>
__device__ int gather(Row & r, Take take) {
    Shared & s = r.s;
    if (threadIdx.x == 0) s.n_local = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < r.here; i += kThreads) {
        if (take(r.x[i], i)) s.local[atomicAdd(&s.n_local, 1u)] = (unsigned long long)key_of(r.x[i]) << 32 | (0xffffffffu - uint32_t(r.first + i));
    }
    cluster_barrier();
    uint32_t n = 0;
    for (uint32_t b = 0; b < r.blocks; b++) {
        const uint32_t m = ld_remote(&s.n_local, b);
        for (uint32_t i = threadIdx.x; i < m; i += kThreads) s.all[n + i] = ld_remote(&s.local[i], b);
        n += m;
    }
    cluster_barrier();
    for (uint32_t i = threadIdx.x; i < n; i += kThreads) {
        const unsigned long long e = s.all[i];
        uint32_t ahead = 0;
        for (uint32_t j = 0; j < n; j++) ahead += s.all[j] > e;
        s.sorted[ahead] = e;
    }
    __syncthreads();
    return int(n);
}

// Where the cumulative weight (of `kind`) over the sorted list's first n elements, on top of `before`, reaches goal(total): the element's place (n: nowhere).
template <class Goal>
__device__ int place_in_list(Row & r, int n, double kind, unsigned long long before, Goal goal, unsigned long long * total) {
    Shared & s = r.s;
    unsigned long long v[2];
    #pragma unroll
    for (int e = 0; e < 2; e++) { const int i = 2 * threadIdx.x + e; v[e] = i < n ? r.weight(value_of(uint32_t(s.sorted[i] >> 32)), kind) : 0ull; }
    const unsigned long long own[2] = {v[0], v[1]};
    scan_pairs(v, s.warp_sum[0]);
    if (threadIdx.x == 0) s.bin = n;
    if (threadIdx.x == kThreads - 1) s.total = before + v[1];
    __syncthreads();
    *total = s.total;
    const unsigned long long g = goal(s.total);
    #pragma unroll
    for (int e = 0; e < 2; e++) {
        const int i = 2 * threadIdx.x + e;
        if (i < n && before + v[e] >= g && before + v[e] - own[e] < g) s.bin = i;
    }
    __syncthreads();
    const int at = s.bin;
    __syncthreads();
    return at;
}

// A histogram over the kept elements that in(v, i) takes, by bin_of(v); leaves in s the first bin where the cumulative weight on top of `before` reaches
// goal(total), what is in front of it, and how many elements it and the bins in front hold. s.bin = kBins: the goal is not reached.
template <class In, class BinOf, class Goal>
__device__ void histogram(Row & r, double kind, unsigned long long before, In in, BinOf bin_of, Goal goal) {
    Shared & s = r.s;
    for (int b = threadIdx.x; b < kBins; b += kThreads) { s.mass[b] = 0; s.count[b] = 0; }
    __syncthreads();
    for (int i = threadIdx.x; i < r.here; i += kThreads) {
        const float v = r.x[i];
        if (!r.kept(v, i) || !in(v)) continue;
        const int b = bin_of(v);
        atomicAdd(&s.count[b], 1u);
        if (kind >= 0) atomicAdd(&s.mass[b], r.weight(v, kind));
    }
    cluster_barrier();
    unsigned long long m[2] = {0, 0}, c[2] = {0, 0};
    for (uint32_t blk = 0; blk < r.blocks; blk++) {
        #pragma unroll
        for (int e = 0; e < 2; e++) {
            const int b = 2 * threadIdx.x + e;
            c[e] += ld_remote(&s.count[b], blk);
            if (kind >= 0) m[e] += ld_remote(&s.mass[b], blk);
        }
    }
    if (kind < 0) { m[0] = c[0]; m[1] = c[1]; }
    const unsigned long long own_m[2] = {m[0], m[1]}, own_c[2] = {c[0], c[1]};
    scan_pairs(m, s.warp_sum[0]);
    scan_pairs(c, s.warp_sum[1]);
    if (threadIdx.x == kThreads - 1) { s.total = before + m[1]; s.total_count = c[1]; s.bin = kBins; }
    __syncthreads();
    const unsigned long long g = goal(s.total);
    #pragma unroll
    for (int e = 0; e < 2; e++) {
        if (before + m[e] >= g && before + m[e] - own_m[e] < g) {
            s.bin = 2 * threadIdx.x + e;
            s.before = before + m[e] - own_m[e];
            s.in_bin = uint32_t(own_c[e]);
            s.list_to = int(min(c[e], (unsigned long long)(kList + 1)));
        }
    }
    cluster_barrier();      // the next step may change the histogram that other blocks have read
}

// The element at which the cumulative weight over what is kept, past the histogram that is in s, reaches the goal: as its (key, index). The goal is reached.
__device__ void resolve(Row & r, double kind, unsigned long long goal, uint32_t * key, uint32_t * index) {
    Shared & s = r.s;
    const int bin = s.bin;
    unsigned long long before = s.before;
    uint32_t count = s.in_bin, lo = 0, hi = 0xffffffffu;
    auto in = [&](float v) { const uint32_t k = key_of(v); return r.bin(v) == bin && k >= lo && k <= hi; };
    while (count > kList) {
        __syncthreads();
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
        cluster_barrier();
        if (lo == hi) {      // one value: the goal falls on its m-th element in the order of the indices
            const unsigned long long w = r.weight(value_of(lo), kind), m = (goal - before + w - 1) / w;
            uint32_t mine = 0;
            for (int i = threadIdx.x; i < r.here; i += kThreads) mine += r.kept(r.x[i], i) && key_of(r.x[i]) == lo;
            if (threadIdx.x == 0) { s.ties = 0; s.index = 0xffffffffu; }
            __syncthreads();
            mine = __reduce_add_sync(0xffffffffu, mine);
            if (threadIdx.x % 32 == 0) atomicAdd(&s.ties, mine);
            cluster_barrier();
            unsigned long long ahead = 0;
            for (uint32_t b = 0; b < r.rank; b++) ahead += ld_remote(&s.ties, b);
            if (ahead < m && m <= ahead + s.ties) {
                unsigned long long seen = ahead;
                for (int base = 0; base < r.here; base += kThreads) {
                    const int i = base + threadIdx.x;
                    const bool is = i < r.here && r.kept(r.x[i], i) && key_of(r.x[i]) == lo;
                    const int total = __syncthreads_count(is);
                    if (seen + total >= m) {
                        // the (m - seen)-th lane that holds one
                        const uint32_t ballot = __ballot_sync(0xffffffffu, is);
                        if (threadIdx.x % 32 == 0) s.count[threadIdx.x / 32] = __popc(ballot);
                        __syncthreads();
                        unsigned long long at = seen + __popc(ballot & ((1u << (threadIdx.x % 32)) - 1u)) + 1;
                        for (int w2 = 0; w2 < int(threadIdx.x / 32); w2++) at += s.count[w2];
                        if (is && at == m) s.index = uint32_t(r.first + i);
                        break;
                    }
                    seen += total;
                }
            }
            cluster_barrier();
            uint32_t found = 0xffffffffu;
            for (uint32_t b = 0; b < r.blocks; b++) found = min(found, ld_remote(&s.index, b));
            cluster_barrier();
            *key = lo;
            *index = found;
            return;
        }
        const int shift = max(0, 32 - __clz(hi - lo) - 10);
        const uint32_t top = hi;
        histogram(r, kind, before, in, [&](float v) { return int((top - key_of(v)) >> shift); }, [&](unsigned long long) { return goal; });
        __syncthreads();
        before = s.before;
        count = s.in_bin;
        hi = top - (uint32_t(s.bin) << shift);
        lo = max(lo, hi - min(hi, (1u << shift) - 1u));
        __syncthreads();
    }
    const int n = gather(r, [&](float v, int i) { return r.kept(v, i) && in(v); });
    unsigned long long total;
    const int at = place_in_list(r, n, kind, before, [&](unsigned long long) { return goal; }, &total);
    const unsigned long long e = s.sorted[min(at, max(n - 1, 0))];
    *key = uint32_t(e >> 32);
    *index = 0xffffffffu - uint32_t(e);
    __syncthreads();
}

__global__ void __launch_bounds__(kThreads) k_sample_rows(const SampleArgs a) {
    extern __shared__ __align__(16) uint8_t smem[];
    Shared & s = *reinterpret_cast<Shared *>(smem);
    float * const x = reinterpret_cast<float *>(smem + sizeof(Shared));
    uint32_t rank, blocks;
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(blocks));
    const int row = int(blockIdx.x / blocks);
    const float * logits = a.logits + int64_t(row) * a.stride;
    const int first = int(rank) * a.slice, here = max(0, min(a.slice, a.n - first));
    float top = -CUDART_INF_F;
    #pragma unroll 8
    for (int i = threadIdx.x; i < here; i += kThreads) {
        float v = __ldg(logits + first + i) + 0.f;      // (one zero)
        v = v == v ? v : -CUDART_INF_F;                 // a NaN never wins
        x[i] = v;
        top = fmaxf(top, v);
    }
    for (int m = 16; m; m >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
    float * const tops = reinterpret_cast<float *>(s.warp_sum[0]);
    if (threadIdx.x % 32 == 0) tops[threadIdx.x / 32] = top;
    __syncthreads();
    if (threadIdx.x == 0) { for (int w = 1; w < kThreads / 32; w++) top = fmaxf(top, tops[w]); s.top = top; s.index = 0xffffffffu; }
    cluster_barrier();
    for (uint32_t b = 0; b < blocks; b++) top = fmaxf(top, ld_cluster(smem_u32(&s.top), b));
    cluster_barrier();      // (s.top and the warps' values have been read)

    Row r{x, first, here, rank, blocks, s, top};
    const float t = a.temperature ? a.temperature[row] : 1.f, top_p = a.top_p ? a.top_p[row] : 1.f, min_p = a.min_p ? a.min_p[row] : 0.f;
    const int k = a.top_k ? a.top_k[row] : 0;
    uint32_t token = 0;
    double chance = 1.0;
    if (!(top > -CUDART_INF_F) || !(t > 0.f)) {
        // the lowest index of the largest logit; a row with nothing above the lowest: the first that is a number, with nothing to draw
        uint32_t found = 0xffffffffu;
        if (top > -CUDART_INF_F) { for (int i = threadIdx.x; i < here; i += kThreads) if (x[i] == top) { found = uint32_t(first + i); break; } }
        else { for (int i = threadIdx.x; i < here; i += kThreads) { const float v = logits[first + i]; if (v == v) { found = uint32_t(first + i); break; } } }
        found = __reduce_min_sync(0xffffffffu, found);
        if (threadIdx.x % 32 == 0) atomicMin(&s.index, found);
        cluster_barrier();
        token = 0xffffffffu;
        for (uint32_t b = 0; b < blocks; b++) token = min(token, ld_remote(&s.index, b));
        if (token == 0xffffffffu) token = 0;
        chance = top > -CUDART_INF_F ? 1.0 : 0.0;
    } else {
        const double kind_t = 1.0 / double(t);
        const bool by_k = k > 0 && k < a.n, by_p = top_p < 1.f;
        if (min_p > 0.f) r.limit = min_p >= 1.f ? 0.0 : -log(double(min_p));
        auto p_goal = [&](unsigned long long total) { return max(1ull, min(total, (unsigned long long)(ceil(double(top_p) * double(total))))); };
        auto u_goal = [&](unsigned long long total) {
            const double u = double(a.uniform[row]) * double(total);
            return u > 0.0 ? min(total, (unsigned long long)u + 1ull) : 1ull;
        };
        const double limit = r.limit;
        auto any = [](float) { return true; };
        auto by_gap = [&](float v) { return r.bin(v); };
        bool listed = false;
        unsigned long long total_p = 0;
        if (by_k) {
            r.limit = kNoLimit;
            histogram(r, -1.0, 0, any, by_gap, [&](unsigned long long) { return (unsigned long long)k; });
            if (s.bin < kBins) {
                listed = s.list_to <= kList;
                if (!listed) { uint32_t ck, ci; resolve(r, -1.0, (unsigned long long)k, &ck, &ci); r.cut_key = ck; r.cut_index = ci; }
            }
        }
        if (by_p && !listed) {
            r.limit = kNoLimit;
            histogram(r, 1.0, 0, any, by_gap, p_goal);
            total_p = s.total;
            listed = s.list_to <= kList;
            if (!listed) { uint32_t ck, ci; resolve(r, 1.0, p_goal(total_p), &ck, &ci); r.cut_key = ck; r.cut_index = ci; }
        }
        r.limit = limit;
        if (listed) {
            const int to = s.bin;
            r.limit = kNoLimit;
            int n = gather(r, [&](float v, int i) { return r.kept(v, i) && r.bin(v) <= to; });
            if (by_k) n = min(n, k);
            unsigned long long total;
            if (by_p) {
                const unsigned long long given = total_p;
                const int at = place_in_list(r, n, 1.0, 0, [&](unsigned long long sum) { return p_goal(given ? given : sum); }, &total);
                n = min(n, at + 1);
            }
            if (limit < kNoLimit) n = max(1, min(n, __syncthreads_count(2 * int(threadIdx.x) < n && r.gap(value_of(uint32_t(s.sorted[2 * threadIdx.x] >> 32))) <= limit) +
                                                      __syncthreads_count(2 * int(threadIdx.x) + 1 < n && r.gap(value_of(uint32_t(s.sorted[2 * threadIdx.x + 1] >> 32))) <= limit)));
            const int at = min(place_in_list(r, n, kind_t, 0, u_goal, &total), n - 1);
            const unsigned long long e = s.sorted[at];
            token = 0xffffffffu - uint32_t(e);
            chance = double(r.weight(value_of(uint32_t(e >> 32)), kind_t)) / double(total);
        } else {
            histogram(r, kind_t, 0, any, by_gap, u_goal);
            const unsigned long long total = s.total;
            uint32_t ck, ci;
            resolve(r, kind_t, u_goal(total), &ck, &ci);
            token = ci;
            chance = double(r.weight(value_of(ck), kind_t)) / double(total);
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
    const int slice = (n + blocks - 1) / blocks;
    if (n < 1 || slice > kMostSlice) return cudaErrorInvalidValue;
    const int bytes = int(sizeof(Shared)) + slice * 4;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_dynamic_smem(k_sample_rows, int(sizeof(Shared)) + kMostSlice * 4, done);
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
