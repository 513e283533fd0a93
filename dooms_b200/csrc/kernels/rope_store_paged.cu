// New rows into a paged cache: the rotary positions of their queries and keys (one axis, or several for the rows of images and video), the queries out as f32 or
// f16 rows, keys and values as f16 into the pages of their sequences.
//
//   pair i of a head, axis x(i) (the sections deal the pairs over the axes in order):  a = position[x(i)] * base^(-2 i / d)
//   (u, w) -> (u cos a - w sin a, u sin a + w cos a), the pair being elements (i, i + d/2) or (2i, 2i + 1)
//
// Angles, sines and cosines are 64-bit (a position of 100 000 leaves an f32 angle two correct decimals) and rounded once to f32; the rotation is f32 and each
// result is rounded once to the type it is stored as.
#include "launch.cuh"
#include "paged.cuh"

namespace dooms {
namespace cuda {

namespace {

constexpr int kThreads = 256, kMostTokens = 4;

struct RopeArgs {
    double log2_base;
    int neox, n_axes, axis_end[4];      // axis x has the pairs [axis_end[x - 1], axis_end[x])
};

__device__ __forceinline__ uint32_t pack(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t *>(&h); }

// A block takes `per_block` rows (1 to 4) and, of their heads, the share blockIdx.y of gridDim.y. It first makes the rows' (cos, sin) in shared memory, one
// thread per pair, then every thread turns units of eight values (four pairs).
template <int D, bool HALF_Q>
__global__ void __launch_bounds__(kThreads) k_rope_store_paged(const PagedView c, const RopeArgs r, const float * __restrict__ qkv, int64_t stride, int n_head, int n_rows,
                                                               const int32_t * __restrict__ sequence, const int32_t * __restrict__ at, const int32_t * __restrict__ positions,
                                                               void * __restrict__ q_out, int per_block) {
    constexpr int kPairs = D / 2, kUnits = D / 8;
    __shared__ float2 cs[kMostTokens][kPairs];
    __shared__ int64_t line[kMostTokens];
    const int row0 = int(blockIdx.x) * per_block, rows = min(per_block, n_rows - row0);
    if (int(threadIdx.x) < rows) {
        const int t = row0 + threadIdx.x, s = sequence[t];
        int64_t where = -1;
        if (s >= 0) {
            const int p = at[t];
            if (s < c.n_sequences && p >= 0 && p < c.capacity()) where = c.row(s, p);
            if (where < 0 && blockIdx.y == 0) c.fail();
        }
        line[threadIdx.x] = where;
    }
    for (int i = threadIdx.x; i < rows * kPairs; i += kThreads) {
        const int t = row0 + i / kPairs, pair = i % kPairs;
        int axis = 0;
        while (axis < r.n_axes - 1 && pair >= r.axis_end[axis]) axis++;
        const double a = double(positions[int64_t(axis) * n_rows + t]) * exp2(r.log2_base * (double(pair) * (-2.0 / D)));
        double s, co;
        sincos(a, &s, &co);
        cs[i / kPairs][pair] = make_float2(float(co), float(s));
    }
    __syncthreads();
    const int heads = n_head + 2 * c.n_kv, units = rows * heads * kUnits;
    for (int u = int(blockIdx.y) * kThreads + threadIdx.x; u < units; u += int(gridDim.y) * kThreads) {
        const int part = u % kUnits, h = (u / kUnits) % heads, b = u / (kUnits * heads);
        const int64_t where = line[b];
        if (where < 0) continue;
        const float * x = qkv + int64_t(row0 + b) * stride + int64_t(h) * D;
        const bool value = h >= n_head + c.n_kv, halves = r.neox && !value;      // (values are taken in order)
        const float4 lo = __ldg(reinterpret_cast<const float4 *>(x + (halves ? part * 4 : part * 8)));
        const float4 hi = __ldg(reinterpret_cast<const float4 *>(x + (halves ? kPairs + part * 4 : part * 8 + 4)));
        float y[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
        if (!value) {
            #pragma unroll
            for (int i = 0; i < 4; i++) {
                const float2 e = cs[b][part * 4 + i];
                const int iu = halves ? i : 2 * i, iw = halves ? 4 + i : 2 * i + 1;
                const float uu = y[iu], ww = y[iw];
                y[iu] = uu * e.x - ww * e.y;
                y[iw] = uu * e.y + ww * e.x;
            }
        }
        const int first = halves ? part * 4 : part * 8, second = halves ? kPairs + part * 4 : part * 8 + 4;
        if (h < n_head && !HALF_Q) {
            float * q = static_cast<float *>(q_out) + (int64_t(row0 + b) * n_head + h) * D;
            *reinterpret_cast<float4 *>(q + first) = make_float4(y[0], y[1], y[2], y[3]);
            *reinterpret_cast<float4 *>(q + second) = make_float4(y[4], y[5], y[6], y[7]);
        } else {
            __half * o = h < n_head ? static_cast<__half *>(q_out) + (int64_t(row0 + b) * n_head + h) * D
                                    : (value ? c.v : c.k) + (where * c.n_kv + (h - n_head - (value ? c.n_kv : 0))) * D;
            *reinterpret_cast<uint2 *>(o + first) = make_uint2(pack(y[0], y[1]), pack(y[2], y[3]));
            *reinterpret_cast<uint2 *>(o + second) = make_uint2(pack(y[4], y[5]), pack(y[6], y[7]));
        }
    }
}

}  // namespace

cudaError_t launch_rope_store_paged(const PagedCache & cache, const RopeSections & rope, const float * qkv, int64_t stride, int n_head, int n_rows, const int32_t * sequence,
                                    const int32_t * at, const int32_t * positions, void * q_out, bool half_q, int * error, cudaStream_t stream) {
    const PagedView c = paged_view(cache, error);
    RopeArgs r{log2(rope.base), rope.neox, rope.n_axes, {0, 0, 0, 0}};
    for (int x = 0, end = 0; x < 4; x++) r.axis_end[x] = end += rope.sections[x];
    const int per_block = n_rows >= kMostTokens * 2 * sm_count() ? kMostTokens : 1;
    const dim3 grid(unsigned((n_rows + per_block - 1) / per_block), 1u);
    auto go = [&](auto kernel) { kernel<<<grid, kThreads, 0, stream>>>(c, r, qkv, stride, n_head, n_rows, sequence, at, positions, q_out, per_block); };
    if (cache.head_dim == 128) half_q ? go(k_rope_store_paged<128, true>) : go(k_rope_store_paged<128, false>);
    else if (cache.head_dim == 64) half_q ? go(k_rope_store_paged<64, true>) : go(k_rope_store_paged<64, false>);
    else return cudaErrorInvalidValue;
    return cudaGetLastError();
}

}  // namespace cuda
}  // namespace dooms
