// New rows into a paged cache: the rotary positions of their queries and keys (one axis, or several for the rows of images and video), the queries out as f32 or
// f16 rows, keys and values as f16 into the pages of their sequences.
//
//   pair i of a head, axis x(i) (the sections deal the pairs over the axes in order):  a = position[x(i)] * base^(-2 i / d)
//   (u, w) -> (u cos a - w sin a, u sin a + w cos a), the pair being elements (i, i + d/2) or (2i, 2i + 1)
//
// An angle is reduced to a turn's fraction in 64 bits (a position of 100 000 leaves an f32 angle two correct decimals); its sine and cosine are those of the fraction
// rounded to f32, corrected by what the rounding left, 1e-7 off at most. The rotation is f32 and each result is rounded once to the type it is stored as.
#include <cmath>

#include "launch.cuh"
#include "paged.cuh"

namespace dooms {
namespace cuda {

using namespace dooms::dev;

namespace {

constexpr int kThreads = 256, kAtOnce = 4;      // kAtOnce: units of a thread whose loads are in flight together

struct RopeArgs {
    double turns[64];                   // base^(-2 i / d) / (2 pi): turns per position
    int n_axes, axis_end[4];            // axis x has the pairs [axis_end[x - 1], axis_end[x])
};

__device__ __forceinline__ uint32_t pack(float a, float b) { const __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<const uint32_t *>(&h); }

// Bound by device memory, and close to being bound by instructions: a row has TPR threads, each of which has the same eight values (four pairs) of every head it takes, so
// that its sines and cosines stay in registers and its addresses are a step apart. (With rows and heads dealt by division and the pairs chosen at run time a unit
// was 325 instructions: 68 us for 6000 rows of 40 + 8 + 8 heads of 128, where this takes 50; their bytes alone take 39.5.) Every thread asks for its first units,
// then the block makes its rows' (cos, sin) in shared memory, one thread per pair, and looks the rows' places up, while those are on their way.
template <int D, bool HALF_Q, bool NEOX, int TPR>
__global__ void __launch_bounds__(kThreads, 4) k_rope_store_paged(const PagedView c, const __grid_constant__ RopeArgs r, const float * __restrict__ qkv, int64_t stride, int n_head,
                                                               int n_rows, const int32_t * __restrict__ sequence, const int32_t * __restrict__ at,
                                                               const int32_t * __restrict__ positions, void * __restrict__ q_out) {
    constexpr int kPairs = D / 2, kUnits = D / 8, kRows = kThreads / TPR, kStep = TPR / kUnits;      // kStep heads apart: a thread's units
    __shared__ __align__(16) float2 cs[kRows][kPairs];
    __shared__ int64_t line[kRows];
    pdl_wait();
    const int row0 = int(blockIdx.x) * kRows, mine = threadIdx.x / TPR, row = row0 + mine, unit = threadIdx.x % TPR, part = unit % kUnits, head0 = unit / kUnits;
    const int heads = n_head + 2 * c.n_kv;
    // where in a head the unit's two times four values begin (a value head is taken the same way, and copied)
    constexpr int kGap = NEOX ? kPairs : 4;
    const int first = NEOX ? part * 4 : part * 8;
    const bool there = row < n_rows;
    const float * from = qkv + int64_t(row) * stride + int64_t(head0) * D + first;
    float4 lo[kAtOnce], hi[kAtOnce];
    auto load = [&](int h0) {
        #pragma unroll
        for (int k = 0; k < kAtOnce; k++) {
            if (there && h0 + k * kStep < heads) {
                lo[k] = __ldg(reinterpret_cast<const float4 *>(from + k * kStep * D));
                hi[k] = __ldg(reinterpret_cast<const float4 *>(from + k * kStep * D + kGap));
            }
        }
        from += kAtOnce * kStep * D;
    };
    load(head0);
    if (threadIdx.x < kRows && row0 + int(threadIdx.x) < n_rows) {
        const int t = row0 + threadIdx.x, s = sequence[t];
        int64_t where = -1;
        if (s >= 0) {
            const int p = at[t];
            if (s < c.n_sequences && p >= 0 && p < c.capacity()) where = c.row(s, p);
            if (where < 0) c.fail();
        }
        line[threadIdx.x] = where;
    }
    for (int i = threadIdx.x; i < kRows * kPairs; i += kThreads) {
        const int t = row0 + i / kPairs, pair = i % kPairs;
        if (t >= n_rows) break;
        int axis = 0;
        while (axis < r.n_axes - 1 && pair >= r.axis_end[axis]) axis++;
        const double turns = double(positions[int64_t(axis) * n_rows + t]) * r.turns[pair], f = turns - rint(turns);
        const float f32 = float(f), rest = float(f - double(f32)) * 6.28318530717958647693f;
        float s, co;
        sincospif(2.f * f32, &s, &co);
        cs[i / kPairs][pair] = make_float2(fmaf(-s, rest, co), fmaf(co, rest, s));
    }
    __syncthreads();
    if (!there) return;
    const int64_t where = line[mine];
    if (where < 0) return;
    const float4 e01 = *reinterpret_cast<const float4 *>(&cs[mine][part * 4]), e23 = *reinterpret_cast<const float4 *>(&cs[mine][part * 4 + 2]);
    const float co[4] = {e01.x, e01.z, e23.x, e23.z}, si[4] = {e01.y, e01.w, e23.y, e23.w};
    __half * const k_to = c.k + where * c.n_kv * D + first, * const v_to = c.v + where * c.n_kv * D + first;
    const int64_t q_at = int64_t(row) * n_head * D + first;
    for (int h0 = head0; h0 < heads; h0 += kAtOnce * kStep) {
        if (h0 != head0) load(h0);
        #pragma unroll
        for (int k = 0; k < kAtOnce; k++) {
            const int h = h0 + k * kStep;
            if (h >= heads) break;
            float a[4], b[4];      // the pairs, and then what they become
            if (NEOX) {
                a[0] = lo[k].x; a[1] = lo[k].y; a[2] = lo[k].z; a[3] = lo[k].w; b[0] = hi[k].x; b[1] = hi[k].y; b[2] = hi[k].z; b[3] = hi[k].w;
            } else {
                a[0] = lo[k].x; b[0] = lo[k].y; a[1] = lo[k].z; b[1] = lo[k].w; a[2] = hi[k].x; b[2] = hi[k].y; a[3] = hi[k].z; b[3] = hi[k].w;
            }
            if (h < n_head + c.n_kv) {
                #pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float u = a[i], w = b[i];
                    a[i] = u * co[i] - w * si[i];
                    b[i] = u * si[i] + w * co[i];
                }
            }
            if (!HALF_Q && h < n_head) {
                float * to = static_cast<float *>(q_out) + q_at + h * D;
                *reinterpret_cast<float4 *>(to) = NEOX ? make_float4(a[0], a[1], a[2], a[3]) : make_float4(a[0], b[0], a[1], b[1]);
                *reinterpret_cast<float4 *>(to + kGap) = NEOX ? make_float4(b[0], b[1], b[2], b[3]) : make_float4(a[2], b[2], a[3], b[3]);
            } else {
                __half * to = h < n_head ? static_cast<__half *>(q_out) + q_at + h * D : h < n_head + c.n_kv ? k_to + (h - n_head) * D : v_to + (h - n_head - c.n_kv) * D;
                if (NEOX) {
                    *reinterpret_cast<uint2 *>(to) = make_uint2(pack(a[0], a[1]), pack(a[2], a[3]));
                    *reinterpret_cast<uint2 *>(to + kGap) = make_uint2(pack(b[0], b[1]), pack(b[2], b[3]));
                } else {
                    *reinterpret_cast<uint4 *>(to) = make_uint4(pack(a[0], b[0]), pack(a[1], b[1]), pack(a[2], b[2]), pack(a[3], b[3]));
                }
            }
        }
    }
}

template <int D, bool HALF_Q, bool NEOX, class... Args>
cudaError_t launch(int heads, int n_rows, cudaStream_t stream, Args... args) {
    // threads per row: so many that a thread has at most four units or so, whose loads all go out at once
    const int units = heads * (D / 8);
    auto go = [&](auto kernel, int rows) { return launch_pdl(kernel, dim3(unsigned((n_rows + rows - 1) / rows)), dim3(kThreads), 0, stream, args...); };
    if (units > 512) return go(k_rope_store_paged<D, HALF_Q, NEOX, 256>, 1);
    if (units > 256) return go(k_rope_store_paged<D, HALF_Q, NEOX, 128>, 2);
    return go(k_rope_store_paged<D, HALF_Q, NEOX, 64>, 4);
}

}  // namespace

cudaError_t launch_rope_store_paged(const PagedCache & cache, const RopeSections & rope, const float * qkv, int64_t stride, int n_head, int n_rows, const int32_t * sequence,
                                    const int32_t * at, const int32_t * positions, void * q_out, bool half_q, int * error, cudaStream_t stream) {
    const PagedView c = paged_view(cache, error);
    // the table of the last base and head size that this thread used: a program has one
    struct Table { double base = 0.0; int head_dim = 0; RopeArgs args; };
    static thread_local Table table;
    if (table.base != rope.base || table.head_dim != cache.head_dim) {
        for (int i = 0; i < cache.head_dim / 2; i++) table.args.turns[i] = std::pow(rope.base, -2.0 * i / cache.head_dim) / 6.28318530717958647693;
        table.base = rope.base;
        table.head_dim = cache.head_dim;
    }
    RopeArgs r = table.args;
    r.n_axes = rope.n_axes;
    for (int x = 0, end = 0; x < 4; x++) r.axis_end[x] = end += rope.sections[x];
    const int heads = n_head + 2 * cache.n_head_kv;
    auto go = [&]<int D>() {
        auto with = [&](auto launcher) { return launcher(heads, n_rows, stream, c, r, qkv, stride, n_head, n_rows, sequence, at, positions, q_out); };
        using L = cudaError_t (*)(int, int, cudaStream_t, PagedView, RopeArgs, const float *, int64_t, int, int, const int32_t *, const int32_t *, const int32_t *, void *);
        const L launchers[4] = {launch<D, false, false>, launch<D, false, true>, launch<D, true, false>, launch<D, true, true>};
        return with(launchers[2 * half_q + (rope.neox != 0)]);
    };
    if (cache.head_dim == 128) return go.template operator()<128>();
    if (cache.head_dim == 64) return go.template operator()<64>();
    return cudaErrorInvalidValue;
}

}  // namespace cuda
}  // namespace dooms
