// Causal attention of packed prompts over a paged cache with grouped heads: query j of a prompt, at position length - queries + j of its sequence, sees the positions
// up to its own: o = sum_p softmax_p(scale q . k_p) v_p.
//
// Bound by the tensor cores and the exponentials: 4 D flops and one exponential per (query head, key), which on heads of 128 take the same time (128 x 128 scores: 512
// cycles of tcgen05.mma for S, 512 for O, 1024 of the special function units). Both run on tcgen05:
//   * A unit is one key / value head and 2 x floor(128 / G) queries: the G query heads that share the head are rows of the same tile (row = query * G + head), so that a
//     unit reads K and V once for all of them and short prompts fill the tile's rows. Its two tiles of 128 rows, A and B, take turns: while one's scores are in the
//     softmax the tensor core works on the other.
//   * One thread issues the MMAs: S = Q K^T (operands by tensor copies in the 128-byte swizzle, accumulator in tensor memory), then O += P V with P (f16) read from
//     tensor memory, where the softmax left it over the scores it came from, and V as it lies in its pages (its 128-byte rows are the N-major form of the
//     operand). One warp brings Q, K and V: a tile of 128 keys is one copy per page and 64 values.
//   * Four warps per tile do the softmax, a thread per row: the row's scores come from tensor memory once, maximum and sum need no other thread. Outputs are scaled
//     back only when a row's maximum has grown by more than 2^8 since they were last (probabilities may stand up to 2^8 higher meanwhile).
// Blocks are persistent, one per SM. The units of all prompts lie end to end, each as long as its last query's keys and a constant for what a unit costs besides; every
// block takes the same length of this line, cutting units between key tiles (where all units are short none is cut): one prompt of 8192 queries, four pieces of 500 behind
// 6000 keys and a single query behind 40000 keep all SMs alike. Of a unit that two blocks share the second, which has its end first thing, leaves its part (f32
// outputs, maxima, sums), and the first, which has its beginning last, adds that to what it has in tensor memory. Where the second has not come within a millisecond (it
// may be waiting for an SM), the first leaves its part too. Of more than two blocks each leaves its part. The last to arrive joins the parts
// in the order of the blocks. (With a part and a join for two as well four pieces of 300 to 512 took 127 us.)
// B200: 8192 queries of 40 / 8 heads of 128 in 760 us (905 TFLOP/s at the 1657 MHz that the power limit leaves; 690 in short runs), four pieces of 300 to 512 behind 1900
// to 4400 keys (32 / 8 heads) in 138 (760 TFLOP/s, 1740 MHz). A pair of steps, one of each tile, takes 4340 cycles of the first (whole time x clock / steps, units' begins
// and ends included) and 5180 of the second; each step more of a unit 4100 to 4500. It is a chain of scores, softmax and weighted sum, and the tensor core works 2048 cycles of it.
// Queries and probabilities are f16 (the type queries come in; a probability's rounding is 2^-12 of it on average, the outputs' own rounding the same again),
// scores, sums and outputs f32.
#include <cuda.h>
#include <math_constants.h>

#include <algorithm>

#include "launch.cuh"
#include "paged.cuh"
#include "ptx.cuh"

namespace dooms {
namespace cuda {

using namespace dooms::dev;

namespace {

constexpr int kRows = 128, kHalf = 64;      // rows of a tile, and keys of a tile
constexpr int kThreads = 320;               // two softmax groups of four warps, the copies' warp, the MMAs' warp
constexpr int kMostBlocks = 160;
constexpr int kUnitCost = 256;              // what a unit costs besides its keys, in keys
constexpr int kShortestSpan = kUnitCost + kRows;      // of the line, per block: a block inside a cut unit has at least two whole tiles
// Where no unit has more than kUncutTiles key tiles none is cut, and a block takes the units that are kUnitCost + kHalf or more inside the line of it: spans that are shorter
// than any unit leave a block one at most. A cut costs 5 to 10 us, which is the work of three to six tiles. Never cut / cut, in us: 8B shape, 1 x 200 queries 17.7 / 28.5,
// 1 x 1000 28.9 / 35, 4 x 64 behind 700 keys 24 / 28, 40 x 120 43 / 42, 16 x 16 behind 900 33 / 29; 0.5B, 30 x 36 behind 200
// 14 / 28. (Two of the six are faster cut. The rule looks at the batch's longest unit alone: one prompt of 1025 keys has every unit cut where it falls.) One unit per block
// at most instead of spans of 384, where no unit has two tiles: 24 questions 13.0 against 15.6.
constexpr int kSpanUncut = 192, kUncutTiles = 8;
constexpr float kRescale = 8.f;             // log2 of the growth of a maximum that is let be
constexpr float kLift = 6.f;                // probabilities are kept times 2^kLift: those of 2^-20 are still normal f16 values, and 2^(kLift + kRescale) is one

struct Args {
    PagedView c;
    const __half * q;
    __half * out;
    int n_head, group, tile_queries, n_prompts, n_rows;      // tile_queries: queries per tile
    const int32_t * sequence, * start, * lengths;
    float scale_log2;
    unsigned long long call;
    Arrivals * arrived;                     // [block]: of the unit cut behind that block, the blocks that have left their part
    float * part;                           // [block][2][tile]: outputs [D / 4][kRows] float4, then (max, sum) [kRows]
};

template <int D> constexpr int kTilePart = kRows * (D + 2);
template <int D> constexpr int kTileBytes = kRows * D * 2;
template <int D> constexpr int kRing = D == 128 ? 2 : 4;          // stages of K, and of V
template <int D> constexpr int kSmem = 1024 + 2 * kTileBytes<D> + 2 * kRing<D> * kTileBytes<D> + (kThreads + 16) * 8 + 256 + 8 * 2048;

// ---- tcgen05 and copies ----
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap * map, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ bool elect_one() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// D (+)= A B with A and B in shared memory
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// the same with A in tensor memory
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(d), "r"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
#define R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define W8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
// 32 columns of this lane's row; the values are there after tc_wait_ld
__device__ __forceinline__ void tc_ld32(uint32_t at, uint32_t * r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : R8(r, 0), R8(r, 8), R8(r, 16), R8(r, 24) : "r"(at) : "memory");
}
__device__ __forceinline__ void tc_st32(uint32_t at, const uint32_t * r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};"
                 ::W8(r, 0), W8(r, 8), W8(r, 16), W8(r, 24), "r"(at) : "memory");
}
__device__ __forceinline__ void tc_st16(uint32_t at, const uint32_t * r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::W8(r, 0), W8(r, 8), "r"(at) : "memory");
}
#undef R8
#undef W8
__device__ __forceinline__ void tc_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
// Ties what tc_ld32 loaded to the wait in front of this: nothing that uses it can be moved before it.
#define T8(r, i) "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7])
__device__ __forceinline__ void tie32(uint32_t * r) { asm volatile("" : T8(r, 0), T8(r, 8), T8(r, 16), T8(r, 24)); }
#undef T8
__device__ __forceinline__ void tc_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// Operand tiles of 128-byte rows in the 128-byte swizzle, groups of 8 rows 1024 bytes apart. K-major (Q, K): a row is 64 values of the reduction, a slice of 16 of
// them is addressed by its byte offset. N-major (V): a row is one key and 64 of the outputs' columns, the next 64 columns lie a whole tile half further.
__device__ __forceinline__ uint64_t desc_k(uint32_t at) { return uint64_t((at & 0x3FFFFu) >> 4) | (uint64_t(1) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61); }
__device__ __forceinline__ uint64_t desc_n(uint32_t at) {
    return uint64_t((at & 0x3FFFFu) >> 4) | (uint64_t((kRows * 128) >> 4) << 16) | (uint64_t(1024 >> 4) << 32) | (uint64_t(1) << 46) | (uint64_t(2) << 61);
}
// f16 operands, f32 accumulator, M = 128, N = n; n_major: B is N-major
constexpr uint32_t idesc(int n, bool n_major) { return (1u << 4) | (n_major ? 1u << 16 : 0u) | (uint32_t(n >> 3) << 17) | (uint32_t(kRows >> 4) << 24); }

__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }

__device__ __forceinline__ float max3(float a, float b, float c) { float r; asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c)); return r; }
// Two f32 at a time.
__device__ __forceinline__ uint64_t pair(float a, float b) { uint64_t r; asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b)); return r; }
__device__ __forceinline__ void halves(uint64_t v, float & a, float & b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) { uint64_t r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c)); return r; }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) { uint64_t r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b)); return r; }
// 2^x of a pair without the special function unit: x = n + f, f in [-1/2, 1/2], a polynomial for 2^f (relative error 4e-6, fitted to it), n added to the exponent. Below
// -120 it stays at 2^-120, which is nothing beside a probability.
__device__ __forceinline__ void ex2_pair(uint64_t x, float & a, float & b) {
    float xa, xb;
    halves(x, xa, xb);
    const uint64_t y = pair(fmaxf(xa, -120.f), fmaxf(xb, -120.f)), magic = pair(12582912.f, 12582912.f), t = add2(y, magic);      // 1.5 2^23: n is in the low bits
    const uint64_t f = fma2(add2(t, pair(-12582912.f, -12582912.f)), pair(-1.f, -1.f), y);
    const uint64_t p = fma2(fma2(fma2(fma2(f, pair(0.009582852013409138f, 0.009582852013409138f), pair(0.055906426161527634f, 0.055906426161527634f)), f, pair(0.24024099111557007f, 0.24024099111557007f)), f, pair(0.6931241750717163f, 0.6931241750717163f)), f, pair(1.f, 1.f));
    float ta, tb, pa, pb;
    halves(t, ta, tb);
    halves(p, pa, pb);
    a = xa == xa ? __uint_as_float(__float_as_uint(pa) + (__float_as_uint(ta) << 23)) : xa;
    b = xb == xb ? __uint_as_float(__float_as_uint(pb) + (__float_as_uint(tb) << 23)) : xb;
}

// ---- the line of units ----
// The part of prompt i that has something to see: its first row, its queries, the keys in front of its first query; no queries for one that is idle or out of range.
struct Prompt { int row, queries, ahead, seq; };
__device__ __forceinline__ Prompt prompt_at(const Args & a, int i, bool * bad = nullptr) {
    const int s = __ldg(a.sequence + i), b = __ldg(a.start + i), e = __ldg(a.start + i + 1), n = __ldg(a.lengths + i);
    const bool fine = s < a.c.n_sequences && n >= 0 && n <= a.c.capacity() && b >= 0 && e >= b && e <= a.n_rows;
    if (bad) *bad = s >= 0 && !fine;
    if (s < 0 || !fine) return {0, 0, 0, s};
    const int unseen = max(0, e - b - n);
    return {b + unseen, e - b - unseen, n - (e - b - unseen), s};
}
struct Unit { int prompt, kvh, tile; };        // tile: of 2 tile_queries queries
// The length of the line up to unit `tile` of a prompt and head.
__device__ __forceinline__ int64_t units_length(const Prompt & p, int wide, int tile) {
    const int last = (p.queries + wide - 1) / wide;      // (the last unit ends with the prompt)
    const int64_t t = tile;
    return t * (p.ahead + kUnitCost) + wide * (t * (t + 1) / 2) - (tile == last ? int64_t(last) * wide - p.queries : 0);
}
__device__ __forceinline__ int64_t prompt_length(const Args & a, const Prompt & p) {
    const int wide = 2 * a.tile_queries;
    return p.queries ? a.c.n_kv * units_length(p, wide, (p.queries + wide - 1) / wide) : 0;
}

// Adds up the parts that blocks b0 to b1 left of a unit, with the eight softmax warps: rows0 and rows1 rows of its tiles A and B; out: its first query's first head. A warp
// takes four rows at a time of two groups of rows, so that the loads of two parts' 2 x D / 32 pieces of 16 bytes are in flight together.
template <int D>
__device__ __forceinline__ void join(const Args & a, int b0, int b1, int rows0, int rows1, __half * out, int warp, int lane) {
    constexpr int kPieces = D / 32, kSets = 2 * kRows / 4;
    const int sub = lane % 4, piece = lane / 4;
    for (int set = warp; set < kSets / 2; set += 8) {      // rows 4 set + sub of tile A, and of tile B
        float4 o[2][kPieces];
        float m[2] = {-CUDART_INF_F, -CUDART_INF_F}, l[2] = {0.f, 0.f};
        const int row = 4 * set + sub;
        const bool there[2] = {row < rows0, row < rows1};
        if (!__any_sync(0xffffffffu, there[0] || there[1])) continue;
        #pragma unroll
        for (int x = 0; x < 2; x++) {
            #pragma unroll
            for (int i = 0; i < kPieces; i++) o[x][i] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        for (int b = b0; b <= b1; b += 2) {
            float2 st[2][2];
            float4 w[2][2][kPieces];
            #pragma unroll
            for (int k = 0; k < 2; k++) {
                #pragma unroll
                for (int x = 0; x < 2; x++) {
                    const float * part = a.part + ((int64_t(b + k) * 2 + (b + k == b0 ? 1 : 0)) * 2 + x) * kTilePart<D>;
                    const bool load = there[x] && b + k <= b1;
                    st[k][x] = load ? __ldcg(reinterpret_cast<const float2 *>(part + kRows * D) + row) : make_float2(-CUDART_INF_F, 0.f);
                    #pragma unroll
                    for (int i = 0; i < kPieces; i++) w[k][x][i] = load ? __ldcg(reinterpret_cast<const float4 *>(part) + (piece + 8 * i) * kRows + row) : make_float4(0.f, 0.f, 0.f, 0.f);
                }
            }
            #pragma unroll
            for (int x = 0; x < 2; x++) {
                const float top = max3(m[x], st[0][x].x, st[1][x].x), minus = top == -CUDART_INF_F ? 0.f : top, keep = ex2(m[x] - minus);
                l[x] *= keep;
                #pragma unroll
                for (int i = 0; i < kPieces; i++) { o[x][i].x *= keep; o[x][i].y *= keep; o[x][i].z *= keep; o[x][i].w *= keep; }
                #pragma unroll
                for (int k = 0; k < 2; k++) {
                    const bool some = st[k][x].x > -CUDART_INF_F;      // (a tile without a step in a part left no outputs there, only that)
                    const float share = ex2(st[k][x].x - minus);
                    l[x] = some ? fmaf(st[k][x].y, share, l[x]) : l[x];
                    #pragma unroll
                    for (int i = 0; i < kPieces; i++) {
                        if (some) {
                            o[x][i].x = fmaf(w[k][x][i].x, share, o[x][i].x); o[x][i].y = fmaf(w[k][x][i].y, share, o[x][i].y);
                            o[x][i].z = fmaf(w[k][x][i].z, share, o[x][i].z); o[x][i].w = fmaf(w[k][x][i].w, share, o[x][i].w);
                        }
                    }
                }
                m[x] = top;
            }
        }
        #pragma unroll
        for (int x = 0; x < 2; x++) {
            if (!there[x]) continue;
            const float by = l[x] > 0.f || l[x] != l[x] ? 1.f / l[x] : 0.f;
            __half * const to = out + ((int64_t(x) * a.tile_queries + row / a.group) * a.n_head + row % a.group) * D;
            #pragma unroll
            for (int i = 0; i < kPieces; i++) {
                const __half2 h[2] = {__floats2half2_rn(o[x][i].x * by, o[x][i].y * by), __floats2half2_rn(o[x][i].z * by, o[x][i].w * by)};
                *reinterpret_cast<uint2 *>(to + (piece + 8 * i) * 4) = *reinterpret_cast<const uint2 *>(h);
            }
        }
    }
}

// Outputs of rows that a value they do not see has spoilt: positions of a unit's later queries lie in the same tiles, and their probability of zero times an infinity
// or NaN is NaN. A warp's rows of one tile, of those in `rows` (a NaN among their outputs, of a finite sum); key0, key1: the segment's keys that the tile had. Such a row whose
// unseen values are at fault is worked out once more, key by key over the segment, against the reference its sum stands for.
struct Spoilt { uint32_t rows; int seq, kvh, q_row, row0, first, key0, key1, queries; };      // row0: the warp's first row; first: the position of the tile's first query
// out: the tile's outputs, f16, times by; else part: the tile's part. Returns the rows that it wrote.
template <int D>
__device__ __noinline__ uint32_t mend_rows(const Args & a, const Spoilt w, float ref, float by, __half * out, float * part) {
    constexpr int kMine = D / 32;
    const int lane = threadIdx.x % 32;
    uint32_t written = 0;
    auto line = [&](int key) { return max(a.c.row(w.seq, key), int64_t(0)) * a.c.n_kv + w.kvh; };
    for (uint32_t rest = w.rows; rest; rest &= rest - 1) {
        const int i = __ffs(rest) - 1, r = w.row0 + i, position = w.first + min(r / a.group, w.queries - 1);
        bool odd = false;
        for (int key = max(position + 1, w.key0); key < w.key1; key++) {
            const __half * v = a.c.v + line(key) * D + lane * kMine;
            for (int d = 0; d < kMine; d++) odd = odd || !(fabsf(__half2float(v[d])) <= 65504.f);
        }
        if (!__any_sync(0xffffffffu, odd)) continue;
        written |= 1u << i;
        const float minus = kLift - __shfl_sync(0xffffffffu, ref, i);
        const __half * q = a.q + ((int64_t(w.q_row) + r / a.group) * a.n_head + w.kvh * a.group + r % a.group) * D;
        float o[kMine] = {};
        const int end = min(w.key1, position + 1);
        for (int k0 = w.key0; k0 < end; k0 += 32) {
            float p = 0.f;
            if (k0 + lane < end) {
                const __half * k = a.c.k + line(k0 + lane) * D;
                float s = 0.f;
                for (int d = 0; d < D; d++) s = fmaf(__half2float(q[d]), __half2float(k[d]), s);
                p = __half2float(__float2half_rn(ex2(fmaf(s, a.scale_log2, minus))));      // (as the other rows' enter the products)
            }
            for (int j = 0; j < min(32, end - k0); j++) {
                const float pj = __shfl_sync(0xffffffffu, p, j);
                const __half * v = a.c.v + line(k0 + j) * D + lane * kMine;
                for (int d = 0; d < kMine; d++) o[d] = fmaf(pj, __half2float(v[d]), o[d]);
            }
        }
        const float by_row = __shfl_sync(0xffffffffu, by, i);
        for (int d = 0; d < kMine; d++) {
            const int c = lane * kMine + d;
            if (out) out[(int64_t(r / a.group) * a.n_head + r % a.group) * D + c] = __float2half_rn(o[d] * by_row);
            else part[((c / 4) * kRows + r) * 4 + c % 4] = o[d];
        }
    }
    __syncwarp();
    return written;
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1) k_attention_prompt(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                                                                  const __grid_constant__ CUtensorMap vmap, const __grid_constant__ Args a) {
    constexpr int S = kRing<D>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t q_at = (smem_u32(smem_raw) + 1023u) & ~1023u, k_at = q_at + 2 * kTileBytes<D>, v_at = k_at + S * kTileBytes<D>;
    int64_t * const sums = reinterpret_cast<int64_t *>(smem_raw + (v_at + S * kTileBytes<D> - smem_u32(smem_raw)));
    int * const flag = reinterpret_cast<int *>(sums + kThreads + 15);
    const uint32_t bars = smem_u32(sums + kThreads + 16);
    const uint32_t q_full = bars, q_empty = bars + 8, s_full = bars + 16, p_full = bars + 32, o_done = bars + 64, k_full = bars + 80, k_empty = k_full + 8 * S, v_full = k_empty + 8 * S,
                   v_empty = v_full + 8 * S, v_fixed = v_empty + 8 * S, tmem_slot = v_fixed + 8 * S, all_done = tmem_slot + 8;
    const uint32_t staged = (bars + 256 + 15u) & ~15u;      // 2 KB per softmax warp
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;      // (a warp's number, as something the whole warp has)
    if (threadIdx.x == 0) {
        mbar_init(q_full, 1); mbar_init(q_empty, 1); mbar_init(all_done, 1);
        for (int x = 0; x < 2; x++) { mbar_init(s_full + 8 * x, 1); mbar_init(p_full + 16 * x, 4); mbar_init(p_full + 16 * x + 8, 4); mbar_init(o_done + 8 * x, 1); }
        for (int s = 0; s < S; s++) { mbar_init(k_full + 8 * s, 1); mbar_init(k_empty + 8 * s, 1); mbar_init(v_full + 8 * s, 1); mbar_init(v_empty + 8 * s, 1); mbar_init(v_fixed + 8 * s, 1); }
        mbar_init_fence();
    }
    if (warp == 9) {      // the MMAs' warp owns the tensor memory
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(tmem_slot) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    } else if (warp == 8 && lane < 3) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(lane == 0 ? &qmap : lane == 1 ? &kmap : &vmap) : "memory");
    }
    pdl_wait();

    // ---- the line: every thread adds up a run of prompts, the block scans the runs ----
    const int wide = 2 * a.tile_queries, per = (a.n_prompts + kThreads - 1) / kThreads;
    bool uncut;
    {
        const int i0 = min(a.n_prompts, int(threadIdx.x) * per), i1 = min(a.n_prompts, i0 + per);
        int64_t mine = 0;
        bool many = false;
        for (int i = i0; i < i1; i++) {
            const Prompt q = prompt_at(a, i);
            mine += prompt_length(a, q);
            const int keys = q.queries ? q.ahead + q.queries : 0;
            many = many || keys > kUncutTiles * kRows;
        }
        int64_t run = mine;
        for (int d = 1; d < 32; d <<= 1) { const int64_t o = __shfl_up_sync(0xffffffffu, run, d); if (lane >= d) run += o; }
        if (lane == 31) sums[kThreads + warp] = run;
        __syncthreads();
        for (int w = 0; w < warp; w++) run += sums[kThreads + w];
        sums[threadIdx.x] = run - mine;
        if (threadIdx.x == kThreads - 1) sums[kThreads + 14] = run;
        tc_fence_before();
        uncut = __syncthreads_or(many) == 0;
        tc_fence_after();
    }
    uint32_t tmem;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(tmem) : "r"(tmem_slot));
    tmem = __shfl_sync(0xffffffffu, tmem, 0);
    const int64_t total = sums[kThreads + 14];
    const int blocks = max(1, int(min(int64_t(gridDim.x), total / (uncut ? kSpanUncut : kShortestSpan))));
    const int64_t each = quotient(total, blocks);
    auto part_at = [&](int b) { return part_of(total, each, b, blocks); };
    const bool idle = total == 0 || int(blockIdx.x) >= blocks;
    const int64_t from = idle ? 0 : part_at(blockIdx.x), to = idle ? 0 : part_at(blockIdx.x + 1);
    Unit u{0, 0, 0};
    Prompt p{0, 0, 0, 0};
    int64_t unit_at = 0;      // where unit u begins
    if (!idle) {
        int th = 0;
        #pragma unroll
        for (int step = 256; step; step >>= 1) if (th + step < kThreads && sums[th + step] <= from) th += step;
        int64_t at = sums[th];
        int i = th * per;
        int64_t n;
        for (;; i++) { p = prompt_at(a, i); n = prompt_length(a, p); if (at + n > from) break; at += n; }
        const int tiles = (p.queries + wide - 1) / wide;
        const int64_t head = units_length(p, wide, tiles);
        const int kvh = int(quotient(from - at, head));
        at += kvh * head;
        int t = 0;
        for (int step = 1 << (31 - __clz(tiles)); step; step >>= 1) if (t + step < tiles && at + units_length(p, wide, t + step) <= from) t += step;
        u = {i, kvh, t};
        unit_at = at + units_length(p, wide, t);
    }
    // The segment of unit u that is this block's: key tiles [t0, t1) of its `tiles`.
    struct Segment { int row, queries, first, keys, tiles, t0, t1; int64_t next; };
    auto tile_of = [&](int64_t x, int tiles) { return uncut ? (x < kUnitCost + kRows / 2 ? 0 : tiles) : int(max(int64_t(0), min(int64_t(tiles), (x - kUnitCost + kRows / 2) / kRows))); };      // (x - kUnitCost < 0 rounds to 0)
    auto segment = [&]() -> Segment {
        const int q0 = u.tile * wide, n = min(wide, p.queries - q0), keys = p.ahead + q0 + n, tiles = (keys + kRows - 1) / kRows;
        const int64_t end = unit_at + keys + kUnitCost;
        return {p.row + q0, n, p.ahead + q0, keys, tiles, from > unit_at ? tile_of(from - unit_at, tiles) : 0, to < end ? tile_of(to - unit_at, tiles) : tiles, end};
    };
    auto next_unit = [&](const Segment & s) {
        unit_at = s.next;
        if (++u.tile * wide < p.queries) return;
        u.tile = 0;
        if (++u.kvh < a.c.n_kv) return;
        u.kvh = 0;
        do { u.prompt++; } while (u.prompt < a.n_prompts && (p = prompt_at(a, u.prompt)).queries == 0);
    };
    // key tiles of the segment that tile x of the unit (its queries [x tile_queries, ..)) takes part in
    auto steps_of = [&](const Segment & s, int x) {
        const int q = min(s.queries, (x + 1) * a.tile_queries);
        if (q <= x * a.tile_queries) return 0;
        return max(0, min(s.t1, (s.first + q + kRows - 1) / kRows) - s.t0);
    };
    bool ok = true;

    if (idle) {
        // (nothing but the end)
    } else if (warp == 8) {
        // ---- the copies ----
        const int box = min(kRows, 1 << a.c.page_shift), piece = lane / (D / 64), half = lane % (D / 64);
        int stage = 0, units = 0, begun = 0;      // begun: copies into the stage at hand (keys, then values)
        uint32_t phase = 0;
        while (unit_at < to && ok) {
            const Segment s = segment();
            if (s.t0 < s.t1) {
                ok = mbar_wait(q_empty, uint32_t(units & 1) ^ 1u);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                units++;
                if (lane == 0) {
                    const int boxes = s.queries > a.tile_queries ? 2 : 1;
                    mbar_arrive_expect_tx(q_full, uint32_t(boxes * a.tile_queries * a.group) * D * 2u);
                    for (int x = 0; x < boxes; x++) {
                        for (int h = 0; h < D / 64; h++) tma_load_3d(q_at + x * kTileBytes<D> + h * (kRows * 128), &qmap, h * 64, u.kvh * a.group, s.row + x * a.tile_queries, q_full);
                    }
                }
                __syncwarp();
                const int32_t * table = a.c.table + int64_t(p.seq) * a.c.max_pages;
                for (int t = s.t0; t < s.t1 && ok; t++) {
                    const int valid = min(kRows, s.keys - t * kRows), used = (valid + box - 1) / box, key = t * kRows + piece * box;
                    int page = 0;
                    if (piece < used) {
                        page = __ldg(table + (key >> a.c.page_shift));
                        if (uint32_t(page) >= uint32_t(a.c.n_pages)) { a.c.fail(); page = 0; }
                    }
                    const int z = (page << a.c.page_shift) + (key & ((1 << a.c.page_shift) - 1));
                    const uint32_t at = stage * kTileBytes<D> + half * (kRows * 128) + piece * box * 128;
                    #pragma unroll
                    for (int kv = 0; kv < 2; kv++) {
                        const uint32_t full = (kv ? v_full : k_full) + 8 * stage;
                        ok = ok && mbar_wait((kv ? v_empty : k_empty) + 8 * stage, phase ^ 1u);
                        ok = __all_sync(0xffffffffu, ok);
                        if (!ok) break;
                        if (lane == 0) mbar_arrive_expect_tx(full, uint32_t(used * box) * D * 2u);
                        __syncwarp();
                        if (piece < used) tma_load_3d((kv ? v_at : k_at) + at, kv ? &vmap : &kmap, half * 64, u.kvh, z, full);
                        begun++;
                    }
                    if (!ok) break;
                    if (valid < kRows) {      // values behind the last key seen are zeros: a probability of zero times what a page may hold there has to stay zero
                        ok = mbar_wait(v_full + 8 * stage, phase);
                        ok = __all_sync(0xffffffffu, ok);
                        for (int i = lane; i < (kRows - valid) * (D / 8); i += 32) {
                            const uint32_t row = uint32_t(valid + i / (D / 8)), c = uint32_t(i % (D / 8));
                            asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(v_at + stage * kTileBytes<D> + (c / 8) * (kRows * 128) + row * 128u + (c % 8) * 16u), "r"(0u) : "memory");
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                        if (lane == 0 && ok) mbar_arrive(v_fixed + 8 * stage);
                    }
                    if (!ok) break;
                    begun = 0;
                    if (++stage == S) { stage = 0; phase ^= 1u; }
                }
            }
            next_unit(s);
        }
        // no copy is under way when the block ends, not behind a wait that ran out either: the last queries, and each stage's last keys and values
        if (units) ok = mbar_wait(q_full, uint32_t(units - 1) & 1u) && ok;
        for (int s = 0; s < S; s++) {
            ok = mbar_wait(k_full + 8 * s, s < stage || (s == stage && begun > 0) ? phase : phase ^ 1u) && ok;
            ok = mbar_wait(v_full + 8 * s, s < stage || (s == stage && begun > 1) ? phase : phase ^ 1u) && ok;
        }
    } else if (warp == 9) {
        // ---- the MMAs: the whole warp walks the steps, so that what describes them stays uniform; one elected thread issues ----
        constexpr uint32_t id_s = idesc(kRows, false), id_o = idesc(D, true);
        int kstage = 0, vstage = 0, units = 0;
        uint32_t kphase = 0, vphase = 0, fixed = 0, done0 = 0, done1 = 0;      // fixed: the phases of v_fixed, a bit per stage; done: probabilities taken
        const bool leader = elect_one();
        auto scores = [&](int x) {
            const uint32_t q = q_at + x * kTileBytes<D>, k = k_at + kstage * kTileBytes<D>, d = tmem + x * kRows;
            if (leader) {
                #pragma unroll
                for (int kk = 0; kk < D / 16; kk++) {
                    const uint32_t at = (kk / 4) * (kRows * 128) + (kk % 4) * 32;
                    mma_ss(d, desc_k(q + at), desc_k(k + at), id_s, kk != 0);
                }
                tc_commit(s_full + 8 * x);
            }
            __syncwarp();
        };
        // one half of the keys, the upper (half = 1) first
        auto outputs = [&](int x, int half, bool add) {
            const uint32_t v = v_at + vstage * kTileBytes<D> + half * (kHalf * 128), p16 = tmem + x * kRows + kHalf + half * 32, d = tmem + 256 + x * kRows;
            if (leader) {
                #pragma unroll
                for (int kk = 0; kk < kHalf / 16; kk++) mma_ts(d, p16 + kk * 8, desc_n(v + kk * (16 * 128)), id_o, add || kk != 0);
                if (half == 0) tc_commit(o_done + 8 * x);
            }
            __syncwarp();
        };
        auto commit = [&](uint32_t bar) {
            if (leader) tc_commit(bar);
            __syncwarp();
        };
        auto wait = [&](uint32_t bar, uint32_t parity) {
            ok = mbar_wait(bar, parity);
            ok = __all_sync(0xffffffffu, ok);
            return ok;
        };
        while (unit_at < to && ok) {
            const Segment s = segment();
            const int n = s.t1 - s.t0;
            if (n > 0) {
                const int steps0 = steps_of(s, 0), steps1 = steps_of(s, 1);
                if (!wait(q_full, uint32_t(units & 1)) || !wait(k_full + 8 * kstage, kphase)) break;
                units++;
                tc_fence_after();
                if (steps0 > 0) scores(0);
                if (steps1 > 0) scores(1);
                commit(k_empty + 8 * kstage);
                if (n == 1) commit(q_empty);
                if (++kstage == S) { kstage = 0; kphase ^= 1u; }
                for (int j = 0; j < n && ok; j++) {
                    bool have_v = false, have_k = false;
                    #pragma unroll
                    for (int x = 0; x < 2; x++) {
                        const int steps = x ? steps1 : steps0;
                        if (ok && j < steps) {
                            const uint32_t parity = (x ? done1 : done0) & 1u;
                            if (!wait(p_full + 16 * x, parity)) break;
                            if (!have_v) {
                                if (!wait(v_full + 8 * vstage, vphase)) break;
                                if (s.keys - (s.t0 + j) * kRows < kRows) { if (!wait(v_fixed + 8 * vstage, fixed >> vstage & 1u)) break; fixed ^= 1u << vstage; }
                                have_v = true;
                            }
                            if (x) done1++; else done0++;
                            tc_fence_after();
                            outputs(x, 1, j != 0);
                            if (!wait(p_full + 16 * x + 8, parity)) break;
                            tc_fence_after();
                            outputs(x, 0, true);
                        }
                        if (ok && j + 1 < steps) {
                            if (!have_k) { if (!wait(k_full + 8 * kstage, kphase)) break; have_k = true; }
                            tc_fence_after();
                            scores(x);
                        }
                    }
                    if (!ok) break;
                    commit(v_empty + 8 * vstage);
                    if (++vstage == S) { vstage = 0; vphase ^= 1u; }
                    if (j + 1 < n) {
                        commit(k_empty + 8 * kstage);
                        if (j + 2 == n) commit(q_empty);
                        if (++kstage == S) { kstage = 0; kphase ^= 1u; }
                    }
                }
            }
            next_unit(s);
        }
        // nor is a product, when the tensor memory is given back
        const bool fine = ok;
        commit(all_done);
        ok = wait(all_done, 0u) && fine;
    } else {
        // ---- softmax: group x (four warps) has tile x, a thread has row r of it ----
        const int x = warp / 4, r = threadIdx.x % kRows;
        const uint32_t lanes = uint32_t((warp % 4) * 32) << 16, s_at = tmem + lanes + x * kRows, o_at = tmem + lanes + 256 + x * kRows;
        const int query = x * a.tile_queries + r / a.group;      // of the unit
        const bool row_there = r < a.tile_queries * a.group;
        uint32_t step = 0;      // scores taken
        while (unit_at < to) {
            const Segment s = segment();
            if (s.t0 < s.t1) {
                const int n = steps_of(s, x);
                float ref = 0.f, sum = 0.f;      // the row's reference (what its probabilities are relative to) and sum
                bool seen = false;
                const int position = s.first + min(query, s.queries - 1), lowest = s.first + x * a.tile_queries;      // the row's, and the tile's first
                for (int j = 0; j < n; j++) {
                    ok = ok && mbar_wait(s_full + 8 * x, step & 1u);
                    ok = __all_sync(0xffffffffu, ok);
                    tc_fence_after();
                    // The scores come in quarters of 32, the last two of which stay in registers; the first two are read again behind the work on those (all 128 held
                    // at once spill). Probabilities go over the second half's place, last quarter first.
                    const int first = (s.t0 + j) * kRows;
                    const bool masked = first + kRows - 1 > lowest;
                    const int limit = position - first;
                    uint32_t va[32], vb[32];
                    auto mask = [&](uint32_t (&v)[32], int c0) {
                        if (masked) {
                            #pragma unroll
                            for (int c = 0; c < 32; c++) v[c] = c0 + c <= limit ? v[c] : 0xff800000u;
                        }
                    };
                    float m4[4];
                    #pragma unroll
                    for (int half = 0; half < 2; half++) {
                        tc_ld32(s_at + half * kHalf, va);
                        tc_ld32(s_at + half * kHalf + 32, vb);
                        tc_wait_ld();
                        tie32(va);
                        tie32(vb);
                        mask(va, half * kHalf);
                        mask(vb, half * kHalf + 32);
                        #pragma unroll
                        for (int c = 0; c < 32; c += 2) {
                            float & m0 = m4[c / 2 % 2], & m1 = m4[2 + c / 2 % 2];
                            m0 = half == 0 && c < 4 ? fmaxf(__uint_as_float(va[c]), __uint_as_float(va[c + 1])) : max3(m0, __uint_as_float(va[c]), __uint_as_float(va[c + 1]));
                            m1 = half == 0 && c < 4 ? fmaxf(__uint_as_float(vb[c]), __uint_as_float(vb[c + 1])) : max3(m1, __uint_as_float(vb[c]), __uint_as_float(vb[c + 1]));
                        }
                    }
                    const float m = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * a.scale_log2;
                    const bool grows = row_there && m > -CUDART_INF_F && (!seen || m > ref + kRescale);
                    if (__any_sync(0xffffffffu, grows && seen)) {
                        // outputs so far, relative to the new reference
                        const float by = grows && seen ? ex2(ref - m) : 1.f;
                        ok = ok && mbar_wait(o_done + 8 * x, (step - 1) & 1u);
                        ok = __all_sync(0xffffffffu, ok);
                        tc_fence_after();
                        #pragma unroll
                        for (int c = 0; c < D; c += 32) {
                            uint32_t o[32];
                            tc_ld32(o_at + c, o);
                            tc_wait_ld();
                            tie32(o);
                            #pragma unroll
                            for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * by);
                            tc_st32(o_at + c, o);
                        }
                        sum *= by;
                    }
                    if (grows) { ref = m; seen = true; }
                    const float minus = kLift - ref;
                    uint64_t sums[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};
                    const uint64_t scale2 = pair(a.scale_log2, a.scale_log2), minus2 = pair(minus, minus);
                    // 32 probabilities from their scores, as f16 pairs in the first half of v: one in eight by the polynomial
                    auto powers = [&](uint32_t (&v)[32]) {
                        #pragma unroll
                        for (int c = 0; c < 32; c += 2) {
                            const uint64_t y = fma2(pair(__uint_as_float(v[c]), __uint_as_float(v[c + 1])), scale2, minus2);
                            float e0, e1;
                            if (c % 16 == 14) {
                                ex2_pair(y, e0, e1);
                            } else {
                                halves(y, e0, e1);
                                e0 = ex2(e0);
                                e1 = ex2(e1);
                            }
                            sums[c / 2 % 2] = add2(sums[c / 2 % 2], pair(e0, e1));
                            const __half2 h = __floats2half2_rn(e0, e1);
                            v[c / 2] = *reinterpret_cast<const uint32_t *>(&h);
                        }
                    };
                    powers(vb);
                    tc_st16(s_at + kHalf + 48, vb);
                    tc_ld32(s_at + 32, vb);
                    powers(va);
                    tc_st16(s_at + kHalf + 32, va);
                    tc_wait_st();      // the upper half's probabilities go ahead
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(p_full + 16 * x);
                    tc_wait_ld();
                    tie32(vb);
                    tc_ld32(s_at, va);
                    mask(vb, 32);
                    powers(vb);
                    tc_st16(s_at + kHalf + 16, vb);
                    tc_wait_ld();
                    tie32(va);
                    mask(va, 0);
                    powers(va);
                    tc_st16(s_at + kHalf, va);
                    float s4[4];
                    halves(sums[0], s4[0], s4[1]);
                    halves(sums[1], s4[2], s4[3]);
                    sum += (s4[0] + s4[1]) + (s4[2] + s4[3]);
                    tc_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(p_full + 16 * x + 8);
                    step++;
                }
                // ---- the unit's outputs, or the segment's part of them ----
                if (n > 0) {
                    ok = ok && mbar_wait(o_done + 8 * x, (step - 1) & 1u);
                    ok = __all_sync(0xffffffffu, ok);
                    tc_fence_after();
                }
                const bool whole = s.t0 == 0 && s.t1 == s.tiles;
                uint64_t odd[2] = {pair(0.f, 0.f), pair(0.f, 0.f)};      // the outputs' sum: NaN if one is
                // 32 columns of the warp's 32 rows, from a thread per row: through shared memory, so that a store is eight rows of 64 bytes and not 32 pieces of 16
                const int last = min(a.tile_queries, s.queries - x * a.tile_queries) * a.group;      // rows of the tile that are there
                __half * const out = a.out + ((int64_t(s.row) + x * a.tile_queries) * a.n_head + u.kvh * a.group) * D;
                auto write_rows = [&](const uint32_t * o, int c) {
                    const uint32_t at = staged + warp * 2048u;
                    #pragma unroll
                    for (uint32_t i = 0; i < 4; i++) {
                        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at + lane * 64u + ((i ^ (uint32_t(lane) >> 1 & 3u)) << 4)), "r"(o[4 * i]), "r"(o[4 * i + 1]), "r"(o[4 * i + 2]),
                                     "r"(o[4 * i + 3]) : "memory");
                    }
                    __syncwarp();
                    #pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t row = uint32_t(lane / 4 + 8 * i), piece = uint32_t(lane % 4);
                        uint4 w;
                        asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w) : "r"(at + row * 64u + ((piece ^ (row >> 1 & 3u)) << 4)) : "memory");
                        const int rr = (warp % 4) * 32 + int(row);
                        if (rr < last) *reinterpret_cast<uint4 *>(out + (int64_t(rr / a.group) * a.n_head + rr % a.group) * D + c + piece * 8) = w;
                    }
                    __syncwarp();
                };
                auto spoilt = [&](float sum) {
                    float a0, a1;
                    halves(add2(odd[0], odd[1]), a0, a1);
                    a0 += a1;
                    const uint32_t rows = __ballot_sync(0xffffffffu, a0 != a0 && sum - sum == 0.f && r < last);
                    const int key0 = s.t0 * kRows;
                    return Spoilt{rows, rows ? __ldg(a.sequence + u.prompt) : 0, u.kvh, s.row + x * a.tile_queries, (warp % 4) * 32, s.first + x * a.tile_queries, key0, min(s.keys, key0 + n * kRows),
                                  s.queries - x * a.tile_queries};
                };
                if (whole) {
                    const float by = sum > 0.f || sum != sum ? 1.f / sum : 0.f;
                    if (n > 0) {
                        #pragma unroll
                        for (int c = 0; c < D; c += 32) {
                            uint32_t o[32];
                            tc_ld32(o_at + c, o);
                            tc_wait_ld();
                            tie32(o);
                            #pragma unroll
                            for (int i = 0; i < 32; i += 2) odd[i / 2 % 2] = add2(odd[i / 2 % 2], pair(__uint_as_float(o[i]), __uint_as_float(o[i + 1])));
                            #pragma unroll
                            for (int i = 0; i < 32; i += 2) {
                                const __half2 h = __floats2half2_rn(__uint_as_float(o[i]) * by, __uint_as_float(o[i + 1]) * by);
                                o[i / 2] = *reinterpret_cast<const uint32_t *>(&h);
                            }
                            write_rows(o, c);
                        }
                        const Spoilt w = spoilt(sum);
                        if (w.rows) mend_rows<D>(a, w, ref, by, out, nullptr);
                    }
                } else {
                    // the blocks that share the unit: those whose tiles are not none
                    int b0 = int(quotient((unit_at + 1) * blocks - 1, total)), b1 = int(quotient(s.next * blocks - 1, total));
                    if (tile_of(part_at(b0 + 1) - unit_at, s.tiles) == 0) b0++;
                    if (tile_of(part_at(b1) - unit_at, s.tiles) == s.tiles) b1--;
                    const bool keeps = b1 == b0 + 1 && s.t0 == 0;      // of two blocks the first adds the other's part to what it has
                    float * const part = a.part + ((int64_t(blockIdx.x) * 2 + (s.t0 == 0 ? 1 : 0)) * 2 + x) * kTilePart<D>;
                    const float2 mine = make_float2(n > 0 && seen ? ref : -CUDART_INF_F, n > 0 ? sum : 0.f);
                    uint32_t mended = 0;
                    if (n > 0) {
                        #pragma unroll
                        for (int c = 0; c < D; c += 32) {
                            uint32_t o[32];
                            tc_ld32(o_at + c, o);
                            tc_wait_ld();
                            tie32(o);
                            #pragma unroll
                            for (int i = 0; i < 32; i += 2) odd[i / 2 % 2] = add2(odd[i / 2 % 2], pair(__uint_as_float(o[i]), __uint_as_float(o[i + 1])));
                            if (!keeps) {
                                #pragma unroll
                                for (int i = 0; i < 8; i++) {
                                    reinterpret_cast<uint4 *>(part)[(c / 4 + i) * kRows + r] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                                }
                            }
                        }
                        const Spoilt w = spoilt(sum);
                        if (w.rows) mended = mend_rows<D>(a, w, ref, 1.f, nullptr, part);
                    }
                    Arrivals * const counter = a.arrived + b0;
                    bool leaves = !keeps;
                    if (keeps) {
                        asm volatile("bar.sync 1, 256;" ::: "memory");
                        if (threadIdx.x == 0) { *flag = paged_counter_wait(counter, a.call, !ok); ok = ok && *flag >= 0; }
                        asm volatile("bar.sync 1, 256;" ::: "memory");
                        const int came = *flag;
                        leaves = came == 0;
                        const bool again = mended >> lane & 1u;      // (this row's outputs were worked out again, into the part)
                        if (came > 0 && n > 0) {      // (the arithmetic of join(), so that it does not matter which of the two it is)
                            __threadfence();
                            const float * const other = a.part + (int64_t(b1) * 4 + x) * kTilePart<D>;
                            const float2 theirs = __ldcg(reinterpret_cast<const float2 *>(other + kRows * D) + r);
                            const float top = fmaxf(mine.x, theirs.x), minus = top == -CUDART_INF_F ? 0.f : top;
                            const bool some = mine.x > -CUDART_INF_F, theirs_some = theirs.x > -CUDART_INF_F;
                            const float share = ex2(mine.x - minus), their_share = ex2(theirs.x - minus);
                            float l = some ? fmaf(mine.y, share, 0.f) : 0.f;
                            l = theirs_some ? fmaf(theirs.y, their_share, l) : l;
                            const float by = l > 0.f || l != l ? 1.f / l : 0.f;
                            #pragma unroll
                            for (int c = 0; c < D; c += 32) {
                                uint32_t o[32];
                                float4 w[8];
                                #pragma unroll
                                for (int i = 0; i < 8; i++) w[i] = theirs_some ? __ldcg(reinterpret_cast<const float4 *>(other) + (c / 4 + i) * kRows + r) : make_float4(0.f, 0.f, 0.f, 0.f);
                                tc_ld32(o_at + c, o);
                                tc_wait_ld();
                                tie32(o);
                                if (again) {
                                    #pragma unroll
                                    for (int i = 0; i < 32; i++) o[i] = __float_as_uint(__ldcg(part + ((c / 4 + i / 4) * kRows + r) * 4 + i % 4));
                                }
                                #pragma unroll
                                for (int i = 0; i < 8; i++) {
                                    float v[4] = {__uint_as_float(o[4 * i]), __uint_as_float(o[4 * i + 1]), __uint_as_float(o[4 * i + 2]), __uint_as_float(o[4 * i + 3])};
                                    const float add[4] = {w[i].x, w[i].y, w[i].z, w[i].w};
                                    #pragma unroll
                                    for (int k = 0; k < 4; k++) v[k] = fmaf(add[k], theirs_some ? their_share : 0.f, some ? fmaf(v[k], share, 0.f) : 0.f) * by;
                                    const __half2 h0 = __floats2half2_rn(v[0], v[1]), h1 = __floats2half2_rn(v[2], v[3]);
                                    o[2 * i] = *reinterpret_cast<const uint32_t *>(&h0);
                                    o[2 * i + 1] = *reinterpret_cast<const uint32_t *>(&h1);
                                }
                                write_rows(o, c);
                            }
                        } else if (leaves && n > 0) {
                            #pragma unroll
                            for (int c = 0; c < D; c += 32) {
                                uint32_t o[32];
                                tc_ld32(o_at + c, o);
                                tc_wait_ld();
                                tie32(o);
                                if (!again) {
                                    #pragma unroll
                                    for (int i = 0; i < 8; i++) {
                                        reinterpret_cast<uint4 *>(part)[(c / 4 + i) * kRows + r] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                                    }
                                }
                            }
                        }
                    }
                    if (leaves) {
                        // (a tile without a step in this segment leaves no outputs, and a maximum that says so)
                        reinterpret_cast<float2 *>(part + kRows * D)[r] = mine;
                        tc_fence_before();
                        __threadfence();
                        asm volatile("bar.sync 1, 256;" ::: "memory");
                        if (threadIdx.x == 0) *flag = paged_counter_arrive(counter, a.call, b1 - b0 + 1, !ok);
                        asm volatile("bar.sync 1, 256;" ::: "memory");
                        if (*flag) {
                            __threadfence();
                            join<D>(a, b0, b1, x == 0 ? last : min(a.tile_queries, s.queries) * a.group, x == 1 ? last : max(0, s.queries - a.tile_queries) * a.group,
                                    a.out + (int64_t(s.row) * a.n_head + u.kvh * a.group) * D, warp, lane);
                        }
                    }
                }
                tc_fence_before();
            }
            next_unit(s);
        }
    }
    if (!ok && lane == 0) a.c.gave_up();
    // ---- what is out of range is reported, queries that see nothing are zero ----
    for (int i = blockIdx.x; i < a.n_prompts; i += gridDim.x) {
        bool bad = false;
        const Prompt q = prompt_at(a, i, &bad);
        if (bad && threadIdx.x == 0) a.c.fail();
        if (bad || q.seq < 0) continue;
        const int b = a.start[i], unseen = (a.start[i + 1] - b) - q.queries;
        for (int64_t v = threadIdx.x; v < int64_t(unseen) * a.n_head * D; v += kThreads) a.out[int64_t(b) * a.n_head * D + v] = __half(0.f);
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 9) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
}

template <int D>
cudaError_t launch(const Args & a, const TensorMap & qmap, const TensorMap & kmap, const TensorMap & vmap, int blocks, cudaStream_t stream) {
    static std::atomic<uint64_t> done{0};
    const cudaError_t e = allow_dynamic_smem(k_attention_prompt<D>, kSmem<D>, done);
    if (e != cudaSuccess) return e;
    return launch_pdl(k_attention_prompt<D>, dim3(unsigned(blocks)), dim3(kThreads), kSmem<D>, stream, reinterpret_cast<const CUtensorMap &>(qmap),
                      reinterpret_cast<const CUtensorMap &>(kmap), reinterpret_cast<const CUtensorMap &>(vmap), a);
}

}  // namespace

size_t attention_prompt_scratch_bytes(int, int, int head_dim) { return size_t(kMostBlocks) * (2 * 2 * kRows * (head_dim + 2) * 4 + 8); }

cudaError_t launch_attention_prompt_paged(const PagedCache & cache, const void * q, void * out, int n_head, int n_rows, int n_prompts, const int32_t * sequence,
                                          const int32_t * start, const int32_t * lengths, float scale, void * scratch, int * error, cudaStream_t stream) {
    Args a{};
    a.c = paged_view(cache, error);
    a.q = static_cast<const __half *>(q);
    a.out = static_cast<__half *>(out);
    a.n_head = n_head; a.group = n_head / cache.n_head_kv; a.tile_queries = kRows / a.group; a.n_prompts = n_prompts; a.n_rows = n_rows;
    a.sequence = sequence; a.start = start; a.lengths = lengths;
    a.scale_log2 = scale * 1.44269504f;
    a.call = paged_call();
    a.arrived = static_cast<Arrivals *>(scratch);
    a.part = reinterpret_cast<float *>(a.arrived + kMostBlocks);
    TensorMap qmap, kmap, vmap;
    const int box = std::min(kRows, cache.page_size);
    cudaError_t e = make_heads_map(&qmap, q, cache.head_dim, n_head, n_rows, a.group, a.tile_queries);
    if (e == cudaSuccess) e = make_heads_map(&kmap, cache.keys, cache.head_dim, cache.n_head_kv, int64_t(cache.n_pages) * cache.page_size, 1, box);
    if (e == cudaSuccess) e = make_heads_map(&vmap, cache.values, cache.head_dim, cache.n_head_kv, int64_t(cache.n_pages) * cache.page_size, 1, box);
    if (e != cudaSuccess) return e;
    const int blocks = std::min(kMostBlocks, sm_count());
    if (cache.head_dim == 128) return launch<128>(a, qmap, kmap, vmap, blocks, stream);
    if (cache.head_dim == 64) return launch<64>(a, qmap, kmap, vmap, blocks, stream);
    return cudaErrorInvalidValue;
}

}  // namespace cuda
}  // namespace dooms
