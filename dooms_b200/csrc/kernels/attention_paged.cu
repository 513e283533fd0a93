// Attention of one new token per row over its sequence's pages: o = sum_j softmax_j(scale q . k_j) v_j over the row's positions j < length, the query heads of a
// key / value head reading it once.
//
// Bound by device memory: 4 D bytes per (key, key / value head), each read once, against 4 G D flops. So the work is dealt by bytes, not by rows: all (row, head
// group) items, cut into tiles of 64 keys, are laid end to end and every block (two per SM) takes the same number of consecutive tiles, whatever the lengths: one
// row of 131071 keys and 256 ragged ones run alike. A block walks its span with one warp that fills a ring of shared-memory stages by tensor copies (the pages' rows
// land in the 128-byte swizzle) and four warps that take 16 keys of each stage; an item that lies whole in a span is written out, of an item that is cut each
// block leaves (max, sum, output), and the last of them to arrive adds them up in the order of the blocks. A block has at most two cut items, so the scratch memory
// depends on the grid alone, and its contents at the start do not matter. B200: 131071 keys of 8 heads of 128, f32, in 95 us (5.7 TB/s), 48 rows of 4000 to 16384 in f16 in
// 327 (6.5 TB/s), 256 rows of 32 to 4096 keys of 2 heads of 64 in 56 (4.7 TB/s); a few thousand keys are a chain of latencies, 10 us.
//
// The G query heads are the eight columns (G > 8: twice eight; more than 16 are several items) of m16n8k16 MMAs, S^T = K Q^T and O^T = V^T P^T, f16 operands, f32
// accumulators: keys and values are their 16-row operands, so that no row is spent on heads that are not there (with the heads as rows a step was twice the
// MMAs, and heads of 128 spilled: 118 against 100 us for one row of 131071 keys). Probabilities enter as f16 value + f16 rest (2^-22 together), with
// f32 queries the query too, after its row was scaled by a power of two, and each tile's products are added to the outputs in f32 (round to nearest; the tensor
// core's own accumulation truncates): as exact as f32 arithmetic. Probabilities are kept times 2^10, so that their second part stays in f16's normal range. (With one
// f16 probability for f16 rows their error against 64 bits was 2.5e-4 where the rounding of the result alone is 2.1e-4. The second product costs nothing at 4 or 5
// heads per key / value head, 1 us at 16 of 64, and 199 against 180 us at 256 rows of 32 to 4096 keys of 64 heads on one.)
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

constexpr int kTile = 64, kWarps = 4, kThreads = (kWarps + 1) * 32;
constexpr int kBlocksPerSm = 2, kMostBlocks = kBlocksPerSm * 160;
constexpr int kHeads = 16;                 // query heads of an item
constexpr float kLift = 10.f;              // probabilities are kept times 2^kLift

struct Args {
    PagedView c;
    const void * q;
    void * out;
    int n_head, group, parts;              // group: query heads per key / value head; parts: items they make
    int n_rows, max_length;
    const int32_t * sequence, * lengths;
    float scale_log2;
    unsigned long long call;               // the call's number, not zero
    Arrivals * arrived;                    // [block]: of the item cut behind that block, the blocks that have left their part
    float * part;                          // [block][2]: outputs [kHeads][D], then (max, sum) [kHeads]
};

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap * map, int x, int y, int z, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The transpose of an 8 x 8 matrix of f16, a row's two neighbours per lane.
__device__ __forceinline__ uint32_t transposed(uint32_t v) {
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
// (a, b) as f16 pairs; *rest: what the rounding left, rounded to f16 too
__device__ __forceinline__ uint32_t split2(float a, float b, uint32_t * rest) {
    const __half2 h = __floats2half2_rn(a, b);
    const float2 f = __half22float2(h);
    const __half2 r = __floats2half2_rn(a - f.x, b - f.y);
    *rest = *reinterpret_cast<const uint32_t *>(&r);
    return *reinterpret_cast<const uint32_t *>(&h);
}

// Probabilities the same way, cut instead of rounded so that the rest has the first part's sign, and never zero beside a first part that is not (at least 2^-24, which
// is 2^-34 of a probability): a value of infinity among those seen gives infinity, not infinity times zero.
__device__ __forceinline__ uint32_t split_p(float a, float b, uint32_t * rest) {
    uint32_t hi;
    asm("cvt.rz.f16x2.f32 %0, %1, %2;" : "=r"(hi) : "f"(b), "f"(a));
    const __half2 h = *reinterpret_cast<const __half2 *>(&hi);
    const float2 f = __half22float2(h);
    const __half2 r = __hmax2(__floats2half2_rn(a - f.x, b - f.y), __hmin2(h, __half2half2(__ushort_as_half(1))));
    *rest = *reinterpret_cast<const uint32_t *>(&r);
    return hi;
}

// Whether row r is one to attend with, and its length; an idle row and one whose entries are out of range have none (-1).
__device__ __forceinline__ int row_length(const Args & a, int r) {
    const int s = __ldg(a.sequence + r), n = __ldg(a.lengths + r);
    return s >= 0 && s < a.c.n_sequences && n >= 0 && n <= min(a.max_length, a.c.capacity()) ? n : -1;
}
__device__ __forceinline__ int64_t row_tiles(const Args & a, int r) { const int n = row_length(a, r); return n > 0 ? (n + kTile - 1) / kTile : 0; }

// A place in the line of all tiles: tile `tile` of item (row, part), of which there are `tiles`.
struct Place { int row, part, tile, tiles; };

// The number of tiles of all rows together; block-wide. Each thread adds up a run of rows; sums[th] becomes the tiles in front of thread th's run.
__device__ int64_t count_tiles(const Args & a, int64_t * sums) {
    const int per = (a.n_rows + kThreads - 1) / kThreads, r0 = min(a.n_rows, int(threadIdx.x) * per), r1 = min(a.n_rows, r0 + per);
    int64_t mine = 0;
    for (int r = r0; r < r1; r++) mine += row_tiles(a, r);
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    int64_t run = mine;
    for (int d = 1; d < 32; d <<= 1) { const int64_t o = __shfl_up_sync(0xffffffffu, run, d); if (lane >= d) run += o; }
    if (lane == 31) sums[kThreads + warp] = run;
    __syncthreads();
    int64_t total = 0;
    for (int w = 0; w <= kWarps; w++) { if (w < warp) run += sums[kThreads + w]; total += sums[kThreads + w]; }
    sums[threadIdx.x] = run - mine;      // tiles in front of this thread's rows
    __syncthreads();
    return total;
}

template <int D> constexpr int kSlot = kHeads * (D + 2);      // floats of a part

// Adds up the parts of a cut item, with the block's 128 threads of the four warps, four values a thread: the first block's second slot, the others' first, sixteen
// parts at a time (their loads in flight together), in the order of the blocks.
template <int D, bool HALF>
__device__ __forceinline__ void join(const Args & a, int first, int count, int row, int head0, int heads) {
    constexpr int kAtOnce = 16;
    for (int u = threadIdx.x; u < heads * (D / 4); u += kWarps * 32) {
        const int h = u / (D / 4), d = u % (D / 4) * 4;
        float m = -CUDART_INF_F, l = 0.f;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int i0 = 0; i0 < count; i0 += kAtOnce) {
            float2 st[kAtOnce];
            float4 x[kAtOnce];
            float top = m;
            #pragma unroll
            for (int i = 0; i < kAtOnce; i++) {
                const bool there = i0 + i < count;
                const float * p = a.part + (int64_t(first + i0 + i) * 2 + (i0 + i == 0 ? 1 : 0)) * kSlot<D>;
                st[i] = there ? __ldcg(reinterpret_cast<const float2 *>(p + kHeads * D + 2 * h)) : make_float2(-CUDART_INF_F, 0.f);
                x[i] = there ? __ldcg(reinterpret_cast<const float4 *>(p + h * D + d)) : make_float4(0.f, 0.f, 0.f, 0.f);
            }
            #pragma unroll
            for (int i = 0; i < kAtOnce; i++) top = fmaxf(top, st[i].x);
            const float minus = top == -CUDART_INF_F ? 0.f : top, keep = ex2(m - minus);
            l *= keep;
            v.x *= keep; v.y *= keep; v.z *= keep; v.w *= keep;
            #pragma unroll
            for (int i = 0; i < kAtOnce; i++) {
                const float share = ex2(st[i].x - minus);
                l = fmaf(st[i].y, share, l);
                v.x = fmaf(x[i].x, share, v.x); v.y = fmaf(x[i].y, share, v.y); v.z = fmaf(x[i].z, share, v.z); v.w = fmaf(x[i].w, share, v.w);
            }
            m = top;
        }
        const float by = l > 0.f || l != l ? 1.f / l : 0.f;
        const int64_t at = (int64_t(row) * a.n_head + head0 + h) * D + d;
        if (HALF) {
            *reinterpret_cast<__half2 *>(static_cast<__half *>(a.out) + at) = __floats2half2_rn(v.x * by, v.y * by);
            *reinterpret_cast<__half2 *>(static_cast<__half *>(a.out) + at + 2) = __floats2half2_rn(v.z * by, v.w * by);
        } else {
            *reinterpret_cast<float4 *>(static_cast<float *>(a.out) + at) = make_float4(v.x * by, v.y * by, v.z * by, v.w * by);
        }
    }
}

template <int D, bool HALF, bool WIDE>      // WIDE: items of more than 8 query heads
struct Kernel {
    static constexpr int kStages = D == 128 ? 3 : 6;
    static constexpr int kStageBytes = kTile * D * 2 * 2;
    static constexpr int NT = WIDE ? 2 : 1, KK = D / 16;
    static constexpr int kMergeBytes = 3 * KK * 32 * 16;       // three warps' results for eight heads
    static constexpr int kSmem = 1024 + kStages * kStageBytes + kMergeBytes + 3 * 8 * 8 + (kThreads + 8) * 8 + 16 * kStages + 32;
};

template <int D, bool HALF, bool WIDE>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm) k_attention_paged(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const Args a) {
    using K = Kernel<D, HALF, WIDE>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t ring = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t * const base = smem_raw + (ring - smem_u32(smem_raw));
    float4 * const merge = reinterpret_cast<float4 *>(base + K::kStages * K::kStageBytes);                       // [3][KK][32]
    float2 * const stats = reinterpret_cast<float2 *>(reinterpret_cast<uint8_t *>(merge) + K::kMergeBytes);     // [3][8] (max, sum)
    int64_t * const sums = reinterpret_cast<int64_t *>(stats + 3 * 8);
    const uint32_t full = smem_u32(sums + kThreads + 8), empty = full + 8 * K::kStages;
    int * const last = reinterpret_cast<int *>(sums + kThreads + 7);
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    if (threadIdx.x == 0) {
        for (int s = 0; s < K::kStages; s++) { mbar_init(full + 8 * s, 1); mbar_init(empty + 8 * s, kWarps); }
        mbar_init_fence();
    }
    if (warp == kWarps && lane < 2) asm volatile("prefetch.tensormap [%0];" ::"l"(lane == 0 ? &kmap : &vmap) : "memory");
    pdl_wait();
    const int items = a.c.n_kv * a.parts;
    const int64_t total = count_tiles(a, sums) * items;
    const int blocks = int(min(int64_t(gridDim.x), total));
    // rows without positions are zero; entries out of range are reported (by the last warp, which has the least to do at the end)
    auto rows_without = [&](int thread, int threads) {
        for (int r = blockIdx.x; r < a.n_rows; r += gridDim.x) {
            const int n = row_length(a, r);
            if (n < 0 && a.sequence[r] >= 0 && thread == 0) a.c.fail();
            if (n == 0) {
                for (int i = thread; i < a.n_head * D; i += threads) {
                    if (HALF) static_cast<__half *>(a.out)[int64_t(r) * a.n_head * D + i] = __half(0.f);
                    else static_cast<float *>(a.out)[int64_t(r) * a.n_head * D + i] = 0.f;
                }
            }
        }
    };
    if (int(blockIdx.x) >= blocks) { rows_without(threadIdx.x, kThreads); return; }
    const int64_t each = quotient(total, blocks);
    const int64_t from = part_of(total, each, blockIdx.x, blocks), to = part_of(total, each, blockIdx.x + 1, blocks);
    Place p;
    int64_t item_at;      // the first tile of the item at hand
    {
        const int per = (a.n_rows + kThreads - 1) / kThreads;
        int th = 0;
        for (int step = 128; step; step >>= 1) if (th + step < kThreads && sums[th + step] * items <= from) th += step;
        int64_t at = sums[th] * items;
        int r = th * per;
        int64_t t = row_tiles(a, r);
        while (at + t * items <= from) { at += t * items; t = row_tiles(a, ++r); }
        p.row = r; p.tiles = int(t); p.part = int(quotient(from - at, t)); p.tile = int(from - at - p.part * t);
        item_at = at + int64_t(p.part) * t;
    }
    auto next_item = [&] {
        item_at += p.tiles;
        p.tile = 0;
        if (++p.part == items) { p.part = 0; do { p.tiles = int(row_tiles(a, ++p.row)); } while (p.tiles == 0); }
    };
    bool ok = true;
    int stage = 0;
    uint32_t phase = 0;
    auto advance = [&] { if (++stage == K::kStages) { stage = 0; phase ^= 1u; } };
    int left = int(to - from);

    if (warp == kWarps) {
        // ---- the copies: lane i brings piece i of a tile (the rows of one page, or 64 of them; half a head of 128), keys and values ----
        const int box = min(kTile, 1 << a.c.page_shift);
        while (left > 0) {
            const int n = row_length(a, p.row), kvh = p.part / a.parts;
            const int32_t * table = a.c.table + int64_t(a.sequence[p.row]) * a.c.max_pages;
            for (; p.tile < p.tiles && left > 0; p.tile++, left--) {
                const int valid = min(kTile, n - p.tile * kTile), used = (valid + box - 1) / box;
                const int piece = lane / (D / 64), half = lane % (D / 64);
                int page = 0;
                const int key = p.tile * kTile + piece * box;
                if (piece < used) {
                    page = __ldg(table + (key >> a.c.page_shift));
                    if (uint32_t(page) >= uint32_t(a.c.n_pages)) { a.c.fail(); page = 0; }
                }
                ok = ok && mbar_wait(empty + 8 * stage, phase ^ 1u);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                if (lane == 0) mbar_arrive_expect_tx(full + 8 * stage, uint32_t(used * box) * D * 4u);
                __syncwarp();
                if (piece < used) {
                    const uint32_t dst = ring + stage * K::kStageBytes + half * (kTile * 128) + piece * box * 128;
                    const int z = (page << a.c.page_shift) + (key & ((1 << a.c.page_shift) - 1));
                    tma_load_3d(dst, &kmap, half * 64, kvh, z, full + 8 * stage);
                    tma_load_3d(dst + kTile * D * 2, &vmap, half * 64, kvh, z, full + 8 * stage);
                }
                advance();
            }
            if (!ok) break;
            if (left > 0) next_item();
        }
        rows_without(lane, 32);
        // no copy is under way when the block ends, not behind a wait that ran out either: each stage's last one (of this turn of the ring in front of `stage`, of the turn before from there on)
        for (int s = 0; s < K::kStages; s++) ok = mbar_wait(full + 8 * s, s < stage ? phase : phase ^ 1u) && ok;
    } else {
        const int g = lane >> 2, t = lane & 3;
        // where this lane's ldmatrix rows lie in a stage: keys 16 warp + .., as rows of the A operand (S^T = K Q^T), and as its columns (O^T = V^T P^T)
        const int krow = warp * 16 + (lane & 7) + ((lane >> 3) & 1) * 8, kchunk = lane >> 4;
        const int vrow = warp * 16 + (lane & 7) + ((lane >> 4) & 1) * 8, vchunk = (lane >> 3) & 1;
        const uint32_t kat = uint32_t(krow) * 128u, vat = uint32_t(vrow) * 128u + kTile * D * 2, sw = uint32_t(lane & 7);
        while (left > 0) {
            const int n = row_length(a, p.row), kvh = p.part / a.parts, head0 = kvh * a.group + (p.part % a.parts) * kHeads;
            const int heads = min(kHeads, a.group - (p.part % a.parts) * kHeads);
            // the item's queries as B operands: this lane has two times two neighbouring values of head g (+ 8 e) in each slice of 16; f: the scale of heads 2t and 2t + 1
            uint32_t qh[K::NT][K::KK][2], ql[HALF ? 1 : K::NT][HALF ? 1 : K::KK][2];
            float f[K::NT][2];
            #pragma unroll
            for (int e = 0; e < K::NT; e++) {
                const bool there = g + 8 * e < heads;
                const int64_t at = (int64_t(p.row) * a.n_head + head0 + g + 8 * e) * D + 2 * t;
                if (HALF) {
                    #pragma unroll
                    for (int kk = 0; kk < K::KK; kk++) {
                        const uint32_t * q = reinterpret_cast<const uint32_t *>(static_cast<const __half *>(a.q) + at + 16 * kk);
                        qh[e][kk][0] = there ? __ldg(q) : 0u;
                        qh[e][kk][1] = there ? __ldg(q + 4) : 0u;
                    }
                    f[e][0] = f[e][1] = a.scale_log2;
                } else {
                    float2 v[K::KK][2];
                    float most = 0.f;
                    #pragma unroll
                    for (int kk = 0; kk < K::KK; kk++) {
                        const float2 * q = reinterpret_cast<const float2 *>(static_cast<const float *>(a.q) + at + 16 * kk);
                        v[kk][0] = there ? __ldg(q) : make_float2(0.f, 0.f);
                        v[kk][1] = there ? __ldg(q + 4) : make_float2(0.f, 0.f);
                        most = fmaxf(fmaxf(most, fmaxf(fabsf(v[kk][0].x), fabsf(v[kk][0].y))), fmaxf(fabsf(v[kk][1].x), fabsf(v[kk][1].y)));
                    }
                    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                    most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                    // a power of two that brings the head's largest value into [1, 2); zeros, subnormals and infinities go as they are
                    const uint32_t ex = __float_as_uint(most) >> 23;
                    const bool fit = ex > 1 && ex < 253;
                    const float down = fit ? __uint_as_float((254u - ex) << 23) : 1.f, up = a.scale_log2 * (fit ? __uint_as_float(ex << 23) : 1.f);
                    f[e][0] = __shfl_sync(0xffffffffu, up, 8 * t);
                    f[e][1] = __shfl_sync(0xffffffffu, up, 8 * t + 4);
                    #pragma unroll
                    for (int kk = 0; kk < K::KK; kk++) {
                        #pragma unroll
                        for (int i = 0; i < 2; i++) qh[e][kk][i] = split2(v[kk][i].x * down, v[kk][i].y * down, &ql[HALF ? 0 : e][HALF ? 0 : kk][i]);
                    }
                }
            }
            float o[K::NT][K::KK][4], top[K::NT][2], sum[K::NT][2];
            #pragma unroll
            for (int e = 0; e < K::NT; e++) {
                #pragma unroll
                for (int j = 0; j < K::KK; j++) o[e][j][0] = o[e][j][1] = o[e][j][2] = o[e][j][3] = 0.f;
                top[e][0] = top[e][1] = -CUDART_INF_F;
                sum[e][0] = sum[e][1] = 0.f;
            }
            const bool starts = p.tile == 0;
            for (; p.tile < p.tiles && left > 0; p.tile++, left--) {
                const int valid = min(kTile, n - p.tile * kTile) - warp * 16;      // of this warp's 16 keys
                ok = ok && mbar_wait(full + 8 * stage, phase);
                ok = __all_sync(0xffffffffu, ok);
                if (valid > 0) {
                    const uint32_t st = ring + stage * K::kStageBytes;
                    // scores of keys g, g + 8 and heads 2t, 2t + 1. f32: sixteen products at a time, added up in f32 (a chain through the accumulator loses 1e-6 of a probability
                    // on heads of 128), the queries' second parts in an accumulator of their own
                    float s[K::NT][4] = {};
                    [[maybe_unused]] float rest[K::NT][4] = {};
                    #pragma unroll
                    for (int kk = 0; kk < K::KK; kk++) {
                        uint32_t k[4];
                        ldsm4(st + kat + (kk / 4) * (kTile * 128) + (((uint32_t(kk % 4) * 2 + kchunk) ^ sw) << 4), k);
                        #pragma unroll
                        for (int e = 0; e < K::NT; e++) {
                            if (HALF) {
                                mma_f16(s[e], k, qh[e][kk][0], qh[e][kk][1]);
                            } else {
                                float c[4] = {0.f, 0.f, 0.f, 0.f};
                                mma_f16(c, k, qh[e][kk][0], qh[e][kk][1]);
                                mma_f16(rest[e], k, ql[HALF ? 0 : e][HALF ? 0 : kk][0], ql[HALF ? 0 : e][HALF ? 0 : kk][1]);
                                #pragma unroll
                                for (int i = 0; i < 4; i++) s[e][i] += c[i];
                            }
                        }
                    }
                    if (valid < 16) {      // the last page's rest: no value (a page may hold anything there), and below no score
                        for (int i = lane; i < (16 - valid) * (D / 8); i += 32) {
                            const uint32_t row = uint32_t(warp * 16 + valid + i / (D / 8)), c = uint32_t(i % (D / 8));
                            asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(st + kTile * D * 2 + (c / 8) * (kTile * 128) + row * 128u + (c % 8) * 16u), "r"(0u) : "memory");
                        }
                        __syncwarp();
                    }
                    uint32_t ph[K::NT][2], pl[K::NT][2];
                    float keep[K::NT][2];
                    #pragma unroll
                    for (int e = 0; e < K::NT; e++) {
                        if (!HALF) {
                            #pragma unroll
                            for (int i = 0; i < 4; i++) s[e][i] += rest[e][i];
                        }
                        if (valid < 16) {
                            #pragma unroll
                            for (int i = 0; i < 4; i++) if (g + 8 * (i / 2) >= valid) s[e][i] = -CUDART_INF_F;
                        }
                        float x[4];
                        #pragma unroll
                        for (int h = 0; h < 2; h++) {
                            const float f_h = f[e][h];
                            float m = fmaxf(s[e][h], s[e][2 + h]) * f_h;
                            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
                            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                            m = fmaxf(m, top[e][h]);
                            const bool none = m == -CUDART_INF_F;
                            const float minus = none ? 0.f : kLift - m;
                            keep[e][h] = ex2(top[e][h] - (none ? 0.f : m));
                            top[e][h] = m;
                            x[h] = ex2(fmaf(s[e][h], f_h, minus));
                            x[2 + h] = ex2(fmaf(s[e][2 + h], f_h, minus));
                            sum[e][h] = fmaf(sum[e][h], keep[e][h], x[h] + x[2 + h]);
                        }
                        // probabilities of key g (+ 8) and heads 2t, 2t + 1 -> of keys 2t, 2t + 1 (+ 8) and head g: the B operand
                        #pragma unroll
                        for (int i = 0; i < 2; i++) {
                            uint32_t low = 0;
                            const uint32_t high = split_p(x[2 * i], x[2 * i + 1], &low);
                            ph[e][i] = transposed(high);
                            pl[e][i] = transposed(low);
                        }
                    }
                    #pragma unroll
                    for (int j = 0; j < K::KK; j++) {
                        uint32_t v[4];
                        ldsm4_t(st + vat + (j / 4) * (kTile * 128) + (((uint32_t(j % 4) * 2 + vchunk) ^ sw) << 4), v);
                        #pragma unroll
                        for (int e = 0; e < K::NT; e++) {
                            float c[4] = {0.f, 0.f, 0.f, 0.f};
                            mma_f16(c, v, ph[e][0], ph[e][1]);
                            mma_f16(c, v, pl[e][0], pl[e][1]);
                            #pragma unroll
                            for (int i = 0; i < 4; i++) o[e][j][i] = fmaf(o[e][j][i], keep[e][i % 2], c[i]);
                        }
                    }
                    if (valid < 16) asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // (the zeros, before a copy may land on them)
                }
                __syncwarp();
                if (lane == 0 && ok) mbar_arrive(empty + 8 * stage);      // (a stage whose copy did not come is not filled again)
                advance();
            }
            const bool ends = p.tile == p.tiles;
            // ---- the four warps' results: warps 1 to 3 hand theirs to warp 0, eight heads at a time ----
            #pragma unroll
            for (int e = 0; e < K::NT; e++) {
                #pragma unroll
                for (int h = 0; h < 2; h++) {
                    #pragma unroll
                    for (int d = 4; d < 32; d *= 2) sum[e][h] += __shfl_xor_sync(0xffffffffu, sum[e][h], d);
                }
                asm volatile("bar.sync 1, 128;" ::: "memory");      // warp 0 is done with the last hand-over
                if (warp > 0) {
                    if (g == 0) {
                        stats[(warp - 1) * 8 + 2 * t] = make_float2(top[e][0], sum[e][0]);
                        stats[(warp - 1) * 8 + 2 * t + 1] = make_float2(top[e][1], sum[e][1]);
                    }
                    #pragma unroll
                    for (int j = 0; j < K::KK; j++) merge[((warp - 1) * K::KK + j) * 32 + lane] = make_float4(o[e][j][0], o[e][j][1], o[e][j][2], o[e][j][3]);
                }
                asm volatile("bar.sync 1, 128;" ::: "memory");
                if (warp == 0) {
                    const bool whole = starts && ends;
                    float * const part = a.part + (int64_t(blockIdx.x) * 2 + (starts ? 1 : 0)) * kSlot<D>;
                    float share[2][4], by[2];
                    #pragma unroll
                    for (int h = 0; h < 2; h++) {
                        float m = top[e][h];
                        #pragma unroll
                        for (int w = 0; w < 3; w++) m = fmaxf(m, stats[w * 8 + 2 * t + h].x);
                        const float minus = m == -CUDART_INF_F ? 0.f : m;
                        share[h][0] = ex2(top[e][h] - minus);
                        float l = sum[e][h] * share[h][0];
                        #pragma unroll
                        for (int w = 0; w < 3; w++) { const float2 x = stats[w * 8 + 2 * t + h]; share[h][w + 1] = ex2(x.x - minus); l += x.y * share[h][w + 1]; }
                        by[h] = whole ? (l > 0.f || l != l ? 1.f / l : 0.f) : 1.f;
                        const int head = 2 * t + h + 8 * e;
                        if (!whole && g == 0 && head < heads) *reinterpret_cast<float2 *>(part + kHeads * D + 2 * head) = make_float2(m, l);
                    }
                    #pragma unroll
                    for (int j = 0; j < K::KK; j++) {
                        float y[4] = {o[e][j][0] * share[0][0], o[e][j][1] * share[1][0], o[e][j][2] * share[0][0], o[e][j][3] * share[1][0]};
                        #pragma unroll
                        for (int w = 0; w < 3; w++) {
                            const float4 x = merge[(w * K::KK + j) * 32 + lane];
                            y[0] = fmaf(x.x, share[0][w + 1], y[0]); y[1] = fmaf(x.y, share[1][w + 1], y[1]);
                            y[2] = fmaf(x.z, share[0][w + 1], y[2]); y[3] = fmaf(x.w, share[1][w + 1], y[3]);
                        }
                        #pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int head = 2 * t + i % 2 + 8 * e, d = 16 * j + g + 8 * (i / 2);
                            if (head < heads) {
                                const float v = y[i] * by[i % 2];
                                const int64_t at = (int64_t(p.row) * a.n_head + head0 + head) * D + d;
                                if (!whole) part[head * D + d] = v;
                                else if (HALF) static_cast<__half *>(a.out)[at] = __float2half_rn(v);
                                else static_cast<float *>(a.out)[at] = v;
                            }
                        }
                    }
                }
            }
            if (!(starts && ends)) {
                const int first = int(quotient((item_at + 1) * blocks - 1, total)), count = int(quotient((item_at + p.tiles) * blocks - 1, total)) - first + 1;
                if (warp == 0) {
                    __threadfence();
                    __syncwarp();
                    if (lane == 0) *last = paged_counter_arrive(a.arrived + first, a.call, count, !ok);
                }
                asm volatile("bar.sync 1, 128;" ::: "memory");
                if (*last) {
                    __threadfence();
                    join<D, HALF>(a, first, count, p.row, head0, heads);
                }
            }
            if (left > 0) next_item();
        }
    }
    if (!ok && lane == 0) a.c.gave_up();
}

template <int D, bool HALF, bool WIDE>
cudaError_t launch(const Args & a, const TensorMap & kmap, const TensorMap & vmap, int blocks, cudaStream_t stream) {
    constexpr int bytes = Kernel<D, HALF, WIDE>::kSmem;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_dynamic_smem(k_attention_paged<D, HALF, WIDE>, bytes, done);
    if (e != cudaSuccess) return e;
    return launch_pdl(k_attention_paged<D, HALF, WIDE>, dim3(unsigned(blocks)), dim3(kThreads), bytes, stream, reinterpret_cast<const CUtensorMap &>(kmap),
                      reinterpret_cast<const CUtensorMap &>(vmap), a);
}

}  // namespace

size_t attention_paged_scratch_bytes(int, int, int head_dim) { return size_t(kMostBlocks) * (2 * kHeads * (head_dim + 2) * 4 + 8); }

cudaError_t launch_attention_paged(const PagedCache & cache, const void * q, void * out, bool half_io, int n_head, int n_rows, const int32_t * sequence, const int32_t * lengths,
                                   int max_length, float scale, void * scratch, int * error, cudaStream_t stream) {
    Args a{};
    a.c = paged_view(cache, error);
    a.q = q; a.out = out;
    a.n_head = n_head; a.group = n_head / cache.n_head_kv; a.parts = (a.group + kHeads - 1) / kHeads;
    a.n_rows = n_rows; a.max_length = max_length;
    a.sequence = sequence; a.lengths = lengths;
    a.scale_log2 = scale * 1.44269504f;
    a.call = paged_call();
    a.arrived = static_cast<Arrivals *>(scratch);
    a.part = reinterpret_cast<float *>(a.arrived + kMostBlocks);
    const int blocks = std::min(kMostBlocks, kBlocksPerSm * sm_count());
    const int64_t rows = int64_t(cache.n_pages) * cache.page_size;
    TensorMap kmap, vmap;
    cudaError_t e = make_heads_map(&kmap, cache.keys, cache.head_dim, cache.n_head_kv, rows, 1, std::min(kTile, cache.page_size));
    if (e == cudaSuccess) e = make_heads_map(&vmap, cache.values, cache.head_dim, cache.n_head_kv, rows, 1, std::min(kTile, cache.page_size));
    if (e != cudaSuccess) return e;
    const bool wide = a.group > 8;
    if (cache.head_dim == 128) {
        if (half_io) return wide ? launch<128, true, true>(a, kmap, vmap, blocks, stream) : launch<128, true, false>(a, kmap, vmap, blocks, stream);
        return wide ? launch<128, false, true>(a, kmap, vmap, blocks, stream) : launch<128, false, false>(a, kmap, vmap, blocks, stream);
    }
    if (cache.head_dim != 64) return cudaErrorInvalidValue;
    if (half_io) return wide ? launch<64, true, true>(a, kmap, vmap, blocks, stream) : launch<64, true, false>(a, kmap, vmap, blocks, stream);
    return wide ? launch<64, false, true>(a, kmap, vmap, blocks, stream) : launch<64, false, false>(a, kmap, vmap, blocks, stream);
}

}  // namespace cuda
}  // namespace dooms
