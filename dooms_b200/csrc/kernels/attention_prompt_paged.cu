// Attention of one new token per row over its sequence's pages: o = sum_j softmax_j(scale q . k_j) v_j over the row's positions j < length. One warp per (row,
// query head): a lane holds D / 32 of the head's values.
#include <math_constants.h>

#include "launch.cuh"
#include "paged.cuh"

namespace dooms {
namespace cuda {

namespace {

// (also the first form of a prompt's attention: a query sees the positions up to its own)
template <int D, class T>
__device__ void one_query(const PagedView & c, int seq, int n, const T * q, T * out, int kvh, float scale, int lane) {
    constexpr int kPer = D / 32;
    float qv[kPer], o[kPer] = {}, top = -CUDART_INF_F, sum = 0.f;
    for (int i = 0; i < kPer; i++) qv[i] = float(q[lane + 32 * i]) * scale;
    for (int j = 0; j < n; j++) {
        const int64_t row = c.row(seq, j);
        if (row < 0) { c.fail(); continue; }
        const __half * k = c.k + (row * c.n_kv + kvh) * D, * v = c.v + (row * c.n_kv + kvh) * D;
        float s = 0.f;
        for (int i = 0; i < kPer; i++) s += qv[i] * __half2float(k[lane + 32 * i]);
        for (int m = 16; m; m >>= 1) s += __shfl_xor_sync(0xffffffffu, s, m);
        const float t = fmaxf(top, s), keep = expf(top - t), e = expf(s - t);
        sum = sum * keep + e;
        for (int i = 0; i < kPer; i++) o[i] = o[i] * keep + e * __half2float(v[lane + 32 * i]);
        top = t;
    }
    for (int i = 0; i < kPer; i++) out[lane + 32 * i] = T(sum > 0.f ? o[i] / sum : 0.f);
}

template <int D>
__global__ void __launch_bounds__(128) k_attention_prompt(const PagedView c, const __half * q, __half * out, int n_head, int n_rows, const int32_t * sequence, const int32_t * start,
                                                          const int32_t * lengths, int n_sequences, float scale) {
    const int64_t w = int64_t(blockIdx.x) * 4 + threadIdx.x / 32;
    const int lane = threadIdx.x % 32;
    if (w >= int64_t(n_rows) * n_head) return;
    const int r = int(w / n_head), h = int(w % n_head);
    int i = 0;
    for (int j = 0; j < n_sequences; j++) if (start[j] < 0 || start[j + 1] < start[j] || start[j + 1] > n_rows) c.fail();
    while (i < n_sequences && !(r >= start[i] && r < start[i + 1] && start[i] >= 0 && start[i + 1] <= n_rows)) i++;
    if (i == n_sequences) return;
    const int seq = sequence[i], n = lengths[i] - (start[i + 1] - 1 - r);
    if (seq < 0) return;
    if (seq >= c.n_sequences || lengths[i] < 0 || lengths[i] > c.capacity()) { c.fail(); return; }
    one_query<D, __half>(c, seq, n, q + w * D, out + w * D, h / (n_head / c.n_kv), scale, lane);
}

}  // namespace

size_t attention_prompt_scratch_bytes(int, int, int) { return 256; }

cudaError_t launch_attention_prompt_paged(const PagedCache & cache, const void * q, void * out, int n_head, int n_rows, int n_sequences, const int32_t * sequence,
                                          const int32_t * start, const int32_t * lengths, float scale, void *, int * error, cudaStream_t stream) {
    const PagedView c = paged_view(cache, error);
    const unsigned blocks = unsigned((int64_t(n_rows) * n_head + 3) / 4);
    auto go = [&](auto kernel) {
        kernel<<<blocks, 128, 0, stream>>>(c, static_cast<const __half *>(q), static_cast<__half *>(out), n_head, n_rows, sequence, start, lengths, n_sequences, scale);
    };
    if (cache.head_dim == 128) go(k_attention_prompt<128>);
    else if (cache.head_dim == 64) go(k_attention_prompt<64>);
    else return cudaErrorInvalidValue;
    return cudaGetLastError();
}

}  // namespace cuda
}  // namespace dooms
