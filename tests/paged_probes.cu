// Kernels that tests of the paged operators put beside them in a stream: a copy that reads as soon as it may be launched, and blocks that keep SMs busy for a while.
#include <cuda_runtime.h>

#include <cstdint>

namespace {

// (no griddepcontrol.wait: a programmatic dependent of another library may read like this)
__global__ void k_copy_at_once(const int32_t * from, int32_t * to, int n) {
    for (int i = blockIdx.x * blockDim.x + threadIdx.x; i < n; i += gridDim.x * blockDim.x) to[i] = *reinterpret_cast<const volatile int32_t *>(from + i);
}

// Ends by itself after `ns` nanoseconds, and after a number of polls whatever the clock says.
__global__ void k_hold(unsigned long long ns) {
    unsigned long long begin, now;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(begin));
    for (int polls = 0; polls < 4000000; polls++) {
        __nanosleep(1000);
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
        if (now - begin > ns) break;
    }
}

}  // namespace

#pragma GCC visibility push(default)
extern "C" {

// `n` words, by a kernel that may start as soon as the one in front of it in the stream lets its dependents go.
int probe_copy_at_once(const void * from, void * to, int n, void * stream) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(1);
    cfg.blockDim = dim3(256);
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return int(cudaLaunchKernelEx(&cfg, k_copy_at_once, static_cast<const int32_t *>(from), static_cast<int32_t *>(to), n));
}

// `blocks` blocks, each an SM of its own (200 KB of its shared memory), for `ns` nanoseconds.
int probe_hold(int blocks, long long ns, void * stream) {
    constexpr int bytes = 200 * 1024;
    const cudaError_t e = cudaFuncSetAttribute(k_hold, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) return int(e);
    k_hold<<<blocks, 32, bytes, static_cast<cudaStream_t>(stream)>>>(static_cast<unsigned long long>(ns));
    return int(cudaGetLastError());
}
}
#pragma GCC visibility pop
