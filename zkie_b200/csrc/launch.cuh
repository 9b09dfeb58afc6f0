// launch.cuh -- launches of the single-token kernels: a cluster dimension, and
// programmatic stream serialization, with which a kernel may start while the
// one before it on the stream still runs (it waits on the device before it
// touches what that one wrote).
#pragma once
#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>

#include "common.cuh"

namespace zk {

constexpr int kSms = 148;

// Raise a kernel's dynamic shared memory limit (and allow clusters of 16) once
// per device; `set` is the kernel's own word, a bit to a device.
inline cudaError_t allow_shared(const void* kernel, size_t bytes, std::atomic<uint64_t>* set, bool wide = false) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = 1ull << (dev & 63);
    if (set->load(std::memory_order_acquire) & bit) return cudaSuccess;
    if (bytes) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess && wide) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess) set->fetch_or(bit, std::memory_order_release);
    return e;
}

// Clusters of `cluster` blocks of a kernel that the present device holds at once: asked for once
// per size and remembered in `known`, a word to a size (devices of one kind in one program).
inline uint32_t clusters_at_once(const void* kernel, int threads, size_t shared, uint32_t cluster,
                                 std::atomic<uint32_t>* known) {
    if (const uint32_t n = known[cluster].load(std::memory_order_relaxed)) return n;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(cluster);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = shared;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = cluster;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int n = 0;
    if (cudaOccupancyMaxActiveClusters(&n, kernel, &cfg) != cudaSuccess) cudaGetLastError();  // not the launch's
    if (n < 1) n = 1;
    known[cluster].store((uint32_t)n, std::memory_order_relaxed);
    return (uint32_t)n;
}

template <typename Args>
int launch(void (*kernel)(const Args), dim3 grid, int threads, size_t shared, uint32_t cluster, cudaStream_t stream,
           const Args& args) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = shared;
    cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.numAttrs = 1;
    if (cluster > 1) {
        attr[1].id = cudaLaunchAttributeClusterDimension;
        attr[1].val.clusterDim.x = cluster;
        attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
        cfg.numAttrs = 2;
    }
    cfg.attrs = attr;
    ZK_TRY(cudaLaunchKernelEx(&cfg, kernel, args));
    return 0;
}

}  // namespace zk
