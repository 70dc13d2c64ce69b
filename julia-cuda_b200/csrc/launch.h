// Launch helpers shared by the kernel translation units: cudaLaunchKernelEx with programmatic stream
// serialization when `pdl`, thread-block clusters, dynamic shared-memory limits.
#pragma once
#include <cuda_runtime.h>
#include <stdlib.h>

#include <atomic>

#include "jc_internal.h"

namespace jc {

inline uint32_t env_u32_early(const char *name, uint32_t dflt) {
    const char *e = getenv(name);
    return e ? (uint32_t)strtoul(e, nullptr, 10) : dflt;
}

// Programmatic dependent launch is on unless the environment sets JC_PDL=0 (for A/B timing).
inline bool pdl_allowed() {
    static const bool on = [] {
        const char *v = getenv("JC_PDL");
        return !(v && v[0] == '0');
    }();
    return on;
}

template <typename... KArgs, typename... Args>
bool launch_ex(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t s, bool pdl,
               const char *what, Args... args) {
    pdl = pdl && pdl_allowed();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = pdl ? attr : nullptr;
    cfg.numAttrs = pdl ? 1 : 0;
    return cuda_ok(cudaLaunchKernelEx(&cfg, kern, args...), what);
}

// launch_ex with the grid grouped into thread-block clusters.
template <typename... KArgs, typename... Args>
bool launch_ex_cluster(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t s,
                       bool pdl, dim3 cluster, const char *what, Args... args) {
    pdl = pdl && pdl_allowed();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    unsigned n = 0;
    if (pdl) {
        attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[n].val.programmaticStreamSerializationAllowed = 1;
        n++;
    }
    if (cluster.x * cluster.y * cluster.z > 1) {
        attr[n].id = cudaLaunchAttributeClusterDimension;
        attr[n].val.clusterDim.x = cluster.x;
        attr[n].val.clusterDim.y = cluster.y;
        attr[n].val.clusterDim.z = cluster.z;
        n++;
    }
    cfg.attrs = n ? attr : nullptr;
    cfg.numAttrs = n;
    return cuda_ok(cudaLaunchKernelEx(&cfg, kern, args...), what);
}

// How many clusters of `size` CTAs along x the current device holds at once.
template <typename K>
bool max_clusters(K kern, int size, int threads, int smem, int *clusters) {
    int dev = 0, sms = 0;
    if (!cuda_ok(cudaGetDevice(&dev), "cudaGetDevice") ||
        !cuda_ok(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev), "sm count"))
        return false;
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)size;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)(sms / size * size));
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (!cuda_ok(cudaOccupancyMaxActiveClusters(clusters, kern, &cfg), "cluster occupancy")) return false;
    if (*clusters > 0) return true;
    set_error("no cluster of a kernel fits this device");
    return false;
}

// Sets a kernel's dynamic shared-memory limit once per device.
template <typename K>
bool ensure_smem(K kern, int bytes, std::atomic<uint64_t> &done_mask) {
    int dev = 0;
    if (!cuda_ok(cudaGetDevice(&dev), "cudaGetDevice")) return false;
    const uint64_t bit = 1ull << (dev & 63);
    if (done_mask.load() & bit) return true;
    if (!cuda_ok(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes),
                 "cudaFuncSetAttribute"))
        return false;
    done_mask.fetch_or(bit);
    return true;
}

}  // namespace jc
