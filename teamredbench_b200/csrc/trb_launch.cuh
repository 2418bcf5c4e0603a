// trb_launch.cuh -- launches with programmatic dependence and clusters.
#pragma once

#include "trb_common.cuh"

namespace trb {

// One launch that may start before the grid before it in the stream is done (griddepcontrol.wait orders what it does).
// cluster: CTAs of a cluster, 0 for the kernel's own; smem: dynamic shared memory, opted in to once for each device
// through attr_set, a flag of the caller's for each.
template <typename Kernel, typename... Args>
static int launch_kernel(Kernel kernel, int grid, int threads, int cluster, size_t smem, int dev, bool (&attr_set)[64],
                         cudaStream_t stream, Args... args) {
    if (dev >= 64 || !attr_set[dev]) {
        TRB_CUDA(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem));
        if (dev < 64) attr_set[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = (unsigned)cluster;
    attr[1].val.clusterDim.y = 1;
    attr[1].val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)grid);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cfg.attrs = attr;
    cfg.numAttrs = cluster > 0 ? 2 : 1;  // 0: the kernel's own cluster size
    TRB_CUDA(cudaLaunchKernelEx(&cfg, kernel, args...));
    return TRB_OK;
}

// Clusters of `cl` CTAs of the kernel that the device holds at once, asked once for each device.  Fewer than the SMs
// divided by cl, since a cluster stays inside a GPC: 33 of 4 and 15 of 8 with one CTA an SM on 148 SMs.
template <typename Kernel>
static int clusters_at_once(Kernel kernel, int threads, size_t smem, int cl, int dev, int (&cache)[64]) {
    if (dev < 64 && cache[dev] > 0) return cache[dev];
    cudaLaunchConfig_t cfg = {};
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = (unsigned)cl;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    cfg.gridDim = dim3((unsigned)cl);
    cfg.blockDim = dim3((unsigned)threads);
    cfg.dynamicSmemBytes = smem;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    int count = 0;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess ||
        cudaOccupancyMaxActiveClusters(&count, kernel, &cfg) != cudaSuccess) {
        (void)cudaGetLastError();  // not split, then
        return 0;
    }
    if (dev < 64) cache[dev] = count;
    return count;
}

}  // namespace trb
