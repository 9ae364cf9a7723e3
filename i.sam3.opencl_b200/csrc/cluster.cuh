// SPDX-License-Identifier: Unlicense
// Host helpers of kernels launched in thread-block clusters.
#pragma once

#include "tmap.cuh"

#include <cuda_runtime.h>

namespace sam3 {

constexpr int kMaxClusterCtas = 16;

// Shared-memory limit and clusters above 8 CTAs, once per kernel and device.
template <auto Kern>
inline cudaError_t cluster_prepare_once(int smem)
{
    static PerDevice done;
    int n = 0;
    cudaError_t e = cudaSuccess;
    done.get(current_device(), n, [&](int &) {
        e = cudaFuncSetAttribute(Kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
        if (e == cudaSuccess)
            e = cudaFuncSetAttribute(Kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        return e == cudaSuccess;
    });
    return e;
}

// Clusters of c CTAs with the kernel's `smem` bytes that run at the same time
// (0: none fits), asked once per kernel and device, after cluster_prepare_once.
template <auto Kern>
inline long clusters_at_once(int c, int threads, int smem)
{
    static PerDevice known[kMaxClusterCtas + 1];
    if (c < 1 || c > kMaxClusterCtas)
        return 0;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = c;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(c);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return clusters_of<Kern>(known[c], cfg);
}

}  // namespace sam3
