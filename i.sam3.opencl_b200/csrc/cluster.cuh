// SPDX-License-Identifier: Unlicense
// Host helpers of kernels launched in thread-block clusters.
#pragma once

#include <cuda_runtime.h>

namespace sam3 {

constexpr int kMaxClusterCtas = 16;

// Shared-memory limit and clusters above 8 CTAs, once per kernel and device.
template <auto Kern>
inline cudaError_t cluster_prepare_once(int smem)
{
    static int done[64];
    int dev = 0;
    const bool known = cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64;
    if (known && done[dev])
        return cudaSuccess;
    cudaError_t e = cudaFuncSetAttribute(Kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess)
        e = cudaFuncSetAttribute(Kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
    if (e == cudaSuccess && known)
        done[dev] = 1;
    return e;
}

// Clusters of c CTAs with the kernel's `smem` bytes that run at the same time
// (0: none fits), asked once per kernel and device, after cluster_prepare_once.
template <auto Kern>
inline long clusters_at_once(int c, int threads, int smem)
{
    static int known[64][kMaxClusterCtas + 1];
    int dev = 0;
    if (c < 1 || c > kMaxClusterCtas || cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64)
        return 0;
    if (!known[dev][c]) {
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
        int n = 0;
        if (cudaOccupancyMaxActiveClusters(&n, Kern, &cfg) != cudaSuccess) {
            (void)cudaGetLastError();
            return 0;
        }
        known[dev][c] = n + 1;
    }
    return known[dev][c] - 1;
}

}  // namespace sam3
