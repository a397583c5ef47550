// Launch of scaled_kernel instances; instantiated in ckb_scaled_inst_*.cu, one file per VMODE and CG.
#pragma once
#include <atomic>

#include "ckb_host.h"
#include "ckb_scaled_kernel.cuh"

namespace ckb {

template <int BN, int CG, int VMODE>
cudaError_t launch_scaled_one(const ScaledParams& p, int grid, cudaStream_t stream, int query_cluster, int* clusters)
{
    constexpr int SMEM = ScaledSmem<BN, CG>::DYN_BYTES;
    static_assert(SMEM <= 227 * 1024, "pipeline does not fit in shared memory");
    auto kern = scaled_kernel<BN, CG, VMODE>;
    static std::atomic<bool> attr_done[64] = {};
    int dev         = 0;
    cudaError_t err = cudaGetDevice(&dev);
    if(err != cudaSuccess)
        return err;
    if(dev < 0 || dev >= 64 || !attr_done[dev])
    {
        err = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
        if(err != cudaSuccess)
            return err;
        if constexpr(ScaledSmem<BN, CG>::SPLIT_REGS)
        {
            // the register shares of the warpgroups are drawn from what the block is launched with
            cudaFuncAttributes fa;
            err = cudaFuncGetAttributes(&fa, kern);
            if(err != cudaSuccess)
                return err;
            if(fa.numRegs * 3 < ScaledSmem<BN, CG>::REGS_LOW + 2 * ScaledSmem<BN, CG>::REGS_HIGH)
                return cudaErrorInvalidConfiguration;
        }
        if(dev >= 0 && dev < 64)
            attr_done[dev] = true;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim            = dim3(grid, 1, 1);
    cfg.blockDim           = dim3(ScaledSmem<BN, CG>::THREADS, 1, 1);
    cfg.dynamicSmemBytes   = SMEM;
    cfg.stream             = stream;
    cudaLaunchAttribute attr[2];
    int n_attr        = 0;
    const int cluster = query_cluster ? query_cluster : CG == 2 ? 2 : p.tiles.ksplit;
    if(cluster > 1)
    {
        attr[n_attr].id               = cudaLaunchAttributeClusterDimension;
        attr[n_attr].val.clusterDim.x = cluster;
        attr[n_attr].val.clusterDim.y = 1;
        attr[n_attr].val.clusterDim.z = 1;
        ++n_attr;
    }
    cfg.attrs = attr;
    if(query_cluster)
    {
        cfg.numAttrs = n_attr;
        return cudaOccupancyMaxActiveClusters(clusters, kern, &cfg);
    }
    host_add_pdl(attr, &n_attr);
    cfg.numAttrs = n_attr;
    return cudaLaunchKernelEx(&cfg, kern, p);
}

// query_cluster = 0: launches.  Otherwise only asks how many clusters of that many CTAs the device holds at once.
template <int VMODE, int CG>
cudaError_t launch_scaled(int bn, const ScaledParams& p, int grid, cudaStream_t stream, int query_cluster, int* clusters)
{
    if constexpr(CG == 2)
        switch(bn)
        {
        case 128: return launch_scaled_one<128, 2, VMODE>(p, grid, stream, query_cluster, clusters);
        case 192: return launch_scaled_one<192, 2, VMODE>(p, grid, stream, query_cluster, clusters);
        case 224: return launch_scaled_one<224, 2, VMODE>(p, grid, stream, query_cluster, clusters);
        case 256: return launch_scaled_one<256, 2, VMODE>(p, grid, stream, query_cluster, clusters);
        default: return cudaErrorInvalidValue;
        }
    else
        switch(bn)
        {
        case 16: return launch_scaled_one<16, 1, VMODE>(p, grid, stream, query_cluster, clusters);
        case 32: return launch_scaled_one<32, 1, VMODE>(p, grid, stream, query_cluster, clusters);
        case 64: return launch_scaled_one<64, 1, VMODE>(p, grid, stream, query_cluster, clusters);
        case 128: return launch_scaled_one<128, 1, VMODE>(p, grid, stream, query_cluster, clusters);
        default: return cudaErrorInvalidValue;
        }
}

#define CKB_SCALED_EXTERN(V, C) extern template cudaError_t launch_scaled<V, C>(int, const ScaledParams&, int, cudaStream_t, int, int*);
CKB_SCALED_EXTERN(0, 1)
CKB_SCALED_EXTERN(1, 1)
CKB_SCALED_EXTERN(0, 2)
CKB_SCALED_EXTERN(1, 2)
#undef CKB_SCALED_EXTERN

} // namespace ckb
