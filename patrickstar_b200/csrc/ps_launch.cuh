// Launches whose set-up may run while the kernel before them in the stream finishes.
//
// Every kernel launched this way calls cudaGridDependencySynchronize() before it
// touches global memory, and cudaTriggerProgrammaticLaunchCompletion() when the
// next one may be set up beside it; the wait is for the end of the kernel before,
// so results are as if one ran after the other.
#ifndef PS_B200_LAUNCH_CUH
#define PS_B200_LAUNCH_CUH

#include "ps_b200.h"
#include "ps_internal.h"

#include <cuda_runtime.h>

#include <atomic>
#include <cstdint>
#include <cstring>

template <typename K, typename... Args>
void launch_behind(K kernel, uint32_t grid, uint32_t threads, uint32_t smem, uint32_t cluster, cudaStream_t st,
                   const Args&... args)
{
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute at[2];
    memset(at, 0, sizeof(at));
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    at[1].id = cudaLaunchAttributeClusterDimension;
    at[1].val.clusterDim.x = cluster, at[1].val.clusterDim.y = 1, at[1].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = cluster > 0 ? 2 : 1;
    cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Lets a kernel have that much shared memory; `seen`: the devices on which that is done.  The limit belongs to the
// kernel, not to a launch: `bytes` is the most that any launch of it asks for, since another thread may be between
// this and its own launch.
template <typename F>
int allow_smem(F kernel, uint32_t bytes, std::atomic<uint64_t>& seen)
{
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    const uint64_t bit = 1ull << (dev & 63);
    if (e == cudaSuccess && dev < 64 && (seen.load(std::memory_order_relaxed) & bit)) return PS_OK;
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e == cudaSuccess) {
        seen.fetch_or(bit, std::memory_order_relaxed);
        return PS_OK;
    }
    ps_internal::set_cuda_error((int)e);
    cudaGetLastError();
    return PS_ERR_CUDA;
}

#endif
