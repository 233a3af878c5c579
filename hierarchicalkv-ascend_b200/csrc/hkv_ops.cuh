// hkv_ops.cuh -- what the row operators (hkv_rows.cu) and the page pool
// (hkv_pages.cu) share: launches, block sums, argument checks, the C ABI frame.
#pragma once

#include <cuda_runtime.h>

#include <string>
#include <utility>

#include "hkv_table.cuh"

namespace hkvb {

void set_last_error(const std::string& m);

// A launch that may be set up while the kernel before it in the stream still
// runs. Every kernel launched so begins with after_previous(), which waits for
// that kernel's end and so, one by one, for all before it: the order of the
// stream holds, only the launch latency between dependent kernels is hidden.
// (cluster > 1: blocks of a cluster.)
template <class... Params, class... Args>
void launch(void (*kernel)(Params...), dim3 grid, unsigned threads, size_t smem, cudaStream_t s,
            unsigned cluster, Args&&... args) {
  cudaLaunchConfig_t c{};
  c.gridDim = grid;
  c.blockDim = dim3(threads);
  c.dynamicSmemBytes = smem;
  c.stream = counted(s);
  cudaLaunchAttribute a[2];
  a[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  a[0].val.programmaticStreamSerializationAllowed = 1;
  a[1].id = cudaLaunchAttributeClusterDimension;
  a[1].val.clusterDim.x = cluster;
  a[1].val.clusterDim.y = a[1].val.clusterDim.z = 1;
  c.attrs = a;
  c.numAttrs = cluster > 1 ? 2 : 1;
  CUDA_TRY(cudaLaunchKernelEx(&c, kernel, std::forward<Args>(args)...));
}

__device__ __forceinline__ void after_previous() {
  cudaGridDependencySynchronize();
  cudaTriggerProgrammaticLaunchCompletion();  // the next one may be set up
}

// Exclusive sum of v over the threads of a block, and the sum of all.
__device__ __forceinline__ uint32_t block_exclusive(uint32_t v, uint32_t* total) {
  __shared__ uint32_t sums[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  uint32_t inc = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t u = __shfl_up_sync(~0u, inc, o);
    if (lane >= o) inc += u;
  }
  __syncthreads();  // the sums of a call before are read
  if (lane == 31) sums[warp] = inc;
  __syncthreads();
  // every warp scans the warps' sums for itself
  uint32_t w = lane < warps ? sums[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t u = __shfl_up_sync(~0u, w, o);
    if (lane >= o) w += u;
  }
  *total = __shfl_sync(~0u, w, 31);
  const uint32_t before = __shfl_sync(~0u, w, warp ? warp - 1 : 0);
  return (warp ? before : 0) + inc - v;
}

// A non-null address that is a multiple of its elements' size.
inline void require(const void* p, size_t align, const char* what) {
  HKV_REQUIRE(p != nullptr, HKV_ERR_INVALID, std::string(what) + " is null");
  HKV_REQUIRE(reinterpret_cast<uintptr_t>(p) % align == 0, HKV_ERR_INVALID,
              std::string(what) + " is not aligned to its elements");
}

}  // namespace hkvb

#define HKV_API_BEGIN try {
#define HKV_API_END                       \
  return HKV_OK;                          \
  }                                       \
  catch (const hkvb::HkvError& e) {       \
    hkvb::set_last_error(e.msg);          \
    return e.code;                        \
  }                                       \
  catch (const std::exception& e) {       \
    hkvb::set_last_error(e.what());       \
    return HKV_ERR_RUNTIME;               \
  }
