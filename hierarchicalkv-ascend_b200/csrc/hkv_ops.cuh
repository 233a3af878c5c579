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
  const cudaError_t e = cudaLaunchKernelEx(&c, kernel, std::forward<Args>(args)...);
  if (e != cudaSuccess) {
    cudaGetLastError();  // not left for the next call to find
    throw HkvError{HKV_ERR_CUDA, std::string("kernel launch: ") + cudaGetErrorString(e)};
  }
}

// Leave for a launch with `smem` bytes of dynamic shared memory. 48 KB need none,
// but hold a kernel's own arrays too (272 bytes at most here): asked for from 46 KB
// on. The limit belongs to the kernel on the device, not to the launch, and other
// host threads launch the same kernel: it is always set to the one value that
// covers every launch (227 KB is the most a block can have), so that no call
// takes away what another one needs.
constexpr size_t kMostShared = 220 * 1024;

template <class K>
void allow_shared(K kernel, size_t smem) {
  if (smem > 46 * 1024)
    CUDA_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  static_cast<int>(kMostShared)));
}

__device__ __forceinline__ void after_previous() {
  cudaGridDependencySynchronize();
  cudaTriggerProgrammaticLaunchCompletion();  // the next one may be set up
}

// Blocks of a cluster. The barrier orders shared and global memory among them.
__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n"
               "barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// word `p` of this block's shared memory, in block `rank` of the cluster
__device__ __forceinline__ uint32_t load_remote(const uint32_t* p, uint32_t rank) {
  uint32_t a = static_cast<uint32_t>(__cvta_generic_to_shared(p)), r, v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(rank));
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(r) : "memory");
  return v;
}

// Exclusive sums of two values over the threads of a block, and the sums of all.
__device__ __forceinline__ void block_exclusive2(uint32_t v, uint32_t u, uint32_t* v_before,
                                                 uint32_t* u_before, uint32_t* v_all,
                                                 uint32_t* u_all) {
  __shared__ uint2 sums[32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  uint32_t a = v, b = u;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t x = __shfl_up_sync(~0u, a, o), y = __shfl_up_sync(~0u, b, o);
    if (lane >= o) {
      a += x;
      b += y;
    }
  }
  __syncthreads();  // the sums of a call before are read
  if (lane == 31) sums[warp] = make_uint2(a, b);
  __syncthreads();
  // every warp scans the warps' sums for itself
  uint2 w = lane < warps ? sums[lane] : make_uint2(0, 0);
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t x = __shfl_up_sync(~0u, w.x, o), y = __shfl_up_sync(~0u, w.y, o);
    if (lane >= o) {
      w.x += x;
      w.y += y;
    }
  }
  *v_all = __shfl_sync(~0u, w.x, 31);
  *u_all = __shfl_sync(~0u, w.y, 31);
  const uint32_t x = __shfl_sync(~0u, w.x, warp ? warp - 1 : 0);
  const uint32_t y = __shfl_sync(~0u, w.y, warp ? warp - 1 : 0);
  *v_before = (warp ? x : 0) + a - v;
  *u_before = (warp ? y : 0) + b - u;
}

__device__ __forceinline__ uint32_t block_exclusive(uint32_t v, uint32_t* total) {
  uint32_t before, zero, none;
  block_exclusive2(v, 0, &before, &zero, total, &none);
  return before;
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
