// serving_common.cuh — helpers shared by the serving operators (paged decode attention,
// beam selection, cache pages): argument checks, warp reductions, programmatic launches.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <atomic>

#include "gdn_b200.h"

namespace gdn_serving {

inline bool aligned(const void* ptr, size_t n) { return reinterpret_cast<uintptr_t>(ptr) % n == 0; }

inline bool overlaps(const void* a, size_t na, const void* b, size_t nb) {
  const uintptr_t pa = reinterpret_cast<uintptr_t>(a), pb = reinterpret_cast<uintptr_t>(b);
  return pa < pb + nb && pb < pa + na;
}

template <typename T> __device__ __forceinline__ T warp_sum(T x) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

constexpr int kSMs = 148;

// x / d for 32-bit x by multiplication with mul and shift from div_constants
__device__ __forceinline__ uint32_t div_by(uint32_t x, uint32_t mul, uint32_t shift) {
  return static_cast<uint32_t>((static_cast<unsigned long long>(__umulhi(x, mul)) + x) >> shift);
}
inline void div_constants(uint32_t d, uint32_t& mul, uint32_t& shift) {
  shift = 0;
  while ((1ull << shift) < d) ++shift;
  mul = static_cast<uint32_t>(((1ull << 32) * ((1ull << shift) - d)) / d + 1);
}

// programmatic dependent launch: a kernel waits for the one before it, or lets the next start
__device__ __forceinline__ void grid_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void grid_trigger() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

// Launches `kernel` as a programmatic dependent of the kernel before it on the stream; it
// must grid_wait() before it reads anything of that kernel's.
template <typename... Args>
cudaError_t launch_after(void (*kernel)(Args...), dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                         const Args&... args) {
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}

// Lets a kernel use `bytes` of dynamic shared memory, once per device: the attribute call
// costs the host microseconds, a decode step's call not many more.
template <auto kKernel> cudaError_t allow_smem(int bytes) {
  static std::atomic<unsigned long long> done{0};       // one bit per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  if (dev < 64 && ((done.load(std::memory_order_relaxed) >> dev) & 1)) return cudaSuccess;
  e = cudaFuncSetAttribute(kKernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess && dev < 64) done.fetch_or(1ull << dev, std::memory_order_relaxed);
  return e;
}

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// 16 bytes to shared memory without a register detour; zeros when !valid (src is not read)
__device__ __forceinline__ void copy16_async(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ float exp2_fast(float x) {   // 2^-22 relative, exp2(-inf) = 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace gdn_serving
