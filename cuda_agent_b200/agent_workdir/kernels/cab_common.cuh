// Shared device/host helpers for the sm_100a kernels in this directory.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <mutex>

#include "../../../include/cuda_agent_b200.h"

namespace cab {

constexpr int kWarp = 32;
constexpr int kNumSMs = 148;  // B200: 2 dies x 74 SMs

__host__ __device__ inline bool aligned_to(const void* p, size_t bytes) {
  return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0;
}

// Status a launcher returns after enqueueing: catches bad launch configurations
// without synchronising the stream.
inline int launch_status() { return cudaGetLastError() == cudaSuccess ? CAB_OK : CAB_ERR_LAUNCH; }

// For small kernels that follow one another: the launch lets the kernel be set up while the one before it in the stream ends, and
// the kernel's first statement waits for that end, with all that was written by then: 1 to 2 us less between two of
// them. What the kernel reads goes through ordinary loads (no __ldg), as it may be there before it is written.
template <typename... P, typename... A>
inline int launch_behind(void (*kernel)(P...), dim3 grid, dim3 block, size_t shared, cudaStream_t stream, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = shared;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...) != cudaSuccess) return CAB_ERR_LAUNCH;
  return launch_status();
}
__device__ __forceinline__ void after_predecessor() {
  cudaTriggerProgrammaticLaunchCompletion();
  cudaGridDependencySynchronize();
}

// Threads for a CTA that walks `chunks` equal pieces of a row, one piece per thread and pass: the largest
// multiple of 32 up to 256 that leaves no thread idle in the last pass (7168 bf16 columns in 16-byte pieces:
// 896 = 4 x 224), else 256.
inline int row_walk_threads(int chunks) {
  for (int t = 256; t >= 128; t -= 32)
    if (chunks % t == 0) return t;
  return 256;
}

// Opt-in to more than 48 KB of dynamic shared memory for `Kernel`. The attribute belongs to the
// (function, device) pair, so it is set once per device with that device current; one process may
// drive several GPUs and several host threads.
constexpr int kMaxDevices = 64;
template <auto Kernel>
inline bool ensure_dynamic_smem(int bytes) {
  static std::mutex mu;
  static bool done[kMaxDevices] = {};
  int dev = -1;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return false;
  std::lock_guard<std::mutex> lock(mu);
  if (!done[dev]) {
    if (cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return false;
    done[dev] = true;
  }
  return true;
}

// SMs of the current device, asked for once per device; 0 on failure.
inline int sm_count() {
  static std::atomic<int> known[kMaxDevices];
  int dev = -1, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return 0;
  n = known[dev].load(std::memory_order_relaxed);
  if (n == 0 && cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) == cudaSuccess)
    known[dev].store(n, std::memory_order_relaxed);
  return n;
}

// The starts of a paged batch's sequences run from 0, never descend, and stay within the T tokens of the call. Whether entry b
// (of `batch`) and the one after it break that.
__device__ __forceinline__ bool wrong_start(const int* q_start, int b, int batch, int T) {
  const int a = q_start[b], e = q_start[b + 1];
  return a > e || (b == 0 && a != 0) || (b == batch - 1 && e > T);
}

__device__ __forceinline__ float warp_sum(float x) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) x += __shfl_xor_sync(0xffffffffu, x, off);
  return x;
}

__device__ __forceinline__ float warp_max(float x) {
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, off));
  return x;
}

// bf16 bits -> fp32 is a 16-bit shift; exact.
__device__ __forceinline__ float bf16_lo(uint32_t packed) { return __uint_as_float(packed << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t packed) {
  return __uint_as_float(packed & 0xffff0000u);
}

// Streaming 128-bit global accesses: data touched once, so it is marked
// evict-first in L1 and L2 instead of displacing anything reusable.
// The load is `asm volatile` so that it is issued exactly once, where it is
// written: a kernel that posts N loads before the first use keeps N in flight.
__device__ __forceinline__ float4 ld_stream(const float4* p) {
  float4 v;
  asm volatile("ld.global.cs.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "l"(p));
  return v;
}
__device__ __forceinline__ void st_stream(float4* p, float4 v) {
  asm volatile("st.global.cs.v4.f32 [%0], {%1, %2, %3, %4};"
               :
               : "l"(p), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
               : "memory");
}

}  // namespace cab
