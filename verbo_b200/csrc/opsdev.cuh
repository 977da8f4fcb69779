// Device helpers of the operators on rows of logits (ops_logits.cu, beam.cu):
// element types, 16-byte vectors, the launch of a chain's next kernel.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "device.cuh"

namespace vb {

constexpr float kNegInf = -__builtin_huge_valf();

template <class T>
__device__ __forceinline__ float to_float(T v);
template <>
__device__ __forceinline__ float to_float(float v) {
  return v;
}
template <>
__device__ __forceinline__ float to_float(__half v) {
  return __half2float(v);
}
template <>
__device__ __forceinline__ float to_float(__nv_bfloat16 v) {
  return __bfloat162float(v);
}

// Elements of a 16-byte vector as floats.
template <class T>
struct Vec {
  static constexpr int N = 16 / sizeof(T);
  uint4 raw;
  __device__ __forceinline__ float get(int i) const;
};
template <>
__device__ __forceinline__ float Vec<float>::get(int i) const {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  return __uint_as_float(w[i]);
}
template <>
__device__ __forceinline__ float Vec<__half>::get(int i) const {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  return __half2float(__ushort_as_half(static_cast<unsigned short>(w[i >> 1] >> (16 * (i & 1)))));
}
template <>
__device__ __forceinline__ float Vec<__nv_bfloat16>::get(int i) const {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
  return __uint_as_float((i & 1) ? (w[i >> 1] & 0xffff0000u) : (w[i >> 1] << 16));
}

// Not the read-only path: a kernel that is launched programmatically has begun
// before the grid whose rows it reads has ended.
__device__ __forceinline__ uint4 ld_stream16(const void* p) {
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.L2::256B.v4.u32 {%0,%1,%2,%3}, [%4];"
               : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
               : "l"(p));
  return v;
}
// Two fp32 numbers in one register pair, for the packed operations (each rounded
// to nearest, two for one instruction).
struct Two {
  unsigned long long v;
};
__device__ __forceinline__ Two two(float lo, float hi) {
  Two r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 parts_of(Two a) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(a.v));
  return r;
}
__device__ __forceinline__ Two add2(Two a, Two b) {
  Two r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two mul2(Two a, Two b) {
  Two r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c) {
  Two r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <class T>
__device__ __forceinline__ uint4 all_neg_inf();
template <>
__device__ __forceinline__ uint4 all_neg_inf<float>() {
  return make_uint4(0xff800000u, 0xff800000u, 0xff800000u, 0xff800000u);
}
template <>
__device__ __forceinline__ uint4 all_neg_inf<__half>() {
  return make_uint4(0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u, 0xfc00fc00u);
}
template <>
__device__ __forceinline__ uint4 all_neg_inf<__nv_bfloat16>() {
  return make_uint4(0xff80ff80u, 0xff80ff80u, 0xff80ff80u, 0xff80ff80u);
}

// The shared memory that a kernel may have on the current device, set at its first
// launch there (devices beyond the 64th: at every launch).
template <auto Kernel>
inline cudaError_t allow_smem(int bytes) {
  static std::atomic<unsigned long long> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
  if (done.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(Kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

// How many clusters of 1, 2, 4 or 8 CTAs of a kernel the current device holds at a time
// (0: it could not be asked); asked once per device.
template <auto Kernel>
inline int clusters_at_once(int cluster, int threads, int smem) {
  static std::atomic<int> known[64][4];
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  const int i = cluster == 8 ? 3 : cluster == 4 ? 2 : cluster == 2 ? 1 : 0;
  if (dev < 64) {
    const int n = known[dev][i].load(std::memory_order_relaxed);
    if (n) return n - 1;
  }
  int n = 0;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(cluster);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute at[1];
  at[0].id = cudaLaunchAttributeClusterDimension;
  at[0].val.clusterDim.x = cluster;
  at[0].val.clusterDim.y = 1;
  at[0].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = 1;
  if (allow_smem<Kernel>(smem) != cudaSuccess || cudaOccupancyMaxActiveClusters(&n, Kernel, &cfg) != cudaSuccess) {
    (void)cudaGetLastError();  // the launch that follows says what is wrong
    return 0;
  }
  if (dev < 64) known[dev][i].store(n + 1, std::memory_order_relaxed);
  return n;
}

// A kernel that may begin before the one before it in the stream has ended
// (grid_wait), with `cluster` CTAs a cluster.
template <class K, class A>
cudaError_t launch_chained(K kernel, unsigned grid, int threads, size_t smem, int cluster, cudaStream_t s, const A& a) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute at[2];
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = cluster;
  at[1].val.clusterDim.y = 1;
  at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, a);
}

}  // namespace vb
