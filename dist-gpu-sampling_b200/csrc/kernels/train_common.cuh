// What the operators of a training step (norm.cu, cross_entropy.cu, adamw.cu) share: element types, vector access with
// values in 32 bits, launches with a shared-memory size, the SM count.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "common.cuh"

namespace dgs {

static inline int dtype_bytes(int32_t dtype) { return dtype == DGS_F32 ? 4 : dtype == DGS_BF16 || dtype == DGS_F16 ? 2 : 0; }

static inline bool aligned_to(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

// SMs of the current device (those of a B200 where there is none: sizes of workspaces may be asked for without a GPU)
static inline int sm_count() {
  constexpr int kMaxDevices = 64;
  static std::atomic<int> known[kMaxDevices] = {};
  int dev = 0;
  constexpr int kB200 = 148;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return kB200;
  int sms = known[dev].load(std::memory_order_relaxed);
  if (sms == 0) {
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return kB200;
    known[dev].store(sms, std::memory_order_relaxed);
  }
  return sms;
}

#ifdef __CUDACC__

template <typename T>
__device__ __forceinline__ float to_float(T v) {
  return static_cast<float>(v);
}
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 v) {
  return __bfloat162float(v);
}
template <>
__device__ __forceinline__ float to_float<__half>(__half v) {
  return __half2float(v);
}
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_float<__half>(float v) {
  return __float2half_rn(v);
}

// VEC elements of T moved as one access of up to 16 bytes (two, for 32 bytes)
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC < 16 ? sizeof(T) * VEC : 16) Vec {
  T v[VEC];
};
template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float (&out)[VEC]) {
  const Vec<T, VEC> t = *reinterpret_cast<const Vec<T, VEC>*>(p);
#pragma unroll
  for (int i = 0; i < VEC; ++i) out[i] = to_float<T>(t.v[i]);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float (&in)[VEC]) {
  Vec<T, VEC> t;
#pragma unroll
  for (int i = 0; i < VEC; ++i) t.v[i] = from_float<T>(in[i]);
  *reinterpret_cast<Vec<T, VEC>*>(p) = t;
}

// One element, or VEC of them, of a type known at run time (the same for all threads of a block)
__device__ __forceinline__ float load_as_float(const void* p, int32_t dtype, int64_t i) {
  if (dtype == DGS_F32) return static_cast<const float*>(p)[i];
  if (dtype == DGS_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_from_float(void* p, int32_t dtype, int64_t i, float v) {
  if (dtype == DGS_F32) static_cast<float*>(p)[i] = v;
  else if (dtype == DGS_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  else static_cast<__half*>(p)[i] = __float2half_rn(v);
}
template <int VEC>
__device__ __forceinline__ void load_vec_as_float(const void* p, int32_t dtype, int64_t i, float (&out)[VEC]) {
  if (dtype == DGS_F32) load_vec<float, VEC>(static_cast<const float*>(p) + i, out);
  else if (dtype == DGS_BF16) load_vec<__nv_bfloat16, VEC>(static_cast<const __nv_bfloat16*>(p) + i, out);
  else load_vec<__half, VEC>(static_cast<const __half*>(p) + i, out);
}
template <int VEC>
__device__ __forceinline__ void store_vec_from_float(void* p, int32_t dtype, int64_t i, const float (&in)[VEC]) {
  if (dtype == DGS_F32) store_vec<float, VEC>(static_cast<float*>(p) + i, in);
  else if (dtype == DGS_BF16) store_vec<__nv_bfloat16, VEC>(static_cast<__nv_bfloat16*>(p) + i, in);
  else store_vec<__half, VEC>(static_cast<__half*>(p) + i, in);
}

// ---- two 32-bit floats in one instruction ---------------------------------------------------------------------------
__device__ __forceinline__ uint64_t two(float lo, float hi) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void split2(uint64_t v, float* lo, float* hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(*lo), "=f"(*hi) : "l"(v)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// launch_chained (common.cuh) with a grid of up to three dimensions, dynamic shared memory and clusters of that many CTAs (0, 1: none)
template <typename... KArgs>
inline cudaError_t launch_clusters(void (*kernel)(KArgs...), dim3 grid, unsigned block, size_t smem, cudaStream_t s, unsigned cluster,
                                   KArgs... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(block, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  cfg.attrs = attr;
  cfg.numAttrs = 0;
  if (chained_launches_enabled(SITE_TRAINING)) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (cluster > 1) {
    attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
    attr[cfg.numAttrs++].val.clusterDim = {cluster, 1, 1};
  }
  return cudaLaunchKernelEx(&cfg, kernel, args...);
}
template <typename... KArgs, typename... Args>
inline cudaError_t launch_training(void (*kernel)(KArgs...), dim3 grid, unsigned block, size_t smem, cudaStream_t s, Args&&... args) {
  return launch_clusters(kernel, grid, block, smem, s, 0u, static_cast<KArgs>(args)...);
}

#endif  // __CUDACC__
}  // namespace dgs
