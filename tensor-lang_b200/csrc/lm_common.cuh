// Helpers of the language-model operators (residual_norm.cu, distill.cu,
// linear_ce.cu): element types, vector access, class indices.
#pragma once

#include <cuda_bf16.h>

#include <atomic>

#include "tl_common.cuh"

namespace tl {

// N consecutive elements as float.  N * sizeof(T) is 16 (one 128-bit access,
// 16-byte aligned address) or N is 1.
template <int N>
__device__ __forceinline__ void ld_vec(const float* p, float (&v)[N]) {
  if constexpr (N == 4) {
    const float4 q = *reinterpret_cast<const float4*>(p);
    v[0] = q.x; v[1] = q.y; v[2] = q.z; v[3] = q.w;
  } else {
    static_assert(N == 1, "one float4 or one float");
    v[0] = *p;
  }
}
template <int N>
__device__ __forceinline__ void ld_vec(const __nv_bfloat16* p, float (&v)[N]) {
  if constexpr (N == 8) {
    const uint4 q = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
    static_assert(N == 1, "eight bf16 or one");
    v[0] = __bfloat162float(*p);
  }
}
__device__ __forceinline__ uint32_t pack2_bf16(float a, float b) {
  const __nv_bfloat162 q = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&q);
}
template <int N>
__device__ __forceinline__ void st_vec(float* p, const float (&v)[N]) {
  if constexpr (N == 4)
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
  else
    *p = v[0];
}
template <int N>
__device__ __forceinline__ void st_vec(__nv_bfloat16* p, const float (&v)[N]) {
  if constexpr (N == 8)
    *reinterpret_cast<uint4*>(p) = make_uint4(pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3]),
                                              pack2_bf16(v[4], v[5]), pack2_bf16(v[6], v[7]));
  else
    *p = __float2bfloat16_rn(v[0]);
}
__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ void from_f32(float* p, float x) { *p = x; }
__device__ __forceinline__ void from_f32(__nv_bfloat16* p, float x) { *p = __float2bfloat16_rn(x); }

// The kernels of these operators overlap their beginnings: each lets the next one start at
// once (griddepcontrol.launch_dependents) and waits for the one before it, whose
// results are visible then, before it touches memory.
__device__ __forceinline__ void wait_for_previous_kernel() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

// Class index i of an index array (TL_IDX_*), or -1 when it is not in [0, n):
// such entries take no part.  A float index is the class the value names
// exactly (cross_entropy's class-index targets, kernel_generator.py:1816-1885,
// are float values); a NaN or a fraction names none.
__device__ __forceinline__ int64_t class_index(const void* p, int type, int64_t i, int64_t n) {
  int64_t v;
  if (type == TL_IDX_F32) {
    const float f = reinterpret_cast<const float*>(p)[i];
    if (!(f >= 0.f && f < 16777216.f) || f != truncf(f)) return -1;
    v = (int64_t)f;
  } else if (type == TL_IDX_I32) {
    v = reinterpret_cast<const int32_t*>(p)[i];
  } else {
    v = reinterpret_cast<const int64_t*>(p)[i];
  }
  return (v >= 0 && v < n) ? v : -1;
}

// Lets a kernel be launched with up to `bytes` of dynamic shared memory on the
// current device: once per kernel and device, since the call costs as much as a
// launch.  (A race of two first calls sets the same value twice.)
template <auto Kern, int Bytes>
int allow_smem() {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  TL_CUDA_TRY(cudaGetDevice(&dev));
  if (dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1)) return TL_OK;
  TL_CUDA_TRY(cudaFuncSetAttribute(Kern, cudaFuncAttributeMaxDynamicSharedMemorySize, Bytes));
  if (dev < 64) done.fetch_or(1ull << dev);
  return TL_OK;
}
// A launch that may begin while the stream's previous kernel runs
// (wait_for_previous_kernel), in clusters of `cluster` CTAs.
template <typename... P, typename... A>
int launch_in_clusters(int cluster, void (*kern)(P...), dim3 grid, int threads, size_t smem,
                       cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at[2] = {};
  at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at[0].val.programmaticStreamSerializationAllowed = 1;
  at[1].id = cudaLaunchAttributeClusterDimension;
  at[1].val.clusterDim.x = (unsigned)cluster;
  at[1].val.clusterDim.y = at[1].val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  TL_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, static_cast<P>(args)...));
  return after_launch();
}
template <typename... P, typename... A>
int launch(void (*kern)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, A... args) {
  return launch_in_clusters(1, kern, grid, threads, smem, st, args...);
}

inline bool aligned_to(const void* p, size_t n) { return ((uintptr_t)p % n) == 0; }
inline size_t elem_bytes(int dtype) { return dtype == TL_BF16 ? 2 : 4; }
inline bool dtype_ok(int dtype) { return dtype == TL_F32 || dtype == TL_BF16; }
inline bool index_ok(int t) { return t == TL_IDX_F32 || t == TL_IDX_I32 || t == TL_IDX_I64; }

}  // namespace tl
