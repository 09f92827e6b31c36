// rowops.cuh -- device helpers of the channel-last row kernels (gated scan, group
// norm, conv step and backward): vectors of channels in and out of registers, sigmoid and
// SiLU, and the second half of sums over all tokens.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "sm100.cuh"

namespace thm {

// VEC consecutive elements of T as one memory access of VEC * sizeof(T) bytes
// (the caller guarantees that alignment), widened to or rounded from fp32.
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

template <typename T, int VEC>
__device__ __forceinline__ void load_vec(const T* p, float* f) {
  const Pack<T, VEC> q = *reinterpret_cast<const Pack<T, VEC>*>(p);
#pragma unroll
  for (int j = 0; j < VEC; ++j) f[j] = to_f32<T>(q.v[j]);
}

template <typename T, int VEC>
__device__ __forceinline__ void store_vec(T* p, const float* f) {
  Pack<T, VEC> q;
#pragma unroll
  for (int j = 0; j < VEC; ++j) q.v[j] = from_f32<T>(f[j]);
  *reinterpret_cast<Pack<T, VEC>*>(p) = q;
}

__device__ __forceinline__ float ex2_approx(float x) {
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// e^x: the hardware exponential where the result is rounded to 16 bits (its error
// grows as |x| 2^-24), expf where fp32 leaves the kernel.
template <typename T>
__device__ __forceinline__ float exp_for(float x) {
  if constexpr (sizeof(T) == 2)
    return __expf(x);
  else
    return expf(x);
}

// 1 / (1 + e^-x): 0 at -inf, 1 at +inf, NaN for NaN. The reciprocal is off by 1 ulp at most.
template <typename T>
__device__ __forceinline__ float sigmoid(float x) {
  return rcp_approx(1.f + exp_for<T>(-x));
}

// silu(x) = x sigmoid(x).
template <typename T>
__device__ __forceinline__ float silu_of(float x) {
  return x * sigmoid<T>(x);
}

// A kernel's blocks say that a launch which was allowed to start early may do so; that one waits
// until all of them have ended and their writes are there.
__device__ __forceinline__ void let_dependents_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void wait_for_predecessor() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// out[map(c)] = sum over the n rows of part [n, M], column c: the second half of a
// reduction over all tokens whose first half left one row per block. 32 threads share a
// column (rows k, k + 32, ... each) and are added in a fixed order, so the result does not
// depend on the order in which blocks ran.
template <typename Map>
__global__ void __launch_bounds__(1024) sum_parts_kernel(const float* __restrict__ part, int n, int M, Map map) {
  __shared__ float sh[32][33];
  wait_for_predecessor();
  const int lane = threadIdx.x & 31, k = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float acc = 0.f;
  if (c < M) {
#pragma unroll 8
    for (int j = k; j < n; j += 32) acc += part[(long long)j * M + c];
  }
  sh[k][lane] = acc;
  __syncthreads();
  // Column k's 32 sums, one a lane of warp k.
  acc = sh[lane][k];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) acc += __shfl_xor_sync(0xffffffffu, acc, o);
  if (lane == 0 && blockIdx.x * 32 + k < M) map(blockIdx.x * 32 + k, acc);
}

// Launched so that it may be set up while the kernel that leaves `part` ends. Returns a thm_status.
template <typename Map>
inline int sum_parts(const float* part, int n, int M, Map map, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  cfg.gridDim = dim3((M + 31) / 32);
  cfg.blockDim = dim3(1024);
  cfg.stream = st;
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, sum_parts_kernel<Map>, part, n, M, map) != cudaSuccess) {
    cudaGetLastError();
    return THM_ERR_CUDA;
  }
  return THM_OK;
}

}  // namespace thm
