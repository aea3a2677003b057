// Device helpers shared by the row kernels (layer norm, activations, token log
// probabilities): element access by type and reductions over a workgroup.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "quant_device.h"

__device__ __forceinline__ float load_elem(const float* p) { return *p; }
__device__ __forceinline__ float load_elem(const uint16_t* p) { return u2f((uint32_t)*p << 16); }
__device__ __forceinline__ void store_elem(float* p, float v) { *p = v; }
__device__ __forceinline__ void store_elem(uint16_t* p, float v) { *p = (uint16_t)f32_to_bf16_rne(v); }

// Element i of an array whose type is known at run time (parameters: [width]
// vectors that stay in the caches).
__device__ __forceinline__ float load_param(const void* p, bool bf16, int64_t i) {
  return bf16 ? load_elem(static_cast<const uint16_t*>(p) + i) : static_cast<const float*>(p)[i];
}
__device__ __forceinline__ void store_param(void* p, bool bf16, int64_t i, float v) {
  if (bf16) store_elem(static_cast<uint16_t*>(p) + i, v);
  else static_cast<float*>(p)[i] = v;
}

// Sum over the lanes of a wave, for every lane.
__device__ __forceinline__ float wave_add(float v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m, 64);
  return v;
}

// Sum over a workgroup of N waves, for every thread.  lds: N floats that
// nothing else uses between the call's barriers.
template <int N>
__device__ __forceinline__ float block_add(float v, float* lds) {
  v = wave_add(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = lds[0];
#pragma unroll
  for (int i = 1; i < N; ++i) s += lds[i];
  return s;
}
