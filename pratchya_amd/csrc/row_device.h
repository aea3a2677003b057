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

// Eight consecutive elements as f32, and back.  The addresses are aligned for one
// element only (rows of odd widths, slices): the vector types say so, and the
// hardware takes 16-byte accesses at any element's address.
typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
constexpr int kVec = 8;

struct Raw16 {
  u32x4_t v;
};
struct Raw32 {
  u32x4_t lo, hi;
};
template <typename T> struct RawOf;
template <> struct RawOf<uint16_t> { typedef Raw16 type; };
template <> struct RawOf<float> { typedef Raw32 type; };

template <bool NT = false>
__device__ __forceinline__ Raw16 load_raw(const uint16_t* p) {
  const u32x4_a2* q = reinterpret_cast<const u32x4_a2*>(p);
  if constexpr (NT) return {__builtin_nontemporal_load(q)};
  else return {*q};
}
template <bool NT = false>
__device__ __forceinline__ Raw32 load_raw(const float* p) {
  const u32x4_a4* q = reinterpret_cast<const u32x4_a4*>(p);
  if constexpr (NT) return {__builtin_nontemporal_load(q), __builtin_nontemporal_load(q + 1)};
  else return {q[0], q[1]};
}
__device__ __forceinline__ void widen(const Raw16& r, float (&v)[kVec]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = u2f(r.v[i] << 16);
    v[2 * i + 1] = u2f(r.v[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void widen(const Raw32& r, float (&v)[kVec]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[i] = u2f(r.lo[i]);
    v[4 + i] = u2f(r.hi[i]);
  }
}
template <bool NT = false>
__device__ __forceinline__ void store_vec(uint16_t* p, const float (&v)[kVec]) {
  const u32x4_t w = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]),
                     pack_bf16x2(v[6], v[7])};
  u32x4_a2* q = reinterpret_cast<u32x4_a2*>(p);
  if constexpr (NT) __builtin_nontemporal_store(w, q);
  else *q = w;
}
template <bool NT = false>
__device__ __forceinline__ void store_vec(float* p, const float (&v)[kVec]) {
  const u32x4_t a = {f2u(v[0]), f2u(v[1]), f2u(v[2]), f2u(v[3])}, b = {f2u(v[4]), f2u(v[5]), f2u(v[6]), f2u(v[7])};
  u32x4_a4* q = reinterpret_cast<u32x4_a4*>(p);
  if constexpr (NT) {
    __builtin_nontemporal_store(a, q);
    __builtin_nontemporal_store(b, q + 1);
  } else {
    q[0] = a;
    q[1] = b;
  }
}
// The first n (0 to 8) of eight elements; the others read as `fill`.
template <typename T>
__device__ __forceinline__ void load_some(const T* p, int64_t n, float fill, float (&v)[kVec]) {
#pragma unroll
  for (int i = 0; i < kVec; ++i) v[i] = i < n ? load_elem(p + i) : fill;
}
template <typename T>
__device__ __forceinline__ void store_some(T* p, int64_t n, const float (&v)[kVec]) {
#pragma unroll
  for (int i = 0; i < kVec; ++i)
    if (i < n) store_elem(p + i, v[i]);
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
