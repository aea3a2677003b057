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

// Element i of an array whose type is known at run time (a parameter's gradient, [width]).
__device__ __forceinline__ void store_param(void* p, bool bf16, int64_t i, float v) {
  if (bf16) store_elem(static_cast<uint16_t*>(p) + i, v);
  else static_cast<float*>(p)[i] = v;
}

// A vector is 16 bytes of a row: kN<T> = 8 bf16 or 4 f32 elements, so neighbouring
// lanes load and store neighbouring pieces in both types (f32 rows in vectors of
// 32 bytes took 417 us where these take 391, 2 GB of logits and their gradient).
// Addresses are aligned for one element only (rows of odd widths, slices): the
// vector types say so, and the hardware takes 16-byte accesses at any element's
// address.
template <typename T>
constexpr int kN = 16 / (int)sizeof(T);
typedef uint32_t u32x4_a2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
template <typename T> struct Unaligned { typedef u32x4_a2 type; };
template <> struct Unaligned<float> { typedef u32x4_a4 type; };

template <bool NT = false, typename T>
__device__ __forceinline__ u32x4_t load_raw(const T* p) {
  const auto* q = reinterpret_cast<const typename Unaligned<T>::type*>(p);
  if constexpr (NT) return __builtin_nontemporal_load(q);
  else return *q;
}
__device__ __forceinline__ void widen(const u32x4_t& r, float (&v)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = u2f(r[i] << 16);
    v[2 * i + 1] = u2f(r[i] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void widen(const u32x4_t& r, float (&v)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = u2f(r[i]);
}
__device__ __forceinline__ u32x4_t narrow(const float (&v)[8]) {
  return u32x4_t{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7])};
}
__device__ __forceinline__ u32x4_t narrow(const float (&v)[4]) {
  return u32x4_t{f2u(v[0]), f2u(v[1]), f2u(v[2]), f2u(v[3])};
}
template <bool NT = false, typename T>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[kN<T>]) {
  auto* q = reinterpret_cast<typename Unaligned<T>::type*>(p);
  if constexpr (NT) __builtin_nontemporal_store(narrow(v), q);
  else *q = narrow(v);
}
// The first n of a vector's elements; the others read as `fill`.
template <typename T, int N>
__device__ __forceinline__ void load_some(const T* p, int64_t n, float fill, float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = i < n ? load_elem(p + i) : fill;
}
template <typename T, int N>
__device__ __forceinline__ void store_some(T* p, int64_t n, const float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < n) store_elem(p + i, v[i]);
}

// The first bf16 piece of an f32 value: its upper half, exactly.
__device__ __forceinline__ float top_piece(float v) { return u2f(f2u(v) & 0xFFFF0000u); }

// Sum over aligned groups of BL lanes, for every lane of the group (the
// exchanges of lane_group_max; every lane adds the same pairs, so all get the
// same bits).
template <int CTRL>
__device__ __forceinline__ float dpp_add_f32(float v) {
  return v + u2f((uint32_t)__builtin_amdgcn_update_dpp(0, (int)f2u(v), CTRL, 0xF, 0xF, true));
}
template <int BL>
__device__ __forceinline__ float lane_group_add(float v) {
  if constexpr (BL >= 2) v = dpp_add_f32<0xB1>(v);   // quad_perm [1,0,3,2]
  if constexpr (BL >= 4) v = dpp_add_f32<0x4E>(v);   // quad_perm [2,3,0,1]
  if constexpr (BL >= 8) v = dpp_add_f32<0x141>(v);  // row_half_mirror
  if constexpr (BL >= 16) v = dpp_add_f32<0x140>(v); // row_mirror
  if constexpr (BL >= 32) {
    const auto p = __builtin_amdgcn_permlane16_swap(f2u(v), f2u(v), false, false);
    v = u2f(p[0]) + u2f(p[1]);
  }
  if constexpr (BL >= 64) {
    const auto p = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
    v = u2f(p[0]) + u2f(p[1]);
  }
  return v;
}
// The largest of the wave's values, for every lane; NaN is passed over.
template <int CTRL>
__device__ __forceinline__ float dpp_max_f32(float v) {
  return fmaxf(v, u2f((uint32_t)__builtin_amdgcn_update_dpp((int)f2u(v), (int)f2u(v), CTRL, 0xF, 0xF, false)));
}
__device__ __forceinline__ float wave_max(float v) {
  v = dpp_max_f32<0xB1>(v);
  v = dpp_max_f32<0x4E>(v);
  v = dpp_max_f32<0x141>(v);
  v = dpp_max_f32<0x140>(v);
  const auto p = __builtin_amdgcn_permlane16_swap(f2u(v), f2u(v), false, false);
  v = fmaxf(u2f(p[0]), u2f(p[1]));
  const auto q = __builtin_amdgcn_permlane32_swap(f2u(v), f2u(v), false, false);
  return fmaxf(u2f(q[0]), u2f(q[1]));
}
// Sum over the lanes of a wave, for every lane.
__device__ __forceinline__ float wave_add(float v) { return lane_group_add<64>(v); }

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

// --------------------------------------------------------------------------
// The 8-bit form of a row's values, a vector of N per lane: blocks of BLK
// elements are BLK / N neighbouring lanes, groups of blocks more of them or the
// same lanes of several vectors.
// --------------------------------------------------------------------------
// max |x| of a vector, as f32 bits.
template <typename T>
__device__ __forceinline__ uint32_t absmax(const u32x4_t& r) {
  return vec_absmax_bits<sizeof(T) == 2>(make_uint4(r[0], r[1], r[2], r[3]));
}

// N payload bytes.
template <int N> struct Payload;
template <> struct Payload<8> { typedef u32x2_t type; };
template <> struct Payload<4> { typedef uint32_t type; };
__device__ __forceinline__ u32x2_t payload_of(uint32_t a, uint32_t b, u32x2_t) { return u32x2_t{a, b}; }
__device__ __forceinline__ uint32_t payload_of(uint32_t a, uint32_t, uint32_t) { return a; }

// The payload of a vector of a block with maximum mb in a group with maximum Gb
// (f32 bits), and the block's e8m0 byte: quantize_impl's (fp8_math.h), by the
// division-free cast of block_scale; values near a bf16 rounding midpoint, and
// clamped blocks and groups that are not finite, by the exact composition.  A
// vector of eight is bf16, whose quotients x / S of two 8-bit significands are no
// midpoint (9 bits) and at least 2^-17 of their size away from one: the cast's few
// ulp do not reach it, and there is nothing to test.
template <int N>
__device__ __forceinline__ typename Payload<N>::type store_form(const float (&v)[N], uint32_t mb, uint32_t Gb,
                                                                uint32_t& e) {
  const float G = u2f(Gb);
  const BlockScale b = block_scale(mb, Gb, __builtin_amdgcn_rcpf(G * 0.0078125f));
  e = b.e;
  bool fast = is_finite_f(G) && !b.clamped;
  uint32_t w[2] = {0, 0};
  if (fast) {
    uint32_t mid = 0xFFFFFFFFu;
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const float t0 = v[i] * b.y, t1 = v[i + 1] * b.y, t2 = v[i + 2] * b.y, t3 = v[i + 3] * b.y;
      w[i / 4] = cvt4_hw(t0, t1, t2, t3);
      if constexpr (N == 4) mid = umin(mid, mid_key4(t0, t1, t2, t3));
    }
    fast = mid > kMidKey;
  }
  if (!fast) {
    e = b.clamped || !is_finite_f(G) ? e8m0_of(u2f(mb), G) : b.e;
    const float S = quant_scale(e, G);
#pragma unroll
    for (int i = 0; i < N; i += 4) w[i / 4] = cvt4_exact(v[i], v[i + 1], v[i + 2], v[i + 3], S);
  }
  return payload_of(w[0], w[1], typename Payload<N>::type());
}

// A vector's payload bytes as numbers; times its block's stored_scale they are what it stands for
// ((q * scale) / 128 in one product: the same but for values beyond 2^118 or below 2^-110).
__device__ __forceinline__ void payload_values(u32x2_t w, float (&v)[8]) {
  fp8_word(w.x, v[0], v[1], v[2], v[3]);
  fp8_word(w.y, v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void payload_values(uint32_t w, float (&v)[4]) { fp8_word(w, v[0], v[1], v[2], v[3]); }
__device__ __forceinline__ float stored_scale(uint32_t e, float G) { return (e8m0_decode(e) * G) * 0.0078125f; }
