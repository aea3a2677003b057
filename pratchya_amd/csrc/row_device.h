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
// The 8-bit form of a row's values, eight consecutive ones per lane: blocks of
// BLK elements are BLK / 8 neighbouring lanes, groups of BLK / 16 blocks (one
// for 16) up to 32 lanes, or for BLK 128 the wave's 64 lanes of two vectors.
// --------------------------------------------------------------------------
__device__ __forceinline__ uint32_t absmax8(const float (&v)[kVec]) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < kVec; ++i) m = umax(m, abs_bits(v[i]));
  return m;
}

// The payload of eight values of a block with maximum mb in a group with
// maximum Gb (f32 bits), and the block's e8m0 byte: quantize_impl's (fp8_math.h),
// by the division-free cast of block_scale; values near a bf16 rounding
// midpoint, and clamped blocks and groups that are not finite, by the exact
// composition.
__device__ __forceinline__ u32x2_t store_form(const float (&v)[kVec], uint32_t mb, uint32_t Gb, uint32_t& e) {
  const float G = u2f(Gb);
  const BlockScale b = block_scale(mb, Gb, __builtin_amdgcn_rcpf(G * 0.0078125f));
  e = b.e;
  bool fast = is_finite_f(G) && !b.clamped;
  u32x2_t w = {0, 0};
  if (fast) {
    float t[kVec];
#pragma unroll
    for (int i = 0; i < kVec; ++i) t[i] = v[i] * b.y;
    w = {cvt4_hw(t[0], t[1], t[2], t[3]), cvt4_hw(t[4], t[5], t[6], t[7])};
    fast = umin(mid_key4(t[0], t[1], t[2], t[3]), mid_key4(t[4], t[5], t[6], t[7])) > kMidKey;
  }
  if (!fast) {
    e = b.clamped || !is_finite_f(G) ? e8m0_of(u2f(mb), G) : b.e;
    const float S = quant_scale(e, G);
    w = {cvt4_exact(v[0], v[1], v[2], v[3], S), cvt4_exact(v[4], v[5], v[6], v[7], S)};
  }
  return w;
}

// What eight payload bytes of a block stand for.
__device__ __forceinline__ void stored_values(u32x2_t w, float scale, float (&v)[kVec]) {
  fp8_word(w.x, v[0], v[1], v[2], v[3]);
  fp8_word(w.y, v[4], v[5], v[6], v[7]);
#pragma unroll
  for (int i = 0; i < kVec; ++i) v[i] = (v[i] * scale) * 0.0078125f;
}
