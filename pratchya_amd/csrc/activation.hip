// Activations whose input is kept in 8 bits for the backward pass, for gfx950.
//
//   relu2  f = max(x, 0)^2            f' = 2 max(x, 0)
//   silu   f = x s, s = 1/(1+e^-x)    f' = s (1 + x (1 - s))
//   gelu   f = x P(x)                 f' = P(x) + x p(x)   (normal distribution and density)
// The forward pass computes f from x itself; the backward pass is dx = f'(x) dy
// with x read as it is or from its quantized form with block grid (1, blk)
// (fp8_math.h).  Arithmetic in f32, one rounding to the result's type.
// Both passes are bound by HBM and read and write past the caches.  With the
// quantizer of the Linear behind it, that reads y at once, this against plain stores:
// 2 MB of bf16 the same, 8 and 16 MB 10.9 -> 9.2 and 16.6 -> 13.0 us, 32 to 192 MB within
// 6% either way, 256 MB 136 -> 149, 512 MB and 1 GB within 2%; f32 and the backward
// pass alike.  One form is kept: only at 256 MB are plain stores clearly ahead.
// [16384, 16384] bf16, forward with the 8-bit form 217 us (1.35 GB, 6.2 TB/s), backward
// from it 211 us (6.4 TB/s); without it 169 and 255 us (6.4 and 6.3 TB/s).  gelu's 20
// operations an element in bf16 show a little with it: [8192, 8192] 61 and 60 us (5.5 and
// 5.6 TB/s); in f32, 31 of them, 104 and 101 us (5.8 and 5.9 TB/s).
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "pratchya_fp8.h"
#include "row_device.h"
#include "row_host.h"

namespace {

constexpr float kLog2e = 1.4426950408889634f;

// P(x) and p(x) of the normal distribution, which share e^(-x^2 / 2).  For a result in
// bf16: with z = |x| / sqrt 2 and t = 1 / (1 + 0.3275911 z), erfc(z) = (a1 t + ... + a5
// t^5) e^(-z^2) to 1.5e-7 (Abramowitz and Stegun, Handbook of Mathematical Functions,
// 7.1.26).  For one in f32, where that is up to 5 times what the roundings of
// x (1 + erf(z)) / 2 leave: P(-|x|) = e^(-x^2 / 2) t Q(t), t = 1 / (1 + 0.35 |x|), with Q
// of degree 8, to 3.2e-8 of itself for |x| up to 14, and for |x| < 1 P = 1/2 + x R(x^2),
// R of degree 5, to 3e-10; Q and R are fitted to the functions' values (least squares,
// weights raised where the error is largest).  The library's erfc in place of both was
// as exact, and a quarter to a third slower in the passes with an 8-bit input ([8192,
// 8192] 131 and 129 us where these take 105 and 99, the shorter form 105 and 98).
template <bool F32>
__device__ __forceinline__ void normal(float x, float& P, float& p) {
  if constexpr (F32) {
    const float a = fabsf(x), sq = x * x;
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.35f, a, 1.0f));
    const float e = __builtin_amdgcn_exp2f(sq * (-0.5f * kLog2e));
    const float Q[] = {0.1396214f, 0.13986185f, 0.119833045f, 0.105507225f, -0.02310781f, 0.15917094f,
                       -0.2557112f, 0.14397009f, -0.029145574f};
    const float R[] = {0.3989423f, -0.06649036f, 0.009973331f, -0.001186353f, 1.13512666e-04f, -7.664675e-06f};
    float c = Q[8], r = R[5];
#pragma unroll
    for (int i = 7; i >= 0; --i) c = __builtin_fmaf(c, t, Q[i]);
#pragma unroll
    for (int i = 4; i >= 0; --i) r = __builtin_fmaf(r, sq, R[i]);
    const float tail = (c * t) * e;
    P = a < 1.0f ? __builtin_fmaf(x, r, 0.5f) : x < 0.0f ? tail : 1.0f - tail;
    p = 0.39894228040143268f * e;
    return;
  }
  const float z = fabsf(x) * 0.70710678118654752f;
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.3275911f, z, 1.0f));
  const float e = __builtin_amdgcn_exp2f(-z * z * kLog2e);
  float c = __builtin_fmaf(1.061405429f, t, -1.453152027f);
  c = __builtin_fmaf(c, t, 1.421413741f);
  c = __builtin_fmaf(c, t, -0.284496736f);
  c = __builtin_fmaf(c, t, 0.254829592f);
  const float tail = 0.5f * c * t * e;       // P(-|x|)
  P = x < 0.0f ? tail : 1.0f - tail;
  p = 0.39894228040143268f * e;
}
// For a result in f32 by the library's exponential, whose argument is not rounded to x
// log2 e first: that rounding is one of |x| units of the sigmoid below 0.
template <bool F32>
__device__ __forceinline__ float sigmoid(float x) {
  return __builtin_amdgcn_rcpf(1.0f + (F32 ? expf(-x) : __builtin_amdgcn_exp2f(-x * kLog2e)));
}

// f of a vector; the kind is the same for the whole launch.
template <int N>
__device__ __forceinline__ void act(float (&v)[N], int kind) {
  if (kind == PRATCHYA_ACT_RELU2) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float r = v[i] < 0.0f ? 0.0f : v[i];
      v[i] = r * r;
    }
  } else if (kind == PRATCHYA_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] *= sigmoid<N == 4>(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float P, p;
      normal<N == 4>(v[i], P, p);
      v[i] *= P;
    }
  }
}

// g *= f'(v).
template <int N>
__device__ __forceinline__ void act_grad(const float (&v)[N], float (&g)[N], int kind) {
  if (kind == PRATCHYA_ACT_RELU2) {
#pragma unroll
    for (int i = 0; i < N; ++i) g[i] *= v[i] < 0.0f ? 0.0f : 2.0f * v[i];
  } else if (kind == PRATCHYA_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float s = sigmoid<N == 4>(v[i]);
      g[i] *= s * (1.0f + v[i] * (1.0f - s));
    }
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float P, p;
      normal<N == 4>(v[i], P, p);
      g[i] *= P + v[i] * p;
    }
  }
}

// Vectors, numbered through all rows; a wave takes 1024 neighbouring elements, a
// vector per lane and step, so a group of stored blocks (at most 1024 elements)
// lies in one wave.  ONE: the array is one row (contiguous rows).
constexpr int kThreads = 256;
template <typename T>
constexpr int kPer = 16 / kN<T>;         // vectors of a thread

struct Rows {
  int64_t ldx, width, vecs_per_row, vecs;
};
struct At {
  int64_t row, c;
  int left;        // elements of the vector, 0 beyond the array
};
template <int N, bool ONE>
__device__ __forceinline__ At place(const Rows& r, int64_t vec) {
  if (vec >= r.vecs) return {0, 0, 0};
  const int64_t row = ONE ? 0 : vec / r.vecs_per_row, c = (ONE ? vec : vec - row * r.vecs_per_row) * N;
  return {row, c, r.width - c < N ? (int)(r.width - c) : N};
}
template <typename T>
__device__ __forceinline__ int64_t first_vec() {
  return ((int64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6)) * (64 * kPer<T>) + (threadIdx.x & 63);
}

// Maxima over groups of K blocks of LB lanes, from the blocks' maxima m of a
// lane's PER vectors (64 lanes apart), for a K of 1, 2, 4 or 8.
template <int LB, int PER, int K>
__device__ __forceinline__ void group_max_of(const uint32_t (&m)[PER], uint32_t (&G)[PER]) {
  constexpr int LG = LB * K, LR = LG < 64 ? LG : 64, GV = LG / LR;
  static_assert(GV <= PER, "a group lies in one wave");
#pragma unroll
  for (int u = 0; u < PER; u += GV) {
    uint32_t g = m[u];
#pragma unroll
    for (int k = 1; k < GV; ++k) g = umax(g, m[u + k]);
    g = lane_group_max<LR>(g);
#pragma unroll
    for (int k = 0; k < GV; ++k) G[u + k] = g;
  }
}
template <int BLK, int N, int PER>
__device__ __forceinline__ void group_max(const uint32_t (&m)[PER], int K, uint32_t (&G)[PER]) {
  constexpr int LB = BLK / N;
  if (K == 1) group_max_of<LB, PER, 1>(m, G);
  if constexpr (BLK >= 32)
    if (K == 2) group_max_of<LB, PER, 2>(m, G);
  if constexpr (BLK >= 64)
    if (K == 4) group_max_of<LB, PER, 4>(m, G);
  if constexpr (BLK >= 128)
    if (K == 8) group_max_of<LB, PER, 8>(m, G);
}

template <typename T, int BLK, bool ONE>
__global__ __launch_bounds__(kThreads) void k_act(const T* __restrict__ x, Rows r, int kind, T* __restrict__ y,
                                                  uint8_t* __restrict__ x8, uint8_t* __restrict__ sc8,
                                                  float* __restrict__ sc32, int K) {
  constexpr int N = kN<T>, PER = kPer<T>;
  const int64_t vec = first_vec<T>();
  At at[PER];
  u32x4_t raw[PER];
  float v[PER][N];
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    at[u] = place<N, ONE>(r, vec + u * 64);
    const T* p = x + at[u].row * r.ldx + at[u].c;
    if (at[u].left == N) {
      raw[u] = load_raw<true>(p);
      widen(raw[u], v[u]);
    } else {
      load_some(p, at[u].left, 0.0f, v[u]);
      raw[u] = narrow(v[u]);
    }
  }
  if constexpr (BLK != 0) {
    uint32_t m[PER], G[PER] = {};
#pragma unroll
    for (int u = 0; u < PER; ++u)
      m[u] = lane_group_max<BLK / N>(absmax<T>(raw[u]));
    group_max<BLK, N>(m, K, G);
#pragma unroll
    for (int u = 0; u < PER; ++u) {
      if (at[u].left == 0) continue;          // blocks divide rows: a vector is whole
      const int64_t e0 = (vec + u * 64) * N;
      uint32_t e;
      const auto q = store_form(v[u], m[u], G[u], e);
      __builtin_nontemporal_store(q, reinterpret_cast<typename Payload<N>::type*>(x8 + e0));
      const int64_t n = e0 / BLK;
      if (e0 % BLK == 0) {
        sc8[n] = (uint8_t)e;
        if ((n & (K - 1)) == 0) sc32[n / K] = u2f(G[u]);
      }
    }
  }
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    act(v[u], kind);
    T* p = y + at[u].row * r.width + at[u].c;
    if (at[u].left == N) store_vec<true>(p, v[u]);
    else store_some(p, at[u].left, v[u]);
  }
}

struct StoredX {
  const uint8_t* x8;
  const uint8_t* sc8;
  const float* sc32;
  int blk_log2, K_log2;
};

template <typename T, bool STORED, bool ONE>
__global__ __launch_bounds__(kThreads) void k_act_bwd(const T* __restrict__ x, Rows r, StoredX s,
                                                      const T* __restrict__ dy, int64_t ldy, int kind,
                                                      T* __restrict__ dx) {
  constexpr int N = kN<T>, PER = kPer<T>;
  typedef typename Payload<N>::type W;
  const int64_t vec = first_vec<T>();
  At at[PER];
  float v[PER][N], g[PER][N];
  W q[PER];
  float scale[PER];
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    at[u] = place<N, ONE>(r, vec + u * 64);
    const T* p = dy + at[u].row * ldy + at[u].c;
    if constexpr (STORED) {
      if (at[u].left) {
        const int64_t e0 = (vec + u * 64) * N, n = e0 >> s.blk_log2;
        q[u] = __builtin_nontemporal_load(reinterpret_cast<const W*>(s.x8 + e0));
        scale[u] = stored_scale(s.sc8[n], s.sc32[n >> s.K_log2]);
      }
    } else {
      const T* px = x + at[u].row * r.ldx + at[u].c;
      if (at[u].left == N) widen(load_raw<true>(px), v[u]);
      else load_some(px, at[u].left, 0.0f, v[u]);
    }
    if (at[u].left == N) widen(load_raw<true>(p), g[u]);
    else load_some(p, at[u].left, 0.0f, g[u]);
  }
#pragma unroll
  for (int u = 0; u < PER; ++u) {
    if (at[u].left == 0) continue;
    if constexpr (STORED) {
      payload_values(q[u], v[u]);
#pragma unroll
      for (int i = 0; i < N; ++i) v[u][i] *= scale[u];
    }
    act_grad(v[u], g[u], kind);
    T* p = dx + at[u].row * r.width + at[u].c;
    if (at[u].left == N) store_vec<true>(p, g[u]);
    else store_some(p, at[u].left, g[u]);
  }
}

int check_args(const char* what, int kind, int dtype, int64_t rows, int64_t width) {
  if (kind < PRATCHYA_ACT_RELU2 || kind > PRATCHYA_ACT_GELU)
    return pratchya_set_error(PRATCHYA_EINVAL, "%s: unknown activation %d", what, kind);
  if (!is_float_dtype(dtype)) return pratchya_set_error(PRATCHYA_EINVAL, "%s: unsupported dtype %d", what, dtype);
  if (rows < 0 || width < 0)
    return pratchya_set_error(PRATCHYA_EINVAL, "%s: negative shape (%lld, %lld)", what, (long long)rows,
                              (long long)width);
  return PRATCHYA_OK;
}

// Rows as one where nothing lies between them.
template <typename T>
Rows make_rows(int64_t ldx, int64_t ldy, int64_t rows, int64_t width, bool& one) {
  one = rows == 1 || (ldx == width && ldy == width);
  const int64_t w = one ? rows * width : width, per = (w + kN<T> - 1) / kN<T>;
  return {ldx, w, per, one ? per : rows * per};
}

template <typename T>
int64_t workgroups(const Rows& r) {
  return (r.vecs + kThreads * kPer<T> - 1) / (kThreads * kPer<T>);
}

template <typename T>
int launch(const void* x, int64_t ldx, int kind, int64_t rows, int64_t width, void* y, uint8_t* x8, uint8_t* sc8,
           float* sc32, int64_t blk, hipStream_t stream) {
  bool one;
  const Rows r = make_rows<T>(ldx, width, rows, width, one);
  const int K = x8 ? (int)gcd64(blk / 16, rows * width / blk) : 1;
  if (!fits_launch(workgroups<T>(r), kThreads))
    return pratchya_set_error(PRATCHYA_EUNSUPPORTED, "activation: more elements than a launch has threads for (2^36)");
#define PRATCHYA_ACT(B)                                                                                              \
  if (one)                                                                                                           \
    hipLaunchKernelGGL((k_act<T, B, true>), dim3((unsigned)workgroups<T>(r)), dim3(kThreads), 0, stream,                \
                       static_cast<const T*>(x), r, kind, static_cast<T*>(y), x8, sc8, sc32, K);                     \
  else                                                                                                               \
    hipLaunchKernelGGL((k_act<T, B, false>), dim3((unsigned)workgroups<T>(r)), dim3(kThreads), 0, stream,               \
                       static_cast<const T*>(x), r, kind, static_cast<T*>(y), x8, sc8, sc32, K)
  if (!x8) { PRATCHYA_ACT(0); }
  else if (blk == 16) { PRATCHYA_ACT(16); }
  else if (blk == 32) { PRATCHYA_ACT(32); }
  else if (blk == 64) { PRATCHYA_ACT(64); }
  else { PRATCHYA_ACT(128); }
#undef PRATCHYA_ACT
  return check_launch("activation");
}

template <typename T, bool STORED>
int launch_bwd(const void* x, int64_t ldx, const StoredX& s, const void* dy, int64_t ldy, int kind, int64_t rows,
               int64_t width, void* dx, hipStream_t stream) {
  bool one;
  const Rows r = make_rows<T>(STORED ? width : ldx, ldy, rows, width, one);
  if (!fits_launch(workgroups<T>(r), kThreads))
    return pratchya_set_error(PRATCHYA_EUNSUPPORTED, "activation_bwd: more elements than a launch has threads for (2^36)");
  const dim3 grid((unsigned)workgroups<T>(r));
  const T* xt = STORED ? nullptr : static_cast<const T*>(x);
  if (one)
    hipLaunchKernelGGL((k_act_bwd<T, STORED, true>), grid, dim3(kThreads), 0, stream, xt, r, s,
                       static_cast<const T*>(dy), ldy, kind, static_cast<T*>(dx));
  else
    hipLaunchKernelGGL((k_act_bwd<T, STORED, false>), grid, dim3(kThreads), 0, stream, xt, r, s,
                       static_cast<const T*>(dy), ldy, kind, static_cast<T*>(dx));
  return check_launch("activation_bwd");
}

}  // namespace

extern "C" int pratchya_activation(const void* x, int64_t ldx, int dtype, int kind, int64_t rows, int64_t width,
                                   void* y, uint8_t* x8, uint8_t* sc8, float* sc32, int64_t blk, hipStream_t stream) {
  const int rc = check_args("activation", kind, dtype, rows, width);
  if (rc) return rc;
  if (x8 && ((blk != 16 && blk != 32 && blk != 64 && blk != 128) || width % blk))
    return pratchya_set_error(PRATCHYA_EINVAL, "activation: blocks of %lld for rows of %lld", (long long)blk,
                              (long long)width);
  if (rows * width == 0) return pratchya_set_error(PRATCHYA_OK, "");
  if (!x || !y || (x8 && (!sc8 || !sc32))) return pratchya_set_error(PRATCHYA_EINVAL, "activation: null buffer");
  if (reinterpret_cast<uintptr_t>(x8) % 8)
    return pratchya_set_error(PRATCHYA_EINVAL, "activation: the payload must be 8-byte aligned");
  return dtype == PRATCHYA_DT_BF16
             ? launch<uint16_t>(x, ldx, kind, rows, width, y, x8, sc8, sc32, blk, stream)
             : launch<float>(x, ldx, kind, rows, width, y, x8, sc8, sc32, blk, stream);
}

extern "C" int pratchya_activation_bwd(const void* x, int64_t ldx, int x_dtype, const uint8_t* sc8, const float* sc32,
                                       int64_t blk, const void* dy, int64_t ldy, int dtype, int kind, int64_t rows,
                                       int64_t width, void* dx, hipStream_t stream) {
  const int rc = check_args("activation_bwd", kind, dtype, rows, width);
  if (rc) return rc;
  const bool stored = x_dtype == PRATCHYA_DT_E4M3;
  if (!stored && x_dtype != dtype)
    return pratchya_set_error(PRATCHYA_EINVAL, "activation_bwd: unsupported dtypes (x %d, dy %d)", x_dtype, dtype);
  if (stored && (blk < 8 || (blk & (blk - 1)) || width % blk))
    return pratchya_set_error(PRATCHYA_EINVAL, "activation_bwd: blocks of %lld for rows of %lld", (long long)blk,
                              (long long)width);
  const int64_t n = rows * width;
  if (n == 0) return pratchya_set_error(PRATCHYA_OK, "");
  if (!x || !dy || !dx || (stored && (!sc8 || !sc32)))
    return pratchya_set_error(PRATCHYA_EINVAL, "activation_bwd: null buffer");
  if (stored && reinterpret_cast<uintptr_t>(x) % 8)
    return pratchya_set_error(PRATCHYA_EINVAL, "activation_bwd: the payload must be 8-byte aligned");
  StoredX s = {nullptr, sc8, sc32, 0, 0};
  if (stored) {
    s.x8 = static_cast<const uint8_t*>(x);
    s.blk_log2 = log2_of(blk);
    s.K_log2 = log2_of(gcd64(blk / 16 > 1 ? blk / 16 : 1, n / blk));
    return dtype == PRATCHYA_DT_BF16 ? launch_bwd<uint16_t, true>(x, ldx, s, dy, ldy, kind, rows, width, dx, stream)
                                     : launch_bwd<float, true>(x, ldx, s, dy, ldy, kind, rows, width, dx, stream);
  }
  return dtype == PRATCHYA_DT_BF16 ? launch_bwd<uint16_t, false>(x, ldx, s, dy, ldy, kind, rows, width, dx, stream)
                                   : launch_bwd<float, false>(x, ldx, s, dy, ldy, kind, rows, width, dx, stream);
}
