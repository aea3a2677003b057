// Activations whose input is kept in 8 bits for the backward pass, for gfx950.
//
//   relu2  f = max(x, 0)^2            f' = 2 max(x, 0)
//   silu   f = x s, s = 1/(1+e^-x)    f' = s (1 + x (1 - s))
//   gelu   f = x P(x)                 f' = P(x) + x p(x)   (normal distribution and density)
// The forward pass computes f from x itself; the backward pass is dx = f'(x) dy
// with x read as it is or from its quantized form with block grid (1, blk)
// (fp8_math.h).  Arithmetic in f32, one rounding to the result's type.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "pratchya_fp8.h"
#include "row_device.h"

int pratchya_set_error(int code, const char* fmt, ...);

namespace {

int64_t gcd64(int64_t x, int64_t y) {
  while (y) {
    const int64_t t = x % y;
    x = y;
    y = t;
  }
  return x;
}

int check_launch(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return pratchya_set_error(PRATCHYA_EHIP, "%s: launch failed: %s", what, hipGetErrorString(e));
  return pratchya_set_error(PRATCHYA_OK, "");
}

bool is_float_dtype(int d) { return d == PRATCHYA_DT_F32 || d == PRATCHYA_DT_BF16; }

__device__ __forceinline__ float act(float x, int kind) {
  if (kind == PRATCHYA_ACT_RELU2) {
    const float r = x < 0.0f ? 0.0f : x;
    return r * r;
  }
  if (kind == PRATCHYA_ACT_SILU) return x / (1.0f + __expf(-x));
  return 0.5f * x * (1.0f + erff(x * 0.70710678118654752f));
}

__device__ __forceinline__ float act_grad(float x, int kind) {
  if (kind == PRATCHYA_ACT_RELU2) return x < 0.0f ? 0.0f : 2.0f * x;
  if (kind == PRATCHYA_ACT_SILU) {
    const float s = 1.0f / (1.0f + __expf(-x));
    return s * (1.0f + x * (1.0f - s));
  }
  return 0.5f * (1.0f + erff(x * 0.70710678118654752f)) + x * 0.39894228040143268f * __expf(-0.5f * x * x);
}

template <typename T>
__global__ __launch_bounds__(256) void k_act(const T* __restrict__ x, int64_t ldx, int64_t width, int64_t n, int kind,
                                             T* __restrict__ y) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / width;
    store_elem(y + i, act(load_elem(x + row * ldx + (i - row * width)), kind));
  }
}

template <typename T>
__global__ __launch_bounds__(256) void k_act_bwd(const T* __restrict__ x, int64_t ldx, const uint8_t* __restrict__ x8,
                                                 const uint8_t* __restrict__ sc8, const float* __restrict__ sc32,
                                                 int64_t blk, int64_t K, const T* __restrict__ dy, int64_t ldy,
                                                 int64_t width, int64_t n, int kind, T* __restrict__ dx) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / width, c = i - row * width;
    float v;
    if (x8) {
      const int64_t k = i / blk;
      v = (e4m3fn_to_f32(x8[i]) * (e8m0_decode(sc8[k]) * sc32[k / K])) * 0.0078125f;
    } else {
      v = load_elem(x + row * ldx + c);
    }
    store_elem(dx + i, act_grad(v, kind) * load_elem(dy + row * ldy + c));
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

unsigned flat_grid(int64_t n) {
  const int64_t g = (n + 255) / 256;
  return (unsigned)(g < 65536 ? g : 65536);
}

}  // namespace

extern "C" int pratchya_activation(const void* x, int64_t ldx, int dtype, int kind, int64_t rows, int64_t width,
                                   void* y, uint8_t* x8, uint8_t* sc8, float* sc32, int64_t blk, hipStream_t stream) {
  const int rc = check_args("activation", kind, dtype, rows, width);
  if (rc) return rc;
  (void)sc8;
  (void)sc32;
  (void)blk;
  if (x8) return pratchya_set_error(PRATCHYA_EUNSUPPORTED, "activation: x is not stored in the same pass");
  const int64_t n = rows * width;
  if (n == 0) return pratchya_set_error(PRATCHYA_OK, "");
  if (!x || !y) return pratchya_set_error(PRATCHYA_EINVAL, "activation: null buffer");
  if (dtype == PRATCHYA_DT_BF16)
    hipLaunchKernelGGL((k_act<uint16_t>), dim3(flat_grid(n)), dim3(256), 0, stream, static_cast<const uint16_t*>(x),
                       ldx, width, n, kind, static_cast<uint16_t*>(y));
  else
    hipLaunchKernelGGL((k_act<float>), dim3(flat_grid(n)), dim3(256), 0, stream, static_cast<const float*>(x), ldx,
                       width, n, kind, static_cast<float*>(y));
  return check_launch("activation");
}

extern "C" int pratchya_activation_bwd(const void* x, int64_t ldx, int x_dtype, const uint8_t* sc8, const float* sc32,
                                       int64_t blk, const void* dy, int64_t ldy, int dtype, int kind, int64_t rows,
                                       int64_t width, void* dx, hipStream_t stream) {
  const int rc = check_args("activation_bwd", kind, dtype, rows, width);
  if (rc) return rc;
  const bool stored = x_dtype == PRATCHYA_DT_E4M3;
  if (!stored && x_dtype != dtype)
    return pratchya_set_error(PRATCHYA_EINVAL, "activation_bwd: unsupported dtypes (x %d, dy %d)", x_dtype, dtype);
  if (stored && (blk < 1 || width % blk))
    return pratchya_set_error(PRATCHYA_EINVAL, "activation_bwd: blocks of %lld do not divide rows of %lld",
                              (long long)blk, (long long)width);
  const int64_t n = rows * width;
  if (n == 0) return pratchya_set_error(PRATCHYA_OK, "");
  if (!x || !dy || !dx || (stored && (!sc8 || !sc32)))
    return pratchya_set_error(PRATCHYA_EINVAL, "activation_bwd: null buffer");
  const int64_t K = stored ? gcd64(blk / 16 > 1 ? blk / 16 : 1, n / blk) : 1;
  const uint8_t* x8 = stored ? static_cast<const uint8_t*>(x) : nullptr;
  if (dtype == PRATCHYA_DT_BF16)
    hipLaunchKernelGGL((k_act_bwd<uint16_t>), dim3(flat_grid(n)), dim3(256), 0, stream,
                       static_cast<const uint16_t*>(x), ldx, x8, sc8, sc32, blk, K, static_cast<const uint16_t*>(dy),
                       ldy, width, n, kind, static_cast<uint16_t*>(dx));
  else
    hipLaunchKernelGGL((k_act_bwd<float>), dim3(flat_grid(n)), dim3(256), 0, stream, static_cast<const float*>(x), ldx,
                       x8, sc8, sc32, blk, K, static_cast<const float*>(dy), ldy, width, n, kind,
                       static_cast<float*>(dx));
  return check_launch("activation_bwd");
}
