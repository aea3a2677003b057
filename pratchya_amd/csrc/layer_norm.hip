// Layer norm over segments of a row and its gradients, for gfx950.
//
// A row of `width` values holds `groups` segments of D = width / groups (one for
// a plain layer norm, one per head for a norm over heads).  Per segment
//   mu = mean(x),  v = mean((x - mu)^2),  r = 1 / sqrt(v + eps),
//   h  = (x - mu) r,  y = h w + b                     (w, b: [width])
// and, with a = w dy,
//   dx = r (a - mean(a) - h mean(a h)),  dw = sum_rows dy h,  db = sum_rows dy.
// The backward reads x itself or, where the forward pass kept it in 8 bits,
// its quantized form with block grid (1, blk) (fp8_math.h); mu and r are the
// unquantized x's either way.  Everything is summed in f32; results are rounded
// to their type once.
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

struct Affine {
  const void* w;
  const void* b;
  bool w16, b16;
};

template <typename T>
__global__ __launch_bounds__(256) void k_layer_norm(const T* __restrict__ x, int64_t ldx, Affine p, int64_t width,
                                                    int64_t groups, float eps, T* __restrict__ y,
                                                    float* __restrict__ stats) {
  __shared__ float lds[4];
  const int64_t D = width / groups, row = blockIdx.x / groups, c0 = (blockIdx.x - row * groups) * D;
  const T* xs = x + row * ldx + c0;
  T* ys = y + row * width + c0;
  float s = 0.0f;
  for (int64_t i = threadIdx.x; i < D; i += 256) s += load_elem(xs + i);
  const float mean = block_add<4>(s, lds) / (float)D;
  float q = 0.0f;
  for (int64_t i = threadIdx.x; i < D; i += 256) {
    const float d = load_elem(xs + i) - mean;
    q += d * d;
  }
  const float rstd = 1.0f / sqrtf(block_add<4>(q, lds) / (float)D + eps);
  for (int64_t i = threadIdx.x; i < D; i += 256) {
    float v = (load_elem(xs + i) - mean) * rstd;
    if (p.w) v *= load_param(p.w, p.w16, c0 + i);
    if (p.b) v += load_param(p.b, p.b16, c0 + i);
    store_elem(ys + i, v);
  }
  if (stats && threadIdx.x == 0) {
    stats[2 * (int64_t)blockIdx.x] = mean;
    stats[2 * (int64_t)blockIdx.x + 1] = rstd;
  }
}

// x as the backward pass reads it: element i of row `row`.
template <typename X>
struct Source {
  const X* x;
  int64_t ldx;
  __device__ __forceinline__ float at(int64_t row, int64_t i) const { return load_elem(x + row * ldx + i); }
};
struct Stored {
  const uint8_t* x8;
  const uint8_t* sc8;
  const float* sc32;
  int64_t width, blk, K;
  __device__ __forceinline__ float at(int64_t row, int64_t i) const {
    const int64_t e = row * width + i, n = e / blk;
    return (e4m3fn_to_f32(x8[e]) * (e8m0_decode(sc8[n]) * sc32[n / K])) * 0.0078125f;
  }
};

template <typename T, typename S>
__global__ __launch_bounds__(256) void k_layer_norm_dx(S src, const T* __restrict__ dy, int64_t ldy, Affine p,
                                                       int64_t width, int64_t groups, const float* __restrict__ stats,
                                                       T* __restrict__ dx) {
  __shared__ float lds[4];
  const int64_t D = width / groups, row = blockIdx.x / groups, c0 = (blockIdx.x - row * groups) * D;
  const float mean = stats[2 * (int64_t)blockIdx.x], rstd = stats[2 * (int64_t)blockIdx.x + 1];
  float s1 = 0.0f, s2 = 0.0f;
  for (int64_t i = threadIdx.x; i < D; i += 256) {
    const float h = (src.at(row, c0 + i) - mean) * rstd;
    float a = load_elem(dy + row * ldy + c0 + i);
    if (p.w) a *= load_param(p.w, p.w16, c0 + i);
    s1 += a;
    s2 += a * h;
  }
  const float m1 = block_add<4>(s1, lds) / (float)D, m2 = block_add<4>(s2, lds) / (float)D;
  for (int64_t i = threadIdx.x; i < D; i += 256) {
    const float h = (src.at(row, c0 + i) - mean) * rstd;
    float a = load_elem(dy + row * ldy + c0 + i);
    if (p.w) a *= load_param(p.w, p.w16, c0 + i);
    store_elem(dx + row * width + c0 + i, rstd * (a - m1 - h * m2));
  }
}

// Column sums over the rows of one of gridDim.y slices: part[slice][0 / 1][width].
template <typename T, typename S>
__global__ __launch_bounds__(256) void k_layer_norm_dp(S src, const T* __restrict__ dy, int64_t ldy, int64_t rows,
                                                       int64_t width, int64_t groups,
                                                       const float* __restrict__ stats, float* __restrict__ part) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= width) return;
  const int64_t g = c / (width / groups);
  float dw = 0.0f, db = 0.0f;
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    const float* st = stats + 2 * (row * groups + g);
    const float v = load_elem(dy + row * ldy + c);
    dw += v * ((src.at(row, c) - st[0]) * st[1]);
    db += v;
  }
  part[(2 * (int64_t)blockIdx.y) * width + c] = dw;
  part[(2 * (int64_t)blockIdx.y + 1) * width + c] = db;
}

__global__ __launch_bounds__(256) void k_layer_norm_join(const float* __restrict__ part, int slices, int64_t width,
                                                         void* dw, bool dw16, void* db, bool db16) {
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= width) return;
  float s = 0.0f, t = 0.0f;
  for (int i = 0; i < slices; ++i) {
    s += part[2 * i * width + c];
    t += part[(2 * i + 1) * width + c];
  }
  if (dw) store_param(dw, dw16, c, s);
  if (db) store_param(db, db16, c, t);
}

constexpr int kSlices = 64;

int check_shape(const char* what, int64_t rows, int64_t width, int64_t groups) {
  if (rows < 0 || width < 0 || groups < 1 || width % groups)
    return pratchya_set_error(PRATCHYA_EINVAL, "%s: %lld groups do not divide rows of %lld (%lld rows)", what,
                              (long long)groups, (long long)width, (long long)rows);
  if (rows > 0 && (rows * groups > 0x7FFFFFFF || width / 256 > 0x7FFFFFFF))
    return pratchya_set_error(PRATCHYA_EUNSUPPORTED, "%s: more than 2^31 segments", what);
  return PRATCHYA_OK;
}

template <typename T, typename S>
int launch_bwd(S src, const void* dy, int64_t ldy, const void* w, int w_dtype, const float* stats, int64_t rows,
               int64_t width, int64_t groups, void* dx, void* dw, int dw_dtype, void* db, int db_dtype, float* part,
               hipStream_t stream) {
  const T* g = static_cast<const T*>(dy);
  const Affine p = {w, nullptr, w_dtype == PRATCHYA_DT_BF16, false};
  if (dx)
    hipLaunchKernelGGL((k_layer_norm_dx<T, S>), dim3((unsigned)(rows * groups)), dim3(256), 0, stream, src, g, ldy, p,
                       width, groups, stats, static_cast<T*>(dx));
  if (dw || db) {
    const int slices = rows < kSlices ? (int)rows : kSlices;
    const dim3 grid((unsigned)((width + 255) / 256), (unsigned)slices);
    hipLaunchKernelGGL((k_layer_norm_dp<T, S>), grid, dim3(256), 0, stream, src, g, ldy, rows, width, groups, stats,
                       part);
    hipLaunchKernelGGL(k_layer_norm_join, dim3(grid.x), dim3(256), 0, stream, part, slices, width, dw,
                       dw_dtype == PRATCHYA_DT_BF16, db, db_dtype == PRATCHYA_DT_BF16);
  }
  return check_launch("layer_norm_bwd");
}

}  // namespace

extern "C" int pratchya_layer_norm_stores(int64_t width, int64_t groups, int64_t blk) {
  (void)width;
  (void)groups;
  (void)blk;
  return 0;
}

extern "C" int pratchya_layer_norm(const void* x, int64_t ldx, int dtype, const void* w, int w_dtype, const void* b,
                                   int b_dtype, int64_t rows, int64_t width, int64_t groups, float eps, void* y,
                                   float* stats, uint8_t* x8, uint8_t* sc8, float* sc32, int64_t blk,
                                   hipStream_t stream) {
  const int rc = check_shape("layer_norm", rows, width, groups);
  if (rc) return rc;
  (void)sc8;
  (void)sc32;
  if (x8 && !pratchya_layer_norm_stores(width, groups, blk))
    return pratchya_set_error(PRATCHYA_EUNSUPPORTED, "layer_norm: blocks of %lld are not stored in the same pass",
                              (long long)blk);
  if (!is_float_dtype(dtype) || (w && !is_float_dtype(w_dtype)) || (b && !is_float_dtype(b_dtype)))
    return pratchya_set_error(PRATCHYA_EINVAL, "layer_norm: unsupported dtypes (x %d, weight %d, bias %d)", dtype,
                              w_dtype, b_dtype);
  if (rows == 0 || width == 0) return pratchya_set_error(PRATCHYA_OK, "");
  if (!x || !y) return pratchya_set_error(PRATCHYA_EINVAL, "layer_norm: null buffer");
  const Affine p = {w, b, w_dtype == PRATCHYA_DT_BF16, b_dtype == PRATCHYA_DT_BF16};
  const dim3 grid((unsigned)(rows * groups));
  if (dtype == PRATCHYA_DT_BF16)
    hipLaunchKernelGGL((k_layer_norm<uint16_t>), grid, dim3(256), 0, stream, static_cast<const uint16_t*>(x), ldx, p,
                       width, groups, eps, static_cast<uint16_t*>(y), stats);
  else
    hipLaunchKernelGGL((k_layer_norm<float>), grid, dim3(256), 0, stream, static_cast<const float*>(x), ldx, p, width,
                       groups, eps, static_cast<float*>(y), stats);
  return check_launch("layer_norm");
}

extern "C" int64_t pratchya_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t width, int64_t groups) {
  (void)groups;
  return (rows < kSlices ? rows : kSlices) * 2 * width * (int64_t)sizeof(float);
}

extern "C" int pratchya_layer_norm_bwd(const void* x, int64_t ldx, int x_dtype, const uint8_t* sc8, const float* sc32,
                                       int64_t blk, const void* dy, int64_t ldy, int dtype, const void* w, int w_dtype,
                                       const float* stats, int64_t rows, int64_t width, int64_t groups, void* dx,
                                       void* dw, int dw_dtype, void* db, int db_dtype, void* workspace,
                                       int64_t workspace_bytes, hipStream_t stream) {
  const int rc = check_shape("layer_norm_bwd", rows, width, groups);
  if (rc) return rc;
  const bool stored = x_dtype == PRATCHYA_DT_E4M3;
  if (!is_float_dtype(dtype) || (!stored && x_dtype != dtype) || (w && !is_float_dtype(w_dtype)) ||
      (dw && !is_float_dtype(dw_dtype)) || (db && !is_float_dtype(db_dtype)))
    return pratchya_set_error(PRATCHYA_EINVAL, "layer_norm_bwd: unsupported dtypes (x %d, dy %d)", x_dtype, dtype);
  if (stored && (blk < 1 || width % blk))
    return pratchya_set_error(PRATCHYA_EINVAL, "layer_norm_bwd: blocks of %lld do not divide rows of %lld",
                              (long long)blk, (long long)width);
  if (rows == 0 || width == 0) return pratchya_set_error(PRATCHYA_OK, "");
  if (!x || !dy || !stats || (stored && (!sc8 || !sc32)))
    return pratchya_set_error(PRATCHYA_EINVAL, "layer_norm_bwd: null buffer");
  const int64_t need = pratchya_layer_norm_bwd_workspace_bytes(rows, width, groups);
  if ((dw || db) && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 4))
    return pratchya_set_error(PRATCHYA_EINVAL, "layer_norm_bwd: workspace of %lld bytes needed, 4-byte aligned",
                              (long long)need);
  float* part = static_cast<float*>(workspace);
#define PRATCHYA_LNB(T, SRC)                                                                                     \
  launch_bwd<T>(SRC, dy, ldy, w, w_dtype, stats, rows, width, groups, dx, dw, dw_dtype, db, db_dtype, part, stream)
  if (stored) {
    const int64_t n_blk = rows * (width / blk);
    const Stored s = {static_cast<const uint8_t*>(x), sc8, sc32, width, blk, gcd64(blk / 16 > 1 ? blk / 16 : 1, n_blk)};
    return dtype == PRATCHYA_DT_BF16 ? PRATCHYA_LNB(uint16_t, s) : PRATCHYA_LNB(float, s);
  }
  if (dtype == PRATCHYA_DT_BF16)
    return PRATCHYA_LNB(uint16_t, (Source<uint16_t>{static_cast<const uint16_t*>(x), ldx}));
  return PRATCHYA_LNB(float, (Source<float>{static_cast<const float*>(x), ldx}));
#undef PRATCHYA_LNB
}
