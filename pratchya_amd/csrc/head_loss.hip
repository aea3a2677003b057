// Cross entropy of an output head whose logits are not kept, with the gradients of
// its input and weight, for gfx950.
//
// Per row of z = x W (x [n, C], W [C, V]) with target t and label smoothing a:
//   l = (1 - a) (lse - z_t) + a (lse - mean z),   lse = log sum_v e^(z_v),
//   dz_v = g (p_v - (1 - a) [v = t] - a / V),     p_v = e^(z_v - lse),
//   dx = dz W^T,   dW = x^T dz.
// A negative target stands for none: l = 0 and dz = 0.  A target of V or more has no
// logit: l is NaN and dz the formula's without its second term.
//
// The vocabulary is taken in pieces: a piece's logits are computed in f32, enter the
// rows' running maxima and sums (forward) or turn into dz (backward, from lse), and
// are overwritten by the next piece's.  In f32 every operand of a product is the sum
// of three exact bf16 planes and a product six products of planes.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "pratchya_fp8.h"
#include "row_device.h"
#include "row_host.h"

namespace {

constexpr float kLowest = -3.4028234663852886e38f;

// --------------------------------------------------------------------------
// operands
// --------------------------------------------------------------------------
__device__ __forceinline__ float top_piece(float v) { return u2f(f2u(v) & 0xFFFF0000u); }

// Planes [P][rows_to][cols_to] of src [rows, cols] (rows ld elements apart, at any
// element's address), zeros around it: bf16 as it is (P 1) or an f32 value's three
// pieces (P 3), 8 columns a thread.
template <typename T, int P>
__global__ __launch_bounds__(256) void k_head_planes(const T* __restrict__ src, int64_t ld, int64_t rows, int64_t cols,
                                                     int64_t rows_to, int64_t cols_to, uint16_t* __restrict__ dst) {
  const int64_t per = cols_to / 8, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows_to * per) return;
  const int64_t r = i / per, c = (i - r * per) * 8;
  uint16_t* to = dst + r * cols_to + c;
  float v[8] = {};
  if (r < rows && c < cols) {
    const T* p = src + r * ld + c;
    if (c + 8 <= cols) {
      constexpr int N = kN<T>;
#pragma unroll
      for (int h = 0; h < 8 / N; ++h) {
        float w[N];
        widen(load_raw(p + h * N), w);
#pragma unroll
        for (int k = 0; k < N; ++k) v[h * N + k] = w[k];
      }
    } else {
      load_some(p, cols - c, 0.0f, v);
    }
  }
#pragma unroll
  for (int q = 0; q < P; ++q) {
    float o[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      o[k] = P == 1 || q == P - 1 ? v[k] : top_piece(v[k]);
      v[k] -= o[k];
    }
    *reinterpret_cast<u32x4_t*>(to + q * rows_to * cols_to) = narrow(o);
  }
}

// --------------------------------------------------------------------------
// rows
// --------------------------------------------------------------------------
// What a row's logits have shown so far: the largest but the target's, m, the sum of
// e^(z - m) without the target's, the target's logit, the sum of all.  With the
// target's term apart a loss near 0 keeps its digits.
struct Seen {
  float m = kLowest, s = 0.0f, zt = -__builtin_inff(), sum = 0.0f;
};

// Loss, and (max, log of the sum about it) for the backward pass.
__device__ __forceinline__ void finish_row(const Seen& a, int64_t target, int64_t vocab, float smooth, float* loss,
                                           float* stats) {
  const bool has = target >= 0 && target < vocab;
  const float M = has && !(a.m > a.zt) ? a.zt : a.m;
  // e^(z_t - M) and the others' sum about M; of infinite or lowest values the sums decide
  const float et = has && a.zt > kLowest ? expf(a.zt - M) : has && a.zt != a.zt ? a.zt : 0.0f;
  const float others = a.s == 0.0f ? 0.0f : a.s * expf(fmaxf(a.m - M, kLowest));
  const float logs = et == 1.0f ? log1pf(others) : logf(et + others);
  if (loss) {
    const float lse = M + logs;
    float l = (M - a.zt) + logs;
    if (smooth != 0.0f) l = (1.0f - smooth) * l + smooth * (lse - a.sum / (float)vocab);
    *loss = target < 0 ? 0.0f : has ? l : __builtin_nanf("");
  }
  if (stats) {
    stats[0] = M;
    stats[1] = logs;
  }
}

// A piece's logits [rows, cols], columns v0 .. of the vocabulary, into the rows'
// states: one workgroup a row.  The last piece's call finishes them.
constexpr int kRowThreads = 256;

__device__ __forceinline__ Seen join_seen(Seen a, float* lds) {
  const float m = wave_max(a.m);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = m;
  __syncthreads();
  float M = lds[0];
#pragma unroll
  for (int w = 1; w < kRowThreads / 64; ++w) M = fmaxf(M, lds[w]);
  a.s = a.s == 0.0f ? 0.0f : a.s * expf(fmaxf(a.m - M, kLowest));
  a.m = M;
  a.s = block_add<kRowThreads / 64>(a.s, lds);
  a.sum = block_add<kRowThreads / 64>(a.sum, lds);
  return a;
}

__global__ __launch_bounds__(kRowThreads) void k_head_rows(const float* __restrict__ z, int64_t ld, int64_t cols,
                                                           const int64_t* __restrict__ targets, int64_t v0,
                                                           int64_t vocab, float smooth, float4* __restrict__ state,
                                                           int first, int last, float* __restrict__ loss,
                                                           float* __restrict__ stats) {
  __shared__ float lds[kRowThreads / 64];
  __shared__ float shared_zt;
  const int64_t row = blockIdx.x, target = targets[row];
  const float* p = z + row * ld;
  // the target's column in this piece, or none
  const int64_t tc = target >= 0 && target < vocab ? target - v0 : -1;
  Seen a;
  for (int64_t c = threadIdx.x * 4; c < cols; c += kRowThreads * 4) {
    float v[4];
    if (c + 4 <= cols) widen(load_raw(p + c), v);
    else load_some(p + c, cols - c, -__builtin_inff(), v);
    float top = a.m;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (c + k < cols) a.sum += v[k];
      if (c + k == tc) {
        shared_zt = v[k];
        v[k] = -__builtin_inff();
      }
      top = fmaxf(top, v[k]);
    }
    if (top > a.m) {
      a.s *= expf(fmaxf(a.m - top, kLowest));
      a.m = top;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) a.s += expf(v[k] - a.m);
  }
  a = join_seen(a, lds);
  if (threadIdx.x) return;
  if (tc >= 0 && tc < cols) a.zt = shared_zt;
  if (!first) {
    const float4 b = state[row];
    const float M = fmaxf(a.m, b.x);
    a.s = (a.s == 0.0f ? 0.0f : a.s * expf(fmaxf(a.m - M, kLowest))) +
          (b.y == 0.0f ? 0.0f : b.y * expf(fmaxf(b.x - M, kLowest)));
    a.m = M;
    if (!(tc >= 0 && tc < cols)) a.zt = b.z;
    a.sum += b.w;
  }
  if (last) finish_row(a, target, vocab, smooth, loss + row, stats ? stats + 2 * row : nullptr);
  else state[row] = make_float4(a.m, a.s, a.zt, a.sum);
}

// dz of a piece's logits as planes [P][rows_to][cols_to], zeros around [rows, cols].
template <int P>
__global__ __launch_bounds__(256) void k_head_grad(const float* __restrict__ z, int64_t ld, int64_t rows, int64_t cols,
                                                   int64_t rows_to, int64_t cols_to, const int64_t* __restrict__ targets,
                                                   int64_t v0, int64_t vocab, float smooth,
                                                   const float* __restrict__ stats, const float* __restrict__ g,
                                                   uint16_t* __restrict__ dst) {
  const int64_t per = cols_to / 8, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows_to * per) return;
  const int64_t r = i / per, c = (i - r * per) * 8;
  uint16_t* to = dst + r * cols_to + c;
  float d[8] = {};
  if (r < rows && targets[r] >= 0) {
    const int64_t target = targets[r];
    const float m = stats[2 * r], logs = stats[2 * r + 1], gr = g[r], even = smooth / (float)vocab;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v[4];
      widen(load_raw(z + r * ld + c + 4 * h), v);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int64_t col = c + 4 * h + k;
        const float p = expf((v[k] - m) - logs) - even - (v0 + col == target ? 1.0f - smooth : 0.0f);
        d[4 * h + k] = col < cols ? gr * p : 0.0f;
      }
    }
  }
#pragma unroll
  for (int q = 0; q < P; ++q) {
    float o[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      o[k] = P == 1 || q == P - 1 ? d[k] : top_piece(d[k]);
      d[k] -= o[k];
    }
    *reinterpret_cast<u32x4_t*>(to + q * rows_to * cols_to) = narrow(o);
  }
}

// out [rows, cols] (contiguous, or ld_out apart) = src [rows, cols], f32 ld_src apart,
// plus the sums of the pieces before (sum, if add); not the last piece: into sum.
template <typename T>
__global__ __launch_bounds__(256) void k_head_out(const float* __restrict__ src, int64_t ld_src, int64_t rows,
                                                  int64_t cols, float* __restrict__ sum, int add, int last,
                                                  T* __restrict__ out, int64_t ld_out) {
  const int64_t per = (cols + 3) / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * per) return;
  const int64_t r = i / per, c = (i - r * per) * 4;
  float v[4];
  widen(load_raw(src + r * ld_src + c), v);
  if (add) {
    float o[4];
    widen(load_raw(sum + r * ld_src + c), o);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] += o[k];
  }
  if (!last) {
    store_vec(sum + r * ld_src + c, v);
    return;
  }
  store_some(out + r * ld_out + c, cols - c < 4 ? cols - c : 4, v);
}

// --------------------------------------------------------------------------
// host
// --------------------------------------------------------------------------
int64_t up64(int64_t v) { return (v + 63) / 64 * 64; }
int64_t round256(int64_t v) { return (v + 255) / 256 * 256; }

// Largest f32 logits of a piece, and the planes of its weight.
constexpr int64_t kPieceBytes = (int64_t)256 << 20;
constexpr int64_t kMaxOffset = (int64_t)0xFFFFFFFF;

// Plane pairs of an f32 product: those of 2^-24 of the product's size or more.
constexpr uint32_t kPairsA = 0x210100, kPairsB = 0x012010;   // (0,0) (0,1) (1,0) (0,2) (1,1) (2,0)

struct Head {
  const void *x, *w;
  int64_t ldx, ldw, n, C, V;
  int dtype;
  bool rows;                     // w is [V, C] (a table's transposed view), not [C, V]
  int P;
  int64_t n64, C64, piece;       // piece: columns of a vocabulary piece, a multiple of 64
  bool x_direct, w_direct;
  // workspace
  int64_t xp, wp, z, dzp, dx_sum, dx_tmp, dw_tmp, split, split_bytes, state, bytes;
};

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Sizes and workspace of a call; direct: whether x and w themselves are operands.
int plan(const char* what, bool bwd, bool want_dx, bool want_dw, Head* h) {
  if (!is_float_dtype(h->dtype)) return pratchya_set_error(PRATCHYA_EINVAL, "%s: unsupported dtype %d", what, h->dtype);
  if (h->n < 0 || h->C < 1 || h->V < 1 || h->ldx < 0 || h->ldw < 0)
    return pratchya_set_error(PRATCHYA_EINVAL, "%s: %lld rows of %lld, a vocabulary of %lld", what, (long long)h->n,
                              (long long)h->C, (long long)h->V);
  h->P = h->dtype == PRATCHYA_DT_BF16 ? 1 : 3;
  h->n64 = up64(h->n);
  h->C64 = up64(h->C);
  const int64_t V64 = up64(h->V);
  // planes are addressed with 32-bit byte offsets
  if (h->n > kMaxOffset || h->C > kMaxOffset || h->V > 0x7FFFFF00 ||
      2 * h->P * (h->n64 + 128) * h->C64 > kMaxOffset || 2 * h->P * 1152 * h->C64 > kMaxOffset ||
      2 * h->P * (h->n64 + 128) * 1024 > kMaxOffset)
    return pratchya_set_error(PRATCHYA_EUNSUPPORTED, "%s: rows or weights beyond 32-bit offsets", what);
  const bool bf = h->dtype == PRATCHYA_DT_BF16;
  if (!fits_launch(h->n, kRowThreads)) return pratchya_set_error(PRATCHYA_EUNSUPPORTED, "%s: 2^24 rows or more", what);
  h->x_direct = bf && h->n % 64 == 0 && h->C % 64 == 0 && h->ldx % 8 == 0 && h->ldx >= h->C && aligned16(h->x) &&
                2 * (h->n + 128) * h->ldx <= kMaxOffset;
  h->w_direct = bf && h->C % 64 == 0 && h->V % 64 == 0 && h->ldw % 8 == 0 && h->ldw >= (h->rows ? h->C : h->V) &&
                aligned16(h->w) && 2 * ((h->rows ? 1152 : h->C + 1) * h->ldw + 128) <= kMaxOffset;
  int64_t piece = kPieceBytes / 4 / (h->n64 ? h->n64 : 64) / 64 * 64;
  const int64_t by_w = 2 * kPieceBytes / (2 * h->P * h->C64) / 64 * 64;       // its planes: 512 MB
  if (!h->w_direct && by_w < piece) piece = by_w;
  const int64_t by_ld = (kMaxOffset / 2 / h->P / (h->n64 > h->C64 ? h->n64 + 128 : h->C64 + 128)) / 64 * 64;
  if (by_ld < piece) piece = by_ld;
  if (piece < 1024) piece = 1024;
  // pieces of one size
  const int64_t pieces = (V64 + piece - 1) / piece;
  h->piece = up64((V64 + pieces - 1) / pieces);
  if (h->piece > V64) h->piece = V64;
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t p = at;
    at += round256(bytes);
    return p;
  };
  const int64_t planes = 2 * h->P, segs = h->P == 1 ? 1 : 6;
  h->xp = take(planes * h->n64 * h->C64);
  h->wp = take(h->w_direct ? 0 : planes * h->C64 * h->piece);
  h->z = take(4 * h->n * h->piece);
  h->state = take(16 * h->n);
  h->split_bytes = 0;
  auto split = [&](int64_t M, int64_t N, int64_t K) {
    const int64_t b = pratchya_gemm_t128_workspace_bytes(M, N, segs * (K / 64), 1);
    if (b > h->split_bytes) h->split_bytes = b;
  };
  const int64_t rest = V64 - (V64 - 1) / h->piece * h->piece;      // the last piece
  for (int64_t Vp : {h->piece, rest}) {
    split(h->n, Vp, h->C64);
    if (bwd && want_dx) split(h->n, h->C64, Vp);
    if (bwd && want_dw) {
      split(h->rows ? Vp : h->C64, h->rows ? h->C64 : Vp, h->n64);
      split(h->rows ? Vp : h->C, h->rows ? h->C : Vp, h->n64);
    }
  }
  h->dzp = h->dx_sum = h->dx_tmp = h->dw_tmp = 0;
  if (bwd) {
    h->dzp = take(planes * h->n64 * h->piece);
    if (want_dx) {
      h->dx_tmp = take(4 * h->n * h->C64);
      h->dx_sum = take(h->piece < h->V ? 4 * h->n * h->C64 : 0);
    }
    if (want_dw) h->dw_tmp = take(4 * h->C64 * h->piece);
  }
  h->split = take(h->split_bytes);
  h->bytes = at;
  return PRATCHYA_OK;
}

struct Call {
  const Head& h;
  char* ws;
  hipStream_t stream;

  uint16_t* planes_at(int64_t off) const { return reinterpret_cast<uint16_t*>(ws + off); }
  float* floats_at(int64_t off) const { return reinterpret_cast<float*>(ws + off); }

  int planes(const void* src, int64_t ld, int64_t rows, int64_t cols, int64_t rows_to, int64_t cols_to,
             uint16_t* dst) const {
    const int64_t blocks = (rows_to * (cols_to / 8) + 255) / 256;
    if (!fits_launch(blocks, 256)) return pratchya_set_error(PRATCHYA_EUNSUPPORTED, "linear_cross_entropy: too large");
    if (h.P == 1)
      hipLaunchKernelGGL((k_head_planes<uint16_t, 1>), dim3((unsigned)blocks), dim3(256), 0, stream,
                         static_cast<const uint16_t*>(src), ld, rows, cols, rows_to, cols_to, dst);
    else
      hipLaunchKernelGGL((k_head_planes<float, 3>), dim3((unsigned)blocks), dim3(256), 0, stream,
                         static_cast<const float*>(src), ld, rows, cols, rows_to, cols_to, dst);
    return check_launch("linear_cross_entropy");
  }
  // C [M, N] = A . B over K; a plane's rows lie lda / ldb apart, planes a_rows * lda.
  int product(const uint16_t* A, int64_t lda, int64_t a_rows, int a_kmajor, const uint16_t* B, int64_t ldb,
              int64_t b_rows, int b_kmajor, int64_t M, int64_t N, int64_t K, void* C, int64_t ldc, int dtype) const {
    const int segs = h.P == 1 ? 1 : 6;
    return pratchya_gemm_bf16_planes(A, lda, a_rows * lda, a_kmajor, h.P, h.P == 1 ? 0 : kPairsA, B, ldb, b_rows * ldb,
                                     b_kmajor, h.P, h.P == 1 ? 0 : kPairsB, h.P == 1 ? 0 : kPairsB, M, N, K, segs, segs,
                                     nullptr, nullptr, 0, 0, 0, C, ldc, dtype, nullptr, 0, 1, 0, 0, 0, 0,
                                     ws + h.split, h.split_bytes, stream);
  }
};

// The operands x and a piece of w, as they are or as planes.
struct Operands {
  const uint16_t *x, *w;
  int64_t ldx, ldw, x_rows, w_rows;
};

int operand_x(const Call& c, Operands* o) {
  const Head& h = c.h;
  o->x_rows = h.n64;
  if (h.x_direct) {
    o->x = static_cast<const uint16_t*>(h.x);
    o->ldx = h.ldx;
    return PRATCHYA_OK;
  }
  o->x = c.planes_at(h.xp);
  o->ldx = h.C64;
  return c.planes(h.x, h.ldx, h.n, h.C, h.n64, h.C64, c.planes_at(h.xp));
}

int operand_w(const Call& c, int64_t v0, int64_t cols, int64_t Vp, Operands* o) {
  const Head& h = c.h;
  const int64_t esz = h.dtype == PRATCHYA_DT_BF16 ? 2 : 4;
  const char* src = static_cast<const char*>(h.w) + v0 * (h.rows ? h.ldw : 1) * esz;
  o->w_rows = h.rows ? Vp : h.C64;
  if (h.w_direct) {
    o->w = reinterpret_cast<const uint16_t*>(src);
    o->ldw = h.ldw;
    return PRATCHYA_OK;
  }
  o->w = c.planes_at(h.wp);
  o->ldw = h.rows ? h.C64 : Vp;
  return h.rows ? c.planes(src, h.ldw, cols, h.C, Vp, h.C64, c.planes_at(h.wp))
                : c.planes(src, h.ldw, h.C, cols, h.C64, Vp, c.planes_at(h.wp));
}

// A piece's logits into the workspace.
int logits(const Call& c, const Operands& o, int64_t Vp) {
  const Head& h = c.h;
  return c.product(o.x, o.ldx, o.x_rows, 0, o.w, o.ldw, o.w_rows, h.rows ? 0 : 1, h.n, Vp, h.C64, c.floats_at(h.z), Vp,
                   PRATCHYA_DT_F32);
}

int forward(const Call& c, const int64_t* targets, float smooth, float* loss, float* stats) {
  const Head& h = c.h;
  Operands o;
  int rc = operand_x(c, &o);
  for (int64_t v0 = 0; v0 < h.V && !rc; v0 += h.piece) {
    const int64_t cols = h.V - v0 < h.piece ? h.V - v0 : h.piece, Vp = up64(cols);
    if ((rc = operand_w(c, v0, cols, Vp, &o)) || (rc = logits(c, o, Vp))) break;
    hipLaunchKernelGGL(k_head_rows, dim3((unsigned)h.n), dim3(kRowThreads), 0, c.stream, c.floats_at(h.z), Vp, cols,
                       targets, v0, h.V, smooth, reinterpret_cast<float4*>(c.ws + h.state), v0 == 0,
                       v0 + h.piece >= h.V, loss, stats);
    rc = check_launch("linear_cross_entropy");
  }
  return rc;
}

template <typename T>
int backward(const Call& c, const int64_t* targets, float smooth, const float* stats, const float* g, T* dx, T* dw) {
  const Head& h = c.h;
  const char* what = "linear_cross_entropy_bwd";
  constexpr int64_t chunk = 16 / sizeof(T);
  Operands o;
  int rc = operand_x(c, &o);
  for (int64_t v0 = 0; v0 < h.V && !rc; v0 += h.piece) {
    const int64_t cols = h.V - v0 < h.piece ? h.V - v0 : h.piece, Vp = up64(cols);
    if ((rc = operand_w(c, v0, cols, Vp, &o)) || (rc = logits(c, o, Vp))) break;
    uint16_t* dz = c.planes_at(h.dzp);
    const int64_t blocks = (h.n64 * (Vp / 8) + 255) / 256;
    if (!fits_launch(blocks, 256)) return pratchya_set_error(PRATCHYA_EUNSUPPORTED, "%s: too large", what);
    auto grad = h.P == 1 ? k_head_grad<1> : k_head_grad<3>;
    hipLaunchKernelGGL(grad, dim3((unsigned)blocks), dim3(256), 0, c.stream, c.floats_at(h.z), Vp, h.n, cols, h.n64, Vp,
                       targets, v0, h.V, smooth, stats, g, dz);
    if ((rc = check_launch(what))) break;
    if (dx) {
      float* tmp = c.floats_at(h.dx_tmp);
      rc = c.product(dz, Vp, h.n64, 0, o.w, o.ldw, o.w_rows, h.rows ? 1 : 0, h.n, h.C64, Vp, tmp, h.C64, PRATCHYA_DT_F32);
      if (rc) break;
      hipLaunchKernelGGL((k_head_out<T>), dim3((unsigned)((h.n * ((h.C + 3) / 4) + 255) / 256)), dim3(256), 0, c.stream,
                         tmp, h.C64, h.n, h.C, c.floats_at(h.dx_sum), v0 > 0, v0 + h.piece >= h.V, dx, h.C);
      if ((rc = check_launch(what))) break;
    }
    if (dw) {
      // [C, V]: rows C, columns cols of them; [V, C]: rows cols, columns C
      const int64_t M = h.rows ? cols : h.C, N = h.rows ? h.C : cols, ld = h.rows ? h.C : h.V;
      T* to = dw + (h.rows ? v0 * h.C : v0);
      const bool direct = M > 32 && M % 8 == 0 && N % 8 == 0 && ld % chunk == 0 && aligned16(to);
      const int64_t Mt = direct ? M : up64(M), Nt = direct ? N : up64(N);
      void* out = direct ? static_cast<void*>(to) : c.ws + h.dw_tmp;
      const int type = direct ? h.dtype : PRATCHYA_DT_F32;
      const int64_t ldo = direct ? ld : Nt;
      rc = h.rows ? c.product(dz, Vp, h.n64, 1, o.x, o.ldx, o.x_rows, 1, Mt, Nt, h.n64, out, ldo, type)
                  : c.product(o.x, o.ldx, o.x_rows, 1, dz, Vp, h.n64, 1, Mt, Nt, h.n64, out, ldo, type);
      if (rc) break;
      if (!direct) {
        hipLaunchKernelGGL((k_head_out<T>), dim3((unsigned)((M * ((N + 3) / 4) + 255) / 256)), dim3(256), 0, c.stream,
                           c.floats_at(h.dw_tmp), Nt, M, N, nullptr, 0, 1, to, ld);
        rc = check_launch(what);
      }
    }
  }
  return rc;
}

__global__ __launch_bounds__(256) void k_head_zero(uint16_t* p, int64_t n) {
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) p[i] = 0;
}

}  // namespace

extern "C" int64_t pratchya_linear_cross_entropy_workspace_bytes(const void* x, int64_t ldx, const void* w, int64_t ldw,
                                                                 int dtype, int w_rows, int64_t n, int64_t width,
                                                                 int64_t vocab, int backward_dx, int backward_dw) {
  Head h = {x, w, ldx, ldw, n, width, vocab, dtype, w_rows != 0};
  return plan("linear_cross_entropy", backward_dx || backward_dw, backward_dx, backward_dw, &h) ? 0 : h.bytes;
}

extern "C" int pratchya_linear_cross_entropy(const void* x, int64_t ldx, const void* w, int64_t ldw, int dtype, int w_rows,
                                             const int64_t* targets, int64_t n, int64_t width, int64_t vocab,
                                             float smoothing, float* loss, float* stats, void* workspace,
                                             int64_t workspace_bytes, hipStream_t stream) {
  const char* what = "linear_cross_entropy";
  Head h = {x, w, ldx, ldw, n, width, vocab, dtype, w_rows != 0};
  const int rc = plan(what, false, false, false, &h);
  if (rc) return rc;
  if (!(smoothing >= 0.0f && smoothing <= 1.0f))
    return pratchya_set_error(PRATCHYA_EINVAL, "%s: label smoothing of %g; expected 0 to 1", what, smoothing);
  if (n == 0) return pratchya_set_error(PRATCHYA_OK, "");
  if (!x || !w || !targets || !loss) return pratchya_set_error(PRATCHYA_EINVAL, "%s: null buffer", what);
  if (!workspace || workspace_bytes < h.bytes || reinterpret_cast<uintptr_t>(workspace) % 256)
    return pratchya_set_error(PRATCHYA_EINVAL, "%s: workspace of %lld bytes needed, 256-byte aligned", what,
                              (long long)h.bytes);
  return forward({h, static_cast<char*>(workspace), stream}, targets, smoothing, loss, stats);
}

extern "C" int pratchya_linear_cross_entropy_bwd(const void* x, int64_t ldx, const void* w, int64_t ldw, int dtype,
                                                 int w_rows, const int64_t* targets, const float* stats, const float* g,
                                                 int64_t n, int64_t width, int64_t vocab, float smoothing, void* dx,
                                                 void* dw, void* workspace, int64_t workspace_bytes,
                                                 hipStream_t stream) {
  const char* what = "linear_cross_entropy_bwd";
  Head h = {x, w, ldx, ldw, n, width, vocab, dtype, w_rows != 0};
  const int rc = plan(what, true, dx != nullptr, dw != nullptr, &h);
  if (rc) return rc;
  if (!(smoothing >= 0.0f && smoothing <= 1.0f))
    return pratchya_set_error(PRATCHYA_EINVAL, "%s: label smoothing of %g; expected 0 to 1", what, smoothing);
  if (!dx && !dw) return pratchya_set_error(PRATCHYA_OK, "");
  if (n == 0) {
    if (dw) {
      hipLaunchKernelGGL(k_head_zero, dim3(1024), dim3(256), 0, stream, static_cast<uint16_t*>(dw),
                         width * vocab * (dtype == PRATCHYA_DT_BF16 ? 1 : 2));
      return check_launch(what);
    }
    return pratchya_set_error(PRATCHYA_OK, "");
  }
  if (!x || !w || !targets || !stats || !g) return pratchya_set_error(PRATCHYA_EINVAL, "%s: null buffer", what);
  if (!workspace || workspace_bytes < h.bytes || reinterpret_cast<uintptr_t>(workspace) % 256)
    return pratchya_set_error(PRATCHYA_EINVAL, "%s: workspace of %lld bytes needed, 256-byte aligned", what,
                              (long long)h.bytes);
  const Call c = {h, static_cast<char*>(workspace), stream};
  return dtype == PRATCHYA_DT_BF16
             ? backward<uint16_t>(c, targets, smoothing, stats, g, static_cast<uint16_t*>(dx), static_cast<uint16_t*>(dw))
             : backward<float>(c, targets, smoothing, stats, g, static_cast<float*>(dx), static_cast<float*>(dw));
}
