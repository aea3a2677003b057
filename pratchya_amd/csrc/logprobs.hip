// Log probabilities of given tokens, entropy, the best alternatives and the
// logits' gradient, for gfx950.
//
// Per row of logits x: m = max x, s = sum e^(x - m), log p_v = (x_v - m) - log s,
//   entropy H = log s - (sum e^(x - m) (x - m)) / s,
//   dx_v = g ([v = token] - p_v) - h p_v (log p_v + H)   (g, h: the cotangents of log p_token and H).
// A logit of -inf is masked: p = 0, and it adds nothing to H or dx.  A row
// that is masked everywhere holds no distribution: its log probabilities are
// -inf, H and dx are 0.  A negative token stands for no token: log probability 0,
// no part in dx; a token beyond the vocabulary gives NaN.
// Alternatives are ranked by their logit (NaN above all numbers), equal ones by
// index; ranking keys hold both in 64 bits, so no two are equal.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "pratchya_fp8.h"
#include "row_device.h"

int pratchya_set_error(int code, const char* fmt, ...);

namespace {

constexpr int kMaxTop = 64;

int check_launch(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return pratchya_set_error(PRATCHYA_EHIP, "%s: launch failed: %s", what, hipGetErrorString(e));
  return pratchya_set_error(PRATCHYA_OK, "");
}

bool is_float_dtype(int d) { return d == PRATCHYA_DT_F32 || d == PRATCHYA_DT_BF16; }

// 32-bit rank of a logit: larger for larger values, equal for 0 and -0, the
// largest for every NaN.
__device__ __forceinline__ uint32_t rank_bits(float x) {
  const uint32_t u = f2u(x + 0.0f);
  if (is_nan_bits(u)) return 0xFFFFFFFEu;   // no key is ~0
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ uint64_t rank_key(float x, int64_t i) {
  return ((uint64_t)rank_bits(x) << 32) | (uint32_t)(0xFFFFFFFFu - (uint32_t)i);
}

template <int N>
__device__ __forceinline__ float block_max(float v, float* lds) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v = fmaxf(v, __shfl_xor(v, m, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = lds[0];
#pragma unroll
  for (int i = 1; i < N; ++i) s = fmaxf(s, lds[i]);
  return s;
}

__device__ __forceinline__ uint64_t umax64(uint64_t a, uint64_t b) { return a > b ? a : b; }

template <typename T>
__global__ __launch_bounds__(256) void k_logprobs(const T* __restrict__ x, int64_t ld,
                                                  const int64_t* __restrict__ tokens, int64_t vocab, int top,
                                                  float* __restrict__ logprobs, float* __restrict__ entropy,
                                                  float* __restrict__ stats, float* __restrict__ top_logprobs,
                                                  int64_t* __restrict__ top_tokens) {
  __shared__ float lds[4];
  __shared__ uint64_t best[4];
  const int64_t row = blockIdx.x;
  const T* xr = x + row * ld;
  float m = -__builtin_inff();
  for (int64_t i = threadIdx.x; i < vocab; i += 256) m = fmaxf(m, load_elem(xr + i));
  m = block_max<4>(m, lds);
  if (m == -__builtin_inff()) m = 0.0f;
  float s = 0.0f, t = 0.0f;
  for (int64_t i = threadIdx.x; i < vocab; i += 256) {
    const float d = load_elem(xr + i) - m, e = __expf(d);
    s += e;
    t += e > 0.0f ? e * d : 0.0f;
  }
  s = block_add<4>(s, lds);
  t = block_add<4>(t, lds);
  const float logs = s == 0.0f ? 0.0f : logf(s), h = s == 0.0f ? 0.0f : logs - t / s;
  if (threadIdx.x == 0) {
    const int64_t tok = tokens[row];
    float lp = 0.0f;
    if (tok >= vocab) lp = __builtin_nanf("");
    else if (tok >= 0) lp = (load_elem(xr + tok) - m) - logs;
    logprobs[row] = lp;
    if (entropy) entropy[row] = s != s ? s : h;
    if (stats) {
      stats[3 * row] = m;
      stats[3 * row + 1] = logs;
      stats[3 * row + 2] = h;
    }
  }
  // one alternative after the other: the largest key below the last one found
  uint64_t last = ~0ull;
  for (int k = 0; k < top; ++k) {
    uint64_t b = 0;
    for (int64_t i = threadIdx.x; i < vocab; i += 256) {
      const uint64_t key = rank_key(load_elem(xr + i), i);
      if (key < last) b = umax64(b, key);
    }
#pragma unroll
    for (int w = 32; w >= 1; w >>= 1) b = umax64(b, __shfl_xor((unsigned long long)b, w, 64));
    __syncthreads();
    if ((threadIdx.x & 63) == 0) best[threadIdx.x >> 6] = b;
    __syncthreads();
    last = umax64(umax64(best[0], best[1]), umax64(best[2], best[3]));
    if (threadIdx.x == 0) {
      const int64_t i = 0xFFFFFFFFu - (uint32_t)last;
      top_tokens[row * top + k] = i;
      top_logprobs[row * top + k] = (load_elem(xr + i) - m) - logs;
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void k_logprobs_bwd(const T* __restrict__ x, int64_t ld,
                                                      const int64_t* __restrict__ tokens,
                                                      const float* __restrict__ stats, const float* __restrict__ g,
                                                      const float* __restrict__ gh, int64_t vocab,
                                                      T* __restrict__ dx) {
  const int64_t row = blockIdx.x;
  const int64_t tok = tokens[row];
  const float m = stats[3 * row], logs = stats[3 * row + 1], H = stats[3 * row + 2];
  const float c = g && tok >= 0 ? g[row] : 0.0f, ch = gh ? gh[row] : 0.0f;
  for (int64_t i = threadIdx.x; i < vocab; i += 256) {
    const float lp = (load_elem(x + row * ld + i) - m) - logs, p = __expf(lp);
    float v = p == 0.0f ? 0.0f : -p * (c + ch * (lp + H));
    if (i == tok) v += c;
    store_elem(dx + row * vocab + i, v);
  }
}

int check_args(const char* what, int dtype, int64_t rows, int64_t vocab) {
  if (!is_float_dtype(dtype)) return pratchya_set_error(PRATCHYA_EINVAL, "%s: unsupported dtype %d", what, dtype);
  if (rows < 0 || vocab < 1 || vocab > 0x7FFFFFFF)
    return pratchya_set_error(PRATCHYA_EINVAL, "%s: %lld rows of %lld logits", what, (long long)rows,
                              (long long)vocab);
  if (rows > 0x7FFFFFFF) return pratchya_set_error(PRATCHYA_EUNSUPPORTED, "%s: more than 2^31 rows", what);
  return PRATCHYA_OK;
}

}  // namespace

extern "C" int pratchya_token_logprobs(const void* logits, int64_t ld, int dtype, const int64_t* tokens, int64_t rows,
                                       int64_t vocab, int top, float* logprobs, float* entropy, float* stats,
                                       float* top_logprobs, int64_t* top_tokens, hipStream_t stream) {
  const int rc = check_args("token_logprobs", dtype, rows, vocab);
  if (rc) return rc;
  if (top < 0 || top > kMaxTop || top > vocab)
    return pratchya_set_error(PRATCHYA_EINVAL, "token_logprobs: %d alternatives of %lld (0 to %d)", top,
                              (long long)vocab, kMaxTop);
  if (rows == 0) return pratchya_set_error(PRATCHYA_OK, "");
  if (!logits || !tokens || !logprobs || (top && (!top_logprobs || !top_tokens)))
    return pratchya_set_error(PRATCHYA_EINVAL, "token_logprobs: null buffer");
  if (dtype == PRATCHYA_DT_BF16)
    hipLaunchKernelGGL((k_logprobs<uint16_t>), dim3((unsigned)rows), dim3(256), 0, stream,
                       static_cast<const uint16_t*>(logits), ld, tokens, vocab, top, logprobs, entropy, stats,
                       top_logprobs, top_tokens);
  else
    hipLaunchKernelGGL((k_logprobs<float>), dim3((unsigned)rows), dim3(256), 0, stream,
                       static_cast<const float*>(logits), ld, tokens, vocab, top, logprobs, entropy, stats,
                       top_logprobs, top_tokens);
  return check_launch("token_logprobs");
}

extern "C" int pratchya_token_logprobs_bwd(const void* logits, int64_t ld, int dtype, const int64_t* tokens,
                                           const float* stats, const float* g_logprobs, const float* g_entropy,
                                           int64_t rows, int64_t vocab, void* d_logits, hipStream_t stream) {
  const int rc = check_args("token_logprobs_bwd", dtype, rows, vocab);
  if (rc) return rc;
  if (rows == 0) return pratchya_set_error(PRATCHYA_OK, "");
  if (!logits || !tokens || !stats || !d_logits)
    return pratchya_set_error(PRATCHYA_EINVAL, "token_logprobs_bwd: null buffer");
  if (dtype == PRATCHYA_DT_BF16)
    hipLaunchKernelGGL((k_logprobs_bwd<uint16_t>), dim3((unsigned)rows), dim3(256), 0, stream,
                       static_cast<const uint16_t*>(logits), ld, tokens, stats, g_logprobs, g_entropy, vocab,
                       static_cast<uint16_t*>(d_logits));
  else
    hipLaunchKernelGGL((k_logprobs_bwd<float>), dim3((unsigned)rows), dim3(256), 0, stream,
                       static_cast<const float*>(logits), ld, tokens, stats, g_logprobs, g_entropy, vocab,
                       static_cast<float*>(d_logits));
  return check_launch("token_logprobs_bwd");
}
