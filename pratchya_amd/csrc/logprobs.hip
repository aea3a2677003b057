// Log probabilities of given tokens, entropy, the best alternatives and the
// logits' gradient, for gfx950.
//
// Per row of logits x: m = max x, s = sum e^(x - m), log p_v = (x_v - m) - log s,
//   entropy H = log s - (sum e^(x - m) (x - m)) / s,
//   dx_v = g ([v = token] - p_v) - h p_v (log p_v + H)   (g, h: the cotangents of log p_token and H).
// A logit of -inf is masked: p = 0, and it adds nothing to H or dx.  A row that is
// masked everywhere holds no distribution: its log probabilities are -inf, H and
// every p in dx are 0.  A negative token stands for no token: log probability 0,
// without a gradient; a token beyond the vocabulary gives NaN (x_token is a NaN that
// no logit holds, so dx is the formula's without its first term, and 0 for g = 0).
// Alternatives are ranked by their logit (NaN above all numbers), equal ones by
// index; ranking keys hold both in 64 bits, so no two are equal.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "pratchya_fp8.h"
#include "row_device.h"
#include "row_host.h"

namespace {

constexpr int kMaxTop = 64;
constexpr float kLowest = -3.4028234663852886e38f;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.69314718055994531f;

// 32-bit rank of a logit: larger for larger values, equal for 0 and -0, the
// largest for every NaN.
__device__ __forceinline__ uint32_t rank_bits(float x) {
  const uint32_t u = f2u(x + 0.0f);
  const uint32_t r = u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
  return x != x ? 0xFFFFFFFEu : r;          // no key is ~0
}
__device__ __forceinline__ uint64_t rank_key(float x, int64_t i) {
  return ((uint64_t)rank_bits(x) << 32) | (uint32_t)(0xFFFFFFFFu - (uint32_t)i);
}
__device__ __forceinline__ int64_t key_index(uint64_t key) { return 0xFFFFFFFFu - (uint32_t)key; }

__device__ __forceinline__ uint64_t umax64(uint64_t a, uint64_t b) { return a > b ? a : b; }
__device__ __forceinline__ uint64_t shfl_xor_u64(uint64_t v, int m) {
  return (uint64_t)__shfl_xor((unsigned long long)v, m, 64);
}

// A thread's running sums over the logits it has seen, relative to the largest, m:
// s = sum 2^((x - m) log2 e), t = sum of the same times (x - m) log2 e.  m moves
// before a larger logit is added, once for several vectors, so the largest one's term
// is 1 and a row's sum 1 or more: no log probability comes out above 0, no entropy
// below, and near 0 they keep a sum's digits.
template <bool ENTROPY>
struct Running {
  float m = kLowest, s = 0.0f, t = 0.0f;

  __device__ __forceinline__ void move(float to) {
    // differences of infinities and lowest values count as lowest: their power is 0
    const float d = fmaxf((m - to) * kLog2e, kLowest), f = __builtin_amdgcn_exp2f(d);
    if constexpr (ENTROPY) t = f * (t + (f > 0.0f ? s * d : 0.0f));
    s *= f;
    m = to;
  }
  // NaN is passed over here; its term makes the sum NaN
  template <int N>
  __device__ __forceinline__ void raise(const float (&v)[N], float& c) const {
#pragma unroll
    for (int i = 0; i < N; ++i) c = fmaxf(c, v[i]);
  }
  template <int N>
  __device__ __forceinline__ void sum(const float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float d = (v[i] - m) * kLog2e, e = __builtin_amdgcn_exp2f(d);
      s += e;
      if constexpr (ENTROPY) t += e * fmaxf(d, kLowest);   // 0, not NaN, for a masked logit
    }
  }
  template <int N>
  __device__ __forceinline__ void add(const float (&v)[N]) {
    float c = m;
    raise(v, c);
    if (c > m) move(c);
    sum(v);
  }
};

// Maximum and sums over the WPR waves of a row, for every thread (lds: 3 * WPR floats).
template <int WPR, bool ENTROPY>
__device__ __forceinline__ void join_running(Running<ENTROPY>& r, float* lds) {
  float m = wave_max(r.m);
  if constexpr (WPR > 1) {
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WPR; ++w) m = fmaxf(m, lds[w]);
  }
  r.move(m);
  r.s = wave_add(r.s);
  if constexpr (ENTROPY) r.t = wave_add(r.t);
  if constexpr (WPR > 1) {
    if ((threadIdx.x & 63) == 0) {
      lds[WPR + (threadIdx.x >> 6)] = r.s;
      if constexpr (ENTROPY) lds[2 * WPR + (threadIdx.x >> 6)] = r.t;
    }
    __syncthreads();
    float s = 0.0f, t = 0.0f;
#pragma unroll
    for (int w = 0; w < WPR; ++w) {
      s += lds[WPR + w];
      if constexpr (ENTROPY) t += lds[2 * WPR + w];
    }
    r.s = s;
    r.t = t;
  }
}

// log s and H of joined sums; a row without any unmasked logit has s = 0.
template <bool ENTROPY>
__device__ __forceinline__ void finish(Running<ENTROPY>& r, float& logs, float& h) {
  logs = r.s == 0.0f ? 0.0f : logf(r.s);
  h = r.s == 0.0f ? 0.0f : logs - (r.t / r.s) * kLn2;
  if (r.s == 0.0f) r.m = 0.0f;
}

__device__ __forceinline__ float token_logprob(float x, float m, float logs) { return (x - m) - logs; }

// Row results from joined sums: for one thread.
__device__ __forceinline__ void store_row(float x_token, int64_t tok, int64_t vocab, int64_t row, float m, float logs,
                                          float h, float* logprobs, float* entropy, float* stats) {
  logprobs[row] = tok < 0 ? 0.0f : tok < vocab ? token_logprob(x_token, m, logs) : __builtin_nanf("");
  if (entropy) entropy[row] = h;
  if (stats) {
    stats[3 * row] = m;
    stats[3 * row + 1] = logs;
    stats[3 * row + 2] = h;
  }
}

// Vectors of one thread in flight: 32 elements, in the backward pass 16 (1000 x
// 8193 f32 15.5 -> 11.3 us, 8192 x 65536 bf16 356 -> 347 us against 32).
template <typename T>
constexpr int kUnroll = 32 / kN<T>;
template <typename T>
constexpr int kBwdUnroll = 16 / kN<T>;

// One row per WPR waves, 4 / WPR rows (at least one) per workgroup: one pass, bound
// by HBM where rows fill the device (8192 x 65536 bf16 167 us, 1.07 GB at 6.4 TB/s, with
// entropies 177 to 213 from run to run and 165 at best; the exponential's quarter rate and
// six operations more a logit are some two thirds of that time), by one compute unit's
// loads for few rows (one row of 131072 in 10 us, whatever the other compute units do),
// which the 16 waves of a row are for.
template <typename T, int WPR, bool ENTROPY, bool NT>
__global__ __launch_bounds__(WPR < 4 ? 256 : WPR * 64) void k_logprobs(
    const T* __restrict__ x, int64_t ld, const int64_t* __restrict__ tokens, int64_t rows, int64_t vocab,
    float* __restrict__ logprobs, float* __restrict__ entropy, float* __restrict__ stats) {
  constexpr int THREADS = WPR * 64, ROWS = WPR < 4 ? 4 / WPR : 1;
  __shared__ float lds[3 * WPR];
  const int tid = threadIdx.x % THREADS;
  const int64_t row = (int64_t)blockIdx.x * ROWS + threadIdx.x / THREADS;
  if (ROWS > 1 && row >= rows) return;      // whole waves; a row of one wave meets no barrier
  const T* xr = x + row * ld;
  constexpr int N = kN<T>, U = kUnroll<T>;
  const int64_t vecs = vocab / N;
  Running<ENTROPY> r;
  int64_t i = tid;
  for (; i + (U - 1) * THREADS < vecs; i += U * THREADS) {
    u32x4_t raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = load_raw<NT>(xr + (i + u * THREADS) * N);
    float v[N], c = r.m;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      widen(raw[u], v);
      r.raise(v, c);
    }
    if (c > r.m) r.move(c);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      widen(raw[u], v);
      r.sum(v);
    }
  }
  for (; i < vecs; i += THREADS) {
    float v[N];
    widen(load_raw(xr + i * N), v);
    r.add(v);
  }
  if (i == vecs && vocab % N) {
    float v[N];
    load_some(xr + vecs * N, vocab - vecs * N, -__builtin_inff(), v);
    r.add(v);
  }
  join_running<WPR>(r, lds);
  float logs, h;
  finish(r, logs, h);
  if (tid == 0) {
    const int64_t tok = tokens[row];
    store_row(tok >= 0 && tok < vocab ? load_elem(xr + tok) : 0.0f, tok, vocab, row, r.m, logs, h, logprobs, entropy,
              stats);
  }
}

// Alternatives.  A row is cut into parts of up to kBlock logits (longer ones where
// that would be more than kParts), a workgroup each, because one compute unit
// alone would take longer over a row than all parts and the join together; a part
// stays in registers, so its logits are read once for the sums and the selection.
// Bound by the selection's instructions and barriers: 20 of one row of 65536 bf16
// 7 us and 5 us for the join, 5 of 256 rows of 32768 f32 14 and 5 us (34 instructions a
// logit), 20 of 512 rows of 131072 bf16 79 us together (1.7 TB/s).
constexpr int kPartThreads = 256, kPartElems = 16, kBlock = kPartThreads * kPartElems, kParts = 64;
constexpr int kKeys = kPartElems + 1;                   // keys of a thread: a block's logits and one kept key

// LDS of a selection among up to kKeys keys per thread.  kCandidates is what
// leaves room for as many workgroups in a compute unit as its registers hold,
// seven (with room for every key four fit: 512 rows of 131072 bf16 117 -> 90 us).
constexpr int kCandidates = 1024;
struct Selection {
  uint64_t cand[kCandidates];
  uint64_t seen[kPartThreads];
  uint32_t above[kPartThreads / 64][64];
  uint64_t bound;
  int found;
};

// The `top` largest of all threads' keys (0: no key) in falling order into
// out[0 .. top), padded with 0, for the whole workgroup.  The top-th largest of
// the maxima of 64 or 128 groups (threads of equal lane, and parity of the wave)
// is a bound that `top` keys reach, if there are so many; the keys that do are
// ranked by counting: some 24 for 20 alternatives, 90 for 64.  A lane's keys lie a
// vector apart from its neighbours', so rows of equal logits leave up to 8 top
// candidates, as rising or falling ones do.  Where there are more than
// kCandidates, the largest key is taken `top` times.  out may hold keys of this
// selection: they are in registers.
constexpr int kFewTop = 32;     // alternatives up to which 64 groups do
__device__ __forceinline__ void select_top(const uint64_t (&keys)[kKeys], int top, Selection& sel, uint64_t* out) {
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  uint64_t best = 0;
#pragma unroll
  for (int i = 0; i < kKeys; ++i) best = umax64(best, keys[i]);
  sel.seen[tid] = best;
  if (tid == 0) {
    sel.found = 0;
    sel.bound = 1;       // where fewer than `top` groups have a key, every key is collected
  }
  __syncthreads();
  // every wave holds all groups, two per lane, and counts how many of a quarter of
  // the groups are larger than each
  const bool few = top <= kFewTop;
  uint64_t k0 = umax64(sel.seen[lane], sel.seen[128 + lane]), k1 = umax64(sel.seen[64 + lane], sel.seen[192 + lane]);
  if (few) k0 = umax64(k0, k1);
  uint32_t above0 = 0, above1 = 0;
#pragma unroll
  for (int g = 0; g < 16; ++g) {
    const int from = wave * 16 + g;
    const uint64_t key = (uint64_t)readlane_u32((uint32_t)(k0 >> 32), from) << 32 | readlane_u32((uint32_t)k0, from);
    above0 += key > k0;
    if (!few) above1 += key > k1;
  }
  if (!few) {
#pragma unroll
    for (int g = 0; g < 16; ++g) {
      const int from = wave * 16 + g;
      const uint64_t key = (uint64_t)readlane_u32((uint32_t)(k1 >> 32), from) << 32 | readlane_u32((uint32_t)k1, from);
      above0 += key > k0;
      above1 += key > k1;
    }
  }
  sel.above[wave][lane] = above0 | above1 << 16;
  __syncthreads();
  if (tid < 64) {
    const uint32_t n = sel.above[0][lane] + sel.above[1][lane] + sel.above[2][lane] + sel.above[3][lane];
    if (k0 != 0 && (int)(n & 0xFFFFu) == top - 1) sel.bound = k0;
    if (!few && k1 != 0 && (int)(n >> 16) == top - 1) sel.bound = k1;
  }
  __syncthreads();
  const uint64_t bound = sel.bound;
  if (best >= bound) {
    int mine = 0;
#pragma unroll
    for (int i = 0; i < kKeys; ++i) mine += keys[i] >= bound;
    int at = atomicAdd(&sel.found, mine);
#pragma unroll
    for (int i = 0; i < kKeys; ++i)
      if (keys[i] >= bound) {
        if (at < kCandidates) sel.cand[at] = keys[i];
        ++at;
      }
  }
  __syncthreads();
  const int n = sel.found;
  if (n <= kCandidates) {
    if (tid >= n && tid < top) out[tid] = 0;
    for (int c = tid; c < n; c += kPartThreads) {
      const uint64_t own = sel.cand[c];
      int above = 0;
#pragma unroll 8
      for (int o = 0; o < n; ++o) above += sel.cand[o] > own;
      if (above < top) out[above] = own;
    }
  } else {
    uint64_t last = ~0ull;
    for (int k = 0; k < top; ++k) {
      uint64_t b = 0;
#pragma unroll
      for (int i = 0; i < kKeys; ++i)
        if (keys[i] < last) b = umax64(b, keys[i]);
#pragma unroll
      for (int w = 32; w >= 1; w >>= 1) b = umax64(b, shfl_xor_u64(b, w));
      if (lane == 0) sel.seen[wave] = b;
      __syncthreads();
      last = umax64(umax64(sel.seen[0], sel.seen[1]), umax64(sel.seen[2], sel.seen[3]));
      if (tid == 0) out[k] = last;
      __syncthreads();
    }
  }
  __syncthreads();
}

struct Out {
  float* logprobs;
  float* entropy;
  float* stats;
  float* top_logprobs;
  int64_t* top_tokens;
};

// One part of a row: its sums and its `top` largest keys, into sums
// [rows][parts][3] and kept [rows][parts][top], or for a row of one part the
// results themselves.
template <typename T, bool ENTROPY>
__global__ __launch_bounds__(kPartThreads, 7) void k_logprobs_part(const T* __restrict__ x, int64_t ld,
                                                                const int64_t* __restrict__ tokens, int64_t vocab,
                                                                int top, int parts, int64_t part_len,
                                                                float* __restrict__ sums, uint64_t* __restrict__ kept,
                                                                Out o) {
  __shared__ float lds[3 * 4];
  __shared__ Selection sel;
  __shared__ uint64_t list[kMaxTop];
  const int tid = threadIdx.x;
  const int64_t row = blockIdx.x / (unsigned)parts;
  const int part = (int)(blockIdx.x - (unsigned)row * (unsigned)parts);
  const T* xr = x + row * ld;
  const int64_t from = part * part_len, to = from + part_len < vocab ? from + part_len : vocab;
  Running<ENTROPY> r;
  if (tid < kMaxTop) list[tid] = 0;
  __syncthreads();
  constexpr int N = kN<T>, VECS = kPartElems / N;
  for (int64_t base = from; base < to; base += kBlock) {
    float v[VECS][N];
#pragma unroll
    for (int u = 0; u < VECS; ++u) {
      const int64_t at = base + (u * kPartThreads + tid) * N;
      if (at + N <= to) widen(load_raw(xr + at), v[u]);
      else load_some(xr + at, to - at, -__builtin_inff(), v[u]);
    }
    // what lies beyond the part reads as masked
    float c = r.m;
#pragma unroll
    for (int u = 0; u < VECS; ++u) r.raise(v[u], c);
    if (c > r.m) r.move(c);
#pragma unroll
    for (int u = 0; u < VECS; ++u)
      if (base + (u * kPartThreads + tid) * N < to) r.sum(v[u]);
    uint64_t keys[kKeys];
#pragma unroll
    for (int u = 0; u < VECS; ++u) {
      const int64_t at = base + (u * kPartThreads + tid) * N;
#pragma unroll
      for (int j = 0; j < N; ++j) keys[u * N + j] = rank_key(v[u][j], at + j);
      if (at + N > to) {
#pragma unroll
        for (int j = 0; j < N; ++j)
          if (at + j >= to) keys[u * N + j] = 0;
      }
    }
    keys[kKeys - 1] = tid < top ? list[tid] : 0;
    select_top(keys, top, sel, list);
  }
  join_running<4>(r, lds);
  if (parts > 1) {
    const int64_t at = row * parts + part;
    if (tid < top) kept[at * top + tid] = list[tid];
    if (tid < 3) sums[at * 3 + tid] = tid == 0 ? r.m : tid == 1 ? r.s : r.t;
    return;
  }
  float logs, h;
  finish(r, logs, h);
  if (tid == 0) {
    const int64_t tok = tokens[row];
    store_row(tok >= 0 && tok < vocab ? load_elem(xr + tok) : 0.0f, tok, vocab, row, r.m, logs, h, o.logprobs,
              o.entropy, o.stats);
  }
  if (tid < top) {
    const int64_t i = key_index(list[tid]);
    o.top_tokens[row * top + tid] = i;
    o.top_logprobs[row * top + tid] = token_logprob(load_elem(xr + i), r.m, logs);
  }
}

// The parts of a row (at most kParts) together.
template <typename T, bool ENTROPY>
__global__ __launch_bounds__(kPartThreads) void k_logprobs_join(const T* __restrict__ x, int64_t ld,
                                                                const int64_t* __restrict__ tokens, int64_t vocab,
                                                                int top, int parts, const float* __restrict__ sums,
                                                                const uint64_t* __restrict__ kept, Out o) {
  __shared__ Selection sel;
  __shared__ uint64_t list[kMaxTop];
  static_assert(kParts * kMaxTop <= kPartThreads * kKeys, "a thread's keys hold every part's");
  const int tid = threadIdx.x, lane = tid & 63;
  const int64_t row = blockIdx.x;
  const T* xr = x + row * ld;
  uint64_t keys[kKeys];
#pragma unroll
  for (int i = 0; i < kKeys; ++i) {
    const int at = i * kPartThreads + tid;
    keys[i] = at < parts * top ? kept[row * parts * top + at] : 0;
  }
  // every wave joins the sums: a part per lane
  Running<ENTROPY> r;
  if (lane < parts) {
    const float* p = sums + (row * parts + lane) * 3;
    r.m = p[0];
    r.s = p[1];
    r.t = p[2];
  }
  join_running<1>(r, nullptr);
  float logs, h;
  finish(r, logs, h);
  if (tid == 0) {
    const int64_t tok = tokens[row];
    store_row(tok >= 0 && tok < vocab ? load_elem(xr + tok) : 0.0f, tok, vocab, row, r.m, logs, h, o.logprobs,
              o.entropy, o.stats);
  }
  select_top(keys, top, sel, list);
  if (tid < top) {
    const int64_t i = key_index(list[tid]);
    o.top_tokens[row * top + tid] = i;
    o.top_logprobs[row * top + tid] = token_logprob(load_elem(xr + i), r.m, logs);
  }
}

// dx of 16 TPR logits of a row per TPR threads: elementwise, one
// read and one write of each logit, bound by HBM: 8192 x 65536 bf16 347 to 367 us (2.15 GB,
// 5.9 to 6.2 TB/s), 1000 x 50021 f32 61 us (6.6 TB/s).
template <typename T, int TPR, bool NT>
__global__ __launch_bounds__(256) void k_logprobs_bwd(const T* __restrict__ x, int64_t ld,
                                                      const int64_t* __restrict__ tokens,
                                                      const float* __restrict__ stats, const float* __restrict__ g,
                                                      const float* __restrict__ gh, int64_t rows, int64_t vocab,
                                                      unsigned pieces, T* __restrict__ dx) {
  constexpr int N = kN<T>, U = kBwdUnroll<T>;
  const int tid = threadIdx.x % TPR;
  // several rows per workgroup are rows of one piece
  const int64_t row = TPR < 256 ? (int64_t)blockIdx.x * (256 / TPR) + threadIdx.x / TPR : blockIdx.x / pieces;
  const int64_t first = TPR < 256 ? tid : (int64_t)(blockIdx.x - (unsigned)row * pieces) * (TPR * U) + tid;
  if (row >= rows) return;
  const int64_t tok = tokens[row];
  const float m = stats[3 * row], logs = stats[3 * row + 1];
  const float c = g && tok >= 0 ? g[row] : 0.0f, ch = gh ? gh[row] : 0.0f, H = stats[3 * row + 2];
  const T* xr = x + row * ld;
  T* dr = dx + row * vocab;
  auto grad = [&](float (&v)[N], int64_t at) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float lp = (v[i] - m) - logs, p = __builtin_amdgcn_exp2f(lp * kLog2e);
      v[i] = -p * (c + ch * (fmaxf(lp, -1000.0f) + H));   // a masked logit: p = 0 times a finite number
    }
    if ((uint64_t)(tok - at) < (uint64_t)N) {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (at + i == tok) v[i] += c;
    }
  };
  // whole pieces without a test per vector: its branches between the loads took
  // 1000 x 50021 f32 from 82 to 122 us
  if ((first - tid + TPR * U) * N <= vocab) {
    u32x4_t raw[U];
#pragma unroll
    for (int u = 0; u < U; ++u) raw[u] = load_raw<NT>(xr + (first + u * TPR) * N);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float v[N];
      widen(raw[u], v);
      grad(v, (first + u * TPR) * N);
      store_vec<NT>(dr + (first + u * TPR) * N, v);
    }
    return;
  }
  for (int u = 0; u < U; ++u) {
    const int64_t at = (first + u * TPR) * N, left = vocab - at;
    if (left <= 0) break;
    float v[N];
    if (left >= N) widen(load_raw(xr + at), v);
    else load_some(xr + at, left, 0.0f, v);
    grad(v, at);
    if (left >= N) store_vec(dr + at, v);
    else store_some(dr + at, left, v);
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

// Logits of a row that one wave takes, four rows a workgroup.
constexpr int64_t kOneWave = 2048;

// Accesses past the caches.  Forward, for logits that the last-level cache (256 MB)
// cannot hold: 8192 x 65536 bf16 188 -> 167 us, but 1000 x 50021 f32, 200 MB, 37.6 ->
// 40.2 us.  Backward, for more than the L2 caches hold: a gradient left in the
// last-level cache is written back while the next pass's logits are read; both
// passes over 1000 x 50021 f32 one after the other 119 -> 97 us.
constexpr int64_t kFwdStream = (int64_t)256 << 20, kBwdStream = (int64_t)32 << 20;

// How a row with alternatives is cut.
struct Cut {
  int parts;
  int64_t len;
};
Cut cut_row(int64_t vocab) {
  const int64_t blocks = (vocab + kBlock - 1) / kBlock, per = (blocks + kParts - 1) / kParts;
  return {(int)((blocks + per - 1) / per), per * kBlock};
}
// The keys of all rows' parts, then their sums.
int64_t keys_bytes(int64_t rows, int parts, int top) { return rows * parts * top * (int64_t)sizeof(uint64_t); }

template <typename T, bool ENTROPY>
int launch(const void* logits, int64_t ld, const int64_t* tokens, int64_t rows, int64_t vocab, int top, Out o,
           void* workspace, hipStream_t stream) {
  const T* x = static_cast<const T*>(logits);
  if (top) {
    const Cut cut = cut_row(vocab);
    if (!fits_launch(rows * cut.parts, kPartThreads))
      return pratchya_set_error(PRATCHYA_EUNSUPPORTED, "token_logprobs: more parts of rows than a launch has threads for (2^24)");
    uint64_t* kept = static_cast<uint64_t*>(workspace);
    float* sums = reinterpret_cast<float*>(static_cast<char*>(workspace) + keys_bytes(rows, cut.parts, top));
    hipLaunchKernelGGL((k_logprobs_part<T, ENTROPY>), dim3((unsigned)(rows * cut.parts)), dim3(kPartThreads), 0, stream,
                       x, ld, tokens, vocab, top, cut.parts, cut.len, sums, kept, o);
    if (cut.parts > 1)
      hipLaunchKernelGGL((k_logprobs_join<T, ENTROPY>), dim3((unsigned)rows), dim3(kPartThreads), 0, stream, x, ld,
                         tokens, vocab, top, cut.parts, sums, kept, o);
    return check_launch("token_logprobs");
  }
  const int rows_per = vocab <= kOneWave ? 4 : 1;
  const int64_t groups = (rows + rows_per - 1) / rows_per;
  if (!fits_launch(groups, 256))
    return pratchya_set_error(PRATCHYA_EUNSUPPORTED, "token_logprobs: more rows than a launch has threads for (2^%d)",
                              rows_per == 4 ? 26 : 24);
#define PRATCHYA_LP(WPR, NT)                                                                                          \
  hipLaunchKernelGGL((k_logprobs<T, WPR, ENTROPY, NT>), dim3((unsigned)groups),                                       \
                     dim3(WPR < 4 ? 256 : WPR * 64), 0, stream, x, ld, tokens, rows, vocab, o.logprobs, o.entropy,    \
                     o.stats)
  const bool nt = rows * vocab > kFwdStream / (int64_t)sizeof(T);
  if (vocab <= kOneWave) PRATCHYA_LP(1, false);
  else if (rows < 512) PRATCHYA_LP(16, false);
  else if (nt) PRATCHYA_LP(4, true);
  else PRATCHYA_LP(4, false);
#undef PRATCHYA_LP
  return check_launch("token_logprobs");
}

template <typename T>
int launch_bwd(const void* logits, int64_t ld, const int64_t* tokens, const float* stats, const float* g,
               const float* gh, int64_t rows, int64_t vocab, void* dx, hipStream_t stream) {
  constexpr int64_t per = kN<T> * kBwdUnroll<T>;          // logits of a thread
  const int tpr = vocab <= 64 * per ? 64 : 256;
  const int64_t pieces = (vocab + tpr * per - 1) / (tpr * per);
  const int64_t blocks = (rows * pieces + 256 / tpr - 1) / (256 / tpr);
  if (!fits_launch(blocks, 256))
    return pratchya_set_error(PRATCHYA_EUNSUPPORTED, "token_logprobs_bwd: more pieces of rows than a launch has threads for (2^24)");
#define PRATCHYA_LPB(TPR, NT)                                                                                         \
  hipLaunchKernelGGL((k_logprobs_bwd<T, TPR, NT>), dim3((unsigned)blocks), dim3(256), 0, stream,                      \
                     static_cast<const T*>(logits), ld, tokens, stats, g, gh, rows, vocab, (unsigned)pieces,          \
                     static_cast<T*>(dx))
  if (tpr == 64) PRATCHYA_LPB(64, false);
  else if (rows * vocab > kBwdStream / (int64_t)sizeof(T)) PRATCHYA_LPB(256, true);
  else PRATCHYA_LPB(256, false);
#undef PRATCHYA_LPB
  return check_launch("token_logprobs_bwd");
}

}  // namespace

extern "C" int64_t pratchya_token_logprobs_workspace_bytes(int64_t rows, int64_t vocab, int top) {
  if (rows < 1 || vocab < 1 || vocab > 0x7FFFFFFF || top < 1) return 0;
  const Cut cut = cut_row(vocab);
  return cut.parts > 1 ? keys_bytes(rows, cut.parts, top) + rows * cut.parts * 3 * (int64_t)sizeof(float) : 0;
}

extern "C" int pratchya_token_logprobs(const void* logits, int64_t ld, int dtype, const int64_t* tokens, int64_t rows,
                                       int64_t vocab, int top, float* logprobs, float* entropy, float* stats,
                                       float* top_logprobs, int64_t* top_tokens, void* workspace,
                                       int64_t workspace_bytes, hipStream_t stream) {
  const int rc = check_args("token_logprobs", dtype, rows, vocab);
  if (rc) return rc;
  if (top < 0 || top > kMaxTop || top > vocab)
    return pratchya_set_error(PRATCHYA_EINVAL, "token_logprobs: %d alternatives of %lld (0 to %d)", top,
                              (long long)vocab, kMaxTop);
  if (rows == 0) return pratchya_set_error(PRATCHYA_OK, "");
  if (!logits || !tokens || !logprobs || (top && (!top_logprobs || !top_tokens)))
    return pratchya_set_error(PRATCHYA_EINVAL, "token_logprobs: null buffer");
  const int64_t need = pratchya_token_logprobs_workspace_bytes(rows, vocab, top);
  if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 8))
    return pratchya_set_error(PRATCHYA_EINVAL, "token_logprobs: workspace of %lld bytes needed, 8-byte aligned",
                              (long long)need);
  const Out o = {logprobs, entropy, stats, top_logprobs, top_tokens};
#define PRATCHYA_LPT(T, E) launch<T, E>(logits, ld, tokens, rows, vocab, top, o, workspace, stream)
  if (dtype == PRATCHYA_DT_BF16) return entropy ? PRATCHYA_LPT(uint16_t, true) : PRATCHYA_LPT(uint16_t, false);
  return entropy ? PRATCHYA_LPT(float, true) : PRATCHYA_LPT(float, false);
#undef PRATCHYA_LPT
}

extern "C" int pratchya_token_logprobs_bwd(const void* logits, int64_t ld, int dtype, const int64_t* tokens,
                                           const float* stats, const float* g_logprobs, const float* g_entropy,
                                           int64_t rows, int64_t vocab, void* d_logits, hipStream_t stream) {
  const int rc = check_args("token_logprobs_bwd", dtype, rows, vocab);
  if (rc) return rc;
  if (rows == 0) return pratchya_set_error(PRATCHYA_OK, "");
  if (!logits || !tokens || !stats || !d_logits)
    return pratchya_set_error(PRATCHYA_EINVAL, "token_logprobs_bwd: null buffer");
  return dtype == PRATCHYA_DT_BF16
             ? launch_bwd<uint16_t>(logits, ld, tokens, stats, g_logprobs, g_entropy, rows, vocab, d_logits, stream)
             : launch_bwd<float>(logits, ld, tokens, stats, g_logprobs, g_entropy, rows, vocab, d_logits, stream);
}
