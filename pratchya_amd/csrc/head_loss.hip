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
// From 256 rows on, of more than 192 columns and words of a vocabulary, where x's planes lie
// within 2^31 bytes, logits are not written: the product's epilogue (head_product) takes each row's maximum and
// sum of 128 columns, which k_head_join joins, or turns its tile into dz (backward, from lse),
// of which a piece of the vocabulary is held at a time.  Elsewhere, and for the vocabulary's
// end that main_of leaves out, a piece's f32 logits are computed, read by k_head_rows or
// k_head_grad and overwritten by the next piece's.  In bf16 dz is rounded once, in units of the
// largest cotangent (k_head_unit): half a step of its own, 2^-9, stands in both gradients before
// their own rounding, and where dz is alike in all rows (probabilities far below a smoothed
// label's share) it stands in all alike.  In f32 every operand of a product is the sum of three
// exact bf16 planes and a product six products of planes.
//
// Bound: the MFMAs' rate on 256-row tiles, 1.1 PFLOP/s of four products (logits twice) where
// a large product alone reaches 1.27 and the library's 1.5: [8192, 4096] . [4096, 65536] in
// bf16, both passes, 16.0 ms (19.4 with the logits written and 128-row tiles); f32
// [1000, 1027] . [1027, 50021] 3.0 ms.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "gemm_head.h"
#include "pratchya_fp8.h"
#include "row_device.h"
#include "row_host.h"

namespace {

constexpr float kLowest = -3.4028234663852886e38f;

// --------------------------------------------------------------------------
// operands
// --------------------------------------------------------------------------
// Planes [P][rows_to][cols_to] of src [rows, cols] (rows ld elements apart, at any
// element's address), zeros around it: bf16 as it is (P 1) or an f32 value's three
// pieces (P 3), 8 columns a thread.  Rows whose target (targets, if not null) is negative
// are zeros: 0 times what padding holds would be NaN in the weight's gradient.
template <typename T, int P>
__global__ __launch_bounds__(256) void k_head_planes(const T* __restrict__ src, int64_t ld, int64_t rows, int64_t cols,
                                                     int64_t rows_to, int64_t cols_to,
                                                     const int64_t* __restrict__ targets, uint16_t* __restrict__ dst) {
  const int64_t per = cols_to / 8, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows_to * per) return;
  const int64_t r = i / per, c = (i - r * per) * 8;
  uint16_t* to = dst + r * cols_to + c;
  float v[8] = {};
  if (r < rows && c < cols && !(targets && targets[r] < 0)) {
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

// Statistics of kRowColumns of a row's logits, as the products' epilogue gives them of 128
// (gemm_head.h): one workgroup a row and part of a piece [rows, cols], whose column 0 is
// v0 of the vocabulary.  (128 rows of 32768 by a workgroup each took 22 us.)
constexpr int kRowThreads = 256, kRowColumns = 4096;

__global__ __launch_bounds__(kRowThreads) void k_head_rows(const float* __restrict__ z, int64_t ld, int64_t cols,
                                                           const int64_t* __restrict__ targets, int64_t v0,
                                                           float2* __restrict__ part, float* __restrict__ part_sum,
                                                           int64_t ld_part, float* __restrict__ target_value) {
  __shared__ float lds[kRowThreads / 64];
  const int64_t row = blockIdx.x, target = targets[row], tc = target < 0 ? -1 : target - v0;
  const int64_t lo = (int64_t)blockIdx.y * kRowColumns, hi = lo + kRowColumns < cols ? lo + kRowColumns : cols;
  const float* p = z + row * ld;
  float v[kRowColumns / kRowThreads / 4][4], m = kLowest, s = 0.0f, sum = 0.0f;
#pragma unroll
  for (int i = 0; i < kRowColumns / kRowThreads / 4; ++i) {
    const int64_t c = lo + (i * kRowThreads + threadIdx.x) * 4;
    if (c + 4 <= hi) widen(load_raw(p + c), v[i]);
    else load_some(p + c, hi - c, -__builtin_inff(), v[i]);
  }
#pragma unroll
  for (int i = 0; i < kRowColumns / kRowThreads / 4; ++i) {
    const int64_t c = lo + (i * kRowThreads + threadIdx.x) * 4;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if (c + k < hi) sum += v[i][k];
      if (c + k == tc && c + k < hi) {
        target_value[row] = v[i][k];
        v[i][k] = -__builtin_inff();
      }
      m = fmaxf(m, v[i][k]);
    }
  }
  m = wave_max(m);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = m;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < kRowThreads / 64; ++w) m = fmaxf(m, lds[w]);
#pragma unroll
  for (int i = 0; i < kRowColumns / kRowThreads / 4; ++i)
#pragma unroll
    for (int k = 0; k < 4; ++k) s += expf(v[i][k] - m);
  s = block_add<kRowThreads / 64>(s, lds);
  if (part_sum) sum = block_add<kRowThreads / 64>(sum, lds);
  if (threadIdx.x) return;
  const int64_t at = blockIdx.y * ld_part + row;
  part[at] = make_float2(m, s);
  if (part_sum) part_sum[at] = sum;
}

// The rows' losses from the statistics of their parts, [held][ld]: 64 rows a workgroup, a
// lane a row and a wave every kJoinWaves-th part.
constexpr int kJoinWaves = 16;

__global__ __launch_bounds__(64 * kJoinWaves) void k_head_join(const float2* __restrict__ part,
                                                               const float* __restrict__ part_sum, int64_t ld, int held,
                                                               const float* __restrict__ target_value, int64_t n,
                                                               const int64_t* __restrict__ targets, int64_t vocab,
                                                               float smooth, float* __restrict__ loss,
                                                               float* __restrict__ stats) {
  __shared__ float ms[kJoinWaves][64], ss[kJoinWaves][64], sums[kJoinWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t row = (int64_t)blockIdx.x * 64 + lane, r = row < n ? row : n - 1;
  Seen a;
  constexpr int AHEAD = 8;
  for (int i = wave; i < held; i += AHEAD * kJoinWaves) {
    float2 v[AHEAD];
    float t[AHEAD], m = a.m;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      const int at = i + k * kJoinWaves;
      v[k] = at < held ? part[at * ld + r] : make_float2(kLowest, 0.0f);
      t[k] = part_sum && at < held ? part_sum[at * ld + r] : 0.0f;
    }
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) m = fmaxf(m, v[k].x);
    a.s = a.s == 0.0f ? 0.0f : a.s * expf(fmaxf(a.m - m, kLowest));
    a.m = m;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
      a.s += v[k].y == 0.0f ? 0.0f : v[k].y * expf(fmaxf(v[k].x - m, kLowest));
      a.sum += t[k];
    }
  }
  ms[wave][lane] = a.m;
  ss[wave][lane] = a.s;
  sums[wave][lane] = a.sum;
  __syncthreads();
  if (wave || row >= n) return;
  for (int w = 1; w < kJoinWaves; ++w) a.m = fmaxf(a.m, ms[w][lane]);
  a.s = a.sum = 0.0f;
  for (int w = 0; w < kJoinWaves; ++w) {
    const float s = ss[w][lane];
    a.s += s == 0.0f ? 0.0f : s * expf(fmaxf(ms[w][lane] - a.m, kLowest));
    a.sum += sums[w][lane];
  }
  const int64_t target = targets[row];
  if (target >= 0 && target < vocab) a.zt = target_value[row];
  finish_row(a, target, vocab, smooth, loss + row, stats ? stats + 2 * row : nullptr);
}

// What gradients in bf16 are measured in: the largest |g| of rows with a target times their
// targets' part (head_part), and 1 / that |g|; 1 and 1 if none is a normal number.  With 1 / n for g, as a
// mean has it, and no unit, the rounding of -g itself, up to 2^-8, stood in all rows' gradients.
__global__ __launch_bounds__(1024) void k_head_unit(const float* __restrict__ g, const int64_t* __restrict__ targets,
                                                    int64_t n, float part, float* __restrict__ unit) {
  __shared__ float lds[16];
  float m = 0.0f;
  for (int64_t i = threadIdx.x; i < n; i += 1024) {
    const float v = __builtin_fabsf(g[i]);
    if (targets[i] >= 0 && v < 3e38f) m = fmaxf(m, v);
  }
  m = wave_max(m);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = m;
  __syncthreads();
  if (threadIdx.x) return;
  for (int w = 0; w < 16; ++w) m = fmaxf(m, lds[w]);
  const bool usual = m > 1e-30f && m < 1e30f;
  unit[0] = usual ? m * part : part;
  unit[1] = usual ? 1.0f / m : 1.0f;
}

// Zeros in the planes' rows [rows, rows_to), which the product of the gradients reads.
__global__ __launch_bounds__(256) void k_head_zero_rows(uint16_t* __restrict__ dst, int64_t plane, int64_t ld, int64_t rows,
                                                        int64_t rows_to) {
  const int64_t per = ld / 8, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (rows_to - rows) * per) return;
  *reinterpret_cast<u32x4_t*>(dst + blockIdx.y * plane + (rows + i / per) * ld + i % per * 8) = u32x4_t{};
}

// dz of a piece's logits as planes [P][rows_to][cols_to], rows ld_dst apart, zeros around
// [rows, cols].
template <int P>
__global__ __launch_bounds__(256) void k_head_grad(const float* __restrict__ z, int64_t ld, int64_t rows, int64_t cols,
                                                   int64_t rows_to, int64_t cols_to, const int64_t* __restrict__ targets,
                                                   int64_t v0, int64_t vocab, float smooth,
                                                   const float* __restrict__ stats, const float* __restrict__ g,
                                                   uint16_t* __restrict__ dst, int64_t ld_dst,
                                                   const float* __restrict__ unit, float part) {
  const int64_t per = cols_to / 8, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows_to * per) return;
  const int64_t r = i / per, c = (i - r * per) * 8;
  uint16_t* to = dst + r * ld_dst + c;
  float d[8] = {};
  if (r < rows && targets[r] >= 0) {
    const int64_t target = targets[r];
    const float m = stats[2 * r], logs = stats[2 * r + 1], gr = unit ? g[r] * unit[1] : g[r],
                even = smooth / (float)vocab / part, keep = (1.0f - smooth) / part, one = 1.0f / part;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v[4];
      widen(load_raw(z + r * ld + c + 4 * h), v);
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int64_t col = c + 4 * h + k;
        const float p = expf((v[k] - m) - logs) * one - even - (v0 + col == target ? keep : 0.0f);
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
    *reinterpret_cast<u32x4_t*>(to + q * rows_to * ld_dst) = narrow(o);
  }
}

// out [rows, cols] (contiguous, or ld_out apart) = src [slices][rows, cols], f32 ld_src
// apart, summed,
// plus the sums of the pieces before (sum, if add); not the last piece: into sum.
template <typename T>
__global__ __launch_bounds__(256) void k_head_out(const float* __restrict__ src, int64_t ld_src, int64_t rows,
                                                  int64_t cols, float* __restrict__ sum, int add, int last,
                                                  T* __restrict__ out, int64_t ld_out, int slices,
                                                  const float* __restrict__ unit) {
  const int64_t per = (cols + 3) / 4, i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= rows * per) return;
  const int64_t r = i / per, c = (i - r * per) * 4;
  float v[4];
  widen(load_raw(src + r * ld_src + c), v);
  for (int s = 1; s < slices; ++s) {
    float o[4];
    widen(load_raw(src + s * rows * ld_src + r * ld_src + c), o);
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] += o[k];
  }
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
  if (unit) {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] *= unit[0];
  }
  store_some(out + r * ld_out + c, cols - c < 4 ? cols - c : 4, v);
}

// --------------------------------------------------------------------------
// host
// --------------------------------------------------------------------------
int64_t up64(int64_t v) { return (v + 63) / 64 * 64; }
int64_t up128(int64_t v) { return (v + 127) / 128 * 128; }
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
  // rows of dz lie apart from each other's memory channels ([4096, 65536] . [65536, 2048]
  // 4183 us of a step without, 4117 with)
  int64_t pad() const { return fused ? 64 : 0; }
  bool fused;                    // logits on 256-row tiles, what follows them in the product's epilogue
  int64_t parts, ld_part;        // what statistics are taken of: of a row of a piece; from one to the next (rows)
  int64_t parts_of(int64_t cols) const {
    const int64_t main = fused ? main_of(cols) : 0, rest = main < cols ? cols - main : 0;
    return 2 * ((main + 255) / 256) + (rest + kRowColumns - 1) / kRowColumns;
  }
  // pieces before the last one are whole
  int64_t all_parts() const {
    const int64_t last = (V - 1) / piece;
    return last * parts + parts_of(V - last * piece);
  }
  // Columns of a piece's logits on the 256-row tiles: all (a multiple of 64 behind the
  // piece's end), or those of full rounds of tiles on the 256 compute units, where the last
  // round would be a third full or less and a tile has 48 steps of K or more; the others go the
  // way of few rows, in four launches more.  Loss alone of [1000, C] . [C, 50176], 784 tiles, and
  // [4096, C] . [C, 33792], 2112, in bf16, all on tiles and the end apart, us:
  //   C 1024   164 150   332 352      C 2048   272 248   582 604      C 4096   522 450   1115 1098
  // f32 [1000, 1024] . [1024, 50176], 96 steps, both passes 2926 and 2686.
  int64_t main_of(int64_t cols) const {
    const int64_t all = (cols + 63) / 64 * 64, tm = (n + 255) / 256, tn = (all + 255) / 256, full = tm * tn / 256;
    if (full < 1 || tm * tn % 256 == 0 || tm * tn % 256 > 85 || C64 / 64 * (P == 1 ? 1 : 6) < 48) return all;
    const int64_t main = full * 256 / tm * 256;
    return main >= 256 && main < all && (tn * 256 - main) / 256 * tm <= 85 ? main : all;
  }
  // Whether the 128-row tiles store the weight's gradient of a piece's columns themselves, at
  // a 16-byte aligned address; else it goes through f32 sums, of dw_cols columns at a time.
  // ([128, 4096] . [4096, 65536] in bf16, both passes: 653 us, all of it through f32 1014.)
  bool dw_plain(int64_t cols) const {
    const int64_t M = rows ? cols : C, N = rows ? C : cols, ld = rows ? C : V;
    return M > 32 && M % 8 == 0 && N % 8 == 0 && ld % (P == 1 ? 8 : 4) == 0;
  }
  int64_t dw_cols;
  // workspace
  int64_t part, part_sum, zt, unit;
  int64_t xp, wp, z, dzp, dx_sum, dx_tmp, dw_tmp, split, split_bytes, bytes;
};

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// Slices of K for which a product of [M, N] over `steps` goes to the 256-row tiles, 0 if it
// does not.  One workgroup a compute unit takes one tile of one slice after the other; where
// 3/10 of the last round are idle, the 128-row tiles, which take K in slices too, are as
// fast ([4096, 65536] . [65536, 2048] in bf16: 1186 us there, 128 tiles in two slices here
// 1117 and 17 to join them; f32 [1000, 50021] . [50021, 1027] 815 there, 700 here).
int on256(const Head& h, int64_t M, int64_t N, int64_t steps, int most) {
  if (!h.fused || M < 256 || N < 256) return 0;
  const int64_t tiles = ((M + 255) / 256) * ((N + 255) / 256);
  int best = 0;
  double best_use = 0.699;
  for (int s = 1; s <= most && (s == 1 || steps / s >= 16); ++s) {
    if (steps % s) continue;
    const int64_t units = tiles * s, rounds = (units + 255) / 256;
    const double use = (double)units / (double)(rounds * 256);
    if (use > best_use + 0.03) {
      best = s;
      best_use = use;
    }
  }
  return best;
}

// The gradient of x from a piece of Vp columns.
int dx256(const Head& h, int64_t Vp) { return on256(h, h.n, h.C64, (h.P == 1 ? 1 : 6) * (Vp / 64), 16); }
// The weight's gradient of a piece of Vp columns.
bool dw256(const Head& h, int64_t Vp) {
  return on256(h, h.rows ? Vp : h.C64, h.rows ? h.C64 : Vp, 1, 1) != 0;
}

// C [M, N] = A . B over K; a plane's rows lie lda / ldb apart, planes a_rows * lda: what both
// kinds of tiles take.
HeadProduct operands(const Head& h, const uint16_t* A, int64_t lda, int64_t a_rows, bool a_kmajor, const uint16_t* B, int64_t ldb,
                     int64_t b_rows, bool b_kmajor, int64_t M, int64_t N, int64_t K) {
  HeadProduct p{};
  p.a = A;
  p.b = B;
  p.lda = lda;
  p.ldb = ldb;
  p.a_plane = h.P == 1 ? 0 : a_rows * lda;
  p.b_plane = h.P == 1 ? 0 : b_rows * ldb;
  p.a_kmajor = a_kmajor;
  p.b_kmajor = b_kmajor;
  p.a_planes = h.P == 1 ? 0 : kPairsA;
  p.b_planes = h.P == 1 ? 0 : kPairsB;
  p.segs = h.P == 1 ? 1 : 6;
  p.splits = 1;
  p.planes = h.P;
  p.M = M;
  p.N = N;
  p.K = K;
  p.rows = M;
  p.cols = N;
  return p;
}

// The operands x and a piece of w, as they are or as planes.
struct Operands {
  const uint16_t *x, *w;
  int64_t ldx, ldw, x_rows, w_rows;
};

// How they lie, of a piece of Vp columns.
Operands layout_of(const Head& h, int64_t Vp) {
  return {nullptr, nullptr, h.x_direct ? h.ldx : h.C64, h.w_direct ? h.ldw : h.rows ? h.C64 : Vp, h.n64, h.rows ? Vp : h.C64};
}

// Whether the tiles take all products of a piece of Vp columns.
bool products_fit(const Head& h, bool bwd, bool want_dx, bool want_dw, int64_t Vp) {
  const Operands o = layout_of(h, Vp);
  const int64_t main = h.fused ? h.main_of(Vp) : 0, ldz = Vp + h.pad(), n64 = h.n64;
  auto logits = [&](int64_t N) { return operands(h, nullptr, o.ldx, o.x_rows, false, nullptr, o.ldw, o.w_rows, !h.rows, h.n, N, h.C64); };
  if (main && !head_product_fits(logits(main))) return false;
  if (main < Vp && !head_product128_fits(logits(Vp - main))) return false;
  if (bwd && want_dx) {
    const HeadProduct p = operands(h, nullptr, ldz, n64, false, nullptr, o.ldw, o.w_rows, h.rows, h.n, h.C64, Vp);
    if (!(dx256(h, Vp) ? head_product_fits(p) : head_product128_fits(p))) return false;
  }
  if (bwd && want_dw) {
    const HeadProduct p = h.rows ? operands(h, nullptr, ldz, n64, true, nullptr, o.ldx, o.x_rows, true, Vp, h.C64, n64)
                                 : operands(h, nullptr, o.ldx, o.x_rows, true, nullptr, ldz, n64, true, h.C64, Vp, n64);
    if (!(dw256(h, Vp) ? head_product_fits(p) : head_product128_fits(p))) return false;
  }
  return true;
}

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
  h->x_direct = bf && !(bwd && want_dw) && h->n % 64 == 0 && h->C % 64 == 0 && h->ldx % 8 == 0 && h->ldx >= h->C && aligned16(h->x) &&
                2 * (h->n + 128) * h->ldx <= kMaxOffset;
  h->w_direct = bf && h->C % 64 == 0 && h->V % 64 == 0 && h->ldw % 8 == 0 && h->ldw >= (h->rows ? h->C : h->V) &&
                aligned16(h->w) && (h->rows ? 2 * (1152 * (h->ldw + 1)) : 2 * (up128(h->C) + 1) * (h->ldw + 1) + 256) <= kMaxOffset;
  // on 256-row tiles, whose operands' offsets have 31 bits: x and w themselves, or copies as planes
  // where they are larger ([8192, 8192] . [8192, 131072] in bf16, both passes: 67 ms, 77 on the
  // 128-row tiles with w in place)
  const int64_t planes = 2 * h->P, segs = h->P == 1 ? 1 : 6, wide = h->n64 > h->C64 ? h->n64 : h->C64;
  h->fused = h->n >= 256 && h->C64 >= 256 && V64 >= 256 && planes * wide * 2560 <= INT32_MAX &&
             planes * h->n64 * h->C64 <= INT32_MAX;
  if (h->fused) {
    h->x_direct = h->x_direct && 2 * h->n * h->ldx <= INT32_MAX;
    h->w_direct = h->w_direct && 2 * (h->rows ? 2560 : h->C) * h->ldw <= INT32_MAX;
  }
  const int64_t unit = h->fused ? 256 : 64;
  // what of a piece is kept: f32 logits, or only the planes of their gradient; the planes
  // of its weight: 512 MB
  int64_t piece = !h->fused ? kPieceBytes / 4 / (h->n64 ? h->n64 : 64) : bwd ? 2 * kPieceBytes / planes / h->n64 : V64;
  auto bound = [&](int64_t by) { piece = by < piece ? by : piece; };
  if (!h->w_direct) bound(2 * kPieceBytes / planes / h->C64);
  if (!h->fused) bound(kMaxOffset / planes / (wide + 128));
  if (h->w_direct && h->rows) bound(h->fused ? INT32_MAX / 4 / h->ldw : kMaxOffset / 2 / (h->ldw + 1) - 256);
  if (piece < V64) piece = piece / unit * unit;
  if (piece < 1024) piece = 1024;
  // pieces of one size
  const int64_t pieces = (V64 + piece - 1) / piece;
  h->piece = ((V64 + pieces - 1) / pieces + unit - 1) / unit * unit;
  if (h->fused)
    while (h->piece < V64 && (V64 - 1) % h->piece + 1 < 256) h->piece += 256;      // the last one: a tile or more
  if (h->piece > V64) h->piece = V64;
  const int64_t rest = V64 - (V64 - 1) / h->piece * h->piece;      // the last piece
  if (h->n && !(products_fit(*h, bwd, want_dx, want_dw, h->piece) && products_fit(*h, bwd, want_dx, want_dw, rest)))
    return pratchya_set_error(PRATCHYA_EUNSUPPORTED, "%s: operands beyond 32-bit offsets", what);
  int64_t at = 0;
  auto take = [&](int64_t bytes) {
    const int64_t p = at;
    at += round256(bytes);
    return p;
  };
  h->xp = take(planes * h->n64 * h->C64);
  h->wp = take(h->w_direct ? 0 : planes * h->C64 * h->piece);
  h->parts = h->parts_of(h->piece);
  h->ld_part = h->n64;
  const int64_t parts = h->all_parts();
  if (parts > INT32_MAX) return pratchya_set_error(PRATCHYA_EUNSUPPORTED, "%s: too large", what);
  h->part = take(bwd ? 0 : 8 * parts * h->ld_part);
  h->part_sum = take(bwd ? 0 : 4 * parts * h->ld_part);
  h->zt = take(bwd ? 0 : 4 * h->n);
  h->unit = take(bwd ? 8 : 0);
  int64_t by_rows = h->piece;                                      // columns of f32 logits
  if (h->fused) {
    by_rows = 0;
    for (int64_t Vp : {h->piece, rest})
      if (Vp - h->main_of(Vp) > by_rows) by_rows = Vp - h->main_of(Vp);
  }
  h->z = take(4 * h->n * by_rows);
  const int64_t last = h->V - (h->V - 1) / h->piece * h->piece;
  const int64_t tmp = h->dw_plain(last) && (last == h->V || h->dw_plain(h->piece)) ? kPieceBytes / 8 : kPieceBytes;
  h->dw_cols = tmp / 4 / h->C64 / 64 * 64;
  if (h->dw_cols < 64) h->dw_cols = 64;
  if (h->dw_cols > h->piece) h->dw_cols = h->piece;
  h->split_bytes = 0;
  auto split = [&](int64_t M, int64_t N, int64_t K) {
    const int64_t b = pratchya_gemm_t128_workspace_bytes(M, N, segs * (K / 64), 1);
    if (b > h->split_bytes) h->split_bytes = b;
  };
  for (int64_t Vp : {h->piece, rest}) {
    const int64_t main = h->fused ? h->main_of(Vp) : 0;
    if (main < Vp) split(h->n, Vp - main, h->C64);
    if (bwd && want_dx && !dx256(*h, Vp)) split(h->n, h->C64, Vp);
    if (bwd && want_dw && !dw256(*h, Vp)) {
      split(h->rows ? Vp : h->C, h->rows ? h->C : Vp, h->n64);
      for (int64_t wide : {Vp < h->dw_cols ? Vp : h->dw_cols, Vp % h->dw_cols})
        if (wide) split(h->rows ? wide : h->C64, h->rows ? h->C64 : wide, h->n64);
    }
  }
  h->dzp = h->dx_sum = h->dx_tmp = h->dw_tmp = 0;
  if (bwd) {
    h->dzp = take(planes * h->n64 * (h->piece + h->pad()));
    if (want_dx) {
      int64_t slices = 0;
      for (int64_t Vp : {h->piece, rest}) {
        const int s = dx256(*h, Vp);
        const int64_t need = s == 1 ? 0 : s ? s : 1;
        if (need > slices) slices = need;
      }
      h->dx_tmp = take(4 * slices * h->n * h->C64);
      h->dx_sum = take(h->piece < h->V ? 4 * h->n * h->C64 : 0);
    }
    if (want_dw && !(dw256(*h, h->piece) && dw256(*h, rest))) h->dw_tmp = take(4 * h->C64 * h->dw_cols);
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
             const int64_t* targets, uint16_t* dst) const {
    const int64_t blocks = (rows_to * (cols_to / 8) + 255) / 256;
    if (!fits_launch(blocks, 256)) return pratchya_set_error(PRATCHYA_EUNSUPPORTED, "linear_cross_entropy: too large");
    if (h.P == 1)
      hipLaunchKernelGGL((k_head_planes<uint16_t, 1>), dim3((unsigned)blocks), dim3(256), 0, stream,
                         static_cast<const uint16_t*>(src), ld, rows, cols, rows_to, cols_to, targets, dst);
    else
      hipLaunchKernelGGL((k_head_planes<float, 3>), dim3((unsigned)blocks), dim3(256), 0, stream,
                         static_cast<const float*>(src), ld, rows, cols, rows_to, cols_to, targets, dst);
    return check_launch("linear_cross_entropy");
  }
  // On 128-row tiles, to C in dtype, in bf16 times *unit.
  int product(HeadProduct p, void* C, int64_t ldc, int dtype, const float* unit = nullptr) const {
    p.c = C;
    p.ldc = ldc;
    p.c_bf16 = dtype == PRATCHYA_DT_BF16;
    p.unit = unit;
    return head_product128(p, ws + h.split, h.split_bytes, stream);
  }
};

int operand_x(const Call& c, const int64_t* targets, Operands* o) {
  const Head& h = c.h;
  o->x_rows = h.n64;
  if (h.x_direct) {
    o->x = static_cast<const uint16_t*>(h.x);
    o->ldx = h.ldx;
    return PRATCHYA_OK;
  }
  o->x = c.planes_at(h.xp);
  o->ldx = h.C64;
  return c.planes(h.x, h.ldx, h.n, h.C, h.n64, h.C64, targets, c.planes_at(h.xp));
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
  return h.rows ? c.planes(src, h.ldw, cols, h.C, Vp, h.C64, nullptr, c.planes_at(h.wp))
                : c.planes(src, h.ldw, h.C, cols, h.C64, Vp, nullptr, c.planes_at(h.wp));
}

// A piece's logits from column `from` on into the workspace, [n, Vp - from].
int logits(const Call& c, const Operands& o, int64_t from, int64_t Vp) {
  const Head& h = c.h;
  return c.product(operands(c.h, o.x, o.ldx, o.x_rows, false, o.w + (h.rows ? from * o.ldw : from), o.ldw, o.w_rows, !h.rows, h.n,
                              Vp - from, h.C64), c.floats_at(h.z), Vp - from, PRATCHYA_DT_F32);
}

HeadProduct logits_product(const Call& c, const Operands& o, int64_t v0, int64_t cols, int64_t main,
                           const int64_t* targets, float smooth) {
  const Head& h = c.h;
  HeadProduct p = operands(c.h, o.x, o.ldx, o.x_rows, false, o.w, o.ldw, o.w_rows, !h.rows, h.n, main, h.C64);
  p.rows = h.n;
  p.cols = cols < main ? cols : main;
  p.targets = targets;
  p.v0 = v0;
  p.vocab = h.V;
  p.smooth = smooth;
  return p;
}

int forward(const Call& c, const int64_t* targets, float smooth, float* loss, float* stats) {
  const Head& h = c.h;
  Operands o;
  int rc = operand_x(c, nullptr, &o);
  for (int64_t v0 = 0; v0 < h.V && !rc; v0 += h.piece) {
    const int64_t cols = h.V - v0 < h.piece ? h.V - v0 : h.piece, Vp = up64(cols);
    if ((rc = operand_w(c, v0, cols, Vp, &o))) break;
    const int64_t at = v0 / h.piece * h.parts * h.ld_part;
    float2* part = reinterpret_cast<float2*>(c.ws + h.part) + at;
    float* part_sum = smooth != 0.0f ? c.floats_at(h.part_sum) + at : nullptr;
    const int64_t main = h.fused ? h.main_of(cols) : 0;
    if (main) {
      HeadProduct p = logits_product(c, o, v0, cols, main, targets, smooth);
      p.epilogue = kHeadRows;
      p.part = part;
      p.part_sum = part_sum;
      p.target_value = c.floats_at(h.zt);
      p.ld_part = h.ld_part;
      rc = head_product(p, c.stream);
    }
    if (!rc && main < cols && !(rc = logits(c, o, main, Vp))) {
      const int64_t skip = main / 128 * h.ld_part;
      hipLaunchKernelGGL(k_head_rows, dim3((unsigned)h.n, (unsigned)((cols - main + kRowColumns - 1) / kRowColumns)),
                         dim3(kRowThreads), 0, c.stream, c.floats_at(h.z), Vp - main, cols - main, targets, v0 + main,
                         part + skip, part_sum ? part_sum + skip : nullptr, h.ld_part, c.floats_at(h.zt));
      rc = check_launch("linear_cross_entropy");
    }
  }
  if (rc) return rc;
  hipLaunchKernelGGL(k_head_join, dim3((unsigned)((h.n + 63) / 64)), dim3(64 * kJoinWaves), 0, c.stream,
                     reinterpret_cast<const float2*>(c.ws + h.part), smooth != 0.0f ? c.floats_at(h.part_sum) : nullptr,
                     h.ld_part, (int)h.all_parts(), c.floats_at(h.zt), h.n, targets, h.V, smooth, loss, stats);
  return check_launch("linear_cross_entropy");
}

template <typename T>
int backward(const Call& c, const int64_t* targets, float smooth, const float* stats, const float* g, T* dx, T* dw) {
  const Head& h = c.h;
  const char* what = "linear_cross_entropy_bwd";
  constexpr int64_t chunk = 16 / sizeof(T);
  Operands o;
  int rc = operand_x(c, dw ? targets : nullptr, &o);
  float* unit = h.P == 1 ? c.floats_at(h.unit) : nullptr;
  if (unit && !rc) {
    hipLaunchKernelGGL(k_head_unit, dim3(1), dim3(1024), 0, c.stream, g, targets, h.n, head_part(smooth), unit);
    rc = check_launch(what);
  }
  for (int64_t v0 = 0; v0 < h.V && !rc; v0 += h.piece) {
    const int64_t cols = h.V - v0 < h.piece ? h.V - v0 : h.piece, Vp = up64(cols);
    if ((rc = operand_w(c, v0, cols, Vp, &o))) break;
    const int64_t ldz = Vp + h.pad();
    uint16_t* dz = c.planes_at(h.dzp);
    const int64_t main = h.fused ? h.main_of(cols) : 0;
    if (main) {
      HeadProduct p = logits_product(c, o, v0, cols, main, targets, smooth);
      p.epilogue = kHeadGrad;
      p.c = dz;
      p.ldc = ldz;
      p.plane_c = h.n64 * ldz;
      p.stats = stats;
      p.g = g;
      p.unit = unit;
      if ((rc = head_product(p, c.stream))) break;
      if (h.n64 > h.n) {
        hipLaunchKernelGGL(k_head_zero_rows, dim3((unsigned)(((h.n64 - h.n) * (ldz / 8) + 255) / 256), (unsigned)h.P), dim3(256),
                           0, c.stream, dz, p.plane_c, ldz, h.n, h.n64);
        if ((rc = check_launch(what))) break;
      }
    }
    if (main < cols) {
      if ((rc = logits(c, o, main, Vp))) break;
      const int64_t blocks = (h.n64 * ((Vp - main) / 8) + 255) / 256;
      if (!fits_launch(blocks, 256)) return pratchya_set_error(PRATCHYA_EUNSUPPORTED, "%s: too large", what);
      auto grad = h.P == 1 ? k_head_grad<1> : k_head_grad<3>;
      hipLaunchKernelGGL(grad, dim3((unsigned)blocks), dim3(256), 0, c.stream, c.floats_at(h.z), Vp - main, h.n, cols - main,
                         h.n64, Vp - main, targets, v0 + main, h.V, smooth, stats, g, dz + main, ldz, unit, unit ? head_part(smooth) : 1.0f);
      if ((rc = check_launch(what))) break;
    }
    const int slices = dx ? dx256(h, Vp) : 0;
    if (slices) {
      const bool first = v0 == 0, last = v0 + h.piece >= h.V;
      HeadProduct p = operands(c.h, dz, ldz, h.n64, false, o.w, o.ldw, o.w_rows, h.rows, h.n, h.C64, Vp);
      p.epilogue = kHeadStore;
      if (slices > 1) {
        p.splits = slices;
        p.c = c.floats_at(h.dx_tmp);
        p.ldc = h.C64;
        p.split_c = h.n * h.C64;
      } else {
        p.cols = last ? h.C : h.C64;
        p.c = last ? static_cast<void*>(dx) : c.floats_at(h.dx_sum);
        p.ldc = last ? h.C : h.C64;
        p.c_bf16 = last && h.P == 1;
        p.sums = first ? nullptr : c.floats_at(h.dx_sum);
        p.ld_sums = h.C64;
        p.unit = last ? unit : nullptr;
      }
      if ((rc = head_product(p, c.stream))) break;
      if (slices > 1) {
        hipLaunchKernelGGL((k_head_out<T>), dim3((unsigned)((h.n * ((h.C + 3) / 4) + 255) / 256)), dim3(256), 0, c.stream,
                           c.floats_at(h.dx_tmp), h.C64, h.n, h.C, c.floats_at(h.dx_sum), !first, last, dx, h.C, slices, unit);
        if ((rc = check_launch(what))) break;
      }
    } else if (dx) {
      float* tmp = c.floats_at(h.dx_tmp);
      rc = c.product(operands(c.h, dz, ldz, h.n64, false, o.w, o.ldw, o.w_rows, h.rows, h.n, h.C64, Vp), tmp, h.C64,
                     PRATCHYA_DT_F32);
      if (rc) break;
      hipLaunchKernelGGL((k_head_out<T>), dim3((unsigned)((h.n * ((h.C + 3) / 4) + 255) / 256)), dim3(256), 0, c.stream,
                         tmp, h.C64, h.n, h.C, c.floats_at(h.dx_sum), v0 > 0, v0 + h.piece >= h.V, dx, h.C, 1, unit);
      if ((rc = check_launch(what))) break;
    }
    if (dw) {
      // [C, V]: rows C, columns cols of them; [V, C]: rows cols, columns C
      const int64_t M = h.rows ? cols : h.C, N = h.rows ? h.C : cols, ld = h.rows ? h.C : h.V;
      T* to = dw + (h.rows ? v0 * h.C : v0);
      if (dw256(h, Vp)) {
        HeadProduct p = h.rows ? operands(c.h, dz, ldz, h.n64, true, o.x, o.ldx, o.x_rows, true, Vp, h.C64, h.n64)
                               : operands(c.h, o.x, o.ldx, o.x_rows, true, dz, ldz, h.n64, true, h.C64, Vp, h.n64);
        p.epilogue = kHeadStore;
        p.rows = M;
        p.cols = N;
        p.c = to;
        p.ldc = ld;
        p.c_bf16 = h.P == 1;
        p.unit = unit;
        if ((rc = head_product(p, c.stream))) break;
        continue;
      }
      // columns [b, b + wide) of the piece
      auto dw_of = [&](int64_t b, int64_t Mt, int64_t Nt) {
        return h.rows ? operands(c.h, dz + b, ldz, h.n64, true, o.x, o.ldx, o.x_rows, true, Mt, Nt, h.n64)
                      : operands(c.h, o.x, o.ldx, o.x_rows, true, dz + b, ldz, h.n64, true, Mt, Nt, h.n64);
      };
      if (h.dw_plain(cols) && aligned16(to)) {
        if ((rc = c.product(dw_of(0, M, N), to, ld, h.dtype, unit))) break;
        continue;
      }
      for (int64_t b = 0; b < cols && !rc; b += h.dw_cols) {
        const int64_t wide = Vp - b < h.dw_cols ? Vp - b : h.dw_cols, some = cols - b < wide ? cols - b : wide;
        const int64_t Nt = h.rows ? h.C64 : wide, Mb = h.rows ? some : M, Nb = h.rows ? N : some;
        if ((rc = c.product(dw_of(b, h.rows ? wide : h.C64, Nt), c.ws + h.dw_tmp, Nt, PRATCHYA_DT_F32))) break;
        hipLaunchKernelGGL((k_head_out<T>), dim3((unsigned)((Mb * ((Nb + 3) / 4) + 255) / 256)), dim3(256), 0, c.stream,
                           c.floats_at(h.dw_tmp), Nt, Mb, Nb, nullptr, 0, 1, to + (h.rows ? b * h.C : b), ld, 1, unit);
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
