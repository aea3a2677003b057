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
#include "row_host.h"

namespace {

struct Affine {
  const void* w;
  const void* b;
  bool w16, b16;
};

// A segment that fits P threads of NV vectors of N = kN<T> elements each stays in
// registers.  A workgroup of TB threads holds TB / P such teams; a team keeps one
// segment position of the row (its slice of w and b, and of dw and db) and walks
// over rows: `gt` neighbouring segments side by side, the other teams on
// further rows.  Thread t of a team holds vectors (t / L * NV + j) * L + t % L, L =
// min(P, 64), j < NV: groups of stored blocks lie in one wave.  Streaming accesses
// where they measured faster: the forward pass's stores of results up to kFwdPast, its
// loads of an x that is stored and so not read again (with its backward pass [16384,
// 4096] 138 -> 134.5 us; of other x 25.2 -> 25.7 us where the caches hold it), the
// backward pass's loads (84.3 -> 79.8 us).
template <int P_, int NV_, int TB_>
struct Shape {
  static constexpr int P = P_, NV = NV_, TB = TB_, TEAMS = TB_ / P_, WAVES = P_ > 64 ? P_ / 64 : 1;
  static constexpr int LANES = P_ < 64 ? P_ : 64;
  static constexpr int JOIN = WAVES <= 2 ? WAVES : WAVES <= 4 ? 4 : WAVES <= 8 ? 8 : 16;    // lanes that join them
};

// A thread's place.  What all lanes of a wave share (all but the lane's offset,
// where a team has whole waves) is made a scalar, and with it rows' addresses.
template <typename G>
struct Place {
  int t, team;         // thread in its team, team in the workgroup
  int rl, rt;          // the team's row lane, row lanes
  int64_t g;           // its segment of the row
  bool live;
  __device__ __forceinline__ Place(int64_t groups) {
    t = threadIdx.x % G::P;
    team = threadIdx.x / G::P;
    if constexpr (G::P >= 64) team = __builtin_amdgcn_readfirstlane(team);
    const int gt = groups < G::TEAMS ? (int)groups : G::TEAMS;
    rt = G::TEAMS / gt;
    rl = team / gt;
    g = (int64_t)blockIdx.y * gt + team % gt;
    live = rl < rt && g < groups;
  }
  // first element of vector j, of N elements, in the segment: the wave's, and the lane's offset to it
  template <int N>
  __device__ __forceinline__ int64_t wave_at(int j) const {
    int wave = t / G::LANES;
    if constexpr (G::P >= 64) wave = __builtin_amdgcn_readfirstlane(wave);
    return (int64_t)(wave * G::NV + j) * (G::LANES * N);
  }
  template <int N>
  __device__ __forceinline__ uint32_t lane_at() const { return (uint32_t)(t % G::LANES) * N; }
  template <int N>
  __device__ __forceinline__ int64_t at(int j) const { return wave_at<N>(j) + lane_at<N>(); }
};

// Elements of a vector that lie in the segment.
template <int N>
__device__ __forceinline__ int part_of(int64_t n) { return n < 0 ? 0 : n < N ? (int)n : N; }

// A thread's vector of a segment of D elements: the last `own` of the n elements
// loaded and stored at `off`.  The vector at the end of a segment of an odd length
// is moved back to end with it: its first elements are the thread's before it, left
// out of sums and stored by both, with the same value.  By its elements, each
// load waited for where it was issued, [8192, 4095] bf16 took 34.5 us where it takes 29, in
// the backward pass 99.9 for 50.  Segments below a vector (whole: false) go by elements.
template <int N>
struct Part {
  uint32_t off;
  int own;
  __device__ __forceinline__ void set(int64_t D, int64_t at, bool whole) {
    own = part_of<N>(D - at);
    off = (uint32_t)(at - (own && whole ? N - own : 0));
  }
  __device__ __forceinline__ int n(bool whole) const { return own && whole ? N : own; }
  __device__ __forceinline__ bool owns(int i, bool whole) const { return whole ? i >= N - own : i < own; }
};

// A vector of a row in registers, in its type.
template <typename T, bool NT = false>
struct Held {
  u32x4_t raw;
  __device__ __forceinline__ void load(const T* p, const Part<kN<T>>& at, bool whole) {
    if (whole) {
      raw = u32x4_t{0, 0, 0, 0};
      if (at.own) raw = load_raw<NT>(p + at.off);
    } else {
      float v[kN<T>];
      load_some(p + at.off, at.own, 0.0f, v);
      raw = narrow(v);
    }
  }
  __device__ __forceinline__ void get(float (&v)[kN<T>]) const { widen(raw, v); }
};

template <int N>
__device__ __forceinline__ void load_params(const void* p, bool bf16, int64_t at, int left, float none,
                                            float (&v)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = none;
  if (!p) return;
  if (left == N && !bf16) {
#pragma unroll
    for (int i = 0; i < N; i += 4) {
      const u32x4_t r = load_raw(static_cast<const float*>(p) + at + i);
      v[i] = u2f(r[0]);
      v[i + 1] = u2f(r[1]);
      v[i + 2] = u2f(r[2]);
      v[i + 3] = u2f(r[3]);
    }
  } else if (bf16) {
    load_some(static_cast<const uint16_t*>(p) + at, left, none, v);
  } else {
    load_some(static_cast<const float*>(p) + at, left, none, v);
  }
}

// 1 / sqrt(v): the hardware's approximation and one step of Newton's iteration,
// but for values near the ends of f32's range, where either may not be finite.
__device__ __forceinline__ float rsqrt_of(float v) {
  if (!(v > 1e-30f && v < 1e30f)) return 1.0f / sqrtf(v);
  const float r = __builtin_amdgcn_rsqf(v);
  return r * (1.5f - 0.5f * v * r * r);
}

// Squared deviations q from a mean that was off, about the corrected one: less the
// correction times the deviations' sum.  Not below 0; infinite sums (values whose
// squares overflow) and NaN stay.
__device__ __forceinline__ float without(float q, float less) {
  return less < q ? q - less : q <= 3.4028234663852886e38f ? 0.0f : q;
}

// (x - mean) r, the difference first: x r - mean r in one operation would leave the
// roundings of mean r in a segment of equal values, r = 1 / sqrt(eps) there (0.4 for
// 29952 where 0 is right).
__device__ __forceinline__ float normed(float x, float mean, float rstd) { return (x - mean) * rstd; }

// y and the statistics of whole segments; with BLK, x's stored form beside them
// (groups = 1).  Mean and squared deviations are taken within each wave, from
// registers, and joined by counts, so a mean far from zero costs no digits.  The mean
// of equal values is that value: up to 2^16 bf16 values' sum is exact and the
// quotient's rounding the only one; f32's mean is corrected by the mean of the
// deviations from it, and waves are joined by their distance from the first.
// Bound by HBM, with 16 to 24 vector instructions an element beside it (medians of
// kernel traces): [16384, 4096] bf16 49.5 us (268 MB, 5.4 TB/s), with its 8-bit form 64 us
// (337 MB, 5.3 TB/s), f32 [8192, 4096] 48.5 us (5.5 TB/s), heads of 64 over [8192, 4096]
// 26 to 27 us (134 MB, 5.1 TB/s); one row of 4096 3.4 us.
template <typename T, typename G, int BLK, int AHEAD, bool PAST>
__global__ __launch_bounds__(G::TB) void k_layer_norm(const T* __restrict__ x, int64_t ldx, Affine p, int64_t rows,
                                                      int64_t width, int64_t groups, float eps, T* __restrict__ y,
                                                      float* __restrict__ stats, uint8_t* __restrict__ x8,
                                                      uint8_t* __restrict__ sc8, float* __restrict__ sc32) {
  constexpr int N = kN<T>, NV = G::NV, LANES = G::LANES, SPAN = NV * LANES * N;   // SPAN: elements of a wave
  __shared__ float4 red[2][G::TEAMS * G::WAVES];
  const Place<G> me(groups);
  const int64_t D = width / groups, c0 = me.g * D;
  const bool whole = G::P > 8 || D >= N;    // wider teams hold segments of more than 64
  Part<N> at[NV];
  float w[NV][N], b[NV][N];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    at[j].set(me.live ? D : 0, me.template at<N>(j), whole);
    load_params(p.w, p.w16, c0 + at[j].off, at[j].n(whole), 1.0f, w[j]);
    load_params(p.b, p.b16, c0 + at[j].off, at[j].n(whole), 0.0f, b[j]);
  }
  // elements of the segment in this wave, and its share of the segment
  const int64_t held = D - me.template wave_at<N>(0);
  const float mine = (float)(held < 0 ? 0 : held < SPAN ? held : SPAN), count = mine > 0.0f ? mine : 1.0f;
  const float per_D = 1.0f / (float)D;
  const int64_t step = (int64_t)gridDim.x * me.rt;
  int64_t row = (int64_t)blockIdx.x * me.rt + me.rl;
  // the next AHEAD rows are on their way while one is computed
  typedef Held<T, BLK != 0> Vec;
  Vec cur[NV], next[AHEAD][NV];
  auto fetch = [&](int64_t r, Vec (&to)[NV]) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      Part<N> a = at[j];
      if (r >= rows) a.own = 0;
      to[j].load(x + (r * ldx + c0), a, whole);
    }
  };
#pragma unroll
  for (int d = 0; d < AHEAD; ++d) fetch(row + d * step, next[d]);
  // the workgroup's first team has the first row: all teams make as many rounds
  int buf = 0;
  for (int64_t lead = (int64_t)blockIdx.x * me.rt; lead < rows; lead += step, row += step, buf ^= 1) {
    const bool on = me.live && row < rows;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      cur[j] = next[0][j];
#pragma unroll
      for (int d = 1; d < AHEAD; ++d) next[d - 1][j] = next[d][j];
    }
    fetch(row + AHEAD * step, next[AHEAD - 1]);
    float v[N], s = 0.0f, q = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      cur[j].get(v);
      if (at[j].own == N) {
#pragma unroll
        for (int i = 0; i < N; ++i) s += v[i];
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) s += at[j].owns(i, whole) ? v[i] : 0.0f;
      }
    }
    s = lane_group_add<LANES>(s);
    constexpr bool EXACT = sizeof(T) == 2;      // the sum of equal values
    float mean = s / count, rest = 0.0f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      cur[j].get(v);
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] -= mean;
      if (at[j].own != N) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = at[j].owns(i, whole) ? v[i] : 0.0f;
      }
#pragma unroll
      for (int i = 0; i < N; ++i) {
        q += v[i] * v[i];
        if constexpr (!EXACT) rest += v[i];
      }
    }
    q = lane_group_add<LANES>(q);
    if constexpr (!EXACT) {
      rest = lane_group_add<LANES>(rest);
      const float by = rest / count;      // equal deviations: exact, and so is what q loses
      mean += by;
      q = without(q, by * rest);
    }
    if constexpr (G::WAVES > 1) {
      float4* r = &red[buf][me.team * G::WAVES];
      if ((me.t & 63) == 0) r[me.t >> 6] = make_float4(mean, q, mine * per_D, 0.0f);
      __syncthreads();
      // a wave's numbers per lane, all waves' in every group of lanes
      const float4 k = r[me.t % G::WAVES];
      const float first = r[0].x;
      mean = first + lane_group_add<G::WAVES>(k.z * (k.x - first));
      const float d = k.x - mean;
      q = lane_group_add<G::WAVES>(k.y + (k.z * (float)D) * d * d);
    }
    const float rstd = rsqrt_of(q * per_D + eps);
    if (!on) continue;
    if (stats && me.t == 0) {
      stats[2 * (row * groups + me.g)] = mean;
      stats[2 * (row * groups + me.g) + 1] = rstd;
    }
    T* yr = y + (row * width + c0);
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      cur[j].get(v);
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = normed(v[i], mean, rstd) * w[j][i] + b[j][i];
      if (at[j].n(whole) == N) store_vec<PAST>(yr + at[j].off, v);
      else if (at[j].own) store_some(yr + at[j].off, at[j].own, v);
    }
    if constexpr (BLK != 0) {
      // lanes of a block, of a group, and vectors that a group spans
      constexpr int K = BLK / 16, LB = BLK / N, LG = LB * K, LR = LG < LANES ? LG : LANES, GV = LG / LR;
      uint32_t mb[NV], Gb[NV];
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        mb[j] = lane_group_max<LB>(absmax<T>(cur[j].raw));
        Gb[j] = lane_group_max<LR>(mb[j]);
      }
#pragma unroll
      for (int j = 0; j < NV; j += GV) {
#pragma unroll
        for (int k = 1; k < GV; ++k) Gb[j] = umax(Gb[j], Gb[j + k]);
#pragma unroll
        for (int k = 1; k < GV; ++k) Gb[j + k] = Gb[j];
      }
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (at[j].own == 0) continue;
        cur[j].get(v);
        uint32_t e;
        // groups divide rows: an element's place in its group is its place in the row's
        const int64_t from = row * width;
        const uint32_t in = at[j].off;
        const auto q8 = store_form(v, mb[j], Gb[j], e);
        __builtin_nontemporal_store(q8, reinterpret_cast<typename Payload<N>::type*>(x8 + from + in));
        if (in % BLK == 0) sc8[(from + in) / BLK] = (uint8_t)e;
        if (in % (BLK * K) == 0) sc32[(from + in) / (BLK * K)] = u2f(Gb[j]);
      }
    }
  }
}

// Segments of more than kLongest elements, which a workgroup's registers do not
// hold beside their weights and biases in f32: a workgroup a segment, kLongVecs vectors
// a thread in flight, three passes over the row of which the later two come from the L2
// cache.  [2048, 32768] bf16 90 us, its backward pass 183 us (3.0 and 2.2 TB/s of what goes
// through HBM once); of 32769, on no address of 16 bytes, 117 and 224 us.  Held as raw
// vectors, with the parameters loaded where they are used, 65536 bf16 would fit.
constexpr int kLongThreads = 1024, kLongVecs = 4;

// Calls use(u, part) for this thread's vectors of a segment, after load has been
// called for up to kLongVecs of them.
template <int N, typename Load, typename Use>
__device__ __forceinline__ void sweep(int64_t D, Load load, Use use) {
  for (int64_t i = (int64_t)threadIdx.x * N; i < D; i += (int64_t)kLongVecs * kLongThreads * N) {
    Part<N> at[kLongVecs];
#pragma unroll
    for (int u = 0; u < kLongVecs; ++u) {
      at[u].set(D, i + (int64_t)u * kLongThreads * N, true);
      load(u, at[u]);
    }
#pragma unroll
    for (int u = 0; u < kLongVecs; ++u)
      if (at[u].own) use(u, at[u]);
  }
}

template <typename T>
__global__ __launch_bounds__(kLongThreads) void k_layer_norm_long(const T* __restrict__ x, int64_t ldx, Affine p,
                                                                  int64_t width, int64_t groups, float eps,
                                                                  T* __restrict__ y, float* __restrict__ stats) {
  constexpr int N = kN<T>;
  __shared__ float lds[kLongThreads / 64];
  const int64_t D = width / groups, row = blockIdx.x / (unsigned)groups, c0 = (blockIdx.x - row * groups) * D;
  const T* xs = x + (row * ldx + c0);
  T* ys = y + (row * width + c0);
  Held<T> h[kLongVecs];
  const auto load = [&](int u, const Part<N>& at) { h[u].load(xs, at, true); };
  float v[N], s = 0.0f, q = 0.0f;
  sweep<N>(D, load, [&](int u, const Part<N>& at) {
    h[u].get(v);
#pragma unroll
    for (int i = 0; i < N; ++i) s += at.owns(i, true) ? v[i] : 0.0f;
  });
  float mean = block_add<kLongThreads / 64>(s, lds) / (float)D, rest = 0.0f;
  sweep<N>(D, load, [&](int u, const Part<N>& at) {
    h[u].get(v);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float d = at.owns(i, true) ? v[i] - mean : 0.0f;
      q += d * d;
      rest += d;
    }
  });
  q = block_add<kLongThreads / 64>(q, lds);
  rest = block_add<kLongThreads / 64>(rest, lds);
  const float by = rest / (float)D;       // of a mean of so many values a step or two may be missing
  mean += by;
  const float rstd = rsqrt_of(without(q, by * rest) / (float)D + eps);
  sweep<N>(D, load, [&](int u, const Part<N>& at) {
    float w[N], b[N];
    load_params(p.w, p.w16, c0 + at.off, N, 1.0f, w);
    load_params(p.b, p.b16, c0 + at.off, N, 0.0f, b);
    h[u].get(v);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = normed(v[i], mean, rstd) * w[i] + b[i];
    store_vec(ys + at.off, v);
  });
  if (stats && threadIdx.x == 0) {
    stats[2 * (int64_t)blockIdx.x] = mean;
    stats[2 * (int64_t)blockIdx.x + 1] = rstd;
  }
}

// x as the backward pass reads it: as it is, or its stored form.
template <typename X>
struct Source {
  const X* x;
  int64_t ldx;
};
struct Stored {
  const uint8_t* x8;
  const uint8_t* sc8;
  const float* sc32;
  int64_t width;
  int blk_log2, K_log2;      // elements per block and blocks per group are powers of two
};
template <typename T, bool STORED> struct SourceOf { typedef Source<T> type; };
template <typename T> struct SourceOf<T, true> { typedef Stored type; };

// The backward pass's x of one vector: as it is, or its stored form.
template <typename T, bool STORED> struct HeldSource;
template <typename T> struct HeldSource<T, false> {
  Held<T, true> x;
  __device__ __forceinline__ void load(const Source<T>& s, int64_t row, int64_t c, const Part<kN<T>>& at, bool whole) {
    x.load(s.x + (row * s.ldx + c), at, whole);
  }
  __device__ __forceinline__ void normed_values(float mean, float rstd, float (&v)[kN<T>]) const {
    x.get(v);
#pragma unroll
    for (int i = 0; i < kN<T>; ++i) v[i] = normed(v[i], mean, rstd);
  }
};
template <typename T> struct HeldSource<T, true> {
  typedef typename Payload<kN<T>>::type W;
  W w;
  uint32_t e;
  float G;
  __device__ __forceinline__ void load(const Stored& s, int64_t row, int64_t c, const Part<kN<T>>& at, bool) {
    w = W{};
    e = 0;
    G = 0.0f;
    if (at.own) {   // segments and blocks are multiples of a vector: it lies in one
      const int64_t from = row * s.width + c, n = (from + at.off) >> s.blk_log2;
      w = __builtin_nontemporal_load(reinterpret_cast<const W*>(s.x8 + from + at.off));
      e = s.sc8[n];
      G = s.sc32[n >> s.K_log2];
    }
  }
  __device__ __forceinline__ void normed_values(float mean, float rstd, float (&v)[kN<T>]) const {
    payload_values(w, v);
    const float s = stored_scale(e, G);
#pragma unroll
    for (int i = 0; i < kN<T>; ++i) v[i] = __builtin_fmaf(v[i], s, -mean) * rstd;
  }
};

// dx of whole segments, and the sums of dy h and dy over the rows that a team
// has walked: joined over the workgroup's row lanes and written to
// part[blockIdx.x][0 / 1][width], or as the results where there is one workgroup
// per column.  Bound by HBM; the partial sums, 2 kB a column over 256 workgroups,
// are 5% of it: with the join [16384, 4096] bf16 77 us (402 MB, 5.2 TB/s), from the
// 8-bit form 73 us (337 MB), f32 [8192, 4096] 71 us (402 MB), heads of 64 over [8192, 4096]
// bf16 41 us (201 MB).
template <typename T, typename G, bool STORED, int AHEAD>
__global__ __launch_bounds__(G::TB) void k_layer_norm_bwd(typename SourceOf<T, STORED>::type src,
                                                          const T* __restrict__ dy, int64_t ldy, Affine p,
                                                          int64_t rows, int64_t width, int64_t groups,
                                                          const float* __restrict__ stats, T* __restrict__ dx,
                                                          float* __restrict__ part, void* dw, bool dw16, void* db,
                                                          bool db16) {
  constexpr int N = kN<T>, NV = G::NV, LANES = G::LANES, SUMS = 2 * NV * N;
  __shared__ float red[2][G::TEAMS * G::WAVES][2];
  __shared__ float sums[G::TEAMS > 1 ? SUMS * (G::TB / 2) : 1];
  const Place<G> me(groups);
  const int64_t D = width / groups, c0 = me.g * D;
  const bool whole = G::P > 8 || D >= N;
  const float per_D = 1.0f / (float)D;
  Part<N> at[NV];
  float w[NV][N], aw[NV][N], ab[NV][N];
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    at[j].set(me.live ? D : 0, me.template at<N>(j), whole);
    load_params(p.w, p.w16, c0 + at[j].off, at[j].n(whole), 1.0f, w[j]);
#pragma unroll
    for (int i = 0; i < N; ++i) aw[j][i] = ab[j][i] = 0.0f;
  }
  const int64_t step = (int64_t)gridDim.x * me.rt;
  int64_t row = (int64_t)blockIdx.x * me.rt + me.rl;
  // a row's data; the next AHEAD rows are on their way while one is computed
  struct Row {
    HeldSource<T, STORED> x[NV];
    Held<T, true> g[NV];
    float mean, rstd;
  };
  Row cur, next[AHEAD ? AHEAD : 1];
  auto fetch = [&](int64_t r, Row& to) {
    const bool on = me.live && r < rows;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      Part<N> a = at[j];
      if (!on) a.own = 0;
      to.x[j].load(src, r, c0, a, whole);
      to.g[j].load(dy + (r * ldy + c0), a, whole);
    }
    to.mean = on ? stats[2 * (r * groups + me.g)] : 0.0f;
    to.rstd = on ? stats[2 * (r * groups + me.g) + 1] : 0.0f;
  };
#pragma unroll
  for (int d = 0; d < AHEAD; ++d) fetch(row + d * step, next[d]);
  int buf = 0;
  for (int64_t lead = (int64_t)blockIdx.x * me.rt; lead < rows; lead += step, row += step, buf ^= 1) {
    if constexpr (AHEAD > 0) {
      cur = next[0];
#pragma unroll
      for (int d = 1; d < AHEAD; ++d) next[d - 1] = next[d];
      fetch(row + AHEAD * step, next[AHEAD - 1]);
    } else {
      fetch(row, cur);
    }
    const float mean = cur.mean, rstd = cur.rstd;
    float s1 = 0.0f, s2 = 0.0f, h[N], g[N];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      cur.x[j].normed_values(mean, rstd, h);
      cur.g[j].get(g);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        aw[j][i] += g[i] * h[i];
        ab[j][i] += g[i];
      }
      if (at[j].own == N) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float a = g[i] * w[j][i];
          s1 += a;
          s2 += a * h[i];
        }
      } else if (!STORED) {      // a stored segment has whole vectors or none
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float a = at[j].owns(i, whole) ? g[i] * w[j][i] : 0.0f;
          s1 += a;
          s2 += a * h[i];
        }
      }
    }
    if (dx) {
      s1 = lane_group_add<LANES>(s1);
      s2 = lane_group_add<LANES>(s2);
      if constexpr (G::WAVES > 1) {
        float (*r)[2] = &red[buf][me.team * G::WAVES];
        if ((me.t & 63) == 0) {
          r[me.t >> 6][0] = s1;
          r[me.t >> 6][1] = s2;
        }
        __syncthreads();
        const int wave = me.t % G::JOIN;
        s1 = lane_group_add<G::JOIN>(wave < G::WAVES ? r[wave][0] : 0.0f);
        s2 = lane_group_add<G::JOIN>(wave < G::WAVES ? r[wave][1] : 0.0f);
      }
      const float m1 = rstd * (s1 * per_D), m2 = rstd * (s2 * per_D);
      if (me.live && row < rows) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          cur.x[j].normed_values(mean, rstd, h);
          cur.g[j].get(g);
#pragma unroll
          for (int i = 0; i < N; ++i) g[i] = (g[i] * w[j][i]) * rstd - m1 - h[i] * m2;
          T* to = dx + (row * width + c0) + at[j].off;
          if (at[j].n(whole) == N) store_vec(to, g);
          else if (at[j].own) store_some(to, at[j].own, g);
        }
      }
    }
  }
  if (!dw && !db) return;
  // the row lanes' sums, halves onto halves
  if constexpr (G::TEAMS > 1) {
    const int cols = G::TEAMS / me.rt * G::P;      // threads of one row lane at most
    const int col = (int)threadIdx.x - me.rl * (groups < G::TEAMS ? (int)groups * G::P : G::TB);
    for (int n = me.rt; n > 1;) {
      const int half = (n + 1) / 2;
      if (me.rl >= half && me.rl < n) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < N; ++i) {
            sums[(j * N + i) * (G::TB / 2) + (me.rl - half) * cols + col] = aw[j][i];
            sums[((NV + j) * N + i) * (G::TB / 2) + (me.rl - half) * cols + col] = ab[j][i];
          }
      }
      __syncthreads();
      if (me.rl < n - half) {
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int i = 0; i < N; ++i) {
            aw[j][i] += sums[(j * N + i) * (G::TB / 2) + me.rl * cols + col];
            ab[j][i] += sums[((NV + j) * N + i) * (G::TB / 2) + me.rl * cols + col];
          }
      }
      __syncthreads();
      n = half;
    }
  }
  if (!me.live || me.rl) return;
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const int64_t c = c0 + at[j].off;
    if (gridDim.x > 1) {
      float* to = part + 2 * (int64_t)blockIdx.x * width + c;
      if (at[j].own == N) {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
          *reinterpret_cast<u32x4_a4*>(to + i) =
              u32x4_t{f2u(aw[j][i]), f2u(aw[j][i + 1]), f2u(aw[j][i + 2]), f2u(aw[j][i + 3])};
          *reinterpret_cast<u32x4_a4*>(to + width + i) =
              u32x4_t{f2u(ab[j][i]), f2u(ab[j][i + 1]), f2u(ab[j][i + 2]), f2u(ab[j][i + 3])};
        }
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
          if (at[j].owns(i, whole)) {
            to[i] = aw[j][i];
            to[width + i] = ab[j][i];
          }
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        if (at[j].owns(i, whole)) {
          if (dw) store_param(dw, dw16, c + i, aw[j][i]);
          if (db) store_param(db, db16, c + i, ab[j][i]);
        }
    }
  }
}

// dx of long segments, a workgroup each: two passes.
template <typename T, bool STORED>
__global__ __launch_bounds__(kLongThreads) void k_layer_norm_long_dx(typename SourceOf<T, STORED>::type src,
                                                                     const T* __restrict__ dy, int64_t ldy, Affine p,
                                                                     int64_t width, int64_t groups,
                                                                     const float* __restrict__ stats,
                                                                     T* __restrict__ dx) {
  constexpr int N = kN<T>;
  __shared__ float lds[kLongThreads / 64];
  const int64_t D = width / groups, row = blockIdx.x / (unsigned)groups, c0 = (blockIdx.x - row * groups) * D;
  const float mean = stats[2 * (int64_t)blockIdx.x], rstd = stats[2 * (int64_t)blockIdx.x + 1];
  const T* gs = dy + (row * ldy + c0);
  T* out = dx + (row * width + c0);
  HeldSource<T, STORED> hx[kLongVecs];
  Held<T> hg[kLongVecs];
  const auto load = [&](int u, const Part<N>& at) {
    hx[u].load(src, row, c0, at, true);
    hg[u].load(gs, at, true);
  };
  float h[N], g[N], w[N], s1 = 0.0f, s2 = 0.0f;
  sweep<N>(D, load, [&](int u, const Part<N>& at) {
    load_params(p.w, p.w16, c0 + at.off, N, 1.0f, w);
    hx[u].normed_values(mean, rstd, h);
    hg[u].get(g);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const float a = at.owns(i, true) ? g[i] * w[i] : 0.0f;
      s1 += a;
      s2 += a * h[i];
    }
  });
  const float m1 = rstd * (block_add<kLongThreads / 64>(s1, lds) / (float)D);
  const float m2 = rstd * (block_add<kLongThreads / 64>(s2, lds) / (float)D);
  sweep<N>(D, load, [&](int u, const Part<N>& at) {
    load_params(p.w, p.w16, c0 + at.off, N, 1.0f, w);
    hx[u].normed_values(mean, rstd, h);
    hg[u].get(g);
#pragma unroll
    for (int i = 0; i < N; ++i) g[i] = (g[i] * w[i]) * rstd - m1 - h[i] * m2;
    store_vec(out + at.off, g);
  });
}

// Column sums of long segments over the rows of one of gridDim.y slices, a vector
// of columns per thread: part[slice][0 / 1][width].
template <typename T, bool STORED>
__global__ __launch_bounds__(256) void k_layer_norm_long_dp(typename SourceOf<T, STORED>::type src,
                                                            const T* __restrict__ dy, int64_t ldy, int64_t rows,
                                                            int64_t width, int64_t groups, int64_t tiles,
                                                            const float* __restrict__ stats,
                                                            float* __restrict__ part) {
  constexpr int N = kN<T>;
  const int64_t D = width / groups, g0 = blockIdx.x / (unsigned)tiles, c0 = g0 * D;
  Part<N> at;
  at.set(D, ((blockIdx.x - g0 * tiles) * 256 + threadIdx.x) * N, true);
  if (!at.own) return;
  float dw[N] = {}, db[N] = {}, h[N], g[N];
#pragma unroll 4
  for (int64_t row = blockIdx.y; row < rows; row += gridDim.y) {
    HeldSource<T, STORED> hx;
    Held<T> hg;
    hx.load(src, row, c0, at, true);
    hg.load(dy + (row * ldy + c0), at, true);
    const float mean = stats[2 * (row * groups + g0)], rstd = stats[2 * (row * groups + g0) + 1];
    hx.normed_values(mean, rstd, h);
    hg.get(g);
#pragma unroll
    for (int i = 0; i < N; ++i) {
      dw[i] += g[i] * h[i];
      db[i] += g[i];
    }
  }
  float* to = part + 2 * (int64_t)blockIdx.y * width + c0 + at.off;
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (at.owns(i, true)) {
      to[i] = dw[i];
      to[width + i] = db[i];
    }
}

// dw and db from the slices' sums: kJoinCols columns per workgroup, its waves on
// different slices.  256 slices of 4096 columns 4 us, the launch among them.
constexpr int kJoinCols = 64, kJoinWaves = 16, kJoinThreads = kJoinWaves * 64;
__global__ __launch_bounds__(kJoinThreads) void k_layer_norm_join(const float* __restrict__ part, int slices,
                                                                  int64_t width, void* dw, bool dw16, void* db,
                                                                  bool db16) {
  __shared__ float lds[2][kJoinWaves][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t c = (int64_t)blockIdx.x * kJoinCols + lane;
  float s = 0.0f, t = 0.0f;
  if (c < width) {
#pragma unroll 4
    for (int i = wave; i < slices; i += kJoinWaves) {
      s += part[2 * i * width + c];
      t += part[(2 * i + 1) * width + c];
    }
  }
  lds[0][wave][lane] = s;
  lds[1][wave][lane] = t;
  __syncthreads();
  if (wave > 1 || c >= width) return;
  void* to = wave ? db : dw;
  if (!to) return;
  s = 0.0f;
#pragma unroll
  for (int k = 0; k < kJoinWaves; ++k) s += lds[wave][k][lane];
  store_param(to, wave ? db16 : dw16, c, s);
}

constexpr int64_t kLongest = 16384;     // elements of a segment held in registers
constexpr int kSlices = 64;             // row slices of the long segments' column sums

bool power_of_two(int64_t v) { return v > 0 && (v & (v - 1)) == 0; }

int check_shape(const char* what, int64_t rows, int64_t width, int64_t groups) {
  if (rows < 0 || width < 0 || groups < 1 || width % groups)
    return pratchya_set_error(PRATCHYA_EINVAL, "%s: %lld groups do not divide rows of %lld (%lld rows)", what,
                              (long long)groups, (long long)width, (long long)rows);
  if (rows > 0x7FFFFFFF || groups > (1 << 20) || rows * groups > 0x7FFFFFFF || width > ((int64_t)1 << 31))
    return pratchya_set_error(PRATCHYA_EUNSUPPORTED, "%s: more than 2^31 segments, 2^20 in a row or 2^31 elements in one", what);
  return PRATCHYA_OK;
}

// Threads of a workgroup (more where a team is larger), workgroups of a launch,
// rows on their way.
constexpr int kFwdThreads = 512, kFwdAhead = 1, kBwdThreads = 1024, kBwdAhead = 1;
constexpr int64_t kFwdBlocks = 512, kBwdBlocks = 256;
// Bytes of y up to which the forward pass stores it past the caches.  With the
// quantizer of the Linear behind it, that reads y at once (bf16, rows of 4096): 2 MB as
// fast, 8 and 16 MB 13.2 -> 12.1 and 18.6 -> 14.0 us (with the 8-bit form 14.4 -> 11.9 and
// 21.7 -> 17.8), 32 and 64 MB within 3%.  Between a residual addition before and that
// quantizer, other work and the backward pass behind, 96 and 128 MB are within 1%,
// but 192 MB take 514 us for 501, 256 MB 684 for 667, 512 MB 1332 for 1311; f32 alike.
constexpr int64_t kFwdPast = (int64_t)128 << 20;
// The backward pass's workgroups of 12 waves: two a compute unit from this many rows
// a team on (2048 x 5120, 4 rows: 23.7 -> 25.2 us; 8 rows 35.1 -> 33.9; 16 rows 58.2 -> 52.3)
constexpr int kBwdThin = 768;
constexpr int64_t kThinRows = 8;

// Call f(Shape) with the smallest team that holds a segment of D elements: in the
// forward pass of 16 elements a thread where a wave is full, in the backward pass,
// where an element takes five registers more for its sums and weight, of 8.  bf16's
// backward pass also has teams of 3, 6 and 12 waves in workgroups of 12 waves, two a
// compute unit: [8192, 5120] 59.3 -> 52.3 us, [16384, 1280] 35.4 -> 31.8.  f32's, of
// more registers, does not fit twice and loses 5% (97.5 -> 102.6 us), and the
// forward pass, of two vectors a thread, gains nothing by them (29.6 -> 28.6, 40.7 -> 42.0).
template <typename T, typename F>
auto with_fwd_shape(int64_t D, F f) {
  constexpr int TB = kFwdThreads, V = 8 / kN<T>;      // vectors of 8 elements
  if (D <= 64) return f(Shape<8, V, TB>());
  if (D <= 128) return f(Shape<16, V, TB>());
  if (D <= 256) return f(Shape<32, V, TB>());
  if (D <= 512) return f(Shape<64, V, TB>());
  if (D <= 1024) return f(Shape<64, 2 * V, TB>());
  if (D <= 2048) return f(Shape<128, 2 * V, TB>());
  if (D <= 4096) return f(Shape<256, 2 * V, TB>());
  if (D <= 8192) return f(Shape<512, 2 * V, TB>());
  return f(Shape<1024, 2 * V, 1024>());
}
template <typename T, typename F>
auto with_bwd_shape(int64_t D, F f) {
  constexpr int TB = kBwdThreads, V = 8 / kN<T>;
  if (D <= 64) return f(Shape<8, V, TB>());
  if (D <= 128) return f(Shape<16, V, TB>());
  if (D <= 256) return f(Shape<32, V, TB>());
  if (D <= 512) return f(Shape<64, V, TB>());
  if (D <= 1024) return f(Shape<128, V, TB>());
  if constexpr (sizeof(T) == 2) {
    if (D > 1024 && D <= 192 * 8) return f(Shape<192, V, kBwdThin>());
    if (D > 2048 && D <= 384 * 8) return f(Shape<384, V, kBwdThin>());
    if (D > 4096 && D <= 768 * 8) return f(Shape<768, V, kBwdThin>());
  }
  if (D <= 2048) return f(Shape<256, V, TB>());
  if (D <= 4096) return f(Shape<512, V, TB>());
  if (D <= 8192) return f(Shape<1024, V, TB>());
  return f(Shape<1024, 2 * V, TB>());
}

// Workgroups along the rows and along the segments of a row.
template <typename G>
dim3 grid_of(int64_t rows, int64_t groups, int64_t most) {
  const int64_t gt = groups < G::TEAMS ? groups : G::TEAMS, rt = G::TEAMS / gt;
  const int64_t gy = (groups + gt - 1) / gt, gx = (rows + rt - 1) / rt, cap = most / gy > 1 ? most / gy : 1;
  return dim3((unsigned)(gx < cap ? gx : cap), (unsigned)gy);
}

// The backward pass's workgroups.  Up to kOneBlockRounds rows a team it is one along
// the rows, whose sums are the results without a second launch.
constexpr int64_t kOneBlockRounds = 4;      // 64 x 512 bf16 11.3 -> 9.7 us; 8 rounds, 128 x 512: 11.1 -> 13.2
template <typename G>
dim3 bwd_grid_of(int64_t rows, int64_t groups) {
  const int64_t rt = G::TEAMS / (groups < G::TEAMS ? groups : G::TEAMS);
  int64_t most = kBwdBlocks;
  if (rows <= kOneBlockRounds * rt) most = 1;
  else if (G::TB == kBwdThin && rows >= kThinRows * 2 * kBwdBlocks * rt) most = 2 * kBwdBlocks;
  return grid_of<G>(rows, groups, most);
}

template <typename T>
dim3 bwd_grid(int64_t rows, int64_t width, int64_t groups) {
  return with_bwd_shape<T>(width / groups, [&](auto shape) { return bwd_grid_of<decltype(shape)>(rows, groups); });
}

int too_many(const char* what) {
  return pratchya_set_error(PRATCHYA_EUNSUPPORTED, "%s: more segments or columns than a launch has workgroups for", what);
}

template <typename T, typename G>
int launch_fwd(G, const T* x, int64_t ldx, const Affine& p, int64_t rows, int64_t width, int64_t groups, float eps,
                T* y, float* stats, uint8_t* x8, uint8_t* sc8, float* sc32, int64_t blk, hipStream_t stream) {
  const dim3 grid = grid_of<G>(rows, groups, kFwdBlocks * kFwdThreads / G::TB);
  if (!fits_launch(grid.x, G::TB, grid.y)) return too_many("layer_norm");
#define PRATCHYA_LNP(B, PAST)                                                                                       \
  hipLaunchKernelGGL((k_layer_norm<T, G, B, kFwdAhead, PAST>), grid, dim3(G::TB), 0, stream, x, ldx, p, rows, width,   \
                     groups, eps, y, stats, x8, sc8, sc32)
#define PRATCHYA_LN(B)                                                                                              \
  {                                                                                                                 \
    if (rows * width * (int64_t)sizeof(T) <= kFwdPast) PRATCHYA_LNP(B, true);                                       \
    else PRATCHYA_LNP(B, false);                                                                                    \
  }
  if (!x8) PRATCHYA_LN(0)
  else if (blk == 16) PRATCHYA_LN(16)
  else if (blk == 32) PRATCHYA_LN(32)
  else if (blk == 64) { if constexpr (G::P >= 32) PRATCHYA_LN(64) }
  else { if constexpr (G::P >= 64 && G::NV * kN<T> >= 16) PRATCHYA_LN(128) }
#undef PRATCHYA_LN
#undef PRATCHYA_LNP
  return check_launch("layer_norm");
}

template <typename T>
int layer_norm(const void* x, int64_t ldx, const Affine& p, int64_t rows, int64_t width, int64_t groups, float eps,
               void* y, float* stats, uint8_t* x8, uint8_t* sc8, float* sc32, int64_t blk, hipStream_t stream) {
  const T* xt = static_cast<const T*>(x);
  T* yt = static_cast<T*>(y);
  if (width / groups <= kLongest)
    return with_fwd_shape<T>(width / groups, [&](auto shape) {
      return launch_fwd<T>(shape, xt, ldx, p, rows, width, groups, eps, yt, stats, x8, sc8, sc32, blk, stream);
    });
  if (!fits_launch(rows * groups, kLongThreads)) return too_many("layer_norm");
  hipLaunchKernelGGL((k_layer_norm_long<T>), dim3((unsigned)(rows * groups)), dim3(kLongThreads), 0, stream, xt, ldx, p,
                     width, groups, eps, yt, stats);
  return check_launch("layer_norm");
}

template <typename T, bool STORED>
int layer_norm_bwd(typename SourceOf<T, STORED>::type src, const void* dy, int64_t ldy, const void* w, int w_dtype,
                   const float* stats, int64_t rows, int64_t width, int64_t groups, void* dx, void* dw, int dw_dtype,
                   void* db, int db_dtype, float* part, hipStream_t stream) {
  const T* g = static_cast<const T*>(dy);
  const Affine p = {w, nullptr, w_dtype == PRATCHYA_DT_BF16, false};
  const bool dw16 = dw_dtype == PRATCHYA_DT_BF16, db16 = db_dtype == PRATCHYA_DT_BF16;
  int slices = 1;
  const int64_t joins = (width + kJoinCols - 1) / kJoinCols;
  if (width / groups > kLongest) {
    // both limits before the first launch; the other form joins rows of 2^22 columns at most
    if ((dx && !fits_launch(rows * groups, kLongThreads)) || ((dw || db) && !fits_launch(joins, kJoinThreads)))
      return too_many("layer_norm_bwd");
    if (dx)
      hipLaunchKernelGGL((k_layer_norm_long_dx<T, STORED>), dim3((unsigned)(rows * groups)), dim3(kLongThreads), 0,
                         stream, src, g, ldy, p, width, groups, stats, static_cast<T*>(dx));
    if (dw || db) {
      slices = rows < kSlices ? (int)rows : kSlices;
      const int64_t tiles = (width / groups + 256 * kN<T> - 1) / (256 * kN<T>);
      hipLaunchKernelGGL((k_layer_norm_long_dp<T, STORED>), dim3((unsigned)(groups * tiles), (unsigned)slices),
                         dim3(256), 0, stream, src, g, ldy, rows, width, groups, tiles, stats, part);
    }
  } else {
    const bool fits = with_bwd_shape<T>(width / groups, [&](auto shape) {
      typedef decltype(shape) G;
      // 16 elements a thread leave none of the 128 registers for a row ahead
      constexpr int AHEAD = G::NV * kN<T> == 8 ? kBwdAhead : 0;
      const dim3 grid = bwd_grid_of<G>(rows, groups);
      if (!fits_launch(grid.x, G::TB, grid.y)) return false;
      slices = (int)grid.x;
      hipLaunchKernelGGL((k_layer_norm_bwd<T, G, STORED, AHEAD>), grid, dim3(G::TB), 0, stream, src, g, ldy, p, rows,
                         width, groups, stats, static_cast<T*>(dx), part, dw, dw16, db, db16);
      return true;
    });
    if (!fits) return too_many("layer_norm_bwd");
    if (slices == 1) return check_launch("layer_norm_bwd");
  }
  if (dw || db)
    hipLaunchKernelGGL(k_layer_norm_join, dim3((unsigned)joins), dim3(kJoinThreads), 0, stream, part, slices,
                       width, dw, dw16, db, db16);
  return check_launch("layer_norm_bwd");
}

}  // namespace

extern "C" int pratchya_layer_norm_stores(int64_t width, int64_t groups, int64_t blk) {
  if (groups != 1 || width < 1 || width > kLongest || (blk != 16 && blk != 32 && blk != 64 && blk != 128)) return 0;
  return width % (blk * (blk / 16)) == 0;      // whole groups of blk / 16 blocks in a row
}

extern "C" int pratchya_layer_norm(const void* x, int64_t ldx, int dtype, const void* w, int w_dtype, const void* b,
                                   int b_dtype, int64_t rows, int64_t width, int64_t groups, float eps, void* y,
                                   float* stats, uint8_t* x8, uint8_t* sc8, float* sc32, int64_t blk,
                                   hipStream_t stream) {
  const int rc = check_shape("layer_norm", rows, width, groups);
  if (rc) return rc;
  if (x8 && !pratchya_layer_norm_stores(width, groups, blk))
    return pratchya_set_error(PRATCHYA_EUNSUPPORTED, "layer_norm: blocks of %lld are not stored in the same pass",
                              (long long)blk);
  if (!is_float_dtype(dtype) || (w && !is_float_dtype(w_dtype)) || (b && !is_float_dtype(b_dtype)))
    return pratchya_set_error(PRATCHYA_EINVAL, "layer_norm: unsupported dtypes (x %d, weight %d, bias %d)", dtype,
                              w_dtype, b_dtype);
  if (rows == 0 || width == 0) return pratchya_set_error(PRATCHYA_OK, "");
  if (!x || !y || (x8 && (!sc8 || !sc32))) return pratchya_set_error(PRATCHYA_EINVAL, "layer_norm: null buffer");
  if (reinterpret_cast<uintptr_t>(x8) % 8)
    return pratchya_set_error(PRATCHYA_EINVAL, "layer_norm: the payload must be 8-byte aligned");
  const Affine p = {w, b, w_dtype == PRATCHYA_DT_BF16, b_dtype == PRATCHYA_DT_BF16};
  return dtype == PRATCHYA_DT_BF16
             ? layer_norm<uint16_t>(x, ldx, p, rows, width, groups, eps, y, stats, x8, sc8, sc32, blk, stream)
             : layer_norm<float>(x, ldx, p, rows, width, groups, eps, y, stats, x8, sc8, sc32, blk, stream);
}

extern "C" int64_t pratchya_layer_norm_bwd_workspace_bytes(int64_t rows, int64_t width, int64_t groups) {
  if (rows < 1 || width < 1 || groups < 1 || width % groups) return 0;
  int64_t slices = rows < kSlices ? rows : kSlices;
  if (width / groups <= kLongest) {      // the larger of the two types' grids
    const int64_t s = bwd_grid<float>(rows, width, groups).x;
    slices = bwd_grid<uint16_t>(rows, width, groups).x;
    if (s > slices) slices = s;
  }
  return slices * 2 * width * (int64_t)sizeof(float);
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
  if (stored && (blk < 8 || !power_of_two(blk) || width % blk))
    return pratchya_set_error(PRATCHYA_EINVAL, "layer_norm_bwd: blocks of %lld for rows of %lld", (long long)blk,
                              (long long)width);
  if (stored && reinterpret_cast<uintptr_t>(x) % 8)
    return pratchya_set_error(PRATCHYA_EINVAL, "layer_norm_bwd: the payload must be 8-byte aligned");
  if (stored && (width / groups) % 8)      // a vector of a segment would lie in two blocks
    return pratchya_set_error(PRATCHYA_EUNSUPPORTED, "layer_norm_bwd: stored segments of %lld elements, not of eights",
                              (long long)(width / groups));
  if (rows == 0 || width == 0) return pratchya_set_error(PRATCHYA_OK, "");
  if (!x || !dy || !stats || (stored && (!sc8 || !sc32)))
    return pratchya_set_error(PRATCHYA_EINVAL, "layer_norm_bwd: null buffer");
  const int64_t need = pratchya_layer_norm_bwd_workspace_bytes(rows, width, groups);
  if ((dw || db) && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 4))
    return pratchya_set_error(PRATCHYA_EINVAL, "layer_norm_bwd: workspace of %lld bytes needed, 4-byte aligned",
                              (long long)need);
  float* part = static_cast<float*>(workspace);
#define PRATCHYA_LNB(T, ST, SRC)                                                                                   \
  layer_norm_bwd<T, ST>(SRC, dy, ldy, w, w_dtype, stats, rows, width, groups, dx, dw, dw_dtype, db, db_dtype, part, \
                        stream)
  if (stored) {
    const int64_t K = gcd64(blk / 16 > 1 ? blk / 16 : 1, rows * (width / blk));
    const Stored s = {static_cast<const uint8_t*>(x), sc8, sc32, width, log2_of(blk), log2_of(K)};
    return dtype == PRATCHYA_DT_BF16 ? PRATCHYA_LNB(uint16_t, true, s) : PRATCHYA_LNB(float, true, s);
  }
  if (dtype == PRATCHYA_DT_BF16)
    return PRATCHYA_LNB(uint16_t, false, (Source<uint16_t>{static_cast<const uint16_t*>(x), ldx}));
  return PRATCHYA_LNB(float, false, (Source<float>{static_cast<const float*>(x), ldx}));
#undef PRATCHYA_LNB
}
