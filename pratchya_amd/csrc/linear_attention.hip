// Linear attention with a decay for each head and token, for gfx950: chunks of tokens
// for prompts and training with all gradients, and one token at a time.
//
//   S_t = e^(g_t) S_(t-1) + k_t^T v_t  (S [dk, dv], f32),   o_t = c q_t S_t.
//
// In a chunk with G_i = sum of g up to and with token i, and the state S before it:
//   o_i = c [ sum over j <= i of e^(G_i - G_j) (q_i . k_j) v_j  +  e^(G_i) q_i S ],
//   S'  = e^(G_last) S + sum over j of e^(G_last - G_j) k_j^T v_j.
//
// Gradients.  With R_t = e^(g_(t+1)) R_(t+1) + c q_t^T do_t (R behind the last token is
// the gradient of the state that the call returns): dq_t = c S_t do_t, dk_t = R_t v_t,
// dv_t = k_t R_t.  Each is a linear attention again, of other arrays, the last two
// from the end to the start:
//         queries  keys  values   state
//   o        q      k      v      S
//   dq       do     v      k      S^T       k_mix serves o and dq
//   dk       v      do     q      R^T       backwards, both in k_mix_back
//   dv       k      q      do     R
// A decay scales all that passes from before t to t or later: dg_t = sum over u >= t of
// (q_u . dq_u - k_u . dk_u) + <S_last, R_last>, taken from the end of a segment of the
// sequence, where S and R are known, so that the sum cancels over a segment at most.
//
// Products run on bf16 MFMAs.  Exact bf16 inputs are one plane; f32 values (f32 inputs,
// states, decayed values) are the sum of three, of which products of 2^-24 of the
// largest or more are taken.  States are f32, and what enters them is never rounded to
// less.  The scores and the states that outputs in bf16 read are two planes, 2^-16 of
// themselves: with one, 2^-9, what the terms of a sum lose stands in outputs in which they
// cancel (error of 0.0023 of the norm against 64 bits, 0.0017 now, the output's own rounding;
// both passes of the size below 690 us, 653 with one).  The decays' gradient is f32, and what
// it sums is not rounded: see k_mix_back.
//
// A sequence is cut into segments where heads alone leave the chip idle: the states that
// their parts add first (k_mix without outputs), joined from the first to the last, then
// all segments at once.
//
// Measured, 8 x 4096 tokens of 32 heads of 64 in bf16, both passes 735 us: states 36 us for
// each of S and R, joins 7, o 158, dq 196, k_mix_back 337.  HBM at a copy's rate would take 220
// (1.08 GB).  The MFMAs are busy a sixth of the time, the vector units two fifths (planes,
// weights, masks), LDS a third, and two or three workgroups a compute unit overlap these in
// part.  Without gradients (8192 tokens of 64 heads, 113 us) the walk runs at 3.7 TB/s.  With
// one plane of scores and read states, and values that are not finite not looked for (650),
// dk and dv as walks of their own, as dq, whose scores then need three planes each for the
// decays' sums, took both passes to 991; states of whole segments, a workgroup each, to 693.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "pratchya_fp8.h"
#include "row_device.h"
#include "row_host.h"

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2_a2 __attribute__((ext_vector_type(2), aligned(2)));     // at any element's address
typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) v4s lds_v4s;

// An array [B, T, H, D] (D contiguous).
struct Array {
  void* p;
  int64_t b, t, h;
};

struct MixArgs {
  Array q, k, v, out, x;           // x: the array whose dot products with the output are wanted
  const void* g;                   // log decays [B, T, H]
  int64_t gb, gt, gh;
  int g_bf16;
  const int64_t* lengths;          // [B], or null
  const float* init;               // state before a segment: [B H][nseg] of [.., ..], or null
  float* last;                     // state after the walk; without outputs: of the parts of every segment but the
                                   // walk's last, in the walk's order
  float* decay;                    // without outputs: e^(sum of a part's log decays)
  float* dot;                      // [B H][T]: x times what the output has from the state before the chunk
  int64_t init_seg, last_seg;      // elements from a segment's state to the next one's
  int init_r, init_c, last_r, last_c;   // strides of a state's query and value axes
  int B, T, H, dq, dv, nseg, per;  // per: chunks of a segment
  int parts, per_part;             // without outputs: parts of a segment, chunks of a part
  int rev;                         // without outputs: from the last token to the first
  float scale, kscale;             // of outputs, of what enters the state
};

// A log decay as it counts: e^-10^4 is 0, and sums of such keep their digits.
__device__ __forceinline__ float floor_decay(float g) { return g < -1e4f ? -1e4f : g; }

__device__ __forceinline__ bf16x8_t frag(v2i a, v2i b) { return __builtin_bit_cast(bf16x8_t, v4i{a.x, a.y, b.x, b.y}); }
__device__ __forceinline__ v4f mfma(bf16x8_t a, bf16x8_t b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

// An operand's fragment for a wave: row l % 16 of 16, K values 8 (l / 16) .. + 7 of 32.
// From rows that hold K contiguously:
__device__ __forceinline__ bf16x8_t read_rows(const uint16_t* p, int pitch, int lane) {
  return *reinterpret_cast<const bf16x8_t*>(p + (lane & 15) * pitch + (lane >> 4) * 8);
}
// the same with the K order of a product's own result, 4 (l / 16) .. + 3 of each half of the 32:
__device__ __forceinline__ bf16x8_t read_rows_halves(const uint16_t* p, int pitch, int lane) {
  const uint16_t* r = p + (lane & 15) * pitch + (lane >> 4) * 4;
  return frag(*reinterpret_cast<const v2i*>(r), *reinterpret_cast<const v2i*>(r + 16));
}
// from rows of K (p: K row 0, operand row 0), by the transposing read: lane j of 16
// reads K row j / 4 at operand rows 4 (j % 4) .. + 3, and lane i receives operand row i
// of the four K rows.
__device__ __forceinline__ bf16x8_t read_columns(const uint16_t* p, int pitch, int lane) {
  const int j = lane & 15;
  const uint16_t* r = p + ((lane >> 4) * 8 + (j >> 2)) * pitch + (j & 3) * 4;
  const v4s a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)r);
  const v4s b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s*)(r + 4 * pitch));
  return frag(__builtin_bit_cast(v2i, a), __builtin_bit_cast(v2i, b));
}

// Values as NP planes of pairs: one rounded plane, or the three exact pieces.
template <int NP, int N>
__device__ __forceinline__ void split(float (&v)[N], uint32_t (&o)[NP][N / 2]) {
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      if (p == NP - 1) {
        o[p][i / 2] = pack_bf16x2(v[i], v[i + 1]);
      } else {
        const float a = top_piece(v[i]), b = top_piece(v[i + 1]);
        o[p][i / 2] = (f2u(a) >> 16) | f2u(b);
        v[i] -= a;
        v[i + 1] -= b;
      }
    }
}
__device__ __forceinline__ bf16x8_t frag4(const uint32_t (&w)[4]) {
  return __builtin_bit_cast(bf16x8_t, v4i{(int)w[0], (int)w[1], (int)w[2], (int)w[3]});
}
// c + the products of the planes of a and b that count.
template <int NA, int NB>
__device__ __forceinline__ v4f mfma_planes(const bf16x8_t (&a)[NA], const bf16x8_t (&b)[NB], v4f c) {
#pragma unroll
  for (int i = 0; i < NA; ++i)
#pragma unroll
    for (int j = 0; j < NB; ++j)
      if (i + j < 3) c = mfma(a[i], b[j], c);
  return c;
}
__device__ __forceinline__ float bf16_at(const bf16x8_t& f, int i) {
  const v4i w = __builtin_bit_cast(v4i, f);
  return u2f((i & 1) ? (uint32_t)w[i >> 1] & 0xFFFF0000u : (uint32_t)w[i >> 1] << 16);
}

constexpr int kThreads = 256;        // a walk with one set of outputs; the backward one has two

// By chunk parity: cumulated log decays in two parts, e^(sum from the chunk's start) and
// e^(sum to its end), the chunk's e^sum.
template <int L>
struct Gates {
  alignas(16) float hi[2][L], lo[2][L], start[2][L], rest[2][L];
  float total[2];
};

template <int NPI, int NP, int L, int DP, int EP, bool OUT>
struct Lds {
  // row pitches: 4 words more than whole turns of the 64 banks, or of half of them (a third of the
  // cycles that the LDS is busy are conflicts still; other pitches took as long)
  static constexpr int PD = DP + 8, PE = EP + 8, PT = L + 8;
  alignas(16) uint16_t q[OUT ? NPI : 1][OUT ? L * PD : 8];
  alignas(16) uint16_t k[NPI][L * PD];
  alignas(16) uint16_t v[NPI][L * PE];
  alignas(16) uint16_t t[NP][OUT ? L * PT : 8];
  Gates<L> gates;
  float dot[4][L];
};

// A head's rows of one sequence as a buffer: reads from `rows` on give 0, writes are
// dropped.  For arrays that the hardware's 32-bit offsets and alignment suit (fits_buffer).
// All of an offset is the vector one: a scalar one takes no part in the bounds check.
constexpr int kBufferFlags = 0x00020000;   // raw buffer, 32-bit data format
constexpr uint32_t kOutside = 0x80000000u; // an offset that stays outside with all that is added to it
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_of(const void* p, int64_t rows, int64_t step, int width,
                                                            int elem) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), 0,
                                           rows > 0 ? (int)(((rows - 1) * step + width) * elem) : 0, kBufferFlags);
}

__device__ __forceinline__ void widen4(const u32x2_t& w, float (&x)[4]) {
  x[0] = u2f(w[0] << 16);
  x[1] = u2f(w[0] & 0xFFFF0000u);
  x[2] = u2f(w[1] << 16);
  x[3] = u2f(w[1] & 0xFFFF0000u);
}
__device__ __forceinline__ void widen4(const u32x4_t& w, float (&x)[4]) { widen(w, x); }
__device__ __forceinline__ u32x2_t load_four(const uint16_t* p) { return *reinterpret_cast<const u32x2_a2*>(p); }
__device__ __forceinline__ u32x4_t load_four(const float* p) { return load_raw(p); }
template <typename T>
__device__ __forceinline__ void store4(__amdgpu_buffer_rsrc_t rs, uint32_t at, const float (&o)[4]) {
  if constexpr (sizeof(T) == 2)
    __builtin_amdgcn_raw_buffer_store_b64(u32x2_t{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])}, rs, (int)at, 0, 0);
  else
    __builtin_amdgcn_raw_buffer_store_b128(narrow(o), rs, (int)at, 0, 0);
}

// A vector without its first elements, as many as a row of `width` is short of a multiple
// of it; zeros behind.
template <typename T>
__device__ __forceinline__ u32x4_t drop_first(u32x4_t v, int width) {
  constexpr int N = kN<T>;
  const int n = (N - width % N) % N, words = n * (int)sizeof(T) / 4;
  if (words & 2) v = u32x4_t{v[2], v[3], 0, 0};
  if (words & 1) v = u32x4_t{v[1], v[2], v[3], 0};
  if (sizeof(T) == 2 && (n & 1))
    v = u32x4_t{v[0] >> 16 | v[1] << 16, v[1] >> 16 | v[2] << 16, v[2] >> 16 | v[3] << 16, v[3] >> 16};
  return v;
}

// A thread's vectors of L rows of W (padded) columns of an array.
template <typename T, int L, int W, int THREADS, bool FULL>
struct Rows {
  static constexpr int N = kN<T>, PER = W / N, V = L * PER / THREADS;
  static_assert(THREADS % PER == 0 && V > 0, "a thread's vectors share a column");
  const T* p;
  int64_t step, length;
  int width;
  __amdgpu_buffer_rsrc_t rs;
  uint32_t at;                         // byte offset of the thread's first vector; the others lie THREADS / PER rows on
  u32x4_t raw[V];

  // p: the head's first row; rows from `length` on count as 0
  __device__ __forceinline__ Rows(const Array& a, int b, int h, int64_t length_, int width_)
      : p(static_cast<const T*>(a.p) + b * a.b + h * a.h), step(a.t), length(length_), width(width_) {
    if constexpr (FULL) {
      rs = buffer_of(p, length, step, width, sizeof(T));
      const int r = (int)threadIdx.x / PER, c = (int)threadIdx.x % PER * N;
      at = c < width ? (uint32_t)(r * (int)step + c) * (uint32_t)sizeof(T) : kOutside;
    }
  }
  __device__ __forceinline__ void load(int t0) {
    if constexpr (FULL) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        raw[i] = __builtin_bit_cast(
            u32x4_t, __builtin_amdgcn_raw_buffer_load_b128(
                         rs, (int)(at + (uint32_t)(t0 + i * (THREADS / PER)) * (uint32_t)step * (uint32_t)sizeof(T)), 0, 0));
      return;
    }
    const int rows = (int)max(min(length - t0, (int64_t)L), (int64_t)0);
    const T* first = p + t0 * step;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int at = threadIdx.x + i * THREADS, r = at / PER, c = at % PER * N;
      raw[i] = u32x4_t{};
      if (r < rows && c < width) {
        const T* s = first + r * step + c;
        if (width >= N) {
          // a row's last vector is read up to the row's end, and moved
          const int over = max(c + N - width, 0);
          const u32x4_t r0 = load_raw(s - over);
          raw[i] = over ? drop_first<T>(r0, width) : r0;
        } else {
          float v[N];
          load_some(s, width - c, 0.0f, v);
          raw[i] = narrow(v);
        }
      }
    }
  }
  template <int NPI, int SIZE>
  __device__ __forceinline__ void store(uint16_t (&to)[NPI][SIZE], int pitch) const {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int at = threadIdx.x + i * THREADS, r = at / PER, c = at % PER * N;
      if constexpr (NPI == 1) {
        *reinterpret_cast<u32x4_t*>(to[0] + r * pitch + c) = raw[i];
      } else {
        float v[4];
        widen(raw[i], v);
        uint32_t o[NPI][2];
        split<NPI, 4>(v, o);
#pragma unroll
        for (int p = 0; p < NPI; ++p) *reinterpret_cast<u32x2_t*>(to[p] + r * pitch + c) = u32x2_t{o[p][0], o[p][1]};
      }
    }
  }
};

// Where a lane's 4 values of an array's tokens are: token row l % 16 of a tile, values e ..
template <typename T, bool FULL>
struct Lane4 {
  T* p;
  int64_t step, rows;
  int left;                            // values from e on that exist
  __amdgpu_buffer_rsrc_t rs;
  uint32_t at;

  // rows: reads from there on give 0, writes are dropped
  __device__ __forceinline__ Lane4(const Array& a, int b, int h, int64_t rows_, int width, int e, int l16)
      : p(static_cast<T*>(a.p) + b * a.b + h * a.h + e), step(a.t), rows(rows_), left(width - e) {
    if constexpr (FULL) {
      rs = buffer_of(p - e, rows, step, width, sizeof(T));
      at = left > 0 ? (uint32_t)(l16 * (int)step + e) * (uint32_t)sizeof(T) : kOutside;
    }
  }
  // of token t + l16 (t uniform), `more` values on (a multiple of 16); with buffers ahead
  // of its use by ask()
  using Raw = std::conditional_t<sizeof(T) == 2, u32x2_t, u32x4_t>;
  __device__ __forceinline__ Raw ask(int t, int more) const {
    if constexpr (!FULL) return Raw{};
    else if constexpr (sizeof(T) == 2) return __builtin_bit_cast(Raw, __builtin_amdgcn_raw_buffer_load_b64(rs, (int)at_of(t, more), 0, 0));
    else return __builtin_bit_cast(Raw, __builtin_amdgcn_raw_buffer_load_b128(rs, (int)at_of(t, more), 0, 0));
  }
  __device__ __forceinline__ void load(int t, int l16, int more, const Raw& raw, float (&x)[4]) const {
    if constexpr (FULL) {
      widen4(raw, x);
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = 0.0f;
      if (t + l16 < rows && left > more) {
        const T* from = p + (t + l16) * step + more;
        if (left - more < 4) load_some(from, left - more, 0.0f, x);
        else widen4(load_four(from), x);
      }
    }
  }
  __device__ __forceinline__ void store(int t, int l16, int more, const float (&o)[4]) const {
    if constexpr (FULL) {
      store4<T>(rs, at_of(t, more), o);
    } else if (t + l16 < rows && left > more) {
      T* to = p + (t + l16) * step + more;
      if (left - more < 4) store_some(to, left - more, o);
      else if constexpr (sizeof(T) == 2) *reinterpret_cast<u32x2_a2*>(to) = u32x2_a2{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
      else store_vec(to, o);
    }
  }
  __device__ __forceinline__ uint32_t at_of(int t, int more) const {
    const uint32_t o = at + (uint32_t)t * (uint32_t)step * (uint32_t)sizeof(T) + (uint32_t)more * (uint32_t)sizeof(T);
    return more && left <= more ? kOutside : o;
  }
};

// log decay of a lane's token, 0 from `length` on
__device__ __forceinline__ float load_gate(const void* g, int is_bf16, int64_t at, int64_t step, int64_t t, int64_t length) {
  if (t >= length) return 0.0f;
  const int64_t i = at + t * step;
  return floor_decay(is_bf16 ? load_elem(static_cast<const uint16_t*>(g) + i) : static_cast<const float*>(g)[i]);
}

// A lane's number as the compiler does not know it: what is compared with it is compared
// where it is used, and no results of comparisons are kept over a loop in scalar registers.
__device__ __forceinline__ int opaque(int lane) {
  asm volatile("" : "+v"(lane));
  return lane;
}

// A chunk's Gates by one wave, sums in 64 bits; returns the chunk's sum.
template <int L>
__device__ __forceinline__ double cumulate(float g, Gates<L>& m, int par, int lane) {
  lane = opaque(lane);
  double s = lane < L ? (double)g : 0.0;
#pragma unroll
  for (int k = 1; k < L; k <<= 1) {
    const double o = __shfl_up(s, k, 64);
    if (lane >= k) s += o;
  }
  const double end = __shfl(s, L - 1, 64);
  if (lane < L) {
    const float hi = (float)s;
    m.hi[par][lane] = hi;
    m.lo[par][lane] = (float)(s - (double)hi);
    m.start[par][lane] = expf((float)s);
    m.rest[par][lane] = expf((float)(end - s));
  }
  if (lane == 0) m.total[par] = expf((float)end);
  return end;
}

// A state [16 DT, 64 ET] by four waves, in the layout of the MFMA's results:
// [16 dt + 4 (l / 16) + r][16 (wave ET + et) + l % 16].
template <int DT, int ET>
struct State {
  v4f s[DT][ET] = {};

  // f(value, row, column) for all that exist
  template <typename F>
  __device__ __forceinline__ void each(int rows, int cols, int wave, int lane, F f) {
    lane = opaque(lane);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int et = 0; et < ET; ++et) {
        const int e = (wave * ET + et) * 16 + (lane & 15);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int d = dt * 16 + (lane >> 4) * 4 + r;
          float x = s[dt][et][r];
          if (d < rows && e < cols) f(x, d, e);
          s[dt][et][r] = x;
        }
      }
  }

  // acc[it][et] = the queries' products with the state: token 16 it + l % 16, value
  // 16 (wave ET + et) + 4 (l / 16) + r; NS: planes of the state
  template <int NS, int NPI, int IT, int SIZE>
  __device__ __forceinline__ void read(const uint16_t (&q)[NPI][SIZE], int pitch, int lane, v4f (&acc)[IT][ET]) const {
#pragma unroll
    for (int it = 0; it < IT; ++it)
#pragma unroll
      for (int et = 0; et < ET; ++et) acc[it][et] = v4f{};
#pragma unroll
    for (int ks = 0; ks < DT / 2; ++ks) {
      bf16x8_t a[ET][NS];
#pragma unroll
      for (int et = 0; et < ET; ++et) {
        float w[8];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          w[r] = s[2 * ks][et][r];
          w[4 + r] = s[2 * ks + 1][et][r];
        }
        uint32_t o[NS][4];
        split<NS, 8>(w, o);
#pragma unroll
        for (int x = 0; x < NS; ++x) a[et][x] = frag4(o[x]);
      }
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        bf16x8_t c[NPI];
#pragma unroll
        for (int x = 0; x < NPI; ++x) c[x] = read_rows_halves(q[x] + it * 16 * pitch + ks * 32, pitch, lane);
#pragma unroll
        for (int et = 0; et < ET; ++et) acc[it][et] = mfma_planes(a[et], c, acc[it][et]);
      }
    }
  }

  // s = total s + keys^T (values times w); val: the values' fragments
  template <int KS, int NPI, int SIZE>
  __device__ __forceinline__ void update(const uint16_t (&k)[NPI][SIZE], int pitch, const bf16x8_t (&val)[KS][ET][NPI],
                                         const float* w, float scale, float total, int lane) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int et = 0; et < ET; ++et)
#pragma unroll
        for (int r = 0; r < 4; ++r) s[dt][et][r] *= total;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      const v4f w0 = *reinterpret_cast<const v4f*>(w + ks * 32 + (lane >> 4) * 8) * scale;
      const v4f w1 = *reinterpret_cast<const v4f*>(w + ks * 32 + (lane >> 4) * 8 + 4) * scale;
      bf16x8_t dec[ET][3];
#pragma unroll
      for (int et = 0; et < ET; ++et) {
        float f[8] = {};
#pragma unroll
        for (int x = NPI - 1; x >= 0; --x)
#pragma unroll
          for (int r = 0; r < 8; ++r) f[r] += bf16_at(val[ks][et][x], r);
#pragma unroll
        for (int r = 0; r < 8; ++r) f[r] *= r < 4 ? w0[r] : w1[r - 4];
        uint32_t o[3][4];
        split<3, 8>(f, o);
#pragma unroll
        for (int x = 0; x < 3; ++x) dec[et][x] = frag4(o[x]);
      }
#pragma unroll
      for (int dt = 0; dt < DT; ++dt) {
        bf16x8_t a[NPI];
#pragma unroll
        for (int x = 0; x < NPI; ++x) a[x] = read_columns(k[x] + ks * 32 * pitch + dt * 16, pitch, lane);
#pragma unroll
        for (int et = 0; et < ET; ++et) s[dt][et] = mfma_planes(a, dec[et], s[dt][et]);
      }
    }
  }
};

// The wave's slice of a chunk's values.
template <int KS, int ET, int NPI, int SIZE>
__device__ __forceinline__ void read_values(const uint16_t (&v)[NPI][SIZE], int pitch, int wave, int lane,
                                            bf16x8_t (&val)[KS][ET][NPI]) {
#pragma unroll
  for (int ks = 0; ks < KS; ++ks)
#pragma unroll
    for (int et = 0; et < ET; ++et)
#pragma unroll
      for (int x = 0; x < NPI; ++x)
        val[ks][et][x] = read_columns(v[x] + ks * 32 * pitch + (wave * ET + et) * 16, pitch, lane);
}

// acc += weighted scores t [token][key] times values; keys before (or behind) a token's are not read.
template <bool REV, int IT, int KS, int ET, int NP, int NPI, int SIZE>
__device__ __forceinline__ void add_scores(const uint16_t (&t)[NP][SIZE], int pitch, const bf16x8_t (&val)[KS][ET][NPI],
                                           int lane, v4f (&acc)[IT][ET]) {
#pragma unroll
  for (int it = 0; it < IT; ++it)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      if (REV ? ks < (it >> 1) : ks > (it >> 1)) continue;
      bf16x8_t c[NP];
#pragma unroll
      for (int x = 0; x < NP; ++x) c[x] = read_rows(t[x] + it * 16 * pitch + ks * 32, pitch, lane);
#pragma unroll
      for (int et = 0; et < ET; ++et) acc[it][et] = mfma_planes(val[ks][et], c, acc[it][et]);
    }
}

// Values that are not finite.  A score that its mask makes 0 is multiplied all the same, and 0
// times NaN or infinity is NaN: such values are 0 in the products (drop_odd, which tells
// whether the wave has any) and reach the tokens that they count for in a walk of their own.
// The test and the branch take 6% of the training pass below (690 -> 735 us); with a flag from
// the threads that store the values, or without a branch, it took as much or more.
template <int KS, int ET, int NPI>
__device__ __forceinline__ bool drop_odd(bf16x8_t (&val)[KS][ET][NPI]) {
  auto odd_of = [](uint32_t w) { return ((w & 0x7F807F80u) + 0x00800080u) & 0x80008000u; };      // exponents all ones
  uint32_t any = 0;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks)
#pragma unroll
    for (int et = 0; et < ET; ++et) {
      const v4i w = __builtin_bit_cast(v4i, val[ks][et][0]);
#pragma unroll
      for (int i = 0; i < 4; ++i) any |= odd_of((uint32_t)w[i]);
    }
  if (!__any(any != 0)) return false;
#pragma unroll
  for (int ks = 0; ks < KS; ++ks)
#pragma unroll
    for (int et = 0; et < ET; ++et) {
      const v4i top = __builtin_bit_cast(v4i, val[ks][et][0]);
#pragma unroll
      for (int x = 0; x < NPI; ++x) {
        v4i w = __builtin_bit_cast(v4i, val[ks][et][x]);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t odd = odd_of((uint32_t)top[i]);
          w[i] &= (int)~(odd | (odd - (odd >> 15)));
        }
        val[ks][et][x] = __builtin_bit_cast(bf16x8_t, w);
      }
    }
  return true;
}
// acc += scores t [token][key] times the values v [key][value] that are not finite.
template <bool REV, int L, int IT, int ET, int NP, int NPI, int TS, int VS>
__device__ __forceinline__ void add_odd(const uint16_t (&t)[NP][TS], int pt, const uint16_t (&v)[NPI][VS], int pv, int wave,
                                        int lane, v4f (&acc)[IT][ET]) {
  const int l16 = lane & 15, g4 = lane >> 4;
#pragma unroll 1
  for (int j = 0; j < L; ++j) {
#pragma unroll
    for (int et = 0; et < ET; ++et) {
      float x[4] = {};
#pragma unroll
      for (int c = NPI - 1; c >= 0; --c) {
        float y[4];
        widen4(*reinterpret_cast<const u32x2_t*>(v[c] + j * pv + (wave * ET + et) * 16 + g4 * 4), y);
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] += y[r];
      }
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        const int i = it * 16 + l16;
        if (REV ? j < i : j > i) continue;
        float w = 0.0f;
#pragma unroll
        for (int c = NP - 1; c >= 0; --c) w += load_elem(t[c] + i * pt + j);
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (!((f2u(x[r]) & 0x7F800000u) < 0x7F800000u)) acc[it][et][r] += w * x[r];
      }
    }
  }
}

// 16 x 16 products of two arrays' rows; rows of the result are a's.
template <int DK, int NPI, int SIZE>
__device__ __forceinline__ v4f row_products(const uint16_t (&a)[NPI][SIZE], int ra, const uint16_t (&b)[NPI][SIZE], int rb,
                                            int pitch, int lane) {
  v4f s = {};
#pragma unroll
  for (int ks = 0; ks < DK; ++ks) {
    bf16x8_t x[NPI], y[NPI];
#pragma unroll
    for (int i = 0; i < NPI; ++i) {
      x[i] = read_rows(a[i] + ra * pitch + ks * 32, pitch, lane);
      y[i] = read_rows(b[i] + rb * pitch + ks * 32, pitch, lane);
    }
    s = mfma_planes(x, y, s);
  }
  return s;
}

template <int NP, int SIZE>
__device__ __forceinline__ void write_scores(uint16_t (&t)[NP][SIZE], int at, float (&w)[4]) {
  uint32_t o[NP][2];
  split<NP, 4>(w, o);
#pragma unroll
  for (int x = 0; x < NP; ++x) *reinterpret_cast<u32x2_t*>(t[x] + at) = u32x2_t{o[x][0], o[x][1]};
}

// A segment's chunks, one workgroup; OUT false: its state alone, from zero.
//
// The four waves own slices of the value axis: a slice's state stays in registers, in
// the layout in which the MFMA returns it, and is an operand of the next chunk's
// products as it lies (read_rows_halves gives the other operand in its K order).  The
// scores of a chunk are shared: wave w computes those of its 16 queries, weights and
// masks them, and all read them from LDS.
template <typename T, int NP, int NS, int L, int DP, int EP, bool OUT, bool FULL>
__global__ __launch_bounds__(kThreads, NS <= 2 && DP + EP == 128 ? 3 : 2) void k_mix(MixArgs p) {
  constexpr int NPI = sizeof(T) == 2 ? 1 : 3, IT = L / 16, KS = L / 32, DT = DP / 16, ET = EP / 64;
  constexpr bool DOT = OUT && NS == 3;
  using M = Lds<NPI, NP, L, DP, EP, OUT>;
  __shared__ M m;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g4 = lane >> 4;
  const int units = OUT ? p.nseg : (p.nseg - 1) * p.parts;      // OUT false: the walk's last segment is not needed
  const int bh = blockIdx.x / units, unit = blockIdx.x - bh * units, walk = OUT ? unit : unit / p.parts;
  const int b = bh / p.H, h = bh - b * p.H, seg = !OUT && p.rev ? p.nseg - 1 - walk : walk;
  int64_t length = p.T;
  if (p.lengths) length = min(max(p.lengths[b], (int64_t)0), (int64_t)p.T);
  const int chunks = (p.T + L - 1) / L;
  int c_lo = seg * p.per, c_hi = min(c_lo + p.per, chunks);
  if constexpr (!OUT) {
    const int before = (unit - walk * p.parts) * p.per_part;
    if (p.rev) {
      c_hi -= before;
      c_lo = max(c_lo, c_hi - p.per_part);
    } else {
      c_lo += before;
      c_hi = min(c_hi, c_lo + p.per_part);
    }
  }
  const int n = max(c_hi - c_lo, 0);
  auto first_of = [&](int i) { return (!OUT && p.rev ? c_hi - 1 - i : c_lo + i) * L; };     // chunk i of the walk

  Rows<T, L, DP, kThreads, FULL> rq(OUT ? p.q : p.k, b, h, length, p.dq), rk(p.k, b, h, length, p.dq);
  Rows<T, L, EP, kThreads, FULL> rv(p.v, b, h, length, p.dv);
  auto load = [&](int t0) {
    if constexpr (OUT) rq.load(t0);
    rk.load(t0);
    rv.load(t0);
  };
  auto store = [&] {
    if constexpr (OUT) rq.store(m.q, M::PD);
    rk.store(m.k, M::PD);
    rv.store(m.v, M::PE);
  };
  const int64_t gate_at = b * p.gb + h * p.gh;
  auto gate = [&](int t0) {
    return load_gate(p.g, p.g_bf16, gate_at, p.gt, t0 + lane, min(length, (int64_t)t0 + L));
  };
  double sum_all = 0.0;

  State<DT, ET> S;
  const int64_t state_at = OUT ? ((int64_t)bh * p.nseg + seg) * p.init_seg : 0;
  if (OUT && p.init)
    S.each(p.dq, p.dv, wave, lane, [&](float& s, int d, int e) {
      s = p.init[state_at + (int64_t)d * p.init_r + (int64_t)e * p.init_c];
    });
  [[maybe_unused]] const int e0 = wave * ET * 16 + g4 * 4;
  [[maybe_unused]] const Lane4<T, FULL> out(OUT ? p.out : p.k, b, h, p.T, p.dv, e0, l16);
  [[maybe_unused]] const Lane4<T, FULL> dotted(DOT && p.dot ? p.x : p.k, b, h, length, p.dv, e0, l16);

  float g_next = 0.0f;
  if (n > 0) {
    load(first_of(0));
    if (wave == 0) {
      sum_all += cumulate(gate(first_of(0)), m.gates, 0, lane);
      if (n > 1) g_next = gate(first_of(1));
    }
    store();
  }
  __syncthreads();
  for (int i = 0; i < n; ++i) {
    const int t0 = first_of(i), par = i & 1;
    [[maybe_unused]] typename Lane4<T, FULL>::Raw raw_x[DOT ? IT : 1][ET];
    if (DOT && p.dot) {
#pragma unroll
      for (int it = 0; it < IT; ++it)
#pragma unroll
        for (int et = 0; et < ET; ++et) raw_x[it][et] = dotted.ask(t0 + it * 16, et * 16);
    }
    if (i + 1 < n) load(first_of(i + 1));
    if (wave == 0 && i + 1 < n) {
      sum_all += cumulate(g_next, m.gates, par ^ 1, lane);
      if (i + 2 < n) g_next = gate(first_of(i + 2));
    }
    v4f acc[IT][ET];
    if constexpr (OUT) {
      // scores of queries 16 it .. with keys 16 jt ..: rows of the result are keys
#pragma unroll
      for (int j = 0; j < (L == 64 ? 4 : 1); ++j) {
        const int it = L == 64 ? wave : wave >> 1, jt = L == 64 ? j : wave & 1;
        if (jt > it && (jt >> 1) != (it >> 1)) continue;       // not read
        const int qi = it * 16 + l16, kj = jt * 16 + g4 * 4;
        float w[4] = {};
        if (jt <= it) {
          const v4f s = row_products<DP / 32>(m.k, jt * 16, m.q, it * 16, M::PD, lane);
          const int behind = opaque(qi - kj);
          const float hq = m.gates.hi[par][qi], lq = m.gates.lo[par][qi];
          const v4f hk = *reinterpret_cast<const v4f*>(&m.gates.hi[par][kj]);
          const v4f lk = *reinterpret_cast<const v4f*>(&m.gates.lo[par][kj]);
#pragma unroll
          for (int r = 0; r < 4; ++r)
            w[r] = r <= behind ? s[r] * __expf((hq - hk[r]) + (lq - lk[r])) * p.scale : 0.0f;
        }
        write_scores(m.t, qi * M::PT + kj, w);
      }
      // what the queries read of the state
      S.template read<NS>(m.q, M::PD, lane, acc);
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        const float w = m.gates.start[par][it * 16 + l16] * p.scale;
        float dot = 0.0f;
#pragma unroll
        for (int et = 0; et < ET; ++et) {
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[it][et][r] *= w;
          if (DOT && p.dot) {
            float x[4];
            dotted.load(t0 + it * 16, l16, et * 16, raw_x[DOT ? it : 0][et], x);
#pragma unroll
            for (int r = 0; r < 4; ++r) dot += x[r] * acc[it][et][r];
          }
        }
        if (DOT && p.dot) {
          dot += __shfl_xor(dot, 16, 64);
          dot += __shfl_xor(dot, 32, 64);
          if (g4 == 0) m.dot[wave][it * 16 + l16] = dot;
        }
      }
    }
    bf16x8_t val[KS][ET][NPI];
    read_values(m.v, M::PE, wave, lane, val);
    S.update(m.k, M::PD, val, !OUT && p.rev ? m.gates.start[par] : m.gates.rest[par], p.kscale, m.gates.total[par], lane);
    __syncthreads();                    // scores are whole
    if constexpr (OUT) {
      const bool odd = drop_odd(val);
      add_scores<false>(m.t, M::PT, val, lane, acc);
      if (odd) add_odd<false, L>(m.t, M::PT, m.v, M::PE, wave, lane, acc);
      const int end = (int)min(length - t0, (int64_t)L);
      // acc[it][et][r]: token 16 it + l16, value 16 (wave ET + et) + 4 g4 + r
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        const bool here = it * 16 + opaque(l16) < end;
#pragma unroll
        for (int et = 0; et < ET; ++et) {
          float o[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) o[r] = here ? acc[it][et][r] : 0.0f;
          out.store(t0 + it * 16, l16, et * 16, o);
        }
      }
    }
    if (DOT && p.dot && threadIdx.x < L && t0 + (int)threadIdx.x < p.T)
      p.dot[(int64_t)bh * p.T + t0 + threadIdx.x] =
          (m.dot[0][threadIdx.x] + m.dot[1][threadIdx.x]) + (m.dot[2][threadIdx.x] + m.dot[3][threadIdx.x]);
    __syncthreads();                    // this chunk's arrays are read
    if (i + 1 < n) store();
    __syncthreads();
  }

  if (p.last && (!OUT || walk == p.nseg - 1)) {
    float* to = p.last + (OUT ? (int64_t)bh : (int64_t)blockIdx.x) * p.last_seg;
    S.each(p.dq, p.dv, wave, lane, [&](float& s, int d, int e) { to[(int64_t)d * p.last_r + (int64_t)e * p.last_c] = s; });
  }
  if (!OUT && threadIdx.x == 0) p.decay[blockIdx.x] = (float)exp(sum_all);
}

// The states before the segments, in the walk's order, from the parts' own.
__global__ __launch_bounds__(256) void k_mix_join(float* __restrict__ states, const float* __restrict__ parts,
                                                  const float* __restrict__ decay, const float* __restrict__ init,
                                                  int64_t size, int nseg, int per, int rev) {
  const int64_t bh = blockIdx.x, e = (int64_t)blockIdx.y * 256 + threadIdx.x;
  if (e >= size) return;
  const int64_t first = bh * (nseg - 1) * per;
  float s = init ? init[bh * size + e] : 0.0f;
  for (int w = 0;; ++w) {
    states[(bh * nseg + (rev ? nseg - 1 - w : w)) * size + e] = s;
    if (w + 1 == nseg) return;
#pragma unroll 4
    for (int i = 0; i < per; ++i) {
      const int64_t at = first + w * per + i;
      s = decay[at] * s + parts[at * size + e];
    }
  }
}

// Gradients of k, v and the log decays.
struct BackArgs {
  Array q, k, v, g;                // g: the output's gradient
  Array dk, dv;
  const void* a;                   // log decays [B, T, H]
  int64_t ab, at, ah;
  int a_bf16;
  const int64_t* lengths;
  const float* r_ends;             // R behind the segments, or behind the last token (nseg 1; may be null)
  const float* s_starts;           // S before the segments (nseg > 1)
  const float* s_last;             // S behind the last token; null: R there is 0
  const float* dot_q;              // [B H][T]: q . what dq has from the state before its chunk
  void* da;                        // [B, T, H], or null
  float* dstate;                   // R before the first token, or null
  int B, T, H, dq, dv_, nseg, per;
  float scale;
};

template <int NPI, int NP, int L, int DP, int EP>
struct BackLds {
  static constexpr int PD = DP + 8, PE = EP + 8, PT = L + 8;
  alignas(16) uint16_t q[NPI][L * PD], k[NPI][L * PD], v[NPI][L * PE], g[NPI][L * PE];
  alignas(16) uint16_t ta[NP][L * PT], tb[NP][L * PT];
  Gates<L> gates;
  float rows[L / 16][L], cols[L / 16][L];      // sums of the scores' products P, see k_mix_back
  float dot[4][L];                             // k . what dk has from the state behind its chunk
  double part[4];
};

template <typename T, int L, int DP, int EP, bool FULL, bool KEYS, typename M>
__device__ __forceinline__ void mix_back(const BackArgs& p, M& m) {
  constexpr int NPI = sizeof(T) == 2 ? 1 : 3, NP = sizeof(T) == 2 ? 2 : 3, IT = L / 16, KS = L / 32, THREADS = 2 * kThreads;
  constexpr int TILES = IT * (IT + 1) / 2;
  // the role's products: outputs of EO values from states [DO, EO]
  constexpr int DO = KEYS ? EP : DP, EO = KEYS ? DP : EP, ET = EO / 64;
  const int lane = threadIdx.x & 63, wave8 = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wave = wave8 & 3;
  const int l16 = lane & 15, g4 = lane >> 4;
  const int bh = blockIdx.x / p.nseg, seg = p.nseg - 1 - (blockIdx.x - bh * p.nseg), b = bh / p.H, h = bh - b * p.H;
  int64_t length = p.T;
  if (p.lengths) length = min(max(p.lengths[b], (int64_t)0), (int64_t)p.T);
  const int chunks = (p.T + L - 1) / L, c_lo = seg * p.per, c_hi = min(c_lo + p.per, chunks), n = max(c_hi - c_lo, 0);
  auto first_of = [&](int i) { return (c_hi - 1 - i) * L; };

  Rows<T, L, DP, THREADS, FULL> rq(p.q, b, h, length, p.dq), rk(p.k, b, h, length, p.dq);
  Rows<T, L, EP, THREADS, FULL> rv(p.v, b, h, length, p.dv_), rg(p.g, b, h, length, p.dv_);
  auto load = [&](int t0) {
    rq.load(t0);
    rk.load(t0);
    rv.load(t0);
    rg.load(t0);
  };
  auto store = [&] {
    rq.store(m.q, M::PD);
    rk.store(m.k, M::PD);
    rv.store(m.v, M::PE);
    rg.store(m.g, M::PE);
  };
  const int64_t gate_at = b * p.ab + h * p.ah;
  auto gate = [&](int t0) {
    return load_gate(p.a, p.a_bf16, gate_at, p.at, t0 + lane, min(length, (int64_t)t0 + L));
  };

  // R [dk, dv], or transposed, and <S, R> behind the segment
  const int64_t size = (int64_t)p.dq * p.dv_;
  const float* r_end = p.r_ends ? p.r_ends + ((int64_t)bh * p.nseg + seg) * size : nullptr;
  State<DO / 16, ET> R;
  if (r_end) {
    if constexpr (KEYS) {
      R.each(p.dv_, p.dq, wave, lane, [&](float& s, int d, int e) { s = r_end[(int64_t)e * p.dv_ + d]; });
    } else {
      R.each(p.dq, p.dv_, wave, lane, [&](float& s, int d, int e) { s = r_end[(int64_t)d * p.dv_ + e]; });
    }
  }
  if constexpr (!KEYS) {
    double sum = 0.0;
    const float* S = seg + 1 < p.nseg ? p.s_starts + ((int64_t)bh * p.nseg + seg + 1) * size
                     : p.s_last       ? p.s_last + bh * size
                                      : nullptr;
    if (p.da && r_end && S) {
      float f = 0.0f;
      R.each(p.dq, p.dv_, wave, lane, [&](float& s, int d, int e) { f += s * S[(int64_t)d * p.dv_ + e]; });
      sum = f;
#pragma unroll
      for (int k = 32; k; k >>= 1) sum += __shfl_xor(sum, k, 64);
    }
    if (lane == 0) m.part[wave] = sum;
  }
  // what no tile writes stays 0
  for (int i = threadIdx.x; i < NP * L * M::PT; i += THREADS) (&m.ta[0][0])[i] = (&m.tb[0][0])[i] = 0;
  for (int i = threadIdx.x; i < IT * L; i += THREADS) (&m.rows[0][0])[i] = (&m.cols[0][0])[i] = 0.0f;

  const Lane4<T, FULL> out(KEYS ? p.dk : p.dv, b, h, p.T, KEYS ? p.dq : p.dv_, wave * ET * 16 + g4 * 4, l16);
  constexpr int GATES = 7, SUMS = 6;           // waves with the fewest tiles of scores
  float g_next = 0.0f;
  if (n > 0) {
    load(first_of(0));
    if (wave8 == GATES) {
      cumulate(gate(first_of(0)), m.gates, 0, lane);
      if (n > 1) g_next = gate(first_of(1));
    }
    store();
  }
  __syncthreads();
  [[maybe_unused]] double carry = 0.0;
  if (wave8 == SUMS) carry = (m.part[0] + m.part[1]) + (m.part[2] + m.part[3]);
  for (int i = 0; i < n; ++i) {
    const int t0 = first_of(i), par = i & 1;
    if (i + 1 < n) load(first_of(i + 1));
    if (wave8 == GATES && i + 1 < n) {
      cumulate(g_next, m.gates, par ^ 1, lane);
      if (i + 2 < n) g_next = gate(first_of(i + 2));
    }
    // token of a lane of the wave that sums: the last one first
    [[maybe_unused]] const int ti = L - 1 - opaque(lane);
    [[maybe_unused]] float dq_dot = 0.0f, own = 0.0f;
    [[maybe_unused]] const bool sums = wave8 == SUMS && p.da;
    if (KEYS && sums && ti >= 0 && t0 + ti < length) {
      dq_dot = p.dot_q[(int64_t)bh * p.T + t0 + ti];
      const int64_t at = gate_at + (t0 + ti) * p.at;
      own = p.a_bf16 ? load_elem(static_cast<const uint16_t*>(p.a) + at) : static_cast<const float*>(p.a)[at];
    }
    // tokens i of tile it and behind them j of tile jt: w = c e^(G_j - G_i), a = w (q_j . k_i),
    // b = w (v_i . do_j), P = w (q_j . k_i) (v_i . do_j); rows of a result are j's
#pragma unroll
    for (int u = 0; u < (TILES + 7) / 8; ++u) {
      const int t = wave8 + 8 * u;
      if (t >= TILES) continue;
      // 0 1 2 3 | 1 2 3 | 2 3 | 3 behind 0 | 1 | 2 | 3
      const int it = L == 64 ? (t >= 4) + (t >= 7) + (t >= 9) : t >> 1;
      const int jt = L == 64 ? t - (it == 0 ? 0 : it == 1 ? 3 : it == 2 ? 5 : 6) : (t + 1) >> 1;
      const v4f a = row_products<DP / 32>(m.q, jt * 16, m.k, it * 16, M::PD, lane);
      const v4f o = row_products<EP / 32>(m.g, jt * 16, m.v, it * 16, M::PE, lane);
      const int ii = it * 16 + l16, jj = jt * 16 + g4 * 4;
      const float hi = m.gates.hi[par][ii], li = m.gates.lo[par][ii];
      const v4f hj = *reinterpret_cast<const v4f*>(&m.gates.hi[par][jj]);
      const v4f lj = *reinterpret_cast<const v4f*>(&m.gates.lo[par][jj]);
      const int behind = opaque(ii - jj);
      float wa[4], wb[4], P[4], sum = 0.0f;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const float w = __expf((hj[r] - hi) + (lj[r] - li)) * p.scale;
        const bool in = r >= behind;
        wa[r] = in ? a[r] * w : 0.0f;
        wb[r] = in ? o[r] * w : 0.0f;
        P[r] = in ? a[r] * wb[r] : 0.0f;
        sum += P[r];
      }
      write_scores(m.ta, ii * M::PT + jj, wa);
      write_scores(m.tb, ii * M::PT + jj, wb);
      if (p.da) {
        sum += __shfl_xor(sum, 16, 64);
        sum += __shfl_xor(sum, 32, 64);
        if (g4 == 0) m.cols[jt][ii] = sum;
        // sums over the 16 lanes of a token i: the lanes take r = l16 mod 4 in two steps
        const int l = opaque(l16);
        const bool odd = l & 1, high = l & 2;
        float x = odd ? P[1] : P[0], y = odd ? P[3] : P[2];
        x += __shfl_xor(odd ? P[0] : P[1], 1, 64);
        y += __shfl_xor(odd ? P[2] : P[3], 1, 64);
        float z = high ? y : x;
        z += __shfl_xor(high ? x : y, 2, 64);
        z += __shfl_xor(z, 4, 64);
        z += __shfl_xor(z, 8, 64);
        if (l < 4) m.rows[it][jj + l16] = z;
      }
    }
    // what the tokens read of the state behind the chunk
    v4f acc[IT][ET];
    bf16x8_t val[KS][ET][NPI];
    if constexpr (KEYS) R.template read<3>(m.v, M::PE, lane, acc);
    else R.template read<NP>(m.k, M::PD, lane, acc);
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const float w = m.gates.rest[par][it * 16 + l16];
      float dot = 0.0f;
#pragma unroll
      for (int et = 0; et < ET; ++et)
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[it][et][r] *= w;
      if constexpr (KEYS) {
        if (p.da) {
#pragma unroll
          for (int et = 0; et < ET; ++et) {
            const int e = (wave * ET + et) * 16 + g4 * 4;
            float x[4] = {};
#pragma unroll
            for (int c = NPI - 1; c >= 0; --c) {
              float y[4];
              widen4(*reinterpret_cast<const u32x2_t*>(m.k[c] + (it * 16 + l16) * M::PD + e), y);
#pragma unroll
              for (int r = 0; r < 4; ++r) x[r] += y[r];
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) dot += x[r] * acc[it][et][r];
          }
          dot += __shfl_xor(dot, 16, 64);
          dot += __shfl_xor(dot, 32, 64);
          if (g4 == 0) m.dot[wave][it * 16 + l16] = dot;
        }
      }
    }
    if constexpr (KEYS) {
      read_values(m.q, M::PD, wave, lane, val);
      R.update(m.g, M::PE, val, m.gates.start[par], p.scale, m.gates.total[par], lane);
    } else {
      read_values(m.g, M::PE, wave, lane, val);
      R.update(m.q, M::PD, val, m.gates.start[par], p.scale, m.gates.total[par], lane);
    }
    __syncthreads();                    // scores are whole
    const bool odd = drop_odd(val);
    add_scores<true>(KEYS ? m.tb : m.ta, M::PT, val, lane, acc);
    if (odd) {
      if constexpr (KEYS) add_odd<true, L>(m.tb, M::PT, m.q, M::PD, wave, lane, acc);
      else add_odd<true, L>(m.ta, M::PT, m.g, M::PE, wave, lane, acc);
    }
    const int end = (int)min(length - t0, (int64_t)L);
#pragma unroll
    for (int it = 0; it < IT; ++it) {
      const bool here = it * 16 + opaque(l16) < end;
#pragma unroll
      for (int et = 0; et < ET; ++et) {
        float o[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r] = here ? acc[it][et][r] : 0.0f;
        out.store(t0 + it * 16, l16, et * 16, o);
      }
    }
    if constexpr (KEYS) {
      if (sums) {
        double s = 0.0;
        if (ti >= 0) {
          float r = 0.0f, c = 0.0f;
#pragma unroll
          for (int x = 0; x < IT; ++x) {
            r += m.rows[x][ti];
            c += m.cols[x][ti];
          }
          s = ((double)r - (double)c) + ((double)dq_dot -
              (double)((m.dot[0][ti] + m.dot[1][ti]) + (m.dot[2][ti] + m.dot[3][ti])));
        }
#pragma unroll
        for (int k = 1; k < L; k <<= 1) {
          const double o = __shfl_up(s, k, 64);
          if (L - 1 - ti >= k) s += o;
        }
        s += carry;
        carry = __shfl(s, L - 1, 64);
        if (ti >= 0 && t0 + ti < p.T) {
          // e^a is 0 in f32 below -104: nothing passes
          const float d = t0 + ti < length && !(own < -104.0f) ? (float)s : 0.0f;
          const int64_t at = ((int64_t)b * p.T + t0 + ti) * p.H + h;
          if (p.a_bf16) store_elem(static_cast<uint16_t*>(p.da) + at, d);
          else static_cast<float*>(p.da)[at] = d;
        }
      }
    }
    __syncthreads();                    // this chunk's arrays are read
    if (i + 1 < n) store();
    __syncthreads();
  }
  if constexpr (!KEYS) {
    if (p.dstate && seg == 0)
      R.each(p.dq, p.dv_, wave, lane, [&](float& s, int d, int e) { p.dstate[bh * size + (int64_t)d * p.dv_ + e] = s; });
  }
}

// A segment's gradients of k, v and the decays, from its last chunk to its first: eight
// waves, of which four own slices of R [dk, dv] and give dv, four slices of R^T and dk.
// A chunk's scores are shared among all.  For the decays q . dq and k . dk of tokens of
// one chunk are sums of one matrix' rows and columns: with
// P_ij = c e^(G_j - G_i) (q_j . k_i) (v_i . do_j), i <= j, q_j . dq_j has sum_i P_ij and
// k_i . dk_i sum_j P_ij, which needs no gradient in more than its own type; what comes
// from states is taken from products with three planes of them.
template <typename T, int L, int DP, int EP, bool FULL>
__global__ __launch_bounds__(2 * kThreads, DP + EP == 128 ? 4 : 2) void k_mix_back(BackArgs p) {
  constexpr int NPI = sizeof(T) == 2 ? 1 : 3;
  using M = BackLds<NPI, sizeof(T) == 2 ? 2 : 3, L, DP, EP>;
  __shared__ M m;
  if (__builtin_amdgcn_readfirstlane(threadIdx.x >> 8)) mix_back<T, L, DP, EP, FULL, true>(p, m);
  else mix_back<T, L, DP, EP, FULL, false>(p, m);
}

// One token: S = e^g S + k^T v in place, o = c q S.  A workgroup a head; a thread
// takes 4 values of every 64th (or so) row of the state.  Bound: HBM, the state read
// and written.
struct StepArgs {
  const void *q, *k, *v, *g;
  void* out;
  float* state;
  int64_t qb, qh, kb, kh, vb, vh, gb, gh;
  int g_bf16, H, dk, dv;
  float scale;
};
template <typename T>
__global__ __launch_bounds__(256) void k_mix_step(StepArgs p) {
  __shared__ float qs[128], ks[128];
  __shared__ float part[256 * 4];
  const int bh = blockIdx.x, b = bh / p.H, h = bh - b * p.H, tid = threadIdx.x;
  const int64_t gi = b * p.gb + h * p.gh;
  const float a = expf(p.g_bf16 ? load_elem(static_cast<const uint16_t*>(p.g) + gi) : static_cast<const float*>(p.g)[gi]);
  if (tid < p.dk) qs[tid] = load_elem(static_cast<const T*>(p.q) + b * p.qb + h * p.qh + tid);
  else if (tid >= 128 && tid - 128 < p.dk) ks[tid - 128] = load_elem(static_cast<const T*>(p.k) + b * p.kb + h * p.kh + tid - 128);
  const int cols = (p.dv + 3) / 4, rows = 256 / cols;      // cols 1 .. 32
  const int e = tid % cols * 4, r0 = tid / cols;
  float v[4], o[4] = {};
  load_some(static_cast<const T*>(p.v) + b * p.vb + h * p.vh + e, p.dv - e, 0.0f, v);
  float* S = p.state + (int64_t)bh * p.dk * p.dv;
  __syncthreads();
  if (r0 < rows) {
    if (p.dv % 4 == 0) {
      for (int d = r0; d < p.dk; d += rows) {
        float4* at = reinterpret_cast<float4*>(S + d * p.dv + e);
        float4 s = *at;
        s.x = a * s.x + ks[d] * v[0];
        s.y = a * s.y + ks[d] * v[1];
        s.z = a * s.z + ks[d] * v[2];
        s.w = a * s.w + ks[d] * v[3];
        *at = s;
        o[0] += qs[d] * s.x;
        o[1] += qs[d] * s.y;
        o[2] += qs[d] * s.z;
        o[3] += qs[d] * s.w;
      }
    } else {
      for (int d = r0; d < p.dk; d += rows)
        for (int i = 0; i < 4 && e + i < p.dv; ++i) {
          const float s = a * S[d * p.dv + e + i] + ks[d] * v[i];
          S[d * p.dv + e + i] = s;
          o[i] += qs[d] * s;
        }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) part[tid * 4 + i] = o[i];
  __syncthreads();
  if (tid < p.dv) {
    float s = 0.0f;
    for (int r = 0; r < rows; ++r) s += part[(r * cols + tid / 4) * 4 + tid % 4];
    store_elem(static_cast<T*>(p.out) + (int64_t)bh * p.dv + tid, s * p.scale);
  }
}

// --------------------------------------------------------------------------
// host
// --------------------------------------------------------------------------
constexpr int kMaxHead = 128;

struct Shape {
  int64_t B, T, H, dk, dv;
  int dtype;
  bool train;                      // a backward pass follows, of the same segments
  int L() const { return dtype == PRATCHYA_DT_BF16 ? 64 : 32; }
  int64_t chunks() const { return (T + L() - 1) / L(); }
  // Segments of a sequence: what the compute units hold at once of the kernels that walk
  // them, each of at least four chunks.  (Training, 8 x 4096 tokens of 32 heads of 64, both
  // passes: two workgroups a unit 692 us, three 745, four 783; a prompt of 8192 tokens of
  // 64 heads: two 119, three 105, four 127.)
  int64_t segments() const {
    const int64_t heads = B * H, most = T / (4 * L());
    if (heads < 1) return 1;
    int64_t n = 256 * (!train && dk <= 64 && dv <= 64 ? 3 : 2) / heads;
    if (n > most) n = most;
    if (n < 1) n = 1;
    const int64_t each = (chunks() + n - 1) / n;
    return each ? (chunks() + each - 1) / each : 1;
  }
  int64_t per() const {
    const int64_t n = segments();
    return (chunks() + n - 1) / n;
  }
  int64_t state() const { return dk * dv; }
  // Parts of a segment whose states are taken at once: about four workgroups a compute
  // unit, of two chunks or more.
  int64_t parts() const {
    const int64_t units = B * H * (segments() - 1), most = per() / 2;
    if (units < 1) return 1;
    int64_t n = 1024 / units;
    if (n > most) n = most;
    return n < 1 ? 1 : n;
  }
  // states before the segments; of their parts, with their decays
  int64_t states_floats() const { return segments() > 1 ? B * H * segments() * state() : 0; }
  int64_t parts_floats() const { return B * H * (segments() - 1) * parts() * (state() + 1); }
  int64_t starts_floats() const { return states_floats() + parts_floats(); }
};

int check_shape(const char* what, const Shape& s, int g_dtype) {
  if (!is_float_dtype(s.dtype) || !is_float_dtype(g_dtype))
    return pratchya_set_error(PRATCHYA_EINVAL, "%s: unsupported dtypes %d, %d", what, s.dtype, g_dtype);
  if (s.B < 0 || s.T < 0 || s.H < 1 || s.dk < 1 || s.dv < 1)
    return pratchya_set_error(PRATCHYA_EINVAL, "%s: [%lld, %lld, %lld] of heads of %lld and %lld", what, (long long)s.B,
                              (long long)s.T, (long long)s.H, (long long)s.dk, (long long)s.dv);
  if (s.dk > kMaxHead || s.dv > kMaxHead || s.T > 0x7FFFFF00 || s.B > (1 << 24) || s.H > (1 << 24) ||
      !fits_launch(s.B * s.H * s.segments() * s.parts(), 2 * kThreads))
    return pratchya_set_error(PRATCHYA_EUNSUPPORTED, "%s: heads of more than %d, or 2^24 heads of segments", what, kMaxHead);
  return PRATCHYA_OK;
}

// Whether an array suits buffers: 16-byte vectors, rows that do not overlap, offsets
// below 2^31.
bool fits_buffer(const Array& x, int64_t T, int width, int elem) {
  const int64_t n = 16 / elem;
  return reinterpret_cast<uintptr_t>(x.p) % 16 == 0 && width % n == 0 && x.b % n == 0 && x.t % n == 0 && x.h % n == 0 &&
         x.t >= width && (T + 128) * x.t * elem <= 0x7FFFFFFF;
}

// f of the padded widths that a head's take
template <typename F>
void by_widths(int64_t d, int64_t e, F f) {
  using W64 = std::integral_constant<int, 64>;
  using W128 = std::integral_constant<int, 128>;
  if (d <= 64 && e <= 64) f(W64{}, W64{});
  else if (d <= 64) f(W64{}, W128{});
  else if (e <= 64) f(W128{}, W64{});
  else f(W128{}, W128{});
}

template <typename T, int NP, int NS, int L, bool OUT>
void launch_mix_as(const MixArgs& a, unsigned blocks, hipStream_t stream) {
  constexpr int E = sizeof(T);
  const bool full = fits_buffer(a.k, a.T, a.dq, E) && fits_buffer(a.v, a.T, a.dv, E) &&
                    (!OUT || (fits_buffer(a.q, a.T, a.dq, E) && fits_buffer(a.out, a.T, a.dv, E) &&
                              (!a.dot || fits_buffer(a.x, a.T, a.dv, E))));
  by_widths(a.dq, a.dv, [&](auto d, auto e) {
    constexpr int D = decltype(d)::value, V = decltype(e)::value;
    if (full) hipLaunchKernelGGL((k_mix<T, NP, NS, L, D, V, OUT, true>), dim3(blocks), dim3(kThreads), 0, stream, a);
    else hipLaunchKernelGGL((k_mix<T, NP, NS, L, D, V, OUT, false>), dim3(blocks), dim3(kThreads), 0, stream, a);
  });
}

int launch_mix(const Shape& s, const MixArgs& a, bool out, hipStream_t stream) {
  const int64_t blocks = s.B * s.H * (out ? a.nseg : (a.nseg - 1) * a.parts);
  if (!blocks) return PRATCHYA_OK;
  if (s.dtype == PRATCHYA_DT_BF16) {
    if (!out) launch_mix_as<uint16_t, 1, 1, 64, false>(a, (unsigned)blocks, stream);
    else if (a.dot) launch_mix_as<uint16_t, 2, 3, 64, true>(a, (unsigned)blocks, stream);
    else launch_mix_as<uint16_t, 2, 2, 64, true>(a, (unsigned)blocks, stream);
  } else {
    if (!out) launch_mix_as<float, 3, 3, 32, false>(a, (unsigned)blocks, stream);
    else launch_mix_as<float, 3, 3, 32, true>(a, (unsigned)blocks, stream);
  }
  return check_launch("linear_attention");
}

template <typename T, int L>
int launch_back(const Shape& s, const BackArgs& a, hipStream_t stream) {
  constexpr int E = sizeof(T);
  const unsigned blocks = (unsigned)(s.B * s.H * a.nseg);
  const bool full = fits_buffer(a.q, a.T, a.dq, E) && fits_buffer(a.k, a.T, a.dq, E) && fits_buffer(a.v, a.T, a.dv_, E) &&
                    fits_buffer(a.g, a.T, a.dv_, E) && fits_buffer(a.dk, a.T, a.dq, E) && fits_buffer(a.dv, a.T, a.dv_, E);
  by_widths(a.dq, a.dv_, [&](auto d, auto e) {
    constexpr int D = decltype(d)::value, V = decltype(e)::value;
    if (full) hipLaunchKernelGGL((k_mix_back<T, L, D, V, true>), dim3(blocks), dim3(2 * kThreads), 0, stream, a);
    else hipLaunchKernelGGL((k_mix_back<T, L, D, V, false>), dim3(blocks), dim3(2 * kThreads), 0, stream, a);
  });
  return check_launch("linear_attention_bwd");
}

// What all walks of a call share.
MixArgs base_args(const Shape& s, const void* g, int g_dtype, const int64_t* gs, const int64_t* lengths) {
  MixArgs a = {};
  a.g = g;
  a.gb = gs[0];
  a.gt = gs[1];
  a.gh = gs[2];
  a.g_bf16 = g_dtype == PRATCHYA_DT_BF16;
  a.lengths = lengths;
  a.B = (int)s.B;
  a.T = (int)s.T;
  a.H = (int)s.H;
  a.nseg = (int)s.segments();
  a.per = (int)s.per();
  return a;
}

Array array(const void* p, const int64_t* strides) { return {const_cast<void*>(p), strides[0], strides[1], strides[2]}; }
Array packed(const Shape& s, const void* p, int64_t d) {
  return {const_cast<void*>(p), s.T * s.H * d, s.H * d, d};
}

// The states before the segments (rev: behind them), where there are several.
int segment_states(const Shape& s, MixArgs a, float* starts, float* parts, const float* init, hipStream_t stream) {
  if (a.nseg < 2) return PRATCHYA_OK;
  const int64_t size = s.state(), n = s.B * s.H * (a.nseg - 1) * s.parts();
  a.parts = (int)s.parts();
  a.per_part = (a.per + a.parts - 1) / a.parts;
  a.last = parts;
  a.last_seg = size;
  a.last_r = a.dv;
  a.last_c = 1;
  a.decay = a.last + n * size;
  const int rc = launch_mix(s, a, false, stream);
  if (rc) return rc;
  hipLaunchKernelGGL(k_mix_join, dim3((unsigned)(s.B * s.H), (unsigned)((size + 255) / 256)), dim3(256), 0, stream,
                     starts, a.last, a.decay, init, size, a.nseg, a.parts, a.rev);
  return check_launch("linear_attention");
}

// Outputs from the states before the segments.  transposed: the state is held as
// [value, query] in memory.
int outputs(const Shape& s, MixArgs a, const float* starts, const float* init, bool transposed, float* last,
            hipStream_t stream) {
  a.init = a.nseg > 1 ? starts : init;
  a.init_seg = a.last_seg = s.state();
  a.init_r = a.last_r = transposed ? 1 : a.dv;
  a.init_c = a.last_c = transposed ? a.dq : 1;
  a.last = last;
  return launch_mix(s, a, true, stream);
}

}  // namespace

extern "C" int64_t pratchya_linear_attention_starts_floats(int64_t batch, int64_t length, int64_t heads, int64_t dk,
                                                           int64_t dv, int dtype, int train) {
  const Shape s = {batch, length, heads, dk, dv, dtype, train != 0};
  return check_shape("linear_attention", s, PRATCHYA_DT_F32) ? 0 : s.starts_floats();
}

extern "C" int64_t pratchya_linear_attention_states_floats(int64_t batch, int64_t length, int64_t heads, int64_t dk,
                                                           int64_t dv, int dtype, int train) {
  const Shape s = {batch, length, heads, dk, dv, dtype, train != 0};
  return check_shape("linear_attention", s, PRATCHYA_DT_F32) ? 0 : s.states_floats();
}

extern "C" int pratchya_linear_attention_parts(const void* q, const void* k, const void* v, int dtype, const void* log_decay,
                                               int g_dtype, const int64_t* strides, const int64_t* lengths,
                                               const float* state, int64_t batch, int64_t length, int64_t heads, int64_t dk,
                                               int64_t dv, float scale, int train, void* out, float* state_out,
                                               float* starts, float* parts, hipStream_t stream) {
  const char* what = "linear_attention";
  const Shape s = {batch, length, heads, dk, dv, dtype, train != 0};
  const int rc = check_shape(what, s, g_dtype);
  if (rc) return rc;
  if (batch == 0) return pratchya_set_error(PRATCHYA_OK, "");
  if (!strides || (length && (!q || !k || !v || !log_decay || !out)) || !state_out || (s.starts_floats() && !(starts && parts)))
    return pratchya_set_error(PRATCHYA_EINVAL, "%s: null buffer", what);
  MixArgs a = base_args(s, log_decay, g_dtype, strides + 9, lengths);
  a.q = array(q, strides);
  a.k = array(k, strides + 3);
  a.v = array(v, strides + 6);
  a.out = packed(s, out, dv);
  a.dq = (int)dk;
  a.dv = (int)dv;
  a.scale = scale;
  a.kscale = 1.0f;
  const int rc2 = segment_states(s, a, starts, parts, state, stream);
  return rc2 ? rc2 : outputs(s, a, starts, state, false, state_out, stream);
}

extern "C" int pratchya_linear_attention(const void* q, const void* k, const void* v, int dtype, const void* log_decay,
                                         int g_dtype, const int64_t* strides, const int64_t* lengths, const float* state,
                                         int64_t batch, int64_t length, int64_t heads, int64_t dk, int64_t dv,
                                         float scale, int train, void* out, float* state_out, float* starts,
                                         hipStream_t stream) {
  // the parts' states behind those that a backward pass reads
  float* parts = starts ? starts + pratchya_linear_attention_states_floats(batch, length, heads, dk, dv, dtype, train) : nullptr;
  return pratchya_linear_attention_parts(q, k, v, dtype, log_decay, g_dtype, strides, lengths, state, batch, length, heads, dk,
                                         dv, scale, train, out, state_out, starts, parts, stream);
}

extern "C" int64_t pratchya_linear_attention_bwd_workspace_bytes(int64_t batch, int64_t length, int64_t heads, int64_t dk,
                                                                 int64_t dv, int dtype) {
  const Shape s = {batch, length, heads, dk, dv, dtype, true};
  if (check_shape("linear_attention_bwd", s, PRATCHYA_DT_F32)) return 0;
  return 4 * (s.starts_floats() + batch * heads * length);
}

extern "C" int pratchya_linear_attention_bwd(const void* q, const void* k, const void* v, int dtype,
                                             const void* log_decay, int g_dtype, const int64_t* strides,
                                             const int64_t* lengths, const float* state, const float* state_out,
                                             const float* starts, const void* dout, const float* dstate_out,
                                             int64_t batch, int64_t length, int64_t heads, int64_t dk, int64_t dv,
                                             float scale, void* dq, void* dk_out, void* dv_out, void* dlog_decay,
                                             float* dstate, void* workspace, int64_t workspace_bytes,
                                             hipStream_t stream) {
  const char* what = "linear_attention_bwd";
  const Shape s = {batch, length, heads, dk, dv, dtype, true};
  int rc = check_shape(what, s, g_dtype);
  if (rc) return rc;
  if (batch == 0) return pratchya_set_error(PRATCHYA_OK, "");
  const int64_t need = pratchya_linear_attention_bwd_workspace_bytes(batch, length, heads, dk, dv, dtype);
  if (!strides || (length && (!q || !k || !v || !log_decay || !dout || !dq || !dk_out || !dv_out)) ||
      (s.starts_floats() && !starts) || (dlog_decay && dstate_out && !state_out))
    return pratchya_set_error(PRATCHYA_EINVAL, "%s: null buffer", what);
  if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 4))
    return pratchya_set_error(PRATCHYA_EINVAL, "%s: workspace of %lld bytes needed, 4-byte aligned", what, (long long)need);
  float* rstarts = static_cast<float*>(workspace);
  float* dot_q = rstarts + s.starts_floats();
  const MixArgs base = base_args(s, log_decay, g_dtype, strides + 9, lengths);
  const Array Q = array(q, strides), K = array(k, strides + 3), V = array(v, strides + 6), D = array(dout, strides + 12);
  // dq: queries do, keys v, values k, state S^T
  MixArgs a = base;
  a.q = D;
  a.k = V;
  a.v = K;
  a.out = packed(s, dq, dk);
  a.dq = (int)dv;
  a.dv = (int)dk;
  a.scale = scale;
  a.kscale = 1.0f;
  if (dlog_decay) {
    a.x = Q;
    a.dot = dot_q;
  }
  if ((rc = outputs(s, a, starts, state, true, nullptr, stream))) return rc;
  // R behind the segments: keys q, values do
  a = base;
  a.rev = 1;
  a.k = Q;
  a.v = D;
  a.dq = (int)dk;
  a.dv = (int)dv;
  a.kscale = scale;
  if ((rc = segment_states(s, a, rstarts, rstarts + s.states_floats(), dstate_out, stream))) return rc;
  BackArgs g = {};
  g.q = Q;
  g.k = K;
  g.v = V;
  g.g = D;
  g.dk = packed(s, dk_out, dk);
  g.dv = packed(s, dv_out, dv);
  g.a = log_decay;
  g.ab = strides[9];
  g.at = strides[10];
  g.ah = strides[11];
  g.a_bf16 = base.g_bf16;
  g.lengths = lengths;
  g.r_ends = base.nseg > 1 ? rstarts : dstate_out;
  g.s_starts = starts;
  g.s_last = dstate_out ? state_out : nullptr;
  g.dot_q = dot_q;
  g.da = dlog_decay;
  g.dstate = dstate;
  g.B = base.B;
  g.T = base.T;
  g.H = base.H;
  g.dq = (int)dk;
  g.dv_ = (int)dv;
  g.nseg = base.nseg;
  g.per = base.per;
  g.scale = scale;
  return dtype == PRATCHYA_DT_BF16 ? launch_back<uint16_t, 64>(s, g, stream) : launch_back<float, 32>(s, g, stream);
}

extern "C" int pratchya_linear_attention_step(const void* q, const void* k, const void* v, int dtype,
                                              const void* log_decay, int g_dtype, const int64_t* strides, float* state,
                                              int64_t batch, int64_t heads, int64_t dk, int64_t dv, float scale,
                                              void* out, hipStream_t stream) {
  const char* what = "linear_attention_step";
  const Shape s = {batch, 1, heads, dk, dv, dtype, false};
  const int rc = check_shape(what, s, g_dtype);
  if (rc) return rc;
  if (batch == 0) return pratchya_set_error(PRATCHYA_OK, "");
  if (!q || !k || !v || !log_decay || !strides || !state || !out)
    return pratchya_set_error(PRATCHYA_EINVAL, "%s: null buffer", what);
  if (reinterpret_cast<uintptr_t>(state) % 16)
    return pratchya_set_error(PRATCHYA_EINVAL, "%s: a state that is not 16-byte aligned", what);
  const StepArgs a = {q, k, v, log_decay, out, state, strides[0], strides[1], strides[2], strides[3], strides[4],
                      strides[5], strides[6], strides[7], g_dtype == PRATCHYA_DT_BF16, (int)heads, (int)dk, (int)dv, scale};
  const dim3 grid((unsigned)(batch * heads));
  if (dtype == PRATCHYA_DT_BF16) hipLaunchKernelGGL((k_mix_step<uint16_t>), grid, dim3(256), 0, stream, a);
  else hipLaunchKernelGGL((k_mix_step<float>), grid, dim3(256), 0, stream, a);
  return check_launch(what);
}
