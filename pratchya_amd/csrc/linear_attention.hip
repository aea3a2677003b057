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
//   dq       do     v      k      S^T
//   dk       v      do     q      R^T     backwards
//   dv       k      q      do     R       backwards
// so one kernel serves all four (k_mix).  A decay scales all that passes from before t
// to t or later: dg_t = sum over u >= t of (q_u . dq_u - k_u . dk_u) + <S_last, R_last>,
// taken from the end of a segment of the sequence, where S and R are known, so that the
// sum cancels over a segment at most.
//
// Products run on bf16 MFMAs.  Exact bf16 inputs are one plane; f32 values (f32 inputs,
// states, decayed values) are the sum of three, of which products of 2^-24 of the
// largest or more are taken.  States are f32, and what enters them is never rounded to
// less.  The scores and the state that outputs in bf16 read are rounded to bf16 once
// (each below the rounding of the output itself), but not where the decays' gradient
// is wanted: it is f32, and the dots that it sums read unrounded gradients.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "pratchya_fp8.h"
#include "row_device.h"
#include "row_host.h"

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v2i __attribute__((ext_vector_type(2)));
typedef int v4i __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));
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
  float* last;                     // state after the walk; without outputs: of every segment but its last
  float* decay;                    // without outputs: e^(sum of a segment's log decays), [B H][nseg]
  float* dot;                      // [B H][T]
  int64_t init_seg, last_seg;      // elements from a segment's state to the next one's
  int init_r, init_c, last_r, last_c;   // strides of a state's query and value axes
  int B, T, H, dq, dv, nseg, per;  // per: chunks of a segment
  int rev;
  float tscale, sscale, kscale;
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

__device__ __forceinline__ float top_piece(float v) { return u2f(f2u(v) & 0xFFFF0000u); }
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

constexpr int kThreads = 256;

template <int NPI, int NP, int L, int DP, int EP, bool OUT>
struct Lds {
  static constexpr int PD = DP + 8, PE = EP + 8, PT = L + 8;   // row pitches: no two rows of a read on one bank
  alignas(16) uint16_t q[OUT ? NPI : 1][OUT ? L * PD : 8];
  alignas(16) uint16_t k[NPI][L * PD];
  alignas(16) uint16_t v[NPI][L * PE];
  alignas(16) uint16_t t[NP][OUT ? L * PT : 8];
  // by chunk parity: cumulated log decays in two parts, weights of queries and keys
  float hi[2][L], lo[2][L], qw[2][L], kw[2][L], total[2];
  float dot[4][L];
};

// A thread's vectors of L rows of W (padded) columns.
template <typename T, int L, int W>
struct Rows {
  static constexpr int N = kN<T>, PER = W / N, V = L * PER / kThreads;
  u32x4_t raw[V];

  __device__ __forceinline__ void load(const T* p, int64_t step, int rows, int width) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int at = threadIdx.x + i * kThreads, r = at / PER, c = at % PER * N;
      raw[i] = u32x4_t{};
      if (r < rows && c < width) {
        const T* s = p + r * step + c;
        if (c + N <= width) {
          raw[i] = load_raw(s);
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
      const int at = threadIdx.x + i * kThreads, r = at / PER, c = at % PER * N;
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

// A segment's chunks, one workgroup; OUT false: its state alone, from zero.
//
// The four waves own slices of the value axis: a slice's state stays in registers, in
// the layout in which the MFMA returns it, and is an operand of the next chunk's
// products as it lies (read_rows_halves gives the other operand in its K order).  The
// scores of a chunk are shared: wave w computes those of its 16 queries, weights and
// masks them, and all read them from LDS.
template <typename T, int NP, int L, int DP, int EP, bool OUT>
__global__ __launch_bounds__(kThreads) void k_mix(MixArgs p) {
  constexpr int NPI = sizeof(T) == 2 ? 1 : 3, IT = L / 16, KS = L / 32, DT = DP / 16, DK = DP / 32, ET = EP / 64;
  using M = Lds<NPI, NP, L, DP, EP, OUT>;
  __shared__ M m;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l16 = lane & 15, g4 = lane >> 4;
  const int segs = OUT ? p.nseg : p.nseg - 1;      // OUT false: the walk's last segment is not needed
  const int bh = blockIdx.x / segs, walk = blockIdx.x - bh * segs;
  const int b = bh / p.H, h = bh - b * p.H, seg = p.rev ? p.nseg - 1 - walk : walk;
  int64_t length = p.T;
  if (p.lengths) length = min(max(p.lengths[b], (int64_t)0), (int64_t)p.T);
  const int chunks = (p.T + L - 1) / L, c_lo = seg * p.per, c_hi = min(c_lo + p.per, chunks), n = max(c_hi - c_lo, 0);
  auto at = [&](const Array& a) { return static_cast<const T*>(a.p) + b * a.b + h * a.h; };
  const T *qp = OUT ? at(p.q) : nullptr, *kp = at(p.k), *vp = at(p.v);
  auto first_of = [&](int i) { return (p.rev ? c_hi - 1 - i : c_lo + i) * L; };     // chunk i of the walk
  auto live = [&](int t0) { return (int)max(min(length - t0, (int64_t)L), (int64_t)0); };

  Rows<T, L, DP> rq, rk;
  Rows<T, L, EP> rv;
  auto load = [&](int t0) {
    const int rows = live(t0);
    if constexpr (OUT) rq.load(qp + t0 * p.q.t, p.q.t, rows, p.dq);
    rk.load(kp + t0 * p.k.t, p.k.t, rows, p.dq);
    rv.load(vp + t0 * p.v.t, p.v.t, rows, p.dv);
  };
  auto store = [&] {
    if constexpr (OUT) rq.store(m.q, M::PD);
    rk.store(m.k, M::PD);
    rv.store(m.v, M::PE);
  };
  // log decay of a lane's token of the chunk at t0
  auto load_gate = [&](int t0) -> float {
    if (lane >= live(t0)) return 0.0f;
    const int64_t i = b * p.gb + (t0 + lane) * p.gt + h * p.gh;
    return floor_decay(p.g_bf16 ? load_elem(static_cast<const uint16_t*>(p.g) + i) : static_cast<const float*>(p.g)[i]);
  };
  double sum_all = 0.0;
  // cumulated log decays of a chunk in 64 bits, kept as the sum of two f32
  auto gates = [&](float g, int par) {
    double s = lane < L ? (double)g : 0.0;
#pragma unroll
    for (int k = 1; k < L; k <<= 1) {
      const double o = __shfl_up(s, k, 64);
      if (lane >= k) s += o;
    }
    const double end = __shfl(s, L - 1, 64);
    sum_all += end;
    const float start = expf((float)s), rest = expf((float)(end - s));
    if (lane < L) {
      const float hi = (float)s;
      m.hi[par][lane] = hi;
      m.lo[par][lane] = (float)(s - (double)hi);
      m.qw[par][lane] = (p.rev ? rest : start) * p.sscale;
      m.kw[par][lane] = (p.rev ? start : rest) * p.kscale;
    }
    if (lane == 0) m.total[par] = expf((float)end);
  };

  // state: S[16 dt + 4 g4 + r][16 (wave ET + et) + l16]
  v4f S[DT][ET] = {};
  const int64_t state_at = OUT ? ((int64_t)bh * p.nseg + seg) * p.init_seg : 0;
  if (OUT && p.init) {
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int et = 0; et < ET; ++et) {
        const int e = (wave * ET + et) * 16 + l16;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int d = dt * 16 + g4 * 4 + r;
          if (d < p.dq && e < p.dv) S[dt][et][r] = p.init[state_at + (int64_t)d * p.init_r + (int64_t)e * p.init_c];
        }
      }
  }

  float g_next = 0.0f;
  if (n > 0) {
    load(first_of(0));
    if (wave == 0) {
      gates(load_gate(first_of(0)), 0);
      if (n > 1) g_next = load_gate(first_of(1));
    }
    store();
  }
  __syncthreads();
  for (int i = 0; i < n; ++i) {
    const int t0 = first_of(i), par = i & 1;
    if (i + 1 < n) load(first_of(i + 1));
    if (wave == 0 && i + 1 < n) {
      gates(g_next, par ^ 1);
      if (i + 2 < n) g_next = load_gate(first_of(i + 2));
    }
    v4f acc[IT][ET];
    if constexpr (OUT) {
      // scores of queries 16 it .. with keys 16 jt ..: rows of the result are keys
#pragma unroll
      for (int j = 0; j < (L == 64 ? 4 : 1); ++j) {
        const int it = L == 64 ? wave : wave >> 1, jt = L == 64 ? j : wave & 1;
        const bool none = p.rev ? jt < it : jt > it;
        if (none && (jt >> 1) != (it >> 1)) continue;       // not read
        v4f s = {};
        if (!none) {
#pragma unroll
          for (int ks = 0; ks < DK; ++ks) {
            bf16x8_t a[NPI], c[NPI];
#pragma unroll
            for (int x = 0; x < NPI; ++x) {
              a[x] = read_rows(m.k[x] + jt * 16 * M::PD + ks * 32, M::PD, lane);
              c[x] = read_rows(m.q[x] + it * 16 * M::PD + ks * 32, M::PD, lane);
            }
            s = mfma_planes(a, c, s);
          }
        }
        const int qi = it * 16 + l16, kj = jt * 16 + g4 * 4;
        const float hq = m.hi[par][qi], lq = m.lo[par][qi];
        float w[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const float d = (hq - m.hi[par][kj + r]) + (lq - m.lo[par][kj + r]);
          const bool in = p.rev ? kj + r >= qi : kj + r <= qi;
          w[r] = in && !none ? s[r] * __expf(p.rev ? -d : d) * p.tscale : 0.0f;
        }
        uint32_t o[NP][2];
        split<NP, 4>(w, o);
#pragma unroll
        for (int x = 0; x < NP; ++x) *reinterpret_cast<u32x2_t*>(m.t[x] + qi * M::PT + kj) = u32x2_t{o[x][0], o[x][1]};
      }
      // what the queries read of the state
#pragma unroll
      for (int it = 0; it < IT; ++it)
#pragma unroll
        for (int et = 0; et < ET; ++et) acc[it][et] = v4f{};
#pragma unroll
      for (int ks = 0; ks < DK; ++ks) {
        bf16x8_t a[ET][NP];
#pragma unroll
        for (int et = 0; et < ET; ++et) {
          float w[8];
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            w[r] = S[2 * ks][et][r];
            w[4 + r] = S[2 * ks + 1][et][r];
          }
          uint32_t o[NP][4];
          split<NP, 8>(w, o);
#pragma unroll
          for (int x = 0; x < NP; ++x) a[et][x] = frag4(o[x]);
        }
#pragma unroll
        for (int it = 0; it < IT; ++it) {
          bf16x8_t c[NPI];
#pragma unroll
          for (int x = 0; x < NPI; ++x) c[x] = read_rows_halves(m.q[x] + it * 16 * M::PD + ks * 32, M::PD, lane);
#pragma unroll
          for (int et = 0; et < ET; ++et) acc[it][et] = mfma_planes(a[et], c, acc[it][et]);
        }
      }
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        const float w = m.qw[par][it * 16 + l16];
#pragma unroll
        for (int et = 0; et < ET; ++et)
#pragma unroll
          for (int r = 0; r < 4; ++r) acc[it][et][r] *= w;
      }
    }
    // the wave's values, and the same decayed to the chunk's end
    bf16x8_t val[KS][ET][NPI], dec[KS][ET][3];
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
      float w[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) w[r] = m.kw[par][ks * 32 + g4 * 8 + r];
#pragma unroll
      for (int et = 0; et < ET; ++et) {
        float f[8] = {};
#pragma unroll
        for (int x = NPI - 1; x >= 0; --x) {
          val[ks][et][x] = read_columns(m.v[x] + ks * 32 * M::PE + (wave * ET + et) * 16, M::PE, lane);
#pragma unroll
          for (int r = 0; r < 8; ++r) f[r] += bf16_at(val[ks][et][x], r);
        }
#pragma unroll
        for (int r = 0; r < 8; ++r) f[r] *= w[r];
        uint32_t o[3][4];
        split<3, 8>(f, o);
#pragma unroll
        for (int x = 0; x < 3; ++x) dec[ks][et][x] = frag4(o[x]);
      }
    }
    const float total = m.total[par];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
      for (int et = 0; et < ET; ++et)
#pragma unroll
        for (int r = 0; r < 4; ++r) S[dt][et][r] *= total;
#pragma unroll
      for (int ks = 0; ks < KS; ++ks) {
        bf16x8_t a[NPI];
#pragma unroll
        for (int x = 0; x < NPI; ++x) a[x] = read_columns(m.k[x] + ks * 32 * M::PD + dt * 16, M::PD, lane);
#pragma unroll
        for (int et = 0; et < ET; ++et) S[dt][et] = mfma_planes(a, dec[ks][et], S[dt][et]);
      }
    }
    __syncthreads();                    // scores are whole
    if constexpr (OUT) {
#pragma unroll
      for (int it = 0; it < IT; ++it)
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
          if (p.rev ? ks < (it >> 1) : ks > (it >> 1)) continue;
          bf16x8_t c[NP];
#pragma unroll
          for (int x = 0; x < NP; ++x) c[x] = read_rows(m.t[x] + it * 16 * M::PT + ks * 32, M::PT, lane);
#pragma unroll
          for (int et = 0; et < ET; ++et) acc[it][et] = mfma_planes(val[ks][et], c, acc[it][et]);
        }
      // acc[it][et][r]: token 16 it + l16, value 16 (wave ET + et) + 4 g4 + r
      T* out = static_cast<T*>(p.out.p) + b * p.out.b + h * p.out.h;
      const int rows = live(t0);
#pragma unroll
      for (int it = 0; it < IT; ++it) {
        const int i_ = it * 16 + l16, t = t0 + i_;
        float dot = 0.0f;
#pragma unroll
        for (int et = 0; et < ET; ++et) {
          const int e = (wave * ET + et) * 16 + g4 * 4;
          float o[4];
#pragma unroll
          for (int r = 0; r < 4; ++r) o[r] = i_ < rows ? acc[it][et][r] : 0.0f;
          if (t < p.T && e < p.dv) {
            T* to = out + t * p.out.t + e;
            if (e + 4 <= p.dv && sizeof(T) == 2) {
              typedef uint32_t u32x2_a2 __attribute__((ext_vector_type(2), aligned(2)));
              *reinterpret_cast<u32x2_a2*>(to) = u32x2_a2{pack_bf16x2(o[0], o[1]), pack_bf16x2(o[2], o[3])};
            } else {
              store_some(to, p.dv - e, o);
            }
            if (p.dot && i_ < rows) {
              float x[4];
              load_some(static_cast<const T*>(p.x.p) + b * p.x.b + h * p.x.h + t * p.x.t + e, p.dv - e, 0.0f, x);
#pragma unroll
              for (int r = 0; r < 4; ++r) dot += x[r] * o[r];
            }
          }
        }
        if (p.dot) {
          dot += __shfl_xor(dot, 16, 64);
          dot += __shfl_xor(dot, 32, 64);
          if (g4 == 0) m.dot[wave][i_] = dot;
        }
      }
    }
    __syncthreads();                    // this chunk's arrays are read
    if (OUT && p.dot && threadIdx.x < L && t0 + (int)threadIdx.x < p.T)
      p.dot[(int64_t)bh * p.T + t0 + threadIdx.x] =
          (m.dot[0][threadIdx.x] + m.dot[1][threadIdx.x]) + (m.dot[2][threadIdx.x] + m.dot[3][threadIdx.x]);
    if (i + 1 < n) store();
    __syncthreads();
  }

  if (p.last && (!OUT || walk == p.nseg - 1)) {
    float* to = p.last + (OUT ? (int64_t)bh * p.last_seg : ((int64_t)bh * p.nseg + seg) * p.last_seg);
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
      for (int et = 0; et < ET; ++et) {
        const int e = (wave * ET + et) * 16 + l16;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int d = dt * 16 + g4 * 4 + r;
          if (d < p.dq && e < p.dv) to[(int64_t)d * p.last_r + (int64_t)e * p.last_c] = S[dt][et][r];
        }
      }
  }
  if (!OUT && threadIdx.x == 0) p.decay[(int64_t)bh * p.nseg + seg] = (float)exp(sum_all);
}

// The states before the segments from the segments' own: states[walk] holds what its
// segment adds and becomes the state before it.
__global__ __launch_bounds__(256) void k_mix_join(float* __restrict__ states, const float* __restrict__ decay,
                                                  const float* __restrict__ init, int64_t size, int nseg, int rev) {
  const int64_t bh = blockIdx.x, e = (int64_t)blockIdx.y * 256 + threadIdx.x;
  if (e >= size) return;
  float s = init ? init[bh * size + e] : 0.0f;
  for (int w = 0; w < nseg; ++w) {
    const int seg = rev ? nseg - 1 - w : w;
    float* at = states + (bh * nseg + seg) * size + e;
    const float add = w + 1 < nseg ? *at : 0.0f;
    *at = s;
    if (w + 1 < nseg) s = decay[bh * nseg + seg] * s + add;
  }
}

// Gradient of a segment's log decays: from its last token to its first, the sums of
// q . dq - k . dk, from <S, R> at its end on.
template <typename G>
__global__ __launch_bounds__(64) void k_mix_decay_grad(const float* __restrict__ dot_q, const float* __restrict__ dot_k,
                                                       const float* __restrict__ s_starts,
                                                       const float* __restrict__ s_last, const float* __restrict__ r_end,
                                                       const int64_t* __restrict__ lengths, int T, int H,
                                                       int64_t size, int nseg, int tokens, const G* __restrict__ g,
                                                       int64_t gb, int64_t gt, int64_t gh, G* __restrict__ dg) {
  const int bh = blockIdx.x / nseg, seg = blockIdx.x - bh * nseg, b = bh / H, h = bh - b * H, lane = threadIdx.x;
  const int64_t length = lengths ? min(max(lengths[b], (int64_t)0), (int64_t)T) : T;
  // S and R behind the segment
  const float* S = seg + 1 < nseg ? s_starts + ((int64_t)bh * nseg + seg + 1) * size : s_last ? s_last + bh * size : nullptr;
  const float* R = r_end && S ? r_end + ((int64_t)bh * nseg + seg) * size : nullptr;
  double carry = 0.0;
  if (R) {
    float sum = 0.0f;
    for (int64_t i = lane; i < size; i += 64) sum += S[i] * R[i];
    double d = sum;
#pragma unroll
    for (int k = 32; k; k >>= 1) d += __shfl_xor(d, k, 64);
    carry = d;
  }
  const int lo = seg * tokens, hi = min(lo + tokens, T);
  for (int end = hi; end > lo; end -= 64) {
    const int t = end - 1 - lane;                       // lane 0: the last token
    const bool in = t >= lo, here = in && t < length;
    double s = here ? (double)dot_q[(int64_t)bh * T + t] - (double)dot_k[(int64_t)bh * T + t] : 0.0;
#pragma unroll
    for (int k = 1; k < 64; k <<= 1) {
      const double o = __shfl_up(s, k, 64);
      if (lane >= k) s += o;
    }
    s += carry;
    if (in) {
      // e^g is 0 in f32 below -104: nothing passes
      const float gate = load_elem(g + b * gb + t * gt + h * gh);
      store_elem(dg + ((int64_t)b * T + t) * H + h, here && !(gate < -104.0f) ? (float)s : 0.0f);
    }
    carry = __shfl(s, 63, 64);
  }
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
  int L() const { return dtype == PRATCHYA_DT_BF16 ? 64 : 32; }
  int64_t chunks() const { return (T + L() - 1) / L(); }
  // Segments of a sequence: as many as give every compute unit four workgroups, each of
  // at least 256 tokens.
  int64_t segments() const {
    const int64_t heads = B * H, most = T / 256;
    if (heads < 1) return 1;
    int64_t n = (1024 + heads - 1) / heads;
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
  // states before the segments, and the segments' decays
  int64_t starts_floats() const {
    const int64_t n = segments();
    return n > 1 ? B * H * n * (state() + 1) : 0;
  }
};

int check_shape(const char* what, const Shape& s, int g_dtype) {
  if (!is_float_dtype(s.dtype) || !is_float_dtype(g_dtype))
    return pratchya_set_error(PRATCHYA_EINVAL, "%s: unsupported dtypes %d, %d", what, s.dtype, g_dtype);
  if (s.B < 0 || s.T < 0 || s.H < 1 || s.dk < 1 || s.dv < 1)
    return pratchya_set_error(PRATCHYA_EINVAL, "%s: [%lld, %lld, %lld] of heads of %lld and %lld", what, (long long)s.B,
                              (long long)s.T, (long long)s.H, (long long)s.dk, (long long)s.dv);
  if (s.dk > kMaxHead || s.dv > kMaxHead || s.T > 0x7FFFFF00 || s.B > (1 << 24) || s.H > (1 << 24) ||
      !fits_launch(s.B * s.H * s.segments(), kThreads))
    return pratchya_set_error(PRATCHYA_EUNSUPPORTED, "%s: heads of more than %d, or 2^24 heads of segments", what, kMaxHead);
  return PRATCHYA_OK;
}

template <typename T, int NP, int L, bool OUT>
void launch_dims(const MixArgs& a, unsigned blocks, hipStream_t stream) {
#define PRATCHYA_MIX(D, E) hipLaunchKernelGGL((k_mix<T, NP, L, D, E, OUT>), dim3(blocks), dim3(kThreads), 0, stream, a)
  if (a.dq <= 64) {
    if (a.dv <= 64) PRATCHYA_MIX(64, 64);
    else PRATCHYA_MIX(64, 128);
  } else {
    if (a.dv <= 64) PRATCHYA_MIX(128, 64);
    else PRATCHYA_MIX(128, 128);
  }
#undef PRATCHYA_MIX
}

int launch_mix(const Shape& s, const MixArgs& a, bool out, bool exact, hipStream_t stream) {
  const int64_t blocks = s.B * s.H * (out ? a.nseg : a.nseg - 1);
  if (!blocks) return PRATCHYA_OK;
  if (s.dtype == PRATCHYA_DT_BF16) {
    if (!out) launch_dims<uint16_t, 1, 64, false>(a, (unsigned)blocks, stream);
    else if (exact) launch_dims<uint16_t, 3, 64, true>(a, (unsigned)blocks, stream);
    else launch_dims<uint16_t, 1, 64, true>(a, (unsigned)blocks, stream);
  } else {
    if (!out) launch_dims<float, 3, 32, false>(a, (unsigned)blocks, stream);
    else launch_dims<float, 3, 32, true>(a, (unsigned)blocks, stream);
  }
  return check_launch("linear_attention");
}

int join(const Shape& s, float* starts, const float* init, int rev, hipStream_t stream) {
  const int64_t n = s.segments(), size = s.state();
  hipLaunchKernelGGL(k_mix_join, dim3((unsigned)(s.B * s.H), (unsigned)((size + 255) / 256)), dim3(256), 0, stream,
                     starts, starts + s.B * s.H * n * size, init, size, (int)n, rev);
  return check_launch("linear_attention");
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

// One walk: the segments' states first where there are several, then the outputs.
// starts: where they are kept; known: they are there already.  transposed: the state
// is held as [value, query] in memory.
int walk(const Shape& s, MixArgs a, float* starts, bool known, const float* init, bool transposed, float* last,
         bool exact, hipStream_t stream) {
  const int64_t size = s.state();
  const int r = transposed ? 1 : a.dv, c = transposed ? a.dq : 1;
  int rc;
  if (a.nseg > 1 && !known) {
    MixArgs u = a;
    u.last = starts;
    u.last_seg = size;
    u.last_r = r;
    u.last_c = c;
    u.decay = starts + s.B * s.H * a.nseg * size;
    if ((rc = launch_mix(s, u, false, true, stream)) || (rc = join(s, starts, init, a.rev, stream))) return rc;
  }
  a.init = a.nseg > 1 ? starts : init;
  a.init_seg = size;
  a.init_r = r;
  a.init_c = c;
  a.last = last;
  a.last_seg = size;
  a.last_r = r;
  a.last_c = c;
  return launch_mix(s, a, true, exact, stream);
}

}  // namespace

extern "C" int64_t pratchya_linear_attention_starts_floats(int64_t batch, int64_t length, int64_t heads, int64_t dk,
                                                           int64_t dv, int dtype) {
  const Shape s = {batch, length, heads, dk, dv, dtype};
  return check_shape("linear_attention", s, PRATCHYA_DT_F32) ? 0 : s.starts_floats();
}

extern "C" int pratchya_linear_attention(const void* q, const void* k, const void* v, int dtype, const void* log_decay,
                                         int g_dtype, const int64_t* strides, const int64_t* lengths, const float* state,
                                         int64_t batch, int64_t length, int64_t heads, int64_t dk, int64_t dv,
                                         float scale, void* out, float* state_out, float* starts, hipStream_t stream) {
  const char* what = "linear_attention";
  const Shape s = {batch, length, heads, dk, dv, dtype};
  const int rc = check_shape(what, s, g_dtype);
  if (rc) return rc;
  if (batch == 0) return pratchya_set_error(PRATCHYA_OK, "");
  if (!strides || (length && (!q || !k || !v || !log_decay || !out)) || !state_out || (s.starts_floats() && !starts))
    return pratchya_set_error(PRATCHYA_EINVAL, "%s: null buffer", what);
  MixArgs a = base_args(s, log_decay, g_dtype, strides + 9, lengths);
  a.q = array(q, strides);
  a.k = array(k, strides + 3);
  a.v = array(v, strides + 6);
  a.out = packed(s, out, dv);
  a.dq = (int)dk;
  a.dv = (int)dv;
  a.tscale = a.sscale = scale;
  a.kscale = 1.0f;
  return walk(s, a, starts, false, state, false, state_out, false, stream);
}

extern "C" int64_t pratchya_linear_attention_bwd_workspace_bytes(int64_t batch, int64_t length, int64_t heads, int64_t dk,
                                                                 int64_t dv, int dtype) {
  const Shape s = {batch, length, heads, dk, dv, dtype};
  if (check_shape("linear_attention_bwd", s, PRATCHYA_DT_F32)) return 0;
  return 4 * (s.starts_floats() + 2 * batch * heads * length);
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
  const Shape s = {batch, length, heads, dk, dv, dtype};
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
  float* dot_k = dot_q + batch * heads * length;
  const bool decays = dlog_decay != nullptr;
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
  a.tscale = a.sscale = scale;
  a.kscale = 1.0f;
  if (decays) {
    a.x = Q;
    a.dot = dot_q;
  }
  rc = walk(s, a, const_cast<float*>(starts), true, state, true, nullptr, decays, stream);
  if (rc) return rc;
  // dv: queries k, keys q, values do, state R
  a = base;
  a.rev = 1;
  a.q = K;
  a.k = Q;
  a.v = D;
  a.out = packed(s, dv_out, dv);
  a.dq = (int)dk;
  a.dv = (int)dv;
  a.tscale = a.kscale = scale;
  a.sscale = 1.0f;
  rc = walk(s, a, rstarts, false, dstate_out, false, dstate, false, stream);
  if (rc) return rc;
  // dk: queries v, keys do, values q, state R^T
  a.q = V;
  a.k = D;
  a.v = Q;
  a.out = packed(s, dk_out, dk);
  a.dq = (int)dv;
  a.dv = (int)dk;
  if (decays) {
    a.x = K;
    a.dot = dot_k;
  }
  rc = walk(s, a, rstarts, true, dstate_out, true, nullptr, decays, stream);
  if (rc || !decays || !length) return rc;
  const int64_t n = s.segments(), size = s.state();
  const float* r_end = n > 1 ? rstarts : dstate_out;
#define PRATCHYA_DG(G)                                                                                                \
  hipLaunchKernelGGL((k_mix_decay_grad<G>), dim3((unsigned)(batch * heads * n)), dim3(64), 0, stream, dot_q, dot_k,   \
                     starts, state_out, r_end, lengths, (int)length, (int)heads, size, (int)n,         \
                     (int)(s.per() * s.L()), static_cast<const G*>(log_decay), strides[9], strides[10], strides[11],  \
                     static_cast<G*>(dlog_decay))
  if (g_dtype == PRATCHYA_DT_BF16) PRATCHYA_DG(uint16_t);
  else PRATCHYA_DG(float);
#undef PRATCHYA_DG
  return check_launch(what);
}

extern "C" int pratchya_linear_attention_step(const void* q, const void* k, const void* v, int dtype,
                                              const void* log_decay, int g_dtype, const int64_t* strides, float* state,
                                              int64_t batch, int64_t heads, int64_t dk, int64_t dv, float scale,
                                              void* out, hipStream_t stream) {
  const char* what = "linear_attention_step";
  const Shape s = {batch, 1, heads, dk, dv, dtype};
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
