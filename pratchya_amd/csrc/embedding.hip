// Embedding lookup with scaling and the table's gradient, for gfx950.
//
//   y_i = scale * table[token_i],   dtable_v = scale * sum over i with token_i = v of dy_i
//
// A negative token stands for none: its row of y is 0 and it has no gradient.  A
// token of the vocabulary's size or more has no row: its y is NaN, without a gradient.
// Sums are f32 in the tokens' order, the same bits for the same inputs.
//
// Gradient.  One launch sorts the tokens by value (k_sort_tokens) while its other
// workgroups fill the gradient with zeros; then each row that has tokens is summed
// once: no atomics and no f32 copy of the table.  Bound: HBM, dy read and the table's
// gradient written.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "pratchya_fp8.h"
#include "row_device.h"
#include "row_host.h"

namespace {

// A piece: the columns of a row that one wave takes, U vectors a lane.
template <typename T, int U>
constexpr int kPiece = 64 * U * kN<T>;

template <typename T, int U>
__global__ __launch_bounds__(256) void k_embedding(const T* __restrict__ table, int64_t ld,
                                                   const int64_t* __restrict__ tokens, int64_t units, int64_t vocab,
                                                   int64_t width, int pieces, float scale, T* __restrict__ y) {
  constexpr int N = kN<T>;
  const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (unit >= units) return;
  const int64_t i = unit / pieces, c0 = (unit - i * pieces) * kPiece<T, U> + (threadIdx.x & 63) * N;
  const int64_t t = tokens[i];
  T* out = y + i * width;
  u32x4_t raw[U];
  const bool found = t >= 0 && t < vocab;
  const T* row = table + (found ? t : 0) * ld;
  const float none = t < 0 ? 0.0f : __builtin_nanf("");
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t c = c0 + u * 64 * N;
    if (found && c + N <= width) raw[u] = load_raw(row + c);
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t c = c0 + u * 64 * N;
    if (c >= width) break;
    float v[N];
    if (!found) {
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] = none;
    } else if (c + N <= width) {
      widen(raw[u], v);
    } else {
      load_some(row + c, width - c, 0.0f, v);
    }
    if (found) {
#pragma unroll
      for (int k = 0; k < N; ++k) v[k] *= scale;
    }
    if (c + N <= width) store_vec(out + c, v);
    else store_some(out + c, width - c, v);
  }
}

// Stable sort of the tokens by value, in one launch: workgroup b owns the table's
// rows [b R, (b + 1) R) and reads all tokens, which the L2 caches hold (8 bytes a
// token and workgroup, where the sum reads a whole row of dy a token), counts those
// below its rows, the place of its first one, and those of each of its rows by
// wave, and then places its own in a second reading.  Each wave takes a contiguous
// stretch of the tokens, so the order within a row is the tokens'.
constexpr int kSortWaves = 16, kSortRows = 512, kSortUnroll = 4;

struct Sorted {
  int32_t* pos;      // [n] indices of tokens, by value, then in order
  int32_t* key;      // [n] their values
  int32_t* offs;     // [vocab + 1] first place of each row
};

// The gradient's bytes as a fill sees them: `vectors` of 16 from the first 16-byte
// boundary on, `head` and `tail` elements around them.
struct Fill {
  uint8_t *first, *vec, *last;
  int64_t vectors;
  int head, tail;
};

constexpr int kSortThreads = kSortWaves * 64, kFillUnroll = 4;

__device__ __forceinline__ void fill_zero(const Fill& f, int64_t block) {
  auto* v = reinterpret_cast<u32x4_t*>(f.vec);
  const int64_t at = block * (kSortThreads * kFillUnroll) + threadIdx.x;
#pragma unroll
  for (int u = 0; u < kFillUnroll; ++u) {
    const int64_t i = at + u * kSortThreads;
    if (i < f.vectors) v[i] = u32x4_t{};
  }
  if (block == 0 && threadIdx.x < 32) {
    const int e = threadIdx.x & 15;
    uint8_t* p = threadIdx.x < 16 ? f.first + e : f.last + e;
    if (e < (threadIdx.x < 16 ? f.head : f.tail)) *p = 0;
  }
}

__global__ __launch_bounds__(kSortThreads) void k_sort_tokens(const int64_t* __restrict__ tokens, int n, int vocab,
                                                              int rows, int sorters, Sorted out, Fill fill) {
  if ((int)blockIdx.x >= sorters) {
    fill_zero(fill, (int64_t)blockIdx.x - sorters);
    return;
  }
  __shared__ int count[kSortWaves][kSortRows];
  __shared__ int part[kSortWaves], first[kSortWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int lo = blockIdx.x * rows, mine = min(rows, vocab - lo);
  for (int r = threadIdx.x; r < kSortWaves * kSortRows; r += kSortWaves * 64) (&count[0][0])[r] = 0;
  __syncthreads();
  const int per = ((n + kSortWaves - 1) / kSortWaves + 63) / 64 * 64;
  const int64_t begin = (int64_t)wave * per, end = begin + per < n ? begin + per : n;
  // row of a token among this workgroup's, below 0 for a smaller one
  auto row_of = [&](int64_t i) -> int64_t {
    if (i >= end) return INT64_MAX;
    const int64_t t = tokens[i];
    return t < 0 ? INT64_MAX : t - lo;
  };
  int below = 0;
  for (int64_t at = begin; at < end; at += 64 * kSortUnroll) {
    int64_t r[kSortUnroll];
#pragma unroll
    for (int u = 0; u < kSortUnroll; ++u) r[u] = row_of(at + u * 64 + lane);
#pragma unroll
    for (int u = 0; u < kSortUnroll; ++u) {
      below += r[u] < 0;
      if (r[u] >= 0 && r[u] < mine) atomicAdd(&count[wave][(int)r[u]], 1);
    }
  }
#pragma unroll
  for (int m = 32; m; m >>= 1) below += __shfl_xor(below, m, 64);
  if (lane == 0) part[wave] = below;
  __syncthreads();
  // places of the rows' first tokens: a thread's row, then the waves of 64 rows
  int base = 0;
#pragma unroll
  for (int w = 0; w < kSortWaves; ++w) base += part[w];
  int total = 0, upto = 0;
  const int r = threadIdx.x;
  if (r < kSortRows) {
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) total += count[w][r];
  }
  upto = total;
#pragma unroll
  for (int m = 1; m < 64; m <<= 1) {
    const int v = __shfl_up(upto, m, 64);
    if (lane >= m) upto += v;
  }
  if (lane == 63) first[wave] = upto;
  __syncthreads();
  if (r < kSortRows) {
    int at = base + upto - total;
    for (int w = 0; w < wave; ++w) at += first[w];
    if (r < mine) out.offs[lo + r] = at;
    if (r < mine && lo + r == vocab - 1) out.offs[vocab] = at + total;
    for (int w = 0; w < kSortWaves; ++w) {
      const int c = count[w][r];
      count[w][r] = at;
      at += c;
    }
  }
  __syncthreads();
  volatile int* place = count[wave];           // this wave's alone from here on
  for (int64_t at = begin; at < end; at += 64 * kSortUnroll) {
    int64_t r2[kSortUnroll];
#pragma unroll
    for (int u = 0; u < kSortUnroll; ++u) r2[u] = row_of(at + u * 64 + lane);
#pragma unroll
    for (int u = 0; u < kSortUnroll; ++u) {
      const bool in = r2[u] >= 0 && r2[u] < mine;
      const int row = in ? (int)r2[u] : -1;
      uint64_t left = __ballot(in);
      while (left) {
        const int lead = __builtin_ctzll(left);
        const int v = __shfl(row, lead, 64);
        const uint64_t same = __ballot(row == v);
        if (row == v) {
          const int p = place[v] + __popcll(same & ((1ull << lane) - 1));
          out.pos[p] = (int)(at + u * 64 + lane);
          out.key[p] = lo + v;
          if (lane == lead) place[v] = p + __popcll(same);
        }
        left &= ~same;
      }
    }
  }
}

// Sum of dy's rows pos[first .. first + count), count up to 64, over the lane's
// vectors: the row numbers come in one load, the rows kAhead at a time.
constexpr int kAhead = 8;
template <typename T, int U>
__device__ __forceinline__ void sum_rows(const T* __restrict__ dy, int64_t ldy, const int32_t* __restrict__ pos,
                                         int first, int count, int64_t c0, int64_t width, float (&acc)[U][kN<T>]) {
  constexpr int N = kN<T>;
  const int lane = threadIdx.x & 63;
  const int mine = lane < count ? pos[first + lane] : 0;
  for (int j = 0; j < count; j += kAhead) {
    u32x4_t raw[kAhead][U];
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      const T* row = dy + (int64_t)__builtin_amdgcn_readlane(mine, (j + a) & 63) * ldy;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t c = c0 + u * 64 * N;
        if (j + a < count && c + N <= width) raw[a][u] = load_raw(row + c);
      }
    }
#pragma unroll
    for (int a = 0; a < kAhead; ++a) {
      if (j + a >= count) break;
      const T* row = dy + (int64_t)__builtin_amdgcn_readlane(mine, (j + a) & 63) * ldy;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t c = c0 + u * 64 * N;
        if (c >= width) break;
        float v[N];
        if (c + N <= width) widen(raw[a][u], v);
        else load_some(row + c, width - c, 0.0f, v);
#pragma unroll
        for (int k = 0; k < N; ++k) acc[u][k] += v[k];
      }
    }
  }
}

// Rows of up to kRun tokens are summed by one wave a piece, that of the row's first
// token in sorted order.  Longer ones are cut at the multiples of kRun of that order:
// a tile of kRun sorted tokens holds parts of at most two such rows, whose sums go to
// the tile's first partial (the part that holds its first token) or its second;
// k_join_rows adds a row's partials.
//
// Measured, gradient of [65536, 2048] bf16 from 16384 tokens as text has them (a tenth
// of them the same): fill and sort 36 us (7.4 TB/s), sums 34, join 6; of [50021, 2057]
// f32 from 1001: 68 (6 TB/s), 15, 4.  One vector a lane and 8 rows ahead: two and 4
// ahead took 0.3 and 3% more time of both passes, runs of 64 and 16 instead of 32 3 to
// 8% and -3 to 3%.  With the zeros written by the waves that sum, whose registers
// leave few of them on a compute unit, both passes took 134 us instead of 104.
constexpr int kRun = 32;

template <typename T, int U>
__global__ __launch_bounds__(256) void k_embedding_grad(const T* __restrict__ dy, int64_t ldy, Sorted s,
                                                        int64_t vocab, int64_t width, int pieces, int64_t tile_units,
                                                        float scale, float* __restrict__ partial,
                                                        T* __restrict__ dtable) {
  constexpr int N = kN<T>;
  int64_t unit = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, total = s.offs[vocab];
  if (unit < tile_units) {
    const int64_t tile = unit / pieces, c0 = (unit - tile * pieces) * kPiece<T, U> + lane * N;
    const int at = (int)tile * kRun;
    if (at >= total) return;
    const int here = min(kRun, total - at);
    const int v = lane < here ? s.key[at + lane] : -1;
    for (int j = 0; j < here;) {
      const int row = __builtin_amdgcn_readlane(v, j);
      const int end = min(s.offs[row + 1], at + here) - at;
      if (s.offs[row + 1] - s.offs[row] > kRun) {
        float acc[U][N] = {};
        sum_rows<T, U>(dy, ldy, s.pos, at + j, end - j, c0, width, acc);
        float* to = partial + (2 * tile + (j ? 1 : 0)) * width;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int64_t c = c0 + u * 64 * N;
#pragma unroll
          for (int k = 0; k < N; ++k)
            if (c + k < width) to[c + k] = acc[u][k];
        }
      }
      j = end;
    }
    return;
  }
  unit -= tile_units;
  const int64_t at = unit / pieces, c0 = (unit - at * pieces) * kPiece<T, U> + lane * N;
  if (at >= total) return;
  const int row = s.key[at], first = s.offs[row], count = s.offs[row + 1] - first;
  if (first != at || count > kRun) return;
  float acc[U][N] = {};
  sum_rows<T, U>(dy, ldy, s.pos, first, count, c0, width, acc);
  T* out = dtable + row * width;
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const int64_t c = c0 + u * 64 * N;
    if (c >= width) break;
#pragma unroll
    for (int k = 0; k < N; ++k) acc[u][k] *= scale;
    if (c + N <= width) store_vec(out + c, acc[u]);
    else store_some(out + c, width - c, acc[u]);
  }
}

// The rows of more than kRun tokens from their partials, by the tile that holds the
// row's first token: one column a thread.
template <typename T>
__global__ __launch_bounds__(256) void k_join_rows(Sorted s, int64_t vocab, int64_t width,
                                                   const float* __restrict__ partial, float scale,
                                                   T* __restrict__ dtable) {
  const int at = (int)blockIdx.x * kRun, total = s.offs[vocab];
  if (at >= total) return;
  // the last row that begins in this tile is the only one that may leave it
  const int end = min(at + kRun, total), row = s.key[end - 1], first = s.offs[row], last = s.offs[row + 1];
  if (first < at || last - first <= kRun) {
    return;
  }
  const int64_t c = (int64_t)blockIdx.y * 256 + threadIdx.x;
  if (c >= width) return;
  const int tile = blockIdx.x, tiles = (last - 1) / kRun - tile;
  float sum = partial[(2 * (int64_t)tile + (first > at ? 1 : 0)) * width + c];
  const float* p = partial + 2 * (int64_t)(tile + 1) * width + c;
  int t = 0;
  for (; t + 8 <= tiles; t += 8) {
    float v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = p[2 * (int64_t)(t + k) * width];
#pragma unroll
    for (int k = 0; k < 8; ++k) sum += v[k];
  }
  for (; t < tiles; ++t) sum += p[2 * (int64_t)t * width];
  store_elem(dtable + row * width + c, sum * scale);
}

int check_args(const char* what, int dtype, int64_t n, int64_t vocab, int64_t width, int64_t ld) {
  if (!is_float_dtype(dtype)) return pratchya_set_error(PRATCHYA_EINVAL, "%s: unsupported dtype %d", what, dtype);
  if (n < 0 || vocab < 1 || width < 0 || ld < 0)
    return pratchya_set_error(PRATCHYA_EINVAL, "%s: %lld tokens of a table of [%lld, %lld], rows %lld apart", what,
                              (long long)n, (long long)vocab, (long long)width, (long long)ld);
  if (n > 0x7FFFFF00 || vocab > 0x7FFFFF00 || width > (int64_t)1 << 40)
    return pratchya_set_error(PRATCHYA_EUNSUPPORTED, "%s: more than 2^31 tokens or rows", what);
  return PRATCHYA_OK;
}

// Vectors of a lane (see k_embedding_grad; the lookup takes 22 us for 16384 rows of 4 KB, 5.8 TB/s).
constexpr int kU = 1;

template <typename T>
int64_t pieces_of(int64_t width) {
  return (width + kPiece<T, kU> - 1) / kPiece<T, kU>;
}

template <typename T>
int launch(const void* table, int64_t ld, const int64_t* tokens, int64_t n, int64_t vocab, int64_t width, float scale,
           void* y, hipStream_t stream) {
  const int64_t pieces = pieces_of<T>(width);
  const int64_t units = n * pieces;
  if (pieces > 0x7FFFFFFF || !fits_launch((units + 3) / 4, 256))
    return pratchya_set_error(PRATCHYA_EUNSUPPORTED, "embedding: more pieces of rows than a launch has threads for (2^26)");
  hipLaunchKernelGGL((k_embedding<T, kU>), dim3((unsigned)((units + 3) / 4)), dim3(256), 0, stream,
                     static_cast<const T*>(table), ld, tokens, units, vocab, width, (int)pieces, scale,
                     static_cast<T*>(y));
  return check_launch("embedding");
}

// Workspace: places, values, rows' first places, partials.
int64_t round16(int64_t v) { return (v + 15) & ~(int64_t)15; }
struct Layout {
  int64_t key, offs, partial, bytes;
  Layout(int64_t n, int64_t vocab, int64_t width) {
    key = round16(n * 4);
    offs = 2 * key;
    partial = offs + round16((vocab + 1) * 4);
    bytes = partial + (n > kRun ? 2 * ((n + kRun - 1) / kRun) * width * 4 : 0);
  }
};

template <typename T>
int launch_bwd(const void* dy, int64_t ldy, const int64_t* tokens, int64_t n, int64_t vocab, int64_t width, float scale,
               void* dtable, char* ws, hipStream_t stream) {
  const int64_t pieces = pieces_of<T>(width), tiles = n > kRun ? (n + kRun - 1) / kRun : 0;
  const int64_t units = (tiles + n) * pieces, columns = (width + 255) / 256;
  if (pieces > 0x7FFFFFFF || !fits_launch((units + 3) / 4, 256) || !fits_launch(tiles, 256, columns))
    return pratchya_set_error(PRATCHYA_EUNSUPPORTED, "embedding_bwd: more pieces of rows than a launch has threads for (2^26)");
  const Layout l(n, vocab, width);
  const Sorted s = {reinterpret_cast<int32_t*>(ws), reinterpret_cast<int32_t*>(ws + l.key),
                    reinterpret_cast<int32_t*>(ws + l.offs)};
  float* partial = reinterpret_cast<float*>(ws + l.partial);
  // one workgroup a compute unit, or as many as the rows need
  const int64_t rows = (vocab + 255) / 256 < kSortRows ? (vocab + 255) / 256 : kSortRows;
  const int64_t sorters = (vocab + rows - 1) / rows;
  Fill fill;
  const int64_t size = vocab * width * (int64_t)sizeof(T);
  fill.first = static_cast<uint8_t*>(dtable);
  fill.head = (int)(-reinterpret_cast<intptr_t>(dtable) & 15);
  if (fill.head > size) fill.head = (int)size;
  fill.vec = fill.first + fill.head;
  fill.vectors = (size - fill.head) / 16;
  fill.last = fill.vec + fill.vectors * 16;
  fill.tail = (int)((size - fill.head) % 16);
  const int64_t fillers = (fill.vectors + kSortThreads * kFillUnroll - 1) / (kSortThreads * kFillUnroll);
  if (!fits_launch(sorters + fillers + 1, kSortThreads))
    return pratchya_set_error(PRATCHYA_EUNSUPPORTED, "embedding_bwd: a table of more than 2^38 bytes");
  hipLaunchKernelGGL(k_sort_tokens, dim3((unsigned)(sorters + (fillers ? fillers : 1))), dim3(kSortThreads), 0, stream,
                     tokens, (int)n, (int)vocab, (int)rows, (int)sorters, s, fill);
  int rc = check_launch("embedding_bwd");
  if (rc || n == 0) return rc;
  hipLaunchKernelGGL((k_embedding_grad<T, kU>), dim3((unsigned)((units + 3) / 4)), dim3(256), 0, stream,
                     static_cast<const T*>(dy), ldy, s, vocab, width, (int)pieces, tiles * pieces, scale, partial,
                     static_cast<T*>(dtable));
  rc = check_launch("embedding_bwd");
  if (rc || !tiles) return rc;
  hipLaunchKernelGGL((k_join_rows<T>), dim3((unsigned)tiles, (unsigned)columns), dim3(256), 0, stream, s, vocab, width,
                     partial, scale, static_cast<T*>(dtable));
  return check_launch("embedding_bwd");
}

}  // namespace

extern "C" int pratchya_embedding(const void* table, int64_t ld, int dtype, const int64_t* tokens, int64_t n,
                                  int64_t vocab, int64_t width, float scale, void* y, hipStream_t stream) {
  const int rc = check_args("embedding", dtype, n, vocab, width, ld);
  if (rc) return rc;
  if (n == 0 || width == 0) return pratchya_set_error(PRATCHYA_OK, "");
  if (!table || !tokens || !y) return pratchya_set_error(PRATCHYA_EINVAL, "embedding: null buffer");
  return dtype == PRATCHYA_DT_BF16 ? launch<uint16_t>(table, ld, tokens, n, vocab, width, scale, y, stream)
                                   : launch<float>(table, ld, tokens, n, vocab, width, scale, y, stream);
}

extern "C" int64_t pratchya_embedding_bwd_workspace_bytes(int64_t n, int64_t vocab, int64_t width) {
  if (n < 0 || vocab < 1 || width < 0 || n > 0x7FFFFF00 || vocab > 0x7FFFFF00 || width > (int64_t)1 << 31) return 0;
  return Layout(n, vocab, width).bytes;
}

extern "C" int pratchya_embedding_bwd(const void* dy, int64_t ldy, int dtype, const int64_t* tokens, int64_t n,
                                      int64_t vocab, int64_t width, float scale, void* dtable, void* workspace,
                                      int64_t workspace_bytes, hipStream_t stream) {
  const int rc = check_args("embedding_bwd", dtype, n, vocab, width, ldy);
  if (rc) return rc;
  if (width == 0) return pratchya_set_error(PRATCHYA_OK, "");
  if (width > (int64_t)1 << 31)
    return pratchya_set_error(PRATCHYA_EUNSUPPORTED, "embedding_bwd: rows of more than 2^31 elements");
  const int64_t need = pratchya_embedding_bwd_workspace_bytes(n, vocab, width);
  if ((n && (!dy || !tokens)) || !dtable) return pratchya_set_error(PRATCHYA_EINVAL, "embedding_bwd: null buffer");
  if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16)
    return pratchya_set_error(PRATCHYA_EINVAL, "embedding_bwd: workspace of %lld bytes needed, 16-byte aligned",
                              (long long)need);
  char* ws = static_cast<char*>(workspace);
  return dtype == PRATCHYA_DT_BF16
             ? launch_bwd<uint16_t>(dy, ldy, tokens, n, vocab, width, scale, dtable, ws, stream)
             : launch_bwd<float>(dy, ldy, tokens, n, vocab, width, scale, dtable, ws, stream);
}
