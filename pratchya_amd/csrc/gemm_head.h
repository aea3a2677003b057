// Products of an output head's loss (head_loss.hip) on the 256 x 256 tiles of gemm.hip,
// with what follows a product in its epilogue.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

enum HeadEpilogue {
  kHeadStore,      // C, f32 or bf16, added to earlier sums where there are such
  kHeadRows,       // of each row and 128 columns: maximum, sum about it, sum; the target's value
  kHeadGrad,       // the loss's gradient of each value, as `planes` bf16 planes
};

// C [M, N] = sum over segments of A_s [M, K] . B_s [N, K]^T, bf16 operands, f32 sums:
// segment s multiplies plane (a_planes >> 4 s) & 15 of A with (b_planes >> 4 s) & 15 of B.
struct HeadProduct {
  const uint16_t *a, *b;
  int64_t lda, ldb, a_plane, b_plane;      // elements from a row, a plane to the next
  bool a_kmajor, b_kmajor;                 // [K, M], [K, N] as they lie
  uint32_t a_planes, b_planes;
  int segs, planes;
  int64_t M, N, K;                         // M, N 256 or more, a K-major operand's a multiple of 8; K of 64
  HeadEpilogue epilogue;
  // kHeadStore: C [rows, cols] (rows <= M, cols <= N) at any element's address; sums
  // [M, N], f32, 16-byte aligned rows: what is added, or null.  kHeadGrad: C as bf16
  // planes [planes][..][N], plane_c elements apart, 16-byte aligned rows, 0 from cols on.
  void* c;
  int64_t ldc, plane_c, rows, cols;
  bool c_bf16;
  int splits;                              // kHeadStore: slices of K (of segs K / 64 steps, which they divide), each to
  int64_t split_c;                         // a C of its own
  const float* sums;
  int64_t ld_sums;
  // kHeadRows, kHeadGrad: the rows' targets, column 0 is v0 of the vocabulary
  const int64_t* targets;
  int64_t v0, vocab;
  float smooth;
  float2* part;                            // [..][ld_part], of the rows' 128 columns each
  float* part_sum;                         // likewise, or null
  float* target_value;                     // [rows]
  int64_t ld_part;
  // kHeadStore, 128-row tiles: null, or what the results are multiplied by.  kHeadGrad: null, or behind that
  // 1 / max |g|: C is then dz over the first.
  const float* unit;
  const float *stats, *g;                  // kHeadGrad: (maximum, log of the sum about it), the loss's cotangent
};

// The part of a loss's gradient that its target has: what a gradient is measured in where it is
// held in bf16, so that the target's value, -g of it where its probability is small, has no
// rounding of its own that all rows share.
inline float head_part(float smooth) { return smooth < 0.5f ? 1.0f - smooth : 1.0f; }

// C [M, N], f32 (or bf16 times *unit), on the 128-row tiles of gemm_t128.hip, for any M and N of
// at least a row that pratchya_gemm_bf16_planes takes: a, b, their planes and segs, M, N, K, c,
// ldc, c_bf16 and unit count.  ws: its workspace.
bool head_product128_fits(const HeadProduct& p);      // sizes only
int head_product128(const HeadProduct& p, void* ws, int64_t ws_bytes, hipStream_t stream);

// Whether the operands suit (sizes, alignment, 32-bit offsets).
bool head_product_fits(const HeadProduct& p);
int head_product(const HeadProduct& p, hipStream_t stream);
