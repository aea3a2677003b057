// Host helpers shared by the row operators' entry points (layer norm, activations,
// token log probabilities).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "pratchya_fp8.h"

int pratchya_set_error(int code, const char* fmt, ...);

// What one launch holds: fewer than 2^32 threads along x, at most 65535 workgroups along y.
inline bool fits_launch(int64_t groups_x, int64_t threads, int64_t groups_y = 1) {
  return groups_x <= (((int64_t)1 << 32) - 1) / threads && groups_y <= 65535;
}

inline int check_launch(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return pratchya_set_error(PRATCHYA_EHIP, "%s: launch failed: %s", what, hipGetErrorString(e));
  return pratchya_set_error(PRATCHYA_OK, "");
}

inline bool is_float_dtype(int d) { return d == PRATCHYA_DT_F32 || d == PRATCHYA_DT_BF16; }

inline int64_t gcd64(int64_t x, int64_t y) {
  while (y) {
    const int64_t t = x % y;
    x = y;
    y = t;
  }
  return x;
}

inline int log2_of(int64_t v) {
  int n = 0;
  while (v > 1) {
    v >>= 1;
    ++n;
  }
  return n;
}
