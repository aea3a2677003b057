// Host helpers shared by the row operators' entry points (layer norm, activations,
// token log probabilities).
#pragma once
#include <stdint.h>

// What one launch holds: fewer than 2^32 threads along x, at most 65535 workgroups along y.
inline bool fits_launch(int64_t groups_x, int64_t threads, int64_t groups_y = 1) {
  return groups_x <= (((int64_t)1 << 32) - 1) / threads && groups_y <= 65535;
}
