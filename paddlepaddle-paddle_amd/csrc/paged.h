// Packed tokens of several sequences.
#pragma once
#include "common.h"

namespace pa {

// Largest b with cu[b] <= t: B behind the last sequence, -1 before the first.  By a whole wave, 64 borders a step.
__device__ __forceinline__ int seq_of_token(const int* cu, int B, int t) {
  int lo = 0, n = B + 1;  // cu[0 .. lo) are <= t, cu[lo + n ..) are not
  while (n > 0) {
    const int step = (n + 63) / 64, i = (int)(threadIdx.x & 63) * step + step - 1;  // (a step's last border)
    const int full = __popcll(__ballot(i < n && cu[lo + i] <= t));
    lo += full * step;
    n = step > 1 ? min(step - 1, n - full * step) : 0;
  }
  return lo - 1;
}

}  // namespace pa
