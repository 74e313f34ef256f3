// Ragged batches: token rows of several requests end to end, cu[b] <= t < cu[b + 1] for request b's rows.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace fgw {

// The last request whose offset is at most t, by a converged warp; 0 where there is none.
__device__ __forceinline__ int find_request(const int32_t* cu, int batch, long long t, int lane) {
  int lo = 0, hi = batch;  // the answer is in [lo, hi)
  while (hi - lo > 1) {
    const int step = (hi - lo + 31) / 32;
    const int at = lo + lane * step;
    const uint32_t below = __ballot_sync(0xffffffffu, at < hi && cu[at] <= t);
    const int k = max(__popc(below), 1) - 1;
    hi = min(hi, lo + (k + 1) * step);
    lo += k * step;
  }
  return lo;
}

}  // namespace fgw
