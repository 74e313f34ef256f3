// Index arithmetic of the serving-step kernels: division by fixed numbers, and ragged batches (token rows of several
// requests end to end, cu[b] <= t < cu[b + 1] for request b's rows).
#pragma once

#include <assert.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace fgw {

// Division of 0 <= n < 2^31 by a fixed positive number with a multiplication and shifts (Granlund and Montgomery, "Division
// by invariant integers using multiplication", 1994): m = floor(2^32 (2^l - d) / d) + 1 with 2^l >= d, q = (t + (n - t) / 2)
// / 2^(l - 1) with t = floor(m n / 2^32). A division by a variable takes some 150 cycles, and the kernels' starts are
// chains of them.
struct FastDiv {
  uint32_t mul, shift, one;  // one: the divisor is 1
  int by;
  FastDiv() = default;
  explicit FastDiv(int d) : by(d) {
    assert(d > 0);
    uint32_t l = 0;
    while (l < 31 && (1u << l) < static_cast<uint32_t>(d)) ++l;
    mul = static_cast<uint32_t>(((1ull << 32) * ((1ull << l) - d)) / d + 1);
    shift = l > 0 ? l - 1 : 0;
    one = l == 0;
  }
  __device__ __forceinline__ int quotient(int n) const {
    const uint32_t u = static_cast<uint32_t>(n), t = __umulhi(mul, u);
    return one ? n : static_cast<int>((t + ((u - t) >> 1)) >> shift);
  }
};

// x / y for x >= 0 and y > 0; nearly always the cheap 32-bit one.
__device__ __forceinline__ long long divide(long long x, int y) {
  if (x <= 0x7fffffffll) return static_cast<long long>(static_cast<uint32_t>(x) / static_cast<uint32_t>(y));
  return x / y;
}
// First unit of program p (program_start with the quotient already taken).
__device__ __forceinline__ long long range_start(long long quotient, int remainder, int p) {
  return quotient * p + min(p, remainder);
}

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
