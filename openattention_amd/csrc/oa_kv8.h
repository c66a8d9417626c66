// What the kernels of the 8-bit paged cache share.
#pragma once
#include "oa_common.h"
#include "openattention_kv8.h"

namespace kv8 {

// 2^e, -126 <= e <= 127
__device__ __forceinline__ float power(int e) { return __uint_as_float((unsigned)(127 + e) << 23); }

// The last of B sequences whose begin(b) is at most id, by all lanes of a wave together: two loads one after the other up
// to 4096 sequences.  (Beginnings that decrease, where a caller's starts are not what they should be, give some
// sequence, whose own checks hold.)
template <typename Begin>
__device__ __forceinline__ int sequence_of(int B, int id, Begin begin) {
  const int lane = threadIdx.x & 63;
  int lo = 0, n = B;
  while (n > 1) {
    const int step = (n + 63) >> 6, at = (lane + 1) * step;
    const int c = __popcll(__ballot(at < n && begin(lo + min(at, n - 1)) <= id));
    lo += c * step;
    n = min(step, n - c * step);
  }
  return __builtin_amdgcn_readfirstlane(lo);
}

}  // namespace kv8
