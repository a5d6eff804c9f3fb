// What the kernels over ragged requests with states in slots share (gfx950).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "common.hpp"

namespace bh {

// A step's requests: tokens q_start[r] .. q_start[r + 1] - 1 are request r's, its
// state is read from slot src[r] and written to slot dst[r] of n_slots.
struct Ragged {
  const int32_t *q_start, *src, *dst;
  int32_t *bad_slot;
  int n_tok, n_req, n_slots;
  size_t slot_stride;  // floats

  // Clipped tokens of request r.
  __device__ __forceinline__ void tokens(int r, int *begin, int *n) const {
    const int s = min(max(q_start[r], 0), n_tok), e = min(max(q_start[r + 1], 0), n_tok);
    *begin = s;
    *n = max(e - s, 0);
  }
  // The same of a request that is the wave's, in scalars: what follows from them is too.
  __device__ __forceinline__ void tokens_of(int r, int *begin, int *n) const {
    int s, count;
    tokens(r, &s, &count);
    *begin = __builtin_amdgcn_readfirstlane(s);
    *n = __builtin_amdgcn_readfirstlane(count);
  }
  // Slots of the wave's request r, -1: none (below 0, or past the pool and then noted).
  __device__ __forceinline__ void slots(int r, int *from, int *to) const {
    const int f = __builtin_amdgcn_readfirstlane(src[r]);
    const int t = __builtin_amdgcn_readfirstlane(dst[r]);
    *from = f >= 0 && f < n_slots ? f : -1;
    *to = t >= 0 && t < n_slots ? t : -1;
    if (bad_slot && threadIdx.x == 0) {
      if (f >= n_slots) *bad_slot = f;
      if (t >= n_slots) *bad_slot = t;
    }
  }
};

// The last r < n with pred(r), pred holding up to some r and not behind it; -1 if it
// does not hold for 0.  The wave asks at 64 places at a time: one round of loads for
// up to 64 requests, two for up to 4096.  (Of a pred that goes up and down some r.)
template <class P>
__device__ __forceinline__ int last_request(int n, P pred) {
  const int lane = threadIdx.x & 63;
  int lo = 0, count = n;
  while (true) {
    const int stride = (count + 63) / 64;
    const int64_t i = static_cast<int64_t>(lo) + static_cast<int64_t>(lane) * stride;
    const bool in = static_cast<int64_t>(lane) * stride < count;
    const uint64_t up = __ballot(in && pred(static_cast<int>(in ? i : lo)));
    if (up == 0) return -1;  // (only in the first round)
    const int at = 63 - __builtin_clzll(up);
    lo += at * stride;
    count = min(stride, count - at * stride);
    if (stride == 1) return lo;
  }
}

}  // namespace bh
