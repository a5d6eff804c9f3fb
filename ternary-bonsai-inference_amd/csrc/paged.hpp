// What the kernels over a paged cache share (gfx950).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "../../include/bonsai_hip_serve.h"

namespace bh {

// x / d for 0 <= x < 2^31 by one high product: with s the smallest shift whose
// 2^s >= d and m = floor(2^(31 + s) / d) + 1, m < 2^32 and
// floor(x m / 2^(31 + s)) = floor(x / d): the excess x (m d - 2^(31 + s)) / (d 2^(31 + s))
// is at most x / 2^(31 + s) < 1 / d, as x < 2^31 and d <= 2^s.
struct FastDiv {
  int d = 1;
  uint32_t m = 0;
  int shift = 0;
  FastDiv() = default;
  explicit FastDiv(uint32_t div) : d(static_cast<int>(div)) {
    int s = 0;
    while ((uint64_t{1} << s) < div) ++s;
    m = static_cast<uint32_t>((uint64_t{1} << (31 + s)) / div + 1);
    shift = s;
  }
  __host__ __device__ __forceinline__ int div(int x) const {
    return static_cast<int>((static_cast<uint64_t>(static_cast<uint32_t>(x)) * m) >> (31 + shift));
  }
  __host__ __device__ __forceinline__ int mod(int x) const { return x - div(x) * d; }
};

// Checks a cache's sizes, type and strides; BH_OK, or the status with its text recorded.
int check_paged_cache(const bh_paged_cache &c, const char *who);

}  // namespace bh
