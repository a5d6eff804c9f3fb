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

// Inclusive running totals over the 64 lanes of a wave by DPP: within rows of 16,
// then a row's last into the next, then the lower half's last into the upper half.
// Lanes that get nothing add 0.
template <int CTRL, int ROWS, class T, class Op>
__device__ __forceinline__ T scan_step(T x, Op op) {
  if constexpr (sizeof(T) == 4) {
    return op(x, static_cast<T>(__builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, ROWS, 0xF, false)));
  } else {
    const int lo = __builtin_amdgcn_update_dpp(0, static_cast<int>(x), CTRL, ROWS, 0xF, false);
    const int hi = __builtin_amdgcn_update_dpp(0, static_cast<int>(x >> 32), CTRL, ROWS, 0xF, false);
    return op(x, static_cast<T>(static_cast<uint64_t>(static_cast<uint32_t>(hi)) << 32 |
                                static_cast<uint32_t>(lo)));
  }
}
template <class T, class Op>
__device__ __forceinline__ T lane_scan(T x, Op op) {
  x = scan_step<0x111, 0xF>(x, op);  // row_shr 1, 2, 4, 8
  x = scan_step<0x112, 0xF>(x, op);
  x = scan_step<0x114, 0xF>(x, op);
  x = scan_step<0x118, 0xF>(x, op);
  x = scan_step<0x142, 0xA>(x, op);  // row_bcast 15, 31
  return scan_step<0x143, 0xC>(x, op);
}

// Checks a cache's sizes, type and strides; BH_OK, or the status with its text recorded.
int check_paged_cache(const bh_paged_cache &c, const char *who);

}  // namespace bh
