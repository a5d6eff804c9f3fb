// Log probabilities of given tokens, entropy and top alternatives of rows of
// logits, each logit read once.
//
// With m a running maximum and z = (x - m) inv_temp log2(e), a thread keeps
//   S = sum 2^z and T = sum 2^z z
// over what it has read; a larger maximum m' moves them by d = (m - m') inv_temp
// log2(e) to 2^d S and 2^d (T + d S).  Then log Z = m inv_temp + ln S and the
// entropy is ln S - ln 2 T / S: two terms of one sign, so that nothing cancels for
// a row that is sure of its token.
//
// Alternatives: a logit and its id make one 64-bit key in the order asked for
// (larger first, of equal ones the lower id), so all keys differ.  Each wave
// keeps its best n in LDS.  In a tile of 64 x 16 logits the n-th largest of the
// lanes' own maxima is a bound that the wave's n best all reach, and at most
// 16 n keys do; those join the kept ones, and each key's rank, counted by
// comparing it with all of them, is its place.  Later tiles are only looked at
// where a lane's maximum passes the n-th key kept, and their few keys move into
// the list one by one.
//
// Long rows are split over as many blocks as fill the card; a second launch then
// joins a row's parts.  Bound by reading the logits where there are many (2048 rows
// of 248320 with 5 alternatives 342 us, 5.9 TB/s; 512 rows 101, with 20 107, with
// none 93), by the chain load - exponentials - selection - second launch where
// there are few (8 rows with 20 alternatives 15.2 us, with none 6.5).
#include <hip/hip_runtime.h>

#include <cmath>
#include <string>

#include "../../include/bonsai_hip_serve.h"
#include "common.hpp"

namespace bh {
namespace {

constexpr int kLpThreads = 256, kLpWaves = kLpThreads / 64;
constexpr int kPer = 16;                     // logits of a thread and tile
constexpr int kLpTile = kPer * kLpThreads;   // 4096
constexpr int kMaxParts = 128;               // blocks of a row
// keys of a wave: those kept, and a tile's
constexpr int kKeep = (1 + kPer) * BH_MAX_TOP;
constexpr int kFew = 8;  // up to so many keys of a tile go into the list one by one

struct Part {
  double s, t;
  float m;
};

struct LogprobArgs {
  const float *x;
  const uint32_t *tokens;
  float *logprob, *entropy;
  uint32_t *top_ids;
  float *top_logprobs;
  uint32_t *bad_id;
  size_t row_stride;
  int vocab, n_top, n_parts;
  float inv_temp, k2;  // k2 = inv_temp log2(e)
  Part *parts;         // [n_rows][n_parts]
  uint64_t *keys;      // [n_rows][n_parts][n_top]
};

// Bits that grow with the value; -0 as 0, NaN below every number.
__device__ __forceinline__ uint32_t order_of(float x) {
  uint32_t b = __float_as_uint(x + 0.0f);
  b = b & 0x80000000u ? ~b : b | 0x80000000u;
  return x != x ? 0 : b;
}
__device__ __forceinline__ float value_of_order(uint32_t b) {
  return __uint_as_float(b & 0x80000000u ? b & 0x7fffffffu : ~b);
}
__device__ __forceinline__ uint64_t key_of(float x, uint32_t id) {
  return static_cast<uint64_t>(order_of(x)) << 32 | (~id);
}
__device__ __forceinline__ float value_of(uint64_t key) {
  return value_of_order(static_cast<uint32_t>(key >> 32));
}

struct Max64 {
  __device__ uint64_t operator()(uint64_t a, uint64_t b) const { return a > b ? a : b; }
};

__device__ __forceinline__ uint64_t lane_value(uint64_t x, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(x), lane);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(x >> 32), lane);
  return static_cast<uint64_t>(hi) << 32 | lo;
}

// Orders the wave's LDS writes before its reads (the wave runs in step).
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The n-th largest of the lanes' keys (equal ones, which are 0s, count as one).
__device__ __forceinline__ uint64_t nth_of_lanes(uint64_t key, int n, int lane) {
  int rank = 0;
#pragma unroll 8
  for (int i = 0; i < 64; ++i) rank += lane_value(key, i) > key;
  const uint64_t at = __ballot(rank == n - 1);
  return at ? lane_value(key, __builtin_ffsll(at) - 1) : 0;
}

// The largest b of 16 significant bits that at least n lanes reach: sixteen
// ballots, where the exact n-th takes 64 compares of keys.  It may let a few more
// than n lanes pass, and any number of equal ones.
__device__ __forceinline__ uint32_t bound_of_lanes(uint32_t order, int n) {
  uint32_t b = 0;
#pragma unroll
  for (int bit = 31; bit >= 16; --bit) {
    const uint32_t up = b | 1u << bit;
    if (__popcll(__ballot(order >= up)) >= n) b = up;
  }
  return b;
}

// A wave's best keys in order, lane i holding the i-th; 0 behind the last.
struct Kept {
  uint64_t key = 0;
  int count = 0;

  // Takes in one key: the lanes from its place on move up by one.
  __device__ __forceinline__ void insert(uint64_t x, int n, int lane) {
    const int place = __popcll(__ballot(key > x));
    const uint64_t below = dpp_move<0x138>(key);  // of the lane before
    key = lane < place ? key : lane == place ? x : below;
    if (lane >= n) key = 0;
    count = min(count + 1, n);
  }
  // Takes in buf[0 .. total): each key's place is the number of larger ones.
  __device__ __forceinline__ void replace(const uint64_t *buf, uint64_t *out, int total, int n,
                                          int lane) {
    wave_sync();
    if (lane < n) out[lane] = 0;
    wave_sync();
    for (int k = 0; k < total; k += 64) {
      const uint64_t mine = k + lane < total ? buf[k + lane] : 0;
      int rank = 0;
#pragma unroll 8
      for (int j = 0; j < total; ++j) rank += buf[j] > mine;
      if (mine != 0 && rank < n) out[rank] = mine;
    }
    wave_sync();
    key = lane < n ? out[lane] : 0;
    count = __popcll(__ballot(key != 0));
  }
};

// The waves' ordered lists of n keys (0: none) into the n largest of them all, in
// order; 0 behind the last.  put(place, key) takes one.  A key's place is its own
// in its list and, by halving, that in the three others.
template <class F>
__device__ __forceinline__ void merge_waves(const uint64_t (*lists)[BH_MAX_TOP], int n, F put) {
  const int tid = threadIdx.x;
  if (tid >= kLpWaves * n) return;
  const int own = tid / n;
  const uint64_t mine = lists[own][tid - own * n];
  int above[kLpWaves];
#pragma unroll
  for (int w = 0; w < kLpWaves; ++w) above[w] = 0;
#pragma unroll
  for (int step = BH_MAX_TOP; step > 0; step >>= 1)
#pragma unroll
    for (int w = 0; w < kLpWaves; ++w) {
      const int at = above[w] + step;
      if (at <= n && lists[w][at - 1] > mine) above[w] = at;
    }
  int rank = 0;
#pragma unroll
  for (int w = 0; w < kLpWaves; ++w) rank += above[w];
  if (mine != 0) {
    if (rank < n) put(rank, mine);
  } else {  // the keys are `rank` in all: 0s behind them
    for (int i = rank; i < n; ++i) put(i, 0);
  }
}

// Joins the block's (m, s, t) into one; every thread gets it.
__device__ __forceinline__ Part join_block(float m, double s, double t, float k2, float *fl,
                                           double *dl) {
  Part p;
  p.m = group_reduce<kLpThreads>(m, MaxOp{}, fl);
  if (m == -INFINITY) {  // s, t: 0, or NaN from a NaN logit
    t = s;
  } else {
    const float d = (m - p.m) * k2;
    const double by = __builtin_amdgcn_exp2f(d);
    t = by == 0.0 ? 0.0 : by * (t + d * s);
    s *= by;
  }
  p.s = group_reduce<kLpThreads>(s, SumOp{}, dl);
  __syncthreads();
  p.t = group_reduce<kLpThreads>(t, SumOp{}, dl);
  return p;
}

// The chosen token's logit, loaded by thread 0 ahead of its use.
struct Chosen {
  uint32_t id;
  float x;
  bool in;
};
__device__ __forceinline__ Chosen load_chosen(const LogprobArgs &a, size_t row) {
  Chosen c{0, 0.0f, false};
  if (threadIdx.x == 0 && a.logprob) {
    c.id = a.tokens[row];
    c.in = c.id < static_cast<uint32_t>(a.vocab);
    if (c.in) c.x = a.x[row * a.row_stride + c.id];
  }
  return c;
}

// The row's logprob and entropy from its joined sums; ln S for the alternatives.
__device__ __forceinline__ float finish_row(const LogprobArgs &a, size_t row, const Part &p,
                                            const Chosen &c) {
  const bool bad = !(p.m > -INFINITY && p.m < INFINITY);
  const double ln = log(p.s);
  const float log_s = bad ? NAN : static_cast<float>(ln);
  if (threadIdx.x == 0) {
    if (a.logprob) {
      if (!c.in && a.bad_id) *a.bad_id = c.id;
      a.logprob[row] = c.in ? (c.x - p.m) * a.inv_temp - log_s : NAN;
    }
    if (a.entropy)
      a.entropy[row] = bad ? NAN : static_cast<float>(ln - 0.693147180559945309 * (p.t / p.s));
  }
  return log_s;
}

__device__ __forceinline__ void put_top(const LogprobArgs &a, size_t row, int place, uint64_t key,
                                        float m, float log_s) {
  const size_t o = row * a.n_top + place;
  a.top_ids[o] = ~static_cast<uint32_t>(key);
  a.top_logprobs[o] = (value_of(key) - m) * a.inv_temp - log_s;
}

// A thread's logits of a tile: four pieces of four; -inf outside the row.
__device__ __forceinline__ void load_tile(const LogprobArgs &a, const float *x, int64_t tile,
                                          int64_t n, int skew, float *v) {
  const uint32_t at = static_cast<uint32_t>(tile) * kLpTile + 4 * threadIdx.x - skew;
  if (tile * kLpTile >= skew && (tile + 1) * kLpTile <= n) {
#pragma unroll
    for (int k = 0; k < kPer; k += 4) {
      const float4 p = *reinterpret_cast<const float4 *>(x + at + k * kLpThreads);
      v[k] = p.x, v[k + 1] = p.y, v[k + 2] = p.z, v[k + 3] = p.w;
    }
  } else {
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const uint32_t id = at + (k & ~3) * kLpThreads + (k & 3);
      v[k] = id < static_cast<uint32_t>(a.vocab) ? x[id] : -INFINITY;
    }
  }
}

// Block (row, part): the tiles of a part of a row.  Tiles begin at the row's last
// 16-byte boundary before it, so that whole pieces load at once for any row.
template <bool TOP>
__global__ __launch_bounds__(kLpThreads) void token_logprobs_kernel(LogprobArgs a) {
  __shared__ uint64_t keep[TOP ? kLpWaves : 1][TOP ? kKeep : 1];
  __shared__ uint64_t lists[TOP ? kLpWaves : 1][BH_MAX_TOP];
  __shared__ float fl[kLpWaves];
  __shared__ double dl[kLpWaves];
  __shared__ uint64_t shown[kLpWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const size_t row = blockIdx.x / a.n_parts;
  const int part = blockIdx.x - row * a.n_parts;
  const float *x = a.x + row * a.row_stride;
  const int skew = static_cast<int>(reinterpret_cast<uintptr_t>(x) >> 2 & 3);
  const int64_t n = static_cast<int64_t>(a.vocab) + skew;  // places, of which `skew` before the row
  const int64_t tiles = (n + kLpTile - 1) / kLpTile;
  const int64_t tile0 = tiles * part / a.n_parts, tile1 = tiles * (part + 1) / a.n_parts;

  const bool whole = a.n_parts == 1;
  Chosen chosen{};
  if (whole) chosen = load_chosen(a, row);
  float m = -INFINITY;
  double s = 0.0, t = 0.0;
  Kept kept;
  uint64_t bound = 0;  // the last of the kept keys, once they are n
  bool full = false, strict = true;  // strict: the bound is a key of this wave
  if constexpr (TOP) {
    if (tid < kLpWaves) shown[tid] = 0;
    __syncthreads();
  }
  float ahead[kPer];
  load_tile(a, x, tile0, n, skew, ahead);
  for (int64_t tile = tile0; tile < tile1; ++tile) {
    // id of the thread's first logit; those before the row wrap round to no id
    const uint32_t at = static_cast<uint32_t>(tile) * kLpTile + 4 * tid - skew, vocab = a.vocab;
    float v[kPer];
#pragma unroll
    for (int k = 0; k < kPer; ++k) v[k] = ahead[k];
    if (tile + 1 < tile1) load_tile(a, x, tile + 1, n, skew, ahead);
    float top = v[0];
#pragma unroll
    for (int k = 1; k < kPer; ++k) top = fmaxf(top, v[k]);
    if (top > m) {
      if (m > -INFINITY) {
        const float d = (m - top) * a.k2;
        const double by = __builtin_amdgcn_exp2f(d);
        t = by == 0.0 ? 0.0 : by * (t + d * s);
        s *= by;
      }
      m = top;
    }
    const float ref = m == -INFINITY ? 0.0f : m;
    float es = 0.0f, et = 0.0f;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      const float z = (v[k] - ref) * a.k2;
      const float e = __builtin_amdgcn_exp2f(z);
      es += e;
      et = __builtin_fmaf(e, fmaxf(z, -1000.0f), et);  // -inf has weight 0, and 0 times it
    }
    s += es;
    t += et;

    if constexpr (TOP) {
      // full: n keys are kept, and a later logit has to pass the last one's value.
      // Each wave also shows its ceil(n / 4)-th best: n keys of the block reach the
      // least of the four, which soon lies far above a wave's own n-th.  (A wave
      // may read an older one, which bounds less.)  Another wave's key may stand
      // behind an equal logit of this one, so that bound lets equal ones pass.
      if (full) {
        uint64_t all = ~uint64_t{0};
#pragma unroll
        for (int w = 0; w < kLpWaves; ++w) {
          const uint64_t of =
              __hip_atomic_load(&shown[w], __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
          all = of < all ? of : all;
        }
        if (all > bound) bound = all, strict = false;
      }
      const float last = value_of(bound);
      if (!full || __any(strict ? top > last : top >= last)) {
        // logits from `least` on join the kept ones
        float least = full ? last : -INFINITY;
        const bool many = __popcll(__ballot(strict ? top > least : top >= least)) > a.n_top;
        if (many) {
          const float of_lanes = value_of_order(bound_of_lanes(order_of(top), a.n_top));
          least = of_lanes > least ? of_lanes : least;
        }
        uint64_t pass[kPer];
        int more = 0;
#pragma unroll
        for (int k = 0; k < kPer; ++k) {
          pass[k] = __ballot(many || !full || !strict ? v[k] >= least : v[k] > least);
          more += __popcll(pass[k]);
        }
        uint64_t from = full ? bound + 1 : 1;
        // Too few for the list, or too many equal ones: by keys.  Then NaN logits
        // count too, and the lanes' n-th best is a bound that at most n lanes reach.
        const bool by_key = (!full && (!many || more < a.n_top)) || more > kPer * a.n_top;
        if (by_key) {
          uint64_t best = 0;
#pragma unroll
          for (int k = 0; k < kPer; ++k) {
            const uint32_t id = at + (k & ~3) * kLpThreads + (k & 3);
            const uint64_t key = id < vocab ? key_of(v[k], id) : 0;
            best = key > best ? key : best;
          }
          if (__popcll(__ballot(best >= from)) > a.n_top) {
            const uint64_t nth = nth_of_lanes(best, a.n_top, lane);
            from = nth > from ? nth : from;
          }
#pragma unroll
          for (int k = 0; k < kPer; ++k) {
            const uint32_t id = at + (k & ~3) * kLpThreads + (k & 3);
            pass[k] = __ballot((id < vocab ? key_of(v[k], id) : 0) >= from);
          }
        }
        if (!by_key && more <= kFew) {
#pragma unroll
          for (int k = 0; k < kPer; ++k) {
            if (pass[k] == 0) continue;
            const uint32_t id = at + (k & ~3) * kLpThreads + (k & 3);
            const uint64_t key = id < vocab ? key_of(v[k], id) : 0;
            for (uint64_t left = pass[k]; left != 0; left &= left - 1) {
              const uint64_t x = lane_value(key, __builtin_ffsll(left) - 1);
              if (x >= from) kept.insert(x, a.n_top, lane);
            }
          }
        } else {
          uint64_t *buf = keep[wave];
          int total = kept.count;
          if (lane < total) buf[lane] = kept.key;
#pragma unroll
          for (int k = 0; k < kPer; ++k) {
            if (pass[k] == 0) continue;
            const uint32_t id = at + (k & ~3) * kLpThreads + (k & 3);
            if (pass[k] >> lane & 1) {
              const uint64_t key = key_of(v[k], id);
              buf[total + __popcll(pass[k] & ((uint64_t{1} << lane) - 1))] =
                  id < vocab && key >= from ? key : 0;
            }
            total += __popcll(pass[k]);
          }
          kept.replace(buf, lists[wave], total, a.n_top, lane);
        }
        if (kept.count == a.n_top) {
          const uint64_t own = lane_value(kept.key, a.n_top - 1);
          if (own > bound) bound = own, strict = true;
          if (lane == (a.n_top - 1) / kLpWaves)
            __hip_atomic_store(&shown[wave], kept.key, __ATOMIC_RELAXED,
                               __HIP_MEMORY_SCOPE_WORKGROUP);
        }
        // a NaN at the end gives way to any number
        full = kept.count == a.n_top && bound >> 32 != 0;
      }
    }
  }

  const Part p = join_block(m, s, t, a.k2, fl, dl);
  float log_s = 0.0f;
  if (whole) log_s = finish_row(a, row, p, chosen);
  else if (tid == 0) a.parts[blockIdx.x] = p;
  if constexpr (TOP) {
    if (lane < a.n_top) lists[wave][lane] = kept.key;
    __syncthreads();
    uint64_t *out = a.keys + static_cast<size_t>(blockIdx.x) * a.n_top;
    merge_waves(lists, a.n_top, [&](int place, uint64_t key) {
      if (whole) put_top(a, row, place, key, p.m, log_s);
      else out[place] = key;
    });
  }
}

// A row's parts: their sums joined, their lists' best keys.
template <bool TOP>
__global__ __launch_bounds__(kLpThreads) void token_logprobs_join_kernel(LogprobArgs a) {
  constexpr int kKeys = kMaxParts * BH_MAX_TOP / kLpThreads;  // keys of a thread at most
  __shared__ uint64_t keep[TOP ? kLpWaves : 1][TOP ? kKeep : 1];
  __shared__ uint64_t lists[TOP ? kLpWaves : 1][BH_MAX_TOP];
  __shared__ float fl[kLpWaves];
  __shared__ double dl[kLpWaves];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const size_t row = blockIdx.x;
  uint64_t key[kKeys];
  const int n = a.n_parts * a.n_top;
  if constexpr (TOP) {
#pragma unroll
    for (int k = 0; k < kKeys; ++k)
      key[k] = tid + k * kLpThreads < n ? a.keys[row * n + tid + k * kLpThreads] : 0;
  }
  const Chosen chosen = load_chosen(a, row);
  Part mine{0.0, 0.0, -INFINITY};
  if (tid < a.n_parts) mine = a.parts[row * a.n_parts + tid];
  const Part p = join_block(mine.m, mine.s, mine.t, a.k2, fl, dl);
  const float log_s = finish_row(a, row, p, chosen);
  if constexpr (TOP) {
    uint64_t best = 0;
#pragma unroll
    for (int k = 0; k < kKeys; ++k) best = key[k] > best ? key[k] : best;
    uint64_t from = 1;
    if (n > 64 * kLpWaves) {  // more than a key a lane
      from = static_cast<uint64_t>(bound_of_lanes(static_cast<uint32_t>(best >> 32), a.n_top)) << 32;
      int more = 0;
#pragma unroll
      for (int k = 0; k < kKeys; ++k) more += __popcll(__ballot(key[k] >= from));
      if (more > kKeep) from = nth_of_lanes(best, a.n_top, lane);
      from = from > 1 ? from : 1;
    }
    int count = 0;
#pragma unroll
    for (int k = 0; k < kKeys; ++k) {
      const uint64_t pass = __ballot(key[k] >= from);
      if (pass == 0) continue;
      if (key[k] >= from) keep[wave][count + __popcll(pass & ((uint64_t{1} << lane) - 1))] = key[k];
      count += __popcll(pass);
    }
    Kept kept;
    kept.replace(keep[wave], lists[wave], count, a.n_top, lane);  // and into lists
    __syncthreads();
    merge_waves(lists, a.n_top, [&](int place, uint64_t k) {
      put_top(a, row, place, k, p.m, log_s);
    });
  }
}

int check(const bh_token_logprobs_args &p) {
  if (p.vocab == 0 || p.vocab > 0x7fffffffu)
    return fail(BH_ERR_SHAPE, "token_logprobs: vocab must be 1 .. 2^31 - 1");
  if (p.row_stride < p.vocab)
    return fail(BH_ERR_SHAPE, "token_logprobs: row_stride " + std::to_string(p.row_stride) +
                                  " below vocab " + std::to_string(p.vocab));
  size_t n;
  if (p.n_rows > 0x7fffffffu / kMaxParts || !mul_size(p.n_rows, p.row_stride, sizeof(float), &n))
    return fail(BH_ERR_SHAPE, "token_logprobs: size overflow");
  if (p.n_top > BH_MAX_TOP || p.n_top > p.vocab)
    return fail(BH_ERR_SHAPE, "token_logprobs: n_top " + std::to_string(p.n_top) + " above " +
                                  std::to_string(BH_MAX_TOP) + " or vocab");
  if (!(p.inv_temp > 0.0f) || std::isinf(p.inv_temp * kExpL2E))
    return fail(BH_ERR_ARG, "token_logprobs: inv_temp must be finite and above 0");
  if (p.n_rows != 0) {
    if (reinterpret_cast<uintptr_t>(p.x) % sizeof(float) != 0)
      return fail(BH_ERR_ARG, "token_logprobs: misaligned x");
    if (!p.x || (p.logprob && !p.tokens) || (p.n_top != 0 && (!p.top_ids || !p.top_logprobs)))
      return fail(BH_ERR_ARG, "token_logprobs: null pointer");
  }
  return BH_OK;
}

bool nothing(const bh_token_logprobs_args &p) {
  return p.n_rows == 0 || (!p.logprob && !p.entropy && p.n_top == 0);
}

// Blocks of a row: about four blocks a compute unit in all, a tile each at least.
// 512 rows of 248320 with 5 alternatives, 1 / 2 / 4 / 8 a unit: 121 / 117 / 111 / 123
// us; 64 rows with 20: 58 / 41 / 35 / 36.  A row of few tiles has one block, whose
// time then is about that of the second launch: up to 8 tiles without alternatives
// (256 rows of 32000: 8.4 us, split 12.7; 61 rows: 8.0 and 7.8, and half the
// launches), up to 2 with them (one row of 8192 with 5: 8.6, 11.4 split; 16 rows of
// 16384 with 20: 16.2, 13.9 split).
size_t parts_of(const bh_token_logprobs_args &p) {
  const size_t tiles = (p.vocab + kLpTile - 1) / kLpTile;
  if (tiles <= (p.n_top == 0 ? 8 : 2)) return 1;
  size_t parts = 4 * device_cu_count() / p.n_rows;
  if (parts > tiles) parts = tiles;
  if (parts > static_cast<size_t>(kMaxParts)) parts = kMaxParts;
  return parts < 1 ? 1 : parts;
}

size_t workspace_of(const bh_token_logprobs_args &p) {
  const size_t parts = parts_of(p);
  return parts == 1 ? 0 : p.n_rows * parts * (sizeof(Part) + 8 * p.n_top);
}

}  // namespace
}  // namespace bh

using namespace bh;

extern "C" size_t bh_token_logprobs_workspace(const bh_token_logprobs_args *args) {
  if (!args || check(*args) != BH_OK || nothing(*args)) return 0;
  return workspace_of(*args);
}

extern "C" int bh_token_logprobs(const bh_token_logprobs_args *args, bh_stream stream) {
  if (!args) return fail(BH_ERR_ARG, "token_logprobs: null args");
  const bh_token_logprobs_args &p = *args;
  if (int e = check(p)) return e;
  if (nothing(p)) return ok();
  hipStream_t st = as_stream(stream);
  const size_t need = workspace_of(p), parts = parts_of(p);
  char *ws = static_cast<char *>(p.workspace);
  if (need != 0) {
    if (ws) {
      if (!aligned16(ws) || p.workspace_bytes < need)
        return fail(BH_ERR_SHAPE, "token_logprobs: workspace of " +
                                      std::to_string(p.workspace_bytes) + " bytes, " +
                                      std::to_string(need) + " needed on a 16-byte boundary");
    } else {
      ws = static_cast<char *>(device_scratch(need, kScratchLogprobs, st));
      if (!ws) return BH_ERR_HIP;
    }
  }
  LogprobArgs a{};
  a.x = p.x, a.tokens = p.tokens, a.logprob = p.logprob, a.entropy = p.entropy;
  a.top_ids = p.top_ids, a.top_logprobs = p.top_logprobs, a.bad_id = p.bad_id;
  a.row_stride = p.row_stride, a.vocab = static_cast<int>(p.vocab);
  a.n_top = static_cast<int>(p.n_top), a.n_parts = static_cast<int>(parts);
  a.inv_temp = p.inv_temp, a.k2 = p.inv_temp * kExpL2E;
  a.parts = reinterpret_cast<Part *>(ws);
  a.keys = reinterpret_cast<uint64_t *>(ws + p.n_rows * parts * sizeof(Part));
  const unsigned blocks = static_cast<unsigned>(p.n_rows * parts);
  if (p.n_top) BH_LAUNCH(token_logprobs_kernel<true>, blocks, kLpThreads, 0, st, a);
  else BH_LAUNCH(token_logprobs_kernel<false>, blocks, kLpThreads, 0, st, a);
  if (parts > 1) {
    const unsigned rows = static_cast<unsigned>(p.n_rows);
    if (p.n_top) BH_LAUNCH(token_logprobs_join_kernel<true>, rows, kLpThreads, 0, st, a);
    else BH_LAUNCH(token_logprobs_join_kernel<false>, rows, kLpThreads, 0, st, a);
  }
  return ok();
}
