// Log probabilities of given tokens, entropy and top alternatives of rows of
// logits, each logit read once.
//
// The pass over a row is logits.hpp's.  log Z = m inv_temp + ln S and the entropy is
// ln S - ln 2 T / S: two terms of one sign, so that nothing cancels for a row that is
// sure of its token.
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
#include "logits.hpp"

namespace bh {
namespace {

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

// Blocks of a row.  A row of few tiles has one block, whose
// time then is about that of the second launch: up to 8 tiles without alternatives
// (256 rows of 32000: 8.4 us, split 12.7; 61 rows: 8.0 and 7.8, and half the
// launches), up to 2 with them (one row of 8192 with 5: 8.6, 11.4 split; 16 rows of
// 16384 with 20: 16.2, 13.9 split).
size_t parts_of(const bh_token_logprobs_args &p) {
  const size_t tiles = (p.vocab + kLpTile - 1) / kLpTile;
  if (tiles <= (p.n_top == 0 ? 8 : 2)) return 1;
  return parts_of_rows(p.n_rows, p.vocab);
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
