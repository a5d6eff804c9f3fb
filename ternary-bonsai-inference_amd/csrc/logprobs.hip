// Log probabilities of given tokens, entropy and top alternatives of rows of
// logits.
#include <hip/hip_runtime.h>

#include <cmath>
#include <string>

#include "../../include/bonsai_hip_serve.h"
#include "common.hpp"

namespace bh {
namespace {

struct LogprobArgs {
  const float *x;
  const uint32_t *tokens;
  float *logprob, *entropy;
  uint32_t *top_ids;
  float *top_logprobs;
  uint32_t *bad_id;
  size_t row_stride;
  int vocab, n_top;
  float inv_temp;
};

// A logit and its id as one number that grows with the order of the
// alternatives: larger logits first, of equal ones the lower id; NaN below all.
__device__ __forceinline__ uint64_t key_of(float x, uint32_t id) {
  uint32_t b = __float_as_uint(x + 0.0f);  // -0 becomes 0
  b = b & 0x80000000u ? ~b : b | 0x80000000u;
  if (x != x) b = 0;
  return static_cast<uint64_t>(b) << 32 | (~id);
}

struct Max64 {
  __device__ uint64_t operator()(uint64_t a, uint64_t b) const { return a > b ? a : b; }
};

__global__ __launch_bounds__(256) void token_logprobs_kernel(LogprobArgs a) {
  __shared__ double lds[4];
  __shared__ float fl[4];
  __shared__ uint64_t kl[4];
  const float *x = a.x + blockIdx.x * a.row_stride;
  float m = -INFINITY;
  bool nan = false;
  for (int i = threadIdx.x; i < a.vocab; i += 256) {
    m = x[i] > m ? x[i] : m;
    nan |= x[i] != x[i];
  }
  m = group_reduce<256>(m, MaxOp{}, fl);
  double s = 0.0, t = 0.0;
  for (int i = threadIdx.x; i < a.vocab; i += 256) {
    const float z = (x[i] - m) * a.inv_temp;
    const float e = expf(z);
    s += e;
    if (e > 0.0f) t += static_cast<double>(e) * z;
  }
  s = group_reduce<256>(s, SumOp{}, lds);
  __syncthreads();
  t = group_reduce<256>(t, SumOp{}, lds);
  const bool bad = __syncthreads_or(nan) || !(m > -INFINITY && m < INFINITY);
  const float log_s = bad ? NAN : static_cast<float>(log(s));
  if (threadIdx.x == 0) {
    if (a.logprob) {
      const uint32_t id = a.tokens[blockIdx.x];
      const bool in = id < static_cast<uint32_t>(a.vocab);
      if (!in && a.bad_id) *a.bad_id = id;
      a.logprob[blockIdx.x] = in ? (x[id] - m) * a.inv_temp - log_s : NAN;
    }
    if (a.entropy) a.entropy[blockIdx.x] = bad ? NAN : static_cast<float>(log(s) - t / s);
  }
  uint64_t below = ~uint64_t{0};
  for (int j = 0; j < a.n_top; ++j) {
    uint64_t best = 0;
    for (int i = threadIdx.x; i < a.vocab; i += 256) {
      const uint64_t k = key_of(x[i], i);
      if (k < below && k > best) best = k;
    }
    __syncthreads();
    best = group_reduce<256>(best, Max64{}, kl);
    below = best;
    if (threadIdx.x == 0) {
      const uint32_t id = ~static_cast<uint32_t>(best);
      const size_t o = static_cast<size_t>(blockIdx.x) * a.n_top + j;
      a.top_ids[o] = id;
      a.top_logprobs[o] = (x[id] - m) * a.inv_temp - log_s;
    }
  }
}

int check(const bh_token_logprobs_args &p) {
  if (p.vocab == 0 || p.vocab > 0x7fffffffu)
    return fail(BH_ERR_SHAPE, "token_logprobs: vocab must be 1 .. 2^31 - 1");
  if (p.row_stride < p.vocab)
    return fail(BH_ERR_SHAPE, "token_logprobs: row_stride " + std::to_string(p.row_stride) +
                                  " below vocab " + std::to_string(p.vocab));
  size_t n;
  if (p.n_rows > 0x7fffffffu || !mul_size(p.n_rows, p.row_stride, sizeof(float), &n))
    return fail(BH_ERR_SHAPE, "token_logprobs: size overflow");
  if (p.n_top > BH_MAX_TOP || p.n_top > p.vocab)
    return fail(BH_ERR_SHAPE, "token_logprobs: n_top " + std::to_string(p.n_top) + " above " +
                                  std::to_string(BH_MAX_TOP) + " or vocab");
  if (!(p.inv_temp > 0.0f) || std::isinf(p.inv_temp))
    return fail(BH_ERR_ARG, "token_logprobs: inv_temp must be finite and above 0");
  if (p.n_rows != 0) {
    if (!p.x || (p.logprob && !p.tokens) || (p.n_top != 0 && (!p.top_ids || !p.top_logprobs)))
      return fail(BH_ERR_ARG, "token_logprobs: null pointer");
  }
  return BH_OK;
}

}  // namespace
}  // namespace bh

using namespace bh;

extern "C" size_t bh_token_logprobs_workspace(const bh_token_logprobs_args *args) { return 0; }

extern "C" int bh_token_logprobs(const bh_token_logprobs_args *args, bh_stream stream) {
  if (!args) return fail(BH_ERR_ARG, "token_logprobs: null args");
  const bh_token_logprobs_args &p = *args;
  if (int e = check(p)) return e;
  if (p.n_rows == 0 || (!p.logprob && !p.entropy && p.n_top == 0)) return ok();
  LogprobArgs a{p.x, p.tokens, p.logprob, p.entropy, p.top_ids, p.top_logprobs, p.bad_id,
                p.row_stride, static_cast<int>(p.vocab), static_cast<int>(p.n_top), p.inv_temp};
  BH_LAUNCH(token_logprobs_kernel, static_cast<unsigned>(p.n_rows), 256, 0, as_stream(stream), a);
  return ok();
}
