// Causal conv + SiLU + L2 norms of many requests at once, each with its last k - 1
// inputs in a slot.
//
//   y_t[c] = silu(sum_j w[c][j] x_{t - k + 1 + j}[c]),  j ascending,
// and the first l2_dim channels scaled by 1 / max(sqrt(sum y^2), eps) over groups of
// head_dim (the sum in f64, as bh_l2_norm_rows).  Four operations a byte: it is bound
// by reading x and writing out once.  10240 channels, 2900 tokens of 3 prompts and 21
// decoders: 53.8 us, 4.5 TB/s; 64 decoders 8.1 us, four rounds of loads after one another
// (the search, offsets, slots, then states and inputs) in front of 21 MB.
#include <hip/hip_runtime.h>

#include <string>

#include "../../include/bonsai_hip_batch.h"
#include "common.hpp"
#include "conv.hpp"
#include "ragged.hpp"

namespace bh {
namespace {

constexpr int kBlock = 256;
constexpr int kRun = 8;  // tokens of a run

struct ConvArgs {
  const float *x, *w;
  float *state, *out;
  size_t x_stride;
  int ch, k, l2_dim, head_dim, groups;
  float eps;
  Ragged rag;
};

// k = 4, four channels a lane.  Block (run, 1024 channels): runs of kRun tokens, of
// one request each.  Request r's j-th run is run q_start[r] / kRun + r + j: that
// leaves ceil(n / kRun) runs to a request of n tokens at least, and every block finds
// its request without a table.  A run that is not a request's first has its window
// in x; the first reads the request's slot and leaves the new inputs, so that a slot
// read and written in place is its own lanes' only.
// LANES: lanes of a group that is normalised (1: none in this launch).
template <int LANES>
__global__ __launch_bounds__(kBlock) void conv_ragged4_kernel(ConvArgs a, int parts) {
  const int run = blockIdx.x / parts, part = blockIdx.x - run * parts;
  const Ragged &rag = a.rag;
  const int r = last_request(rag.n_req, [&](int i) {
    return static_cast<int64_t>(min(max(rag.q_start[i], 0), rag.n_tok) / kRun) + i <= run;
  });
  if (r < 0) return;
  int begin, n, from, to;
  rag.tokens_of(r, &begin, &n);
  const int64_t first = (run - (static_cast<int64_t>(begin / kRun) + r)) * kRun;
  if (first < 0 || first >= n) return;
  rag.slots(r, &from, &to);
  const int here = min(kRun, n - static_cast<int>(first));
  const int c0 = (part * kBlock + static_cast<int>(threadIdx.x)) * 4;
  const bool in = c0 < a.ch;
  const int c = in ? c0 : 0;
  const float *x = a.x + (begin + first) * a.x_stride + c;
  f32x4 xr[kRun];
#pragma unroll
  for (int t = 0; t < kRun; ++t)
    if (t < here) xr[t] = *reinterpret_cast<const f32x4 *>(x + t * a.x_stride);
  f32x4 w[4], win[3];  // by tap, by input: four channels each
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const f32x4 of = *reinterpret_cast<const f32x4 *>(a.w + static_cast<size_t>(c + e) * 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j][e] = of[j];
  }
  if (first != 0) {
#pragma unroll
    for (int j = 0; j < 3; ++j) win[j] = *reinterpret_cast<const f32x4 *>(x - (3 - j) * a.x_stride);
  } else {
    f32x4 s[3] = {f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}, f32x4{0, 0, 0, 0}};
    if (from >= 0) {
      const float *p = a.state + from * rag.slot_stride + static_cast<size_t>(c) * 3;
#pragma unroll
      for (int j = 0; j < 3; ++j) s[j] = *reinterpret_cast<const f32x4 *>(p + 4 * j);
    }
    // [channel][input] to [input][channel]
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int j = 0; j < 3; ++j) win[j][e] = s[(3 * e + j) / 4][(3 * e + j) % 4];
    if (to >= 0 && in) {
      // input e of the new ones: token n - 3 + e, or an old one
      f32x4 now[3];
#pragma unroll
      for (int e = 0; e < 3; ++e) {
        const int p = n - 3 + e;
        const f32x4 late = *reinterpret_cast<const f32x4 *>(x + static_cast<size_t>(max(p, 0)) * a.x_stride);
#pragma unroll
        for (int i = 0; i < 4; ++i)
          now[e][i] = p >= 0 ? late[i] : p == -1 ? win[2][i] : win[1][i];
      }
      float *d = a.state + to * rag.slot_stride + static_cast<size_t>(c) * 3;
#pragma unroll
      for (int j = 0; j < 3; ++j) {
        f32x4 o;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[i] = now[(4 * j + i) % 3][(4 * j + i) / 3];
        *reinterpret_cast<f32x4 *>(d + 4 * j) = o;
      }
    }
  }
  float *out = a.out + (begin + first) * static_cast<size_t>(a.ch) + c;
#pragma unroll
  for (int t = 0; t < kRun; ++t) {
    if (t >= here) break;
    f32x4 y;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float acc = ((w[0][e] * win[0][e] + w[1][e] * win[1][e]) + w[2][e] * win[2][e]) +
                        w[3][e] * xr[t][e];
      y[e] = silu_fast(acc);
    }
    if constexpr (LANES > 1) {
      if (part * kBlock * 4 < a.l2_dim) {  // (of all lanes: a sum over lanes follows)
        double sum = 0.0;
#pragma unroll
        for (int e = 0; e < 4; ++e) sum += static_cast<double>(y[e]) * y[e];
        sum = lane_group_reduce<LANES>(sum, SumOp{});
        const float norm = sqrtf(static_cast<float>(sum));
        const float by = 1.0f / (norm < a.eps ? a.eps : norm);  // (a NaN stays)
        if (c < a.l2_dim) y = y * by;
      }
    }
    if (in) *reinterpret_cast<f32x4 *>(out + t * static_cast<size_t>(a.ch)) = y;
    win[0] = win[1], win[1] = win[2], win[2] = xr[t];
  }
}

// Any k and layout: a thread a (token, channel).
__global__ __launch_bounds__(kBlock) void conv_ragged_kernel(ConvArgs a, int parts) {
  const int t = blockIdx.x / parts, c = (blockIdx.x - t * parts) * kBlock + threadIdx.x;
  const Ragged &rag = a.rag;
  const int r = last_request(rag.n_req, [&](int i) { return rag.q_start[i] <= t; });
  if (r < 0) return;
  int begin, n, from, to;
  rag.tokens_of(r, &begin, &n);
  if (t < begin || t >= begin + n) return;
  rag.slots(r, &from, &to);
  if (c >= a.ch) return;
  float acc = 0.0f;
  for (int j = 0; j < a.k; ++j) {
    const int p = t - (a.k - 1) + j;  // token
    float s = 0.0f;
    if (p >= begin) s = a.x[p * a.x_stride + c];
    else if (from >= 0)
      s = a.state[from * rag.slot_stride + static_cast<size_t>(c) * (a.k - 1) + (p - begin + a.k - 1)];
    acc += a.w[static_cast<size_t>(c) * a.k + j] * s;
  }
  a.out[static_cast<size_t>(t) * a.ch + c] = silu(acc);
}

// The groups' norms, in place: a wave a (token, group).
__global__ __launch_bounds__(kBlock) void conv_ragged_l2_kernel(ConvArgs a) {
  const int lane = threadIdx.x & 63;
  const int64_t item = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  const int t = static_cast<int>(item / a.groups), g = static_cast<int>(item % a.groups);
  if (t >= a.rag.n_tok) return;
  const int r = last_request(a.rag.n_req, [&](int i) { return a.rag.q_start[i] <= t; });
  if (r < 0) return;
  int begin, n;
  a.rag.tokens_of(r, &begin, &n);
  if (t < begin || t >= begin + n) return;  // a row of no request
  float *y = a.out + static_cast<size_t>(t) * a.ch + static_cast<size_t>(g) * a.head_dim;
  double sum = 0.0;
  for (int d = lane; d < a.head_dim; d += 64) sum += static_cast<double>(y[d]) * y[d];
  sum = lane_group_reduce<64>(sum, SumOp{});
  const float norm = sqrtf(static_cast<float>(sum));
  const float by = 1.0f / (norm < a.eps ? a.eps : norm);  // (a NaN stays)
  for (int d = lane; d < a.head_dim; d += 64) y[d] *= by;
}

// The slots written, once all outputs are there: a thread a (request, channel).  An
// old input moves to a lower place, which ascending order has read by then.
__global__ __launch_bounds__(kBlock) void conv_ragged_state_kernel(ConvArgs a, int parts) {
  const int r = blockIdx.x / parts, c = (blockIdx.x - r * parts) * kBlock + threadIdx.x;
  int begin, n, from, to;
  a.rag.tokens_of(r, &begin, &n);
  if (n == 0) return;
  a.rag.slots(r, &from, &to);
  if (to < 0 || c >= a.ch) return;
  const size_t at = static_cast<size_t>(c) * (a.k - 1);
  for (int i = 0; i < a.k - 1; ++i) {
    const int64_t p = static_cast<int64_t>(n) - (a.k - 1) + i;
    float s = 0.0f;
    if (p >= 0) s = a.x[(begin + p) * a.x_stride + c];
    else if (from >= 0) s = a.state[from * a.rag.slot_stride + at + (p + a.k - 1)];
    a.state[to * a.rag.slot_stride + at + i] = s;
  }
}

constexpr size_t kMostBlocks = 0xffffff;

int check(const bh_conv_ragged_args &p) {
  if (p.k < 1 || p.k > static_cast<size_t>(kMaxConvK))
    return fail(BH_ERR_SHAPE, "conv1d_silu_ragged: conv kernel size " + std::to_string(p.k) +
                                  " must be in 1.." + std::to_string(kMaxConvK));
  if (p.ch == 0 || p.ch > 0x7fffff00u)
    return fail(BH_ERR_SHAPE, "conv1d_silu_ragged: ch must be 1 .. 2^31 - 256");
  if (p.l2_dim > p.ch || (p.l2_dim != 0 && (p.head_dim == 0 || p.l2_dim % p.head_dim != 0)))
    return fail(BH_ERR_SHAPE, "conv1d_silu_ragged: l2_dim " + std::to_string(p.l2_dim) +
                                  " is above ch or no multiple of head_dim " +
                                  std::to_string(p.head_dim));
  if (p.x_stride < p.ch || (p.n_slots > 1 && p.slot_stride < p.ch * (p.k - 1)))
    return fail(BH_ERR_SHAPE, "conv1d_silu_ragged: a stride is below the rows it steps over");
  const size_t parts = (p.ch + kBlock - 1) / kBlock;
  size_t n;
  if (p.n_tok > 0x7fff0000u || p.n_req > kMostBlocks || !mul_size(p.n_tok + p.n_req, parts, &n) ||
      n > kMostBlocks || !mul_size(p.n_tok, p.x_stride, sizeof(float), &n) ||
      (p.l2_dim != 0 && p.n_tok * (p.l2_dim / p.head_dim) / 4 >= kMostBlocks) ||
      p.n_slots > 0x7fffffffu || !mul_size(p.n_slots, p.slot_stride, sizeof(float), &n))
    return fail(BH_ERR_SHAPE, "conv1d_silu_ragged: size overflow");
  if (p.n_req != 0 && p.n_tok != 0) {
    if (!p.x || !p.w || !p.out || !p.q_start || !p.src_slot || !p.dst_slot ||
        (p.k > 1 && p.n_slots != 0 && !p.state))
      return fail(BH_ERR_ARG, "conv1d_silu_ragged: null pointer");
    if (p.x == p.out)
      return fail(BH_ERR_ARG, "conv1d_silu_ragged: out must not be x (later tokens read it)");
  }
  return BH_OK;
}

}  // namespace
}  // namespace bh

using namespace bh;

extern "C" int bh_conv1d_silu_ragged(const bh_conv_ragged_args *args, bh_stream stream) {
  if (!args) return fail(BH_ERR_ARG, "conv1d_silu_ragged: null args");
  const bh_conv_ragged_args &p = *args;
  if (int e = check(p)) return e;
  if (p.n_req == 0 || p.n_tok == 0) return ok();
  ConvArgs a{};
  a.x = p.x, a.w = p.w, a.state = p.state, a.out = p.out, a.x_stride = p.x_stride;
  a.ch = static_cast<int>(p.ch), a.k = static_cast<int>(p.k);
  a.l2_dim = static_cast<int>(p.l2_dim), a.head_dim = static_cast<int>(p.head_dim);
  a.groups = p.l2_dim == 0 ? 0 : static_cast<int>(p.l2_dim / p.head_dim);
  a.eps = p.eps;
  // (one tap: no state, so that no slot of it is bad)
  a.rag = Ragged{p.q_start, p.src_slot, p.dst_slot, p.k > 1 ? p.bad_slot : nullptr,
                 static_cast<int>(p.n_tok), static_cast<int>(p.n_req),
                 static_cast<int>(p.k > 1 ? p.n_slots : 0), p.slot_stride};
  hipStream_t st = as_stream(stream);
  // lanes of a group: a power of two up to a wave's, whole groups a lane's four channels
  const size_t lanes = p.l2_dim == 0 ? 1 : p.head_dim / 4;
  const bool groups = p.l2_dim == 0 || (p.head_dim % 4 == 0 && lanes >= 2 && lanes <= 64 &&
                                        (lanes & (lanes - 1)) == 0);
  if (p.k == 4 && p.ch % 4 == 0 && p.x_stride % 4 == 0 && p.slot_stride % 4 == 0 && groups &&
      aligned16(p.x) && aligned16(p.out) && aligned16(p.w) && aligned16(p.state)) {
    const int parts = static_cast<int>((p.ch / 4 + kBlock - 1) / kBlock);
    const unsigned blocks = static_cast<unsigned>((p.n_tok / kRun + p.n_req) * parts);
    if (lanes == 1) BH_LAUNCH(conv_ragged4_kernel<1>, blocks, kBlock, 0, st, a, parts);
    else if (lanes == 2) BH_LAUNCH(conv_ragged4_kernel<2>, blocks, kBlock, 0, st, a, parts);
    else if (lanes == 4) BH_LAUNCH(conv_ragged4_kernel<4>, blocks, kBlock, 0, st, a, parts);
    else if (lanes == 8) BH_LAUNCH(conv_ragged4_kernel<8>, blocks, kBlock, 0, st, a, parts);
    else if (lanes == 16) BH_LAUNCH(conv_ragged4_kernel<16>, blocks, kBlock, 0, st, a, parts);
    else if (lanes == 32) BH_LAUNCH(conv_ragged4_kernel<32>, blocks, kBlock, 0, st, a, parts);
    else BH_LAUNCH(conv_ragged4_kernel<64>, blocks, kBlock, 0, st, a, parts);
    return ok();
  }
  const int parts = static_cast<int>((p.ch + kBlock - 1) / kBlock);
  BH_LAUNCH(conv_ragged_kernel, static_cast<unsigned>(p.n_tok * parts), kBlock, 0, st, a, parts);
  if (p.l2_dim != 0) {
    const size_t items = p.n_tok * a.groups;
    BH_LAUNCH(conv_ragged_l2_kernel, static_cast<unsigned>((items + 3) / 4), kBlock, 0, st, a);
  }
  if (p.k > 1)
    BH_LAUNCH(conv_ragged_state_kernel, static_cast<unsigned>(p.n_req * parts), kBlock, 0, st, a,
              parts);
  return ok();
}
