// The gated delta rule of many requests at once, each with its state in a slot.
//
// Per request, v-head h (q/k head h % h_k) and state row j, with m = M[j]:
//   m *= e^gate;  delta = (v[j] - m.k) beta;  m += k delta;  attn[j] = m.q / sqrt(s).
// A row only ever meets its own delta and the head's q and k, so rows are
// independent; with d_k = m.k and d_q = m.q of the row before the token
//   delta = (v - e^gate d_k) beta,  m' = e^gate m + delta k,
//   m'.q = e^gate d_q + delta (k.q),
// so that both dots come from the old row at once.  Decoding reads and writes the
// states, 2 x 4 h_v s^2 bytes a request, and is bound by that.
#include <hip/hip_runtime.h>

#include <string>

#include "../../include/bonsai_hip_batch.h"
#include "common.hpp"
#include "ragged.hpp"

namespace bh {
namespace {

constexpr int kBlock = 256;
constexpr int kAnyMaxS = 1024;

struct GdnArgs {
  const float *q, *k, *v, *gate, *beta;
  float *state, *attn;
  size_t q_stride, k_stride, v_stride;
  int h_k, h_v, s;
  float scale;
  Ragged rag;
};

// Rows of S floats in registers, S / 8 lanes a row and RPG rows a lane, for as many
// tokens as the request has; the next token's inputs load under the present one.
template <int S, int RPG>
__global__ __launch_bounds__(kBlock) void gdn_ragged_step_kernel(GdnArgs a) {
  constexpr int L = S / 8, kRows = kBlock / L * RPG, kTiles = S / kRows;
  static_assert(S % kRows == 0, "a block's rows are of one head");
  const int per = a.h_v * kTiles;
  const int r = blockIdx.x / per, rest = blockIdx.x - r * per;
  const int h = rest / kTiles, kh = h % a.h_k;
  const int sub = threadIdx.x % L, j = (rest - h * kTiles) * kRows + threadIdx.x / L * RPG;
  int t0, n, from, to;
  a.rag.tokens(r, &t0, &n);
  if (n == 0) return;
  a.rag.slots(r, &from, &to);
  const size_t row = (static_cast<size_t>(h) * S + j) * S + 4 * sub;
  f32x4 m[RPG][2];
  if (from >= 0) {
    const float *p = a.state + from * a.rag.slot_stride + row;
#pragma unroll
    for (int i = 0; i < RPG; ++i) {
      m[i][0] = *reinterpret_cast<const f32x4 *>(p + i * S);
      m[i][1] = *reinterpret_cast<const f32x4 *>(p + i * S + S / 2);
    }
  } else {
#pragma unroll
    for (int i = 0; i < RPG; ++i) m[i][0] = m[i][1] = f32x4{0, 0, 0, 0};
  }
  f32x4 k[2], q[2];
  float v[RPG], g, b;
  const auto load = [&](int t) {
    const float *kp = a.k + t * a.k_stride + kh * S + 4 * sub;
    const float *qp = a.q + t * a.q_stride + kh * S + 4 * sub;
    k[0] = *reinterpret_cast<const f32x4 *>(kp);
    k[1] = *reinterpret_cast<const f32x4 *>(kp + S / 2);
    q[0] = *reinterpret_cast<const f32x4 *>(qp);
    q[1] = *reinterpret_cast<const f32x4 *>(qp + S / 2);
#pragma unroll
    for (int i = 0; i < RPG; ++i) v[i] = a.v[t * a.v_stride + h * S + j + i];
    g = a.gate[static_cast<size_t>(t) * a.h_v + h];
    b = a.beta[static_cast<size_t>(t) * a.h_v + h];
  };
  const auto dot = [](f32x4 x, f32x4 y, f32x4 z, f32x4 w) {
    const float lo = fmaf(x.w, y.w, fmaf(x.z, y.z, fmaf(x.y, y.y, x.x * y.x)));
    const float hi = fmaf(z.w, w.w, fmaf(z.z, w.z, fmaf(z.y, w.y, z.x * w.x)));
    return lo + hi;
  };
  load(t0);
  for (int t = 0; t < n; ++t) {
    const f32x4 k0 = k[0], k1 = k[1], q0 = q[0], q1 = q[1];
    float vt[RPG];
#pragma unroll
    for (int i = 0; i < RPG; ++i) vt[i] = v[i];
    const float eg = expf(g), beta = b;
    if (t + 1 < n) load(t0 + t + 1);
    const float kq = lane_group_sum<L>(dot(k0, q0, k1, q1));
    float out[RPG];
#pragma unroll
    for (int i = 0; i < RPG; ++i) {
      const float dk = lane_group_sum<L>(dot(m[i][0], k0, m[i][1], k1));
      const float dq = lane_group_sum<L>(dot(m[i][0], q0, m[i][1], q1));
      const float delta = fmaf(-eg, dk, vt[i]) * beta;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        m[i][0][e] = fmaf(k0[e], delta, eg * m[i][0][e]);
        m[i][1][e] = fmaf(k1[e], delta, eg * m[i][1][e]);
      }
      out[i] = fmaf(eg, dq, delta * kq) * a.scale;
    }
    if (sub == 0) {
      float *o = a.attn + (static_cast<size_t>(t0 + t) * a.h_v + h) * S + j;
#pragma unroll
      for (int i = 0; i < RPG; ++i) o[i] = out[i];
    }
  }
  if (to >= 0) {
    float *p = a.state + to * a.rag.slot_stride + row;
#pragma unroll
    for (int i = 0; i < RPG; ++i) {
      *reinterpret_cast<f32x4 *>(p + i * S) = m[i][0];
      *reinterpret_cast<f32x4 *>(p + i * S + S / 2) = m[i][1];
    }
  }
}

// Any s up to kAnyMaxS and any alignment: a wave a row, 16 of its floats a lane.
__global__ __launch_bounds__(kBlock) void gdn_ragged_any_kernel(GdnArgs a) {
  constexpr int kPer = kAnyMaxS / 64;
  const int rows = a.h_v * a.s, blocks = (rows + 3) / 4;
  const int r = blockIdx.x / blocks, lane = threadIdx.x & 63;
  const int row = (blockIdx.x - r * blocks) * 4 + (threadIdx.x >> 6);
  int t0, n, from, to;
  a.rag.tokens(r, &t0, &n);
  if (n == 0 || row >= rows) return;
  a.rag.slots(r, &from, &to);
  const int h = row / a.s, j = row - h * a.s, kh = h % a.h_k, s = a.s;
  float m[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int d = lane + 64 * i;
    m[i] = 0.0f;
    if (from >= 0 && d < s)
      m[i] = a.state[from * a.rag.slot_stride + static_cast<size_t>(row) * s + d];
  }
  for (int t = t0; t < t0 + n; ++t) {
    const float *kp = a.k + t * a.k_stride + static_cast<size_t>(kh) * s;
    const float *qp = a.q + t * a.q_stride + static_cast<size_t>(kh) * s;
    const size_t at = static_cast<size_t>(t) * a.h_v + h;
    const float eg = expf(a.gate[at]);
    float k[kPer], q[kPer], dk = 0.0f, dq = 0.0f, kq = 0.0f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int d = lane + 64 * i;
      k[i] = d < s ? kp[d] : 0.0f;
      q[i] = d < s ? qp[d] : 0.0f;
      dk = fmaf(m[i], k[i], dk);
      dq = fmaf(m[i], q[i], dq);
      kq = fmaf(k[i], q[i], kq);
    }
    dk = lane_group_sum<64>(dk);
    dq = lane_group_sum<64>(dq);
    kq = lane_group_sum<64>(kq);
    const float delta =
        fmaf(-eg, dk, a.v[t * a.v_stride + static_cast<size_t>(h) * s + j]) * a.beta[at];
#pragma unroll
    for (int i = 0; i < kPer; ++i) m[i] = fmaf(k[i], delta, eg * m[i]);
    if (lane == 0) a.attn[at * s + j] = fmaf(eg, dq, delta * kq) * a.scale;
  }
  if (to < 0) return;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int d = lane + 64 * i;
    if (d < s) a.state[to * a.rag.slot_stride + static_cast<size_t>(row) * s + d] = m[i];
  }
}

// Blocks of a launch: a grid has fewer than 2^32 threads a dimension.
constexpr size_t kMostBlocks = 0xffffff;

int check(const bh_gdn_ragged_args &p) {
  if (p.h_k == 0 || p.h_v == 0 || p.s == 0)
    return fail(BH_ERR_SHAPE, "gdn_ragged: h_k, h_v and s must be above 0");
  if (p.s > static_cast<size_t>(kAnyMaxS))
    return fail(BH_ERR_SHAPE, "gdn_ragged: s " + std::to_string(p.s) + " above " +
                                  std::to_string(kAnyMaxS));
  if (p.h_k > 65535 || p.h_v > 65535)
    return fail(BH_ERR_SHAPE, "gdn_ragged: more than 65535 heads");
  const size_t qk = p.h_k * p.s, vs = p.h_v * p.s, st = vs * p.s;
  if (p.q_stride < qk || p.k_stride < qk || p.v_stride < vs || p.slot_stride < st)
    return fail(BH_ERR_SHAPE, "gdn_ragged: a stride is below the rows it steps over");
  size_t n;
  // a block holds 16 rows at least, or 4 in the form for any s
  if (p.n_tok > 0x7fff0000u || p.n_req > kMostBlocks ||
      !mul_size(p.n_req, (vs + 3) / 4, &n) || n > kMostBlocks ||
      !mul_size(p.n_tok, p.q_stride, sizeof(float), &n) ||
      !mul_size(p.n_tok, p.k_stride, sizeof(float), &n) ||
      !mul_size(p.n_tok, p.v_stride, sizeof(float), &n) || p.n_slots > 0x7fffffffu ||
      !mul_size(p.n_slots, p.slot_stride, sizeof(float), &n))
    return fail(BH_ERR_SHAPE, "gdn_ragged: size overflow");
  if (p.n_req != 0 && p.n_tok != 0) {
    if (!p.q || !p.k || !p.v || !p.gate || !p.beta || !p.attn || !p.q_start || !p.src_slot ||
        !p.dst_slot || (p.n_slots != 0 && !p.state))
      return fail(BH_ERR_ARG, "gdn_ragged: null pointer");
  }
  return BH_OK;
}

}  // namespace
}  // namespace bh

using namespace bh;

extern "C" size_t bh_gdn_ragged_workspace(const bh_gdn_ragged_args *args) {
  if (!args || check(*args) != BH_OK) return 0;
  return 0;
}

extern "C" int bh_gdn_ragged(const bh_gdn_ragged_args *args, bh_stream stream) {
  if (!args) return fail(BH_ERR_ARG, "gdn_ragged: null args");
  const bh_gdn_ragged_args &p = *args;
  if (int e = check(p)) return e;
  if (p.n_req == 0 || p.n_tok == 0) return ok();
  GdnArgs a{};
  a.q = p.q, a.k = p.k, a.v = p.v, a.gate = p.gate, a.beta = p.beta;
  a.state = p.state, a.attn = p.attn;
  a.q_stride = p.q_stride, a.k_stride = p.k_stride, a.v_stride = p.v_stride;
  a.h_k = static_cast<int>(p.h_k), a.h_v = static_cast<int>(p.h_v), a.s = static_cast<int>(p.s);
  a.scale = 1.0f / sqrtf(static_cast<float>(p.s));
  a.rag = Ragged{p.q_start, p.src_slot, p.dst_slot, p.bad_slot, static_cast<int>(p.n_tok),
                 static_cast<int>(p.n_req), static_cast<int>(p.n_slots), p.slot_stride};
  hipStream_t st = as_stream(stream);
  const bool whole = (p.q_stride | p.k_stride | p.slot_stride) % 4 == 0 && aligned16(p.q) &&
                     aligned16(p.k) && aligned16(p.state);
  const auto blocks = [&](size_t rows) { return static_cast<unsigned>(p.n_req * p.h_v * p.s / rows); };
  if (whole && p.s == 128) {
    if (blocks(64) >= 2 * device_cu_count())
      BH_LAUNCH((gdn_ragged_step_kernel<128, 4>), blocks(64), kBlock, 0, st, a);
    else
      BH_LAUNCH((gdn_ragged_step_kernel<128, 1>), blocks(16), kBlock, 0, st, a);
  } else if (whole && p.s == 64) {
    if (blocks(64) >= 2 * device_cu_count())
      BH_LAUNCH((gdn_ragged_step_kernel<64, 2>), blocks(64), kBlock, 0, st, a);
    else
      BH_LAUNCH((gdn_ragged_step_kernel<64, 1>), blocks(32), kBlock, 0, st, a);
  } else {
    BH_LAUNCH(gdn_ragged_any_kernel,
              static_cast<unsigned>(p.n_req * ((p.h_v * p.s + 3) / 4)), kBlock, 0, st, a);
  }
  return ok();
}
