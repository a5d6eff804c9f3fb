// Attention of many requests' new queries over a paged KV cache.
//
// One pass over K and V with a running maximum and sum of the softmax.  The rows of
// a kv head, (token, head of its group) pairs, go through the matrix cores 16 at
// a time; the work of a call, whatever its requests' lengths, is cut into equal
// runs of positions, one a worker, and what was cut is joined by a second launch
// (inside the first it would take counters that are zero at its start, and
// fences across the L2s of eight dies).  Three forms:
//   attn_paged_kernel       few rows a request: the waves of a block split the
//                           positions; bound by reading the cache
//   attn_paged_wide_kernel  many rows over f16: the waves share K and V in LDS;
//                           bound by LDS reads and instruction issue
//   attn_paged_any_kernel   any head size and layout, one block per (token, head),
//                           its waves each over every fourth position
// A position that a query does not see has no effect on it, whatever it holds.
//
// Measured (24 / 4 heads of 256, us of the call, both launches): one token at 100 /
// 5000 / 32768 f16 positions 12 / 15.9 / 30.6 (the last 4.4 TB/s), 64 requests at
// 16384 715 (6.0 TB/s), 64 at 8192 f32 689 (6.2 TB/s), 509 at 500 211 (4.9 TB/s), 1500
// at 100 175 (3.5 TB/s); a copy reaches 5.1 TB/s here.  Of one token's 12 us the wait
// for offsets, table, K and V one after the other is most; K, V, q and the next table
// entry are asked for together.  The generic form, as it is: one token at 5000 1.9-3.0
// ms, 64 at 4096 1.9-3.9 ms (hd 80 to 256), 512 tokens at 4096 6.9-11.5 ms.  Error
// against 64-bit arithmetic 2e-7 to 4e-7.
#include <hip/hip_runtime.h>

#include <string>

#include "../../include/bonsai_hip_serve.h"
#include "common.hpp"
#include "paged.hpp"
#include "paged_attention.hpp"

namespace bh {
namespace {

template <class T>
__global__ __launch_bounds__(256) void attn_paged_any_kernel(PagedArgs a) {
  __shared__ int owner;
  __shared__ float lm[4], ll[4];
  __shared__ float acc_s[4][kAnyMaxHd];
  const int t = blockIdx.x, h = blockIdx.y;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (threadIdx.x == 0) owner = a.n_req;
  __syncthreads();
  for (int r = threadIdx.x; r < a.n_req; r += 256) {
    int q0, n, len;
    request(a, r, &q0, &n, &len);
    if (t >= q0 && t < q0 + n) atomicMin(&owner, r);
  }
  __syncthreads();
  const int r = owner;
  if (r == a.n_req) return;
  int q0, n, len;
  request(a, r, &q0, &n, &len);
  const int seen = len - n + (t - q0) + 1;  // positions 0 .. seen - 1; none if <= 0
  const int32_t *table = a.table + static_cast<size_t>(r) * a.width;
  const size_t head = (h / a.group) * a.head_stride;
  const size_t row = (static_cast<size_t>(t) * a.n_head + h) * a.hd;

  constexpr int kPer = kAnyMaxHd / 64;
  float q[kPer], acc[kPer];
  for (int i = 0; i < kPer; ++i) {
    const int d = lane + 64 * i;
    q[i] = d < a.hd ? a.q[row + d] : 0.0f;
    acc[i] = 0.0f;
  }
  float m = -INFINITY, l = 0.0f;
  bool any = false;  // a visible position of a page of the pool
  for (int p = wave; p < seen; p += 4) {
    const int b = a.page.div(p);
    const int at_page = table[b];
    if (at_page < 0 || at_page >= a.n_pages) {
      if (a.bad_page && lane == 0) *a.bad_page = at_page;
      continue;
    }
    any = true;
    const size_t at = at_page * a.page_stride +
                      static_cast<size_t>(p - b * a.page.d) * a.pos_stride + head;
    const T *k = static_cast<const T *>(a.kc) + at, *v = static_cast<const T *>(a.vc) + at;
    float s = 0.0f;
    for (int i = 0; i < kPer; ++i)
      if (lane + 64 * i < a.hd) s = __builtin_fmaf(q[i], cache_at(k + lane + 64 * i), s);
    s = lane_group_sum<64>(s) * a.scale;
    const float top = s > m ? s : m;
    // before the first score above -inf nothing is scaled
    const float keep = top == -INFINITY ? 1.0f : expf(m - top);
    const float e = s == -INFINITY && top == -INFINITY ? 0.0f : expf(s - top);
    l = l * keep + e;
    for (int i = 0; i < kPer; ++i) {
      acc[i] *= keep;
      if (lane + 64 * i < a.hd)
        acc[i] = __builtin_fmaf(e, cache_at(v + lane + 64 * i), acc[i]);
    }
    m = top;
  }
  if (lane == 0) lm[wave] = any ? m : -INFINITY, ll[wave] = l;
  for (int i = 0; i < kPer; ++i) acc_s[wave][lane + 64 * i] = acc[i];
  const bool some = __syncthreads_or(any);
  float top = lm[0];
  for (int w = 1; w < 4; ++w) top = lm[w] > top ? lm[w] : top;
  float sum = 0.0f, keep[4];
  for (int w = 0; w < 4; ++w) {
    keep[w] = top == -INFINITY ? 1.0f : expf(lm[w] - top);
    sum += keep[w] * ll[w];
  }
  for (int d = threadIdx.x; d < a.hd; d += 256) {
    float o = 0.0f;
    for (int w = 0; w < 4; ++w) o += keep[w] * acc_s[w][d];
    a.out[row + d] = some ? o / sum : 0.0f;
  }
}

}  // namespace
}  // namespace bh

using namespace bh;

extern "C" size_t bh_attention_paged_workspace(const bh_attention_paged_args *args) {
  PagedArgs a{};
  if (!args || prepare(*args, &a, "attention_paged") != BH_OK || !on_matrix_cores(*args)) return 0;
  if (a.n_tok == 0 || a.n_req == 0) return 0;
  Form f[2];
  size_t need = 0;
  for (int i = 0, n = forms_of(*args, f); i < n; ++i) need += workspace_of<false>(a, f[i]);
  return need;
}

extern "C" int bh_attention_paged(const bh_attention_paged_args *args, bh_stream stream) {
  if (!args) return fail(BH_ERR_ARG, "attention_paged: null args");
  const bh_attention_paged_args &p = *args;
  PagedArgs a{};
  if (int e = prepare(p, &a, "attention_paged")) return e;
  if (a.n_tok == 0 || a.n_req == 0) return ok();
  const bool f16 = p.cache.kv_dtype == BH_KV_F16;
  hipStream_t st = as_stream(stream);
  if (on_matrix_cores(p)) {
    Form f[2];
    const int n = forms_of(p, f);
    size_t need = 0, tiles = 0;
    for (int i = 0; i < n; ++i) {
      need += workspace_of<false>(a, f[i]);
      tiles += most_tiles<false>(a, f[i]);
    }
    if (tiles > kMostBlocks)  // (the join has more than a block a tile only of few)
      return fail(BH_ERR_SHAPE, "attention_paged: more row tiles than a launch has blocks");
    char *ws = static_cast<char *>(p.workspace);
    if (ws) {
      if (!aligned16(ws) || p.workspace_bytes < need)
        return fail(BH_ERR_SHAPE, "attention_paged: workspace of " +
                                      std::to_string(p.workspace_bytes) + " bytes, " +
                                      std::to_string(need) + " needed on a 16-byte boundary");
    } else {
      ws = static_cast<char *>(device_scratch(need, kScratchPaged, st));
      if (!ws) return BH_ERR_HIP;
    }
    Join join[2] = {};
    for (int i = 0; i < n; ++i) {
      if (int e = launch_form<false>(a, f16, f[i], ws, st, &join[i])) return e;
      ws += workspace_of<false>(a, f[i]);
    }
    if (int e = launch_join(a, join[0], join[1], st)) return e;
    return ok();
  }
  const dim3 grid(static_cast<unsigned>(a.n_tok), static_cast<unsigned>(a.n_head));
  if (f16)
    BH_LAUNCH(attn_paged_any_kernel<_Float16>, grid, 256, 0, st, a);
  else
    BH_LAUNCH(attn_paged_any_kernel<float>, grid, 256, 0, st, a);
  return ok();
}
