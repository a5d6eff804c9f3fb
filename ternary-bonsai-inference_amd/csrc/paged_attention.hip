// Attention of many requests' new queries over a paged KV cache.
//
// Any head size and layout (attn_paged_any_kernel): one block per (token,
// head), its four waves each over every fourth position with a running
// maximum and sum; a position that the query does not see is never read.
#include <hip/hip_runtime.h>

#include <string>

#include "../../include/bonsai_hip_serve.h"
#include "common.hpp"
#include "paged.hpp"

namespace bh {
namespace {

constexpr int kAnyMaxHd = 512;

struct PagedArgs {
  const float *q;
  float *out;
  const void *kc, *vc;
  const int32_t *q_start, *kv_len, *table;
  int32_t *bad_page;
  size_t page_stride, pos_stride, head_stride;
  int n_tok, n_req, n_head, n_kv, group, hd, width, n_pages, max_len;
  float scale;
  FastDiv page;
};

__device__ __forceinline__ float cache_at(const float *p) { return *p; }
__device__ __forceinline__ float cache_at(const _Float16 *p) { return static_cast<float>(*p); }

// Clipped tokens and length of request r.
__device__ __forceinline__ void request(const PagedArgs &a, int r, int *q0, int *n, int *len) {
  const int s = min(max(a.q_start[r], 0), a.n_tok), e = min(max(a.q_start[r + 1], 0), a.n_tok);
  *q0 = s;
  *n = max(e - s, 0);
  *len = min(max(a.kv_len[r], 0), a.max_len);
}

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

// Checks the arguments and fills `a`.
int prepare(const bh_attention_paged_args &p, PagedArgs *a) {
  const bh_paged_cache &c = p.cache;
  if (int e = check_paged_cache(c, "attention_paged")) return e;
  if (p.n_head == 0 || p.n_head % c.n_kv != 0)
    return fail(BH_ERR_SHAPE, "attention_paged: n_head " + std::to_string(p.n_head) +
                                  " is not a multiple of n_kv " + std::to_string(c.n_kv));
  if (c.hd > kAnyMaxHd)
    return fail(BH_ERR_SHAPE, "attention_paged: hd " + std::to_string(c.hd) + " above " +
                                  std::to_string(kAnyMaxHd));
  size_t n;
  if (p.n_head > 65535 || p.n_tok > 0x7fffffffu || p.n_req > 0x7ffffffeu ||
      !mul_size(p.n_tok, p.n_head * c.hd, sizeof(float), &n) || n > SIZE_MAX / 2)
    return fail(BH_ERR_SHAPE, "attention_paged: size overflow");
  if (p.table_width == 0 || !mul_size(p.table_width, c.page_size, &n) || n > 0x7fffffffu)
    return fail(BH_ERR_SHAPE, "attention_paged: table_width * page_size must be 1 .. 2^31 - 1");
  if (p.n_tok != 0 && p.n_req != 0) {
    if (!p.q || !p.out || !p.q_start || !p.kv_len || !p.block_table)
      return fail(BH_ERR_ARG, "attention_paged: null pointer");
    if (p.q == p.out) return fail(BH_ERR_ARG, "attention_paged: out must not be q");
  }
  a->q = p.q, a->out = p.out, a->kc = c.k, a->vc = c.v;
  a->q_start = p.q_start, a->kv_len = p.kv_len, a->table = p.block_table;
  a->bad_page = p.bad_page;
  a->page_stride = c.page_stride, a->pos_stride = c.pos_stride, a->head_stride = c.head_stride;
  a->n_tok = static_cast<int>(p.n_tok), a->n_req = static_cast<int>(p.n_req);
  a->n_head = static_cast<int>(p.n_head), a->n_kv = static_cast<int>(c.n_kv);
  a->group = a->n_head / a->n_kv, a->hd = static_cast<int>(c.hd);
  a->width = static_cast<int>(p.table_width), a->n_pages = static_cast<int>(c.n_pages);
  a->max_len = static_cast<int>(p.table_width * c.page_size);
  a->scale = 1.0f / sqrtf(static_cast<float>(c.hd));
  a->page = FastDiv(static_cast<uint32_t>(c.page_size));
  return BH_OK;
}

}  // namespace
}  // namespace bh

using namespace bh;

extern "C" size_t bh_attention_paged_workspace(const bh_attention_paged_args *args) {
  return 0;
}

extern "C" int bh_attention_paged(const bh_attention_paged_args *args, bh_stream stream) {
  if (!args) return fail(BH_ERR_ARG, "attention_paged: null args");
  PagedArgs a{};
  if (int e = prepare(*args, &a)) return e;
  if (a.n_tok == 0 || a.n_req == 0) return ok();
  const dim3 grid(static_cast<unsigned>(a.n_tok), static_cast<unsigned>(a.n_head));
  if (args->cache.kv_dtype == BH_KV_F16)
    BH_LAUNCH(attn_paged_any_kernel<_Float16>, grid, 256, 0, as_stream(stream), a);
  else
    BH_LAUNCH(attn_paged_any_kernel<float>, grid, 256, 0, as_stream(stream), a);
  return ok();
}
