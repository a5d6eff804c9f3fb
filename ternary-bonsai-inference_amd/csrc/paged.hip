// The bookkeeping of a step over a paged KV cache, and the append.
//
// bh_paged_plan: the requests' lengths become pages (popped from or pushed on a
// stack of free ones), the ragged offsets of the step's tokens, and each
// token's slot and position.  All of it follows from three running totals over
// the requests (new pages, new tokens, released pages):
//
//   request i is refused when its running total of new pages passes what the
//   stack holds or that of its new tokens passes n_tok; as both totals grow, a
//   request that is admitted and takes pages has no refused one before it, so
//   its pages begin at the plain running total and only the tokens need a
//   second one, over the admitted requests.
//
// One workgroup does it: every step needs the totals of all requests, and the
// data is a few hundred KB at most.  It is bound by the chain of dependent
// steps (load, scan, scan, pages, tokens), not by bytes.
#include <hip/hip_runtime.h>

#include <string>

#include "../../include/bonsai_hip_serve.h"
#include "common.hpp"
#include "paged.hpp"

namespace bh {
namespace {

constexpr int kPlanThreads = 1024;
constexpr int kPlanPer = BH_PAGED_MAX_REQ / kPlanThreads;  // requests of a thread

struct PlanArgs {
  const int32_t *cached, *n_new, *n_free;
  int32_t *table, *free_pages, *kv_len, *q_start, *slots, *pos, *n_free_out, *n_refused;
  int n_req, n_tok, width, n_pages;
  FastDiv page;
};

// Exclusive running total over the block in thread order; *total gets the sum.
__device__ __forceinline__ int64_t block_scan(int64_t v, int64_t *lds, int64_t *total) {
  int64_t run = v;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int d = 1; d < 64; d <<= 1) {
    const int64_t o = __shfl_up(run, d);
    if (lane >= d) run += o;
  }
  __syncthreads();
  if (lane == 63) lds[wave] = run;
  __syncthreads();
  int64_t before = 0, all = 0;
  for (int w = 0; w < kPlanThreads / 64; ++w) {
    if (w < wave) before += lds[w];
    all += lds[w];
  }
  *total = all;
  return before + run - v;
}

// The request r with start[r] <= x < start[r + 1], for 0 <= x < start[n].
__device__ __forceinline__ int find(const int *start, int n, int x) {
  int lo = 0, hi = n;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (start[mid] <= x) lo = mid;
    else hi = mid;
  }
  return lo;
}

__global__ __launch_bounds__(kPlanThreads) void paged_plan_kernel(PlanArgs a) {
  __shared__ int64_t part[kPlanThreads / 64];
  __shared__ int start[BH_PAGED_MAX_REQ + 1];
  __shared__ int lens[BH_PAGED_MAX_REQ];
  const int tid = threadIdx.x;
  const int64_t page = a.page.d;

  int cached[kPlanPer], grow[kPlanPer], have[kPlanPer], need[kPlanPer];
  bool gone[kPlanPer], refused[kPlanPer];
  int64_t sn = 0, sg = 0, sb = 0;
  for (int k = 0; k < kPlanPer; ++k) {
    const int i = tid * kPlanPer + k;
    cached[k] = grow[k] = have[k] = need[k] = 0;
    gone[k] = refused[k] = false;
    if (i >= a.n_req) continue;
    const int c = max(a.cached[i], 0), n = a.n_new[i];
    gone[k] = n < 0;
    cached[k] = c;
    have[k] = a.page.div(c) + (a.page.mod(c) != 0);
    if (!gone[k]) {
      const int64_t len = static_cast<int64_t>(c) + n;
      if (len > a.width * page) {
        refused[k] = true;
      } else {
        const int l = static_cast<int>(len);
        grow[k] = n;
        need[k] = a.page.div(l) + (a.page.mod(l) != 0) - have[k];
      }
    }
    have[k] = min(have[k], a.width);
    sn += need[k];
    sg += grow[k];
    sb += gone[k] ? have[k] : 0;
  }
  const int n_free = min(max(*a.n_free, 0), a.n_pages);
  int64_t tn, tg, tb;
  int64_t on = block_scan(sn, part, &tn), og = block_scan(sg, part, &tg);
  int64_t ob = block_scan(sb, part, &tb);

  // the released pages go on the stack
  for (int k = 0; k < kPlanPer; ++k) {
    const int i = tid * kPlanPer + k;
    if (i <= a.n_req) start[i] = static_cast<int>(min<int64_t>(ob, a.n_pages));
    if (i < a.n_req && gone[k]) ob += have[k];
  }
  if (tid == 0 && a.n_req == BH_PAGED_MAX_REQ)
    start[a.n_req] = static_cast<int>(min<int64_t>(tb, a.n_pages));
  __syncthreads();
  const int n_back = static_cast<int>(min<int64_t>(tb, a.n_pages - n_free));
  for (int p = tid; p < n_back; p += kPlanThreads) {
    const int r = find(start, a.n_req, p);
    a.free_pages[n_free + p] = a.table[static_cast<size_t>(r) * a.width + (p - start[r])];
  }
  const int avail = n_free + n_back;

  // who fits
  int64_t taken = 0, admitted = 0, out = 0;
  const int64_t first = on;
  for (int k = 0; k < kPlanPer; ++k) {
    on += need[k];
    og += grow[k];
    if ((need[k] > 0 && on > avail) || (grow[k] > 0 && og > a.n_tok)) refused[k] = true;
    if (refused[k]) {
      need[k] = grow[k] = 0;
      ++out;
    }
    taken += need[k];
    admitted += grow[k];
  }
  int64_t all_taken, n_out, n_admitted;
  block_scan(taken, part, &all_taken);
  block_scan(out, part, &n_out);
  int64_t at = block_scan(admitted, part, &n_admitted);

  // the pages taken, from the top of the stack; start: where a request's begin
  int64_t base = first;
  for (int k = 0; k < kPlanPer; ++k) {
    const int i = tid * kPlanPer + k;
    // a refused request's range is empty: it begins where the taken ones end
    if (i <= a.n_req) start[i] = static_cast<int>(min(base, all_taken));
    if (i < a.n_req) lens[i] = have[k];
    base += need[k];
  }
  if (tid == 0 && a.n_req == BH_PAGED_MAX_REQ) start[a.n_req] = static_cast<int>(all_taken);
  __syncthreads();
  for (int p = tid; p < static_cast<int>(all_taken); p += kPlanThreads) {
    const int r = find(start, a.n_req, p);
    a.table[static_cast<size_t>(r) * a.width + lens[r] + (p - start[r])] =
        a.free_pages[avail - 1 - p];
  }
  __syncthreads();

  // offsets, lengths, tokens
  for (int k = 0; k < kPlanPer; ++k) {
    const int i = tid * kPlanPer + k;
    if (i <= a.n_req) a.q_start[i] = start[i] = static_cast<int>(at);
    if (i < a.n_req) a.kv_len[i] = lens[i] = gone[k] || refused[k] ? 0 : cached[k] + grow[k];
    at += grow[k];
  }
  if (tid == 0) {
    *a.n_free_out = avail - static_cast<int>(all_taken);
    if (a.n_refused) *a.n_refused = static_cast<int>(n_out);
    if (a.n_req == BH_PAGED_MAX_REQ)
      a.q_start[a.n_req] = start[a.n_req] = static_cast<int>(n_admitted);
  }
  __syncthreads();
  const int live = static_cast<int>(n_admitted);
  for (int t = tid; t < a.n_tok; t += kPlanThreads) {
    int p = 0, slot = -1;
    if (t < live) {
      const int r = find(start, a.n_req, t);
      p = lens[r] - start[r + 1] + t;
      const int b = a.page.div(p);
      const int at_page = a.table[static_cast<size_t>(r) * a.width + b];
      if (at_page >= 0 && at_page < a.n_pages) slot = at_page * a.page.d + (p - b * a.page.d);
    }
    a.slots[t] = slot;
    if (a.pos) *reinterpret_cast<int4 *>(a.pos + static_cast<size_t>(t) * 4) = make_int4(p, p, p, p);
  }
}

// ---- append ------------------------------------------------------------------

// The f16 bits of bh_kv_store: round to nearest even by the hardware, a NaN as
// its sign and a quiet bit.
__device__ __forceinline__ uint16_t store_half(float v) {
  const _Float16 h = static_cast<_Float16>(v);
  if (v != v) return static_cast<uint16_t>((__float_as_uint(v) >> 16 & 0x8000u) | 0x7e00u);
  return __builtin_bit_cast(uint16_t, h);
}

struct StoreArgs {
  const float *k, *v;
  const int32_t *slots;
  void *kc, *vc;
  size_t page_stride, pos_stride, head_stride;
  int n_tok, n_slots, elems, hd;
  FastDiv page;
};

template <class T>
__global__ __launch_bounds__(256) void kv_store_paged_kernel(StoreArgs a) {
  const int t = blockIdx.x;
  const int slot = a.slots[t];
  if (slot < 0 || slot >= a.n_slots) return;
  const int b = a.page.div(slot);
  const size_t at = b * a.page_stride + static_cast<size_t>(slot - b * a.page.d) * a.pos_stride;
  T *kc = static_cast<T *>(a.kc) + at, *vc = static_cast<T *>(a.vc) + at;
  for (int e = threadIdx.x; e < a.elems; e += 256) {
    const int h = e / a.hd;
    const size_t o = h * a.head_stride + (e - h * a.hd);
    const size_t i = static_cast<size_t>(t) * a.elems + e;
    if constexpr (sizeof(T) == 2) {
      kc[o] = store_half(a.k[i]);
      vc[o] = store_half(a.v[i]);
    } else {
      kc[o] = a.k[i];
      vc[o] = a.v[i];
    }
  }
}

}  // namespace

int check_paged_cache(const bh_paged_cache &c, const char *who) {
  const std::string w = std::string(who) + ": ";
  if (c.kv_dtype != BH_KV_F32 && c.kv_dtype != BH_KV_F16)
    return fail(BH_ERR_ARG, w + "kv_dtype must be BH_KV_F32 or BH_KV_F16");
  if (c.n_pages == 0 || c.page_size == 0 || c.n_kv == 0 || c.hd == 0)
    return fail(BH_ERR_SHAPE, w + "n_pages, page_size, n_kv and hd must be above 0");
  size_t n, row, s0, s1, s2;
  if (!mul_size(c.n_pages, c.page_size, &n) || n > 0x7fffffffu)
    return fail(BH_ERR_SHAPE, w + "n_pages " + std::to_string(c.n_pages) + " of " +
                                  std::to_string(c.page_size) + " positions pass 2^31");
  if (!mul_size(c.n_kv, c.hd, &row) || row > 0x7fffffffu)
    return fail(BH_ERR_SHAPE, w + "n_kv * hd passes 2^31");
  const size_t esz = c.kv_dtype == BH_KV_F16 ? 2 : 4;
  if (!mul_size(c.n_pages - 1, c.page_stride, esz, &s0) ||
      !mul_size(c.page_size - 1, c.pos_stride, esz, &s1) ||
      !mul_size(c.n_kv - 1, c.head_stride, esz, &s2) || s0 > SIZE_MAX / 8 || s1 > SIZE_MAX / 8 ||
      s2 > SIZE_MAX / 8)
    return fail(BH_ERR_SHAPE, w + "the cache's strides overflow");
  if ((c.n_pages > 1 && c.page_stride == 0) || (c.page_size > 1 && c.pos_stride < c.hd) ||
      (c.n_kv > 1 && c.head_stride < c.hd))
    return fail(BH_ERR_SHAPE, w + "the cache's strides let rows overlap");
  if (!c.k || !c.v) return fail(BH_ERR_ARG, w + "null cache");
  if ((reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v)) & (esz - 1))
    return fail(BH_ERR_ARG, w + "misaligned cache");
  return BH_OK;
}

}  // namespace bh

using namespace bh;

extern "C" int bh_paged_plan(const bh_paged_plan_args *args, bh_stream stream) {
  if (!args) return fail(BH_ERR_ARG, "paged_plan: null args");
  const bh_paged_plan_args &p = *args;
  if (p.n_req > BH_PAGED_MAX_REQ)
    return fail(BH_ERR_SHAPE, "paged_plan: n_req " + std::to_string(p.n_req) + " above " +
                                  std::to_string(BH_PAGED_MAX_REQ));
  if (p.page_size == 0 || p.n_pages == 0 || p.table_width == 0)
    return fail(BH_ERR_SHAPE, "paged_plan: page_size, n_pages and table_width must be above 0");
  size_t n;
  if (!mul_size(p.n_pages, p.page_size, &n) || n > 0x7fffffffu)
    return fail(BH_ERR_SHAPE, "paged_plan: n_pages * page_size passes 2^31");
  if (!mul_size(p.table_width, p.page_size, &n) || n > 0x7fffffffu)
    return fail(BH_ERR_SHAPE, "paged_plan: table_width * page_size passes 2^31");
  if (p.n_tok > 0x7fffffffu - kPlanThreads)
    return fail(BH_ERR_SHAPE, "paged_plan: n_tok passes 2^31");
  if (!p.q_start || !p.n_free || !p.n_free_out || !p.free_pages || (p.n_tok != 0 && !p.slots) ||
      (p.n_req != 0 && (!p.cached || !p.n_new || !p.block_table || !p.kv_len)))
    return fail(BH_ERR_ARG, "paged_plan: null pointer");
  if (p.kv_len == p.cached && p.n_req != 0)
    return fail(BH_ERR_ARG, "paged_plan: kv_len must not be cached (a refused request keeps that)");
  if (p.pos && !aligned16(p.pos)) return fail(BH_ERR_ARG, "paged_plan: pos must be 16-byte aligned");
  PlanArgs a{};
  a.cached = p.cached, a.n_new = p.n_new, a.n_free = p.n_free;
  a.table = p.block_table, a.free_pages = p.free_pages;
  a.kv_len = p.kv_len, a.q_start = p.q_start, a.slots = p.slots, a.pos = p.pos;
  a.n_free_out = p.n_free_out, a.n_refused = p.n_refused;
  a.n_req = static_cast<int>(p.n_req), a.n_tok = static_cast<int>(p.n_tok);
  a.width = static_cast<int>(p.table_width), a.n_pages = static_cast<int>(p.n_pages);
  a.page = FastDiv(static_cast<uint32_t>(p.page_size));
  BH_LAUNCH(paged_plan_kernel, 1, kPlanThreads, 0, as_stream(stream), a);
  return ok();
}

extern "C" int bh_kv_store_paged(const bh_paged_cache *cache, const float *k, const float *v,
                                 const int32_t *slots, size_t n_tok, bh_stream stream) {
  if (!cache) return fail(BH_ERR_ARG, "kv_store_paged: null cache");
  if (int e = check_paged_cache(*cache, "kv_store_paged")) return e;
  if (n_tok == 0) return ok();
  size_t n;
  if (n_tok > 0x7fffffffu || !mul_size(n_tok, cache->n_kv * cache->hd, sizeof(float), &n))
    return fail(BH_ERR_SHAPE, "kv_store_paged: size overflow");
  if (!k || !v || !slots) return fail(BH_ERR_ARG, "kv_store_paged: null pointer");
  StoreArgs a{};
  a.k = k, a.v = v, a.slots = slots, a.kc = cache->k, a.vc = cache->v;
  a.page_stride = cache->page_stride, a.pos_stride = cache->pos_stride;
  a.head_stride = cache->head_stride;
  a.n_tok = static_cast<int>(n_tok);
  a.n_slots = static_cast<int>(cache->n_pages * cache->page_size);
  a.elems = static_cast<int>(cache->n_kv * cache->hd), a.hd = static_cast<int>(cache->hd);
  a.page = FastDiv(static_cast<uint32_t>(cache->page_size));
  if (cache->kv_dtype == BH_KV_F16)
    BH_LAUNCH(kv_store_paged_kernel<uint16_t>, static_cast<unsigned>(n_tok), 256, 0,
              as_stream(stream), a);
  else
    BH_LAUNCH(kv_store_paged_kernel<float>, static_cast<unsigned>(n_tok), 256, 0,
              as_stream(stream), a);
  return ok();
}
