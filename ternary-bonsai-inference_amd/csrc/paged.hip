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
// data is a few hundred KB at most.  It is bound by the chain of dependent steps
// (load, scan, scan, pages, tokens), not by bytes; so few requests take one wave,
// whose barriers cost nothing (16 requests: 3.6 us, with 16 waves 4.6 us), as long as
// their tokens are few too (64 requests, 129 token slots: 0.6 us more than 128).  509
// requests of 8192 tokens: 14.4 us.  Two or four pages and tokens of a thread side
// by side were slower (4.3, 6.0 and 15.9, 16.6 us): the searches are LDS reads.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>

#include "../../include/bonsai_hip_serve.h"
#include "common.hpp"
#include "paged.hpp"

namespace bh {
namespace {

constexpr int kMost = 0x7fffffff;  // where running totals stop: past every limit

struct PlanArgs {
  const int32_t *cached, *n_new, *n_free;
  int32_t *table, *free_pages, *kv_len, *q_start, *slots, *pos, *n_free_out, *n_refused;
  int n_req, n_tok, width, n_pages;
  FastDiv page;
};

__device__ __forceinline__ int add_most(int a, int b) {
  const uint32_t s = static_cast<uint32_t>(a) + static_cast<uint32_t>(b);
  return s > static_cast<uint32_t>(kMost) ? kMost : static_cast<int>(s);
}

struct AddMost {
  __device__ int operator()(int a, int b) const { return add_most(a, b); }
};
__device__ __forceinline__ int wave_scan(int x) { return lane_scan(x, AddMost{}); }

struct Three {
  int a, b, c;
};

// Exclusive running totals of three numbers over the block in thread order;
// *total gets the sums.
template <int WAVES>
__device__ __forceinline__ Three block_scan(Three v, Three *lds, Three *total) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Three run{wave_scan(v.a), wave_scan(v.b), wave_scan(v.c)};
  // the lane before's, 0 for lane 0
  Three out{dpp_move<0x138>(run.a), dpp_move<0x138>(run.b), dpp_move<0x138>(run.c)};
  if constexpr (WAVES == 1) {
    *total = Three{__builtin_amdgcn_readlane(run.a, 63), __builtin_amdgcn_readlane(run.b, 63),
                   __builtin_amdgcn_readlane(run.c, 63)};
    return out;
  }
  __syncthreads();
  if (lane == 63) lds[wave] = run;
  __syncthreads();
  Three w = lane < WAVES ? lds[lane] : Three{0, 0, 0};
  w = Three{wave_scan(w.a), wave_scan(w.b), wave_scan(w.c)};
  *total = Three{__builtin_amdgcn_readlane(w.a, 63), __builtin_amdgcn_readlane(w.b, 63),
                 __builtin_amdgcn_readlane(w.c, 63)};
  if (wave > 0) {
    out.a = add_most(out.a, __builtin_amdgcn_readlane(w.a, wave - 1));
    out.b = add_most(out.b, __builtin_amdgcn_readlane(w.b, wave - 1));
    out.c = add_most(out.c, __builtin_amdgcn_readlane(w.c, wave - 1));
  }
  return out;
}

// The last r < n with start[r] <= x (start[0] = 0, x >= 0); `top`: the power of two
// from which to halve, at least n.
__device__ __forceinline__ int find(const int *start, int n, int top, int x) {
  int r = 0;
  for (int step = top; step > 0; step >>= 1) {
    const int at = r + step;
    if (at < n && start[at] <= x) r = at;
  }
  return r;
}

template <int THREADS, int PER>
__global__ __launch_bounds__(THREADS) void paged_plan_kernel(PlanArgs a) {
  constexpr int kReq = THREADS * PER;
  __shared__ Three part[THREADS / 64];
  __shared__ int start[kReq + 1], lens[kReq];
  const int tid = threadIdx.x;
  const int64_t page = a.page.d;

  int cached[PER], grow[PER], have[PER], need[PER];
  bool gone[PER], refused[PER];
  Three own{0, 0, 0};  // new pages, new tokens, released pages
  int n_free = *a.n_free;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int i = tid * PER + k;
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
    own.a = add_most(own.a, need[k]);
    own.b = add_most(own.b, grow[k]);
    own.c = add_most(own.c, gone[k] ? have[k] : 0);
  }
  n_free = min(max(n_free, 0), a.n_pages);
  Three all;
  Three run = block_scan<THREADS / 64>(own, part, &all);
  int top = 1;
  while (top < a.n_req) top <<= 1;

  // the released pages go on the stack
  const int n_back = min(all.c, a.n_pages - n_free), avail = n_free + n_back;
  if (n_back > 0) {
    int at = run.c;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      if (tid * PER + k < a.n_req) start[tid * PER + k] = at;
      if (gone[k]) at = add_most(at, have[k]);
    }
    __syncthreads();
    // (unsigned: n_back may be within a round of 2^31)
    for (uint32_t p = tid; p < static_cast<uint32_t>(n_back); p += THREADS) {
      const int r = find(start, a.n_req, top, static_cast<int>(p));
      a.free_pages[n_free + p] = a.table[static_cast<size_t>(r) * a.width + (p - start[r])];
    }
    __syncthreads();
  }

  // who fits
  const int first = run.a;
  Three fit{0, 0, 0};  // pages taken, tokens admitted, requests refused
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    run.a = add_most(run.a, need[k]);
    run.b = add_most(run.b, grow[k]);
    if ((need[k] > 0 && run.a > avail) || (grow[k] > 0 && run.b > a.n_tok)) refused[k] = true;
    if (refused[k]) {
      need[k] = grow[k] = 0;
      ++fit.c;
    }
    fit.a += need[k];
    fit.b += grow[k];
  }
  Three sums;
  const Three before = block_scan<THREADS / 64>(fit, part, &sums);

  // the pages taken, from the top of the stack
  if (sums.a > 0) {
    int at = first;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int i = tid * PER + k;
      // a refused request's range is empty: it begins where the taken ones end
      if (i < a.n_req) start[i] = min(at, sums.a), lens[i] = have[k];
      at = add_most(at, need[k]);
    }
    __syncthreads();
    for (int p = tid; p < sums.a; p += THREADS) {
      const int entry = a.free_pages[avail - 1 - p];
      const int r = find(start, a.n_req, top, p);
      a.table[static_cast<size_t>(r) * a.width + lens[r] + (p - start[r])] = entry;
    }
    __syncthreads();
  }

  // offsets and lengths
  {
    int at = before.b;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      const int i = tid * PER + k;
      if (i < a.n_req) {
        const int len = gone[k] || refused[k] ? 0 : cached[k] + grow[k];
        a.q_start[i] = start[i] = at;
        a.kv_len[i] = len;
        lens[i] = len;
      }
      at += grow[k];
    }
  }
  const int live = sums.b;
  if (tid == 0) {
    start[a.n_req] = a.q_start[a.n_req] = live;
    *a.n_free_out = avail - sums.a;
    if (a.n_refused) *a.n_refused = sums.c;
  }
  __syncthreads();

  // tokens
  for (int t = tid; t < a.n_tok; t += THREADS) {
    int p = 0, slot = -1;
    if (t < live) {
      const int r = find(start, a.n_req, top, t);
      p = lens[r] - start[r + 1] + t;
      const int entry = a.table[static_cast<size_t>(r) * a.width + a.page.div(p)];
      if (entry >= 0 && entry < a.n_pages) slot = entry * a.page.d + a.page.mod(p);
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
  int n_tok, n_slots, elems, hd, pieces;
  FastDiv page, row, head;  // row, head: pieces of four elements
};

// Four elements a thread, for heads, strides and pointers of whole pieces: as many
// bytes in flight a wave as a copy has.  4001 rows of 4 x 256 in f32: 11.2 us, 5.9
// TB/s; 32 rows in f16: 2.8, the latency of the slot and of the store.
template <class T>
__global__ __launch_bounds__(256) void kv_store_paged_pieces_kernel(StoreArgs a) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i >= a.pieces) return;
  const int t = a.row.div(i), e = i - t * a.row.d, h = a.head.div(e);
  const float4 k = reinterpret_cast<const float4 *>(a.k)[i];  // fresh from the call before: cached
  const float4 v = reinterpret_cast<const float4 *>(a.v)[i];
  const int slot = a.slots[t];
  if (slot < 0 || slot >= a.n_slots) return;
  const int b = a.page.div(slot);
  const size_t at = b * a.page_stride + static_cast<size_t>(slot - b * a.page.d) * a.pos_stride +
                    h * a.head_stride + 4 * (e - h * a.head.d);
  if constexpr (sizeof(T) == 2) {
    typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));
    *reinterpret_cast<u16x4 *>(static_cast<T *>(a.kc) + at) =
        u16x4{store_half(k.x), store_half(k.y), store_half(k.z), store_half(k.w)};
    *reinterpret_cast<u16x4 *>(static_cast<T *>(a.vc) + at) =
        u16x4{store_half(v.x), store_half(v.y), store_half(v.z), store_half(v.w)};
  } else {
    *reinterpret_cast<float4 *>(static_cast<T *>(a.kc) + at) = k;
    *reinterpret_cast<float4 *>(static_cast<T *>(a.vc) + at) = v;
  }
}

// Any layout: a block a token (and every kStoreBlocks-th after it).  4001 rows of 4 x 256
// with an odd stride: f32 12.0 us, 5.4 TB/s (whole pieces 10.9), f16 10.9 (8.9).
constexpr int kStoreBlocks = 1 << 20;

template <class T>
__global__ __launch_bounds__(256) void kv_store_paged_kernel(StoreArgs a) {
  for (int64_t t = blockIdx.x; t < a.n_tok; t += kStoreBlocks) {
    const int slot = a.slots[t];
    if (slot < 0 || slot >= a.n_slots) continue;
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
  // in the order of their strides, each dimension steps over all that lies within it
  struct Dim {
    size_t n, stride;
  } dims[3] = {{c.n_pages, c.page_stride}, {c.page_size, c.pos_stride}, {c.n_kv, c.head_stride}};
  std::sort(dims, dims + 3, [](const Dim &x, const Dim &y) { return x.stride < y.stride; });
  size_t span = c.hd;
  for (const Dim &d : dims) {
    if (d.n == 1) continue;
    if (d.stride < span) return fail(BH_ERR_SHAPE, w + "the cache's strides let rows overlap");
    span += (d.n - 1) * d.stride;
  }
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
  if (p.n_tok > 0x7fffffffu - 4096)
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
  hipStream_t st = as_stream(stream);
  if (p.n_req <= 64 && p.n_tok <= 128) BH_LAUNCH((paged_plan_kernel<64, 1>), 1, 64, 0, st, a);
  else if (p.n_req <= 1024) BH_LAUNCH((paged_plan_kernel<1024, 1>), 1, 1024, 0, st, a);
  else BH_LAUNCH((paged_plan_kernel<1024, 4>), 1, 1024, 0, st, a);
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
  const size_t pieces = n_tok * (cache->n_kv * cache->hd / 4);
  const size_t piece = cache->kv_dtype == BH_KV_F16 ? 8 : 16;
  const auto whole = [](const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; };
  if (cache->hd % 4 == 0 && pieces <= 0x7fffff00u && (cache->page_stride | cache->pos_stride |
      cache->head_stride) % 4 == 0 && whole(cache->k, piece) && whole(cache->v, piece) &&
      whole(k, 16) && whole(v, 16)) {
    a.pieces = static_cast<int>(pieces);
    a.row = FastDiv(static_cast<uint32_t>(cache->n_kv * cache->hd / 4));
    a.head = FastDiv(static_cast<uint32_t>(cache->hd / 4));
    const unsigned blocks = static_cast<unsigned>((pieces + 255) / 256);
    if (cache->kv_dtype == BH_KV_F16)
      BH_LAUNCH(kv_store_paged_pieces_kernel<uint16_t>, blocks, 256, 0, as_stream(stream), a);
    else
      BH_LAUNCH(kv_store_paged_pieces_kernel<float>, blocks, 256, 0, as_stream(stream), a);
    return ok();
  }
  const unsigned blocks = static_cast<unsigned>(n_tok < kStoreBlocks ? n_tok : kStoreBlocks);
  if (cache->kv_dtype == BH_KV_F16)
    BH_LAUNCH(kv_store_paged_kernel<uint16_t>, blocks, 256, 0, as_stream(stream), a);
  else
    BH_LAUNCH(kv_store_paged_kernel<float>, blocks, 256, 0, as_stream(stream), a);
  return ok();
}
