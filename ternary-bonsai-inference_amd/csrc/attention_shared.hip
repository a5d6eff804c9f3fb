// Attention of requests that share a prefix: the prefix's keys and values are read
// once a tile of 16 to 128 rows of all requests of a group, not once a request.
//
// With o, m and l of a set of positions P the sums of a softmax over it (m the
// largest score, l = sum e^(s - m), o = sum e^(s - m) v), those of two sets join as
//   m' = max(m1, m2),  l' = e^(m1 - m') l1 + e^(m2 - m') l2,  o' likewise.
// So a group's prefix is one more request of the walk (paged_attention.hpp), whose
// tokens are those of all the group's requests and see all of it, and a request's own
// walk begins where its prefix ends.  Both stand in one list that is cut into equal
// runs, so that a long prefix and many short tails fill the card together; the join
// takes each row's parts from its own tile and from its tile of the prefix.
// 8 requests behind 4096 positions (24 / 4 heads of 256, f16): 18.1 us and 7.0 of the join, the
// prefix read by three tiles, from memory once; bh_attention_paged reads 8 times as much; 64
// behind 8192, tails to 2000: 66, 44 and 16.
#include <hip/hip_runtime.h>

#include <string>

#include "../../include/bonsai_hip_batch.h"
#include "common.hpp"
#include "paged.hpp"
#include "paged_attention.hpp"

namespace bh {
namespace {

// The tiles of a group's prefix: which launch has them and where they begin there.
struct Prefix {
  int q0 = 0, n = 0, base = 0, tiles = 0;
  uint32_t rows = 1, most = 0;  // of a tile; tiles of the launch
  bool two = false;
};

// A row's tile of the prefix: its parts' first place and number (0: none), and the
// row's number in it.
struct At {
  int slot = 0, parts = 0, row = 0;
};

template <int HD>
__global__ __launch_bounds__(kThreads) void attn_shared_join_kernel(PagedArgs a, Join one, Join two) {
  constexpr int kAt = kThreads / 16, kSlices = HD / 64, kAhead = 8;
  __shared__ float part[kAt][64], sums[kAt], tops[kAt];
  const bool of_two = blockIdx.x >= one.blocks;
  const unsigned block = blockIdx.x - (of_two ? one.blocks : 0);
  const Split sp = of_two ? two.sp : one.sp;
  const int share = of_two ? two.share : one.share, R = of_two ? two.rows : one.rows;
  const int tile = block / share, tid = threadIdx.x;
  const SharedCut cut = static_cast<const SharedCut *>(sp.cut)[tile];
  // (past n_tiles cut holds nothing; a prefix's tiles have no rows of their own)
  if (tile >= *sp.n_tiles || cut.r < a.n_group) return;
  Prefix pre;
  if (cut.group >= 0) {
    const PrefixOf of_group = a.prefix[cut.group];
    pre.q0 = of_group.q0, pre.n = of_group.n, pre.base = of_group.base, pre.two = of_group.launch != 0;
    const int64_t rows = static_cast<int64_t>(pre.n) * a.group;
    const Split &of = pre.two ? two.sp : one.sp;
    pre.rows = pre.two ? two.rows : one.rows;
    pre.tiles = static_cast<int>((rows + pre.rows - 1) / pre.rows);
    pre.most = min(static_cast<uint32_t>(*of.n_tiles), of.most_cut);
  }
  const Split psp = pre.two ? two.sp : one.sp;
  const auto prefix_of = [&](int row) {  // of the tile
    At at;
    if (pre.n == 0) return at;
    const int q_row = cut.row0 + row, tok = a.grp.div(q_row), t = cut.q0 + tok - pre.q0;
    if (t < 0 || t >= pre.n) return at;
    const uint32_t p_row = static_cast<uint32_t>(t * a.group + (q_row - tok * a.group));
    const uint32_t i = static_cast<uint32_t>(pre.base + cut.head * pre.tiles) + p_row / pre.rows;
    if (i >= pre.most) return at;
    const SharedCut &c = static_cast<const SharedCut *>(psp.cut)[i];
    at.row = static_cast<int>(p_row % pre.rows);
    at.slot = c.tile + c.first;
    at.parts = c.last - c.first + 1;
    return at;
  };
  const int own = cut.last - cut.first + 1, own_slot = cut.tile + cut.first;
  // groups of 16 lanes that share a row, the same number for the block
  const int most = own + max(prefix_of(0).parts, prefix_of(cut.rows - 1).parts);
  int p = 1;
  while (kAhead * p < most && p < kAt) p <<= 1;
  const int group = tid >> 4, mine = group & (p - 1), d = (tid & 15) * 4;
  const int items = cut.rows * kSlices, at_once = kAt / p;
  for (int i0 = (block - tile * share) * at_once; i0 < items; i0 += share * at_once) {
    const int item = i0 + group / p;
    const bool live = item < items;
    const int row = live ? item / kSlices : 0, dim = item % kSlices * 64 + d;
    const At pr = prefix_of(row);
    const int parts = own + pr.parts;
    struct Place {
      const float *m, *l, *o;
    };
    const auto at = [&](int x) {
      const bool is_own = x < own;
      const Split &of = is_own ? sp : psp;
      const size_t o = is_own ? static_cast<size_t>(own_slot + x) * R + row
                              : static_cast<size_t>(pr.slot + x - own) * pre.rows + pr.row;
      return Place{of.pm + o, of.pl + o, of.pacc + o * HD + dim};
    };
    f32x4 ahead[kAhead];
    float pm[kAhead], pl[kAhead];
#pragma unroll
    for (int x = 0; x < kAhead; ++x) {
      // past the last part: the last again, at no weight
      if (x * p >= most) break;
      const Place w = at(min(mine + x * p, parts - 1));
      ahead[x] = *reinterpret_cast<const f32x4 *>(w.o);
      pm[x] = *w.m;
      pl[x] = *w.l;
    }
    float top = -INFINITY;
#pragma unroll
    for (int x = 0; x < kAhead; ++x) {
      if (x * p >= most) break;
      top = fmaxf(top, pm[x]);
    }
    for (int x = mine + kAhead * p; x < parts; x += p) top = fmaxf(top, *at(x).m);
    if (p > 1) {
      if (d == 0) tops[group] = top;
      __syncthreads();
      for (int k = 0; k < p; ++k) top = fmaxf(top, tops[(group - mine) + k]);
    }
    const float ref = top == -INFINITY ? 0.0f : top;
    f32x4 o = {0, 0, 0, 0};
    float sum = 0.0f;
#pragma unroll
    for (int x = 0; x < kAhead; ++x) {
      if (x * p >= most) break;
      if (mine + x * p >= parts) continue;
      const float keep = __builtin_amdgcn_exp2f(pm[x] - ref);
      sum += keep * pl[x];
      o += keep * ahead[x];
    }
#pragma unroll 4
    for (int x = mine + kAhead * p; x < parts; x += p) {
      const Place w = at(x);
      const float keep = __builtin_amdgcn_exp2f(*w.m - ref);
      sum += keep * *w.l;
      o += keep * *reinterpret_cast<const f32x4 *>(w.o);
    }
    if (p > 1) {
      *reinterpret_cast<f32x4 *>(&part[group][d]) = o;
      if (d == 0) sums[group] = sum;
      __syncthreads();
    }
    if (mine == 0 && live) {
      for (int k = 1; k < p; ++k) {
        o += *reinterpret_cast<const f32x4 *>(&part[group + k][d]);
        sum += sums[group + k];
      }
      const int q_row = cut.row0 + row, tok = a.grp.div(q_row);
      *reinterpret_cast<f32x4 *>(
          a.out + (static_cast<size_t>(cut.q0 + tok) * a.n_head + cut.head * a.group +
                   (q_row - tok * a.group)) * HD + dim) = o * (top == -INFINITY ? 0.0f : 1.0f / sum);
    }
    if (p > 1) __syncthreads();  // for the next rows
  }
}

int launch_shared_join(const PagedArgs &a, const Join &one, const Join &two, hipStream_t st) {
  const unsigned blocks = one.blocks + two.blocks;
  if (a.hd == 64) BH_LAUNCH(attn_shared_join_kernel<64>, blocks, kThreads, 0, st, a, one, two);
  else if (a.hd == 128) BH_LAUNCH(attn_shared_join_kernel<128>, blocks, kThreads, 0, st, a, one, two);
  else BH_LAUNCH(attn_shared_join_kernel<256>, blocks, kThreads, 0, st, a, one, two);
  return BH_OK;
}

// As forms_of, the prefix of a group being a request of all the group's rows; but the
// tiles of a prefix read the same pages, which then come from the last level cache, so
// that small tiles, whose steps are shorter, cost less than there, and one launch saves
// more than the wide form's larger tiles while the work is small.  What counts is the work
// as far as the host knows it: rows of the call times positions of the table, in millions.
// Measured, us of the call, in order: as in forms_of, one row tile, two; "rows" of a group.
//   up to 64 rows.  hd 256, f16: 0.2 32, 26, 32; 0.8 50, 46, 51; 1.0 54, 57, 54; 2.0 72, 86, 74
//     f32: 0.5 73, 65, 70; 0.6 82, 83, 82; 1.0 81, 98, 84
//     hd 128, f16: 0.07 24, 21, 21; 0.3 34, 34, 33; 0.4 32, 38, 31; 1.1 44, 56, 45
//     f32: 0.05 25, 22, 25; 0.13 28, 29, 29; 0.5 50, 55, 50
//     hd 64, f16: 0.3 18, 16, 18; 1.1 21, 21, 21; 8.5 41, 49, 41; f32: 0.3 20, 18, 19; 1.9 38, 36, 38;
//     3.2 38, 47, 38
//   more.  hd 256, f16: 0.4 46, 26, 31; 0.8 71, 47, 56; 1.3 66, 62, 58; 2.5 64, 68, 58; 3.1 106, 128, 116
//     f32: 0.4 86, 38, 39; 0.8 96, 81, 73; 2.1 171, 153, 134; 6.4 321, 492, 322
//     hd 128, f16: 0.3 47, 32, 34; 0.8 52, 44, 41; 3.3 114, 138, 93; 4.3 102, 176, 106
//     f32: 0.3 74, 47, 52; 0.8 80, 83, 65; 4.3 228, 342, 207
//     hd 64, f16: 1.1 31, 21, 23; 2.8 44, 29, 30; 4.1 50, 34, 31; 8.5 59, 52, 44
//     f32: 1.1 40, 25, 27; 2.1 45, 35, 34; 8.5 88, 104, 77
//
// A tile has whole runs (Walk::run) where few requests and groups have few units a worker:
// us of the call without and with, f16 hd 256 at 6 units a worker 60 and 46, at 7 71 and 63;
// hd 128 at 7 54 and 39; hd 64 at 4 28 and 26; f32 102 and 84, 53 and 49, 39 and 33.
// Where runs are longer, or tiles many, the walk's further registers only cost, up to 4 per
// cent: the host leaves out what can be told from the table, the rows and the requests.
bool whole_runs_pay(const bh_attention_paged_args &q, size_t n_group, const Form &f) {
  const size_t n = q.n_req + n_group, most = f.workers() / kRunPads;
  if (n > 64 || n * q.cache.n_kv > most) return false;
  const size_t tiles = q.n_tok * (q.n_head / q.cache.n_kv) / f.rows() + n_group;
  const int unit = q.cache.kv_dtype == BH_KV_F16 && q.cache.hd <= 128 ? 128 : 64;  // Shape::U
  return static_cast<double>(tiles * q.cache.n_kv) * static_cast<double>(q.table_width * q.cache.page_size) <=
         1.25 * kRunUnits * unit * f.workers();
}

int shared_forms(const bh_attention_shared_args &p, Form *f) {
  bh_attention_paged_args q = p.paged;
  const size_t own = q.max_new == 0 || q.max_new > q.n_tok ? q.n_tok : q.max_new;
  const size_t all = p.max_group_new == 0 || p.max_group_new > q.n_tok ? q.n_tok : p.max_group_new;
  q.max_new = all > own ? all : own;
  q.n_req = 2;  // not one request's: both sorts are there
  const size_t group = q.n_head / q.cache.n_kv, rows = q.max_new * group;
  const double work = 1e-6 * static_cast<double>(q.n_tok * group) *
                      static_cast<double>(q.table_width * q.cache.page_size);
  // up to which one tile is taken: up to 64 rows, of more; two tiles of more
  struct Line {
    double few, one, two;
  };
  const bool f16 = q.cache.kv_dtype == BH_KV_F16;
  const Line line = q.cache.hd == 256   ? (f16 ? Line{0.9, 1.0, 2.6} : Line{0.55, 0.6, 6})
                    : q.cache.hd == 128 ? (f16 ? Line{0.3, 0.5, 4.2} : Line{0.13, 0.5, 5})
                                        : (f16 ? Line{1.1, 3, 16} : Line{2, 2, 12});
  constexpr int kAll = 0x7fffffff;
  if (work <= (rows <= 64 ? line.few : line.one)) {
    f[0] = Form{1, false, 0, kAll, 2};
    f[0].runs = whole_runs_pay(p.paged, p.n_group, f[0]);
    return 1;
  }
  if (rows > 64 && work <= line.two) {
    f[0] = Form{2, false, 0, kAll, q.cache.hd == 256 ? 1 : 2};  // (E::kBlocks)
    f[0].runs = whole_runs_pay(p.paged, p.n_group, f[0]);
    return 1;
  }
  const int n = forms_of(q, f);
  if (n == 1 && !f[0].wide) f[0].runs = whole_runs_pay(p.paged, p.n_group, f[0]);
  return n;
}

size_t prefix_bytes(const PagedArgs &a) { return align256(a.n_group * sizeof(PrefixOf)); }

int prepare_shared(const bh_attention_shared_args &p, PagedArgs *a) {
  if (int e = prepare(p.paged, a, "attention_shared")) return e;
  if (p.n_group > 0x7fff0000u || p.paged.n_req + p.n_group > 0x7fff0000u)
    return fail(BH_ERR_SHAPE, "attention_shared: size overflow");
  if (p.n_group != 0 && p.paged.n_tok != 0 && p.paged.n_req != 0 &&
      (!p.group || !p.group_start || !p.shared_len))
    return fail(BH_ERR_ARG, "attention_shared: null pointer");
  a->group_of = p.group, a->group_start = p.group_start, a->shared_len = p.shared_len;
  a->n_group = static_cast<int>(p.n_group);
  return BH_OK;
}

}  // namespace
}  // namespace bh

using namespace bh;

extern "C" size_t bh_attention_shared_workspace(const bh_attention_shared_args *args) {
  PagedArgs a{};
  if (!args || prepare_shared(*args, &a) != BH_OK) return 0;
  if (a.n_group == 0 || !on_matrix_cores(args->paged))
    return bh_attention_paged_workspace(&args->paged);
  if (a.n_tok == 0 || a.n_req == 0) return 0;
  Form f[2];
  size_t need = 0;
  for (int i = 0, n = shared_forms(*args, f); i < n; ++i) need += workspace_of<true>(a, f[i]);
  return need + prefix_bytes(a);
}

extern "C" int bh_attention_shared(const bh_attention_shared_args *args, bh_stream stream) {
  if (!args) return fail(BH_ERR_ARG, "attention_shared: null args");
  const bh_attention_shared_args &p = *args;
  PagedArgs a{};
  if (int e = prepare_shared(p, &a)) return e;
  if (a.n_tok == 0 || a.n_req == 0) return ok();
  if (a.n_group == 0 || !on_matrix_cores(p.paged)) return bh_attention_paged(&p.paged, stream);
  const bool f16 = p.paged.cache.kv_dtype == BH_KV_F16;
  hipStream_t st = as_stream(stream);
  Form f[2];
  const int n = shared_forms(p, f);
  size_t need = prefix_bytes(a), tiles = 0;
  for (int i = 0; i < n; ++i) {
    need += workspace_of<true>(a, f[i]);
    tiles += most_tiles<true>(a, f[i]);
  }
  if (tiles > kMostBlocks)  // (the join has more than a block a tile only of few)
    return fail(BH_ERR_SHAPE, "attention_shared: more row tiles than a launch has blocks");
  char *ws = static_cast<char *>(p.paged.workspace);
  if (ws) {
    if (!aligned16(ws) || p.paged.workspace_bytes < need)
      return fail(BH_ERR_SHAPE, "attention_shared: workspace of " +
                                    std::to_string(p.paged.workspace_bytes) + " bytes, " +
                                    std::to_string(need) + " needed on a 16-byte boundary");
  } else {
    ws = static_cast<char *>(device_scratch(need, kScratchPaged, st));
    if (!ws) return BH_ERR_HIP;
  }
  Join join[2] = {};
  a.prefix = reinterpret_cast<PrefixOf *>(ws);
  ws += prefix_bytes(a);
  for (int i = 0; i < n; ++i) {
    a.launch = i;
    if (int e = launch_form<true>(a, f16, f[i], ws, st, &join[i])) return e;
    ws += workspace_of<true>(a, f[i]);
  }
  if (int e = launch_shared_join(a, join[0], join[1], st)) return e;
  return ok();
}
