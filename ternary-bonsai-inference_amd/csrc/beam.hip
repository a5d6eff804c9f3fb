// Beam search: the selection of a step, and the beams' storage in the new order.
//
// Selection.  Every continuation of a group's beams has the score
//   score[row] + (x - m) inv_temp - ln S,  m and S of its row of logits,
// and the n_best largest are wanted.  The pass over the logits (logits.hpp) leaves, a
// part of a row, m, S and the part's n_best largest logits in order; the n_best best
// of a group are among these, as a row's continuations are in the order of its
// logits.  One block a group then forms the rows' ln S, and with them the score of
// each part's logits.  Where n_best of them reach a bound, only keys that reach it
// matter: a few more than n_best, whose ranks, counted against one another, are
// their places.  Scores are compared in f64: a step of f32 at a score of -100 is 8e-6, and
// what rounds before is ln S, which is the same for a beam's own continuations.  Its
// exponentials are f32's, of arguments z log2(e) that round three times: |z| 3 2^-24, and
// terms that matter have z down to -20: within 4e-6, commonly 1e-7.
// Bound by reading the logits: 256 rows of 248320 in 32 groups, best 16: 57.0 us, 4.5 TB/s,
// and 8.2 for the groups (30 with 256 threads that went through their lists one key after
// the other); 4 rows 8.8 and 4.6.
#include <hip/hip_runtime.h>

#include <cmath>
#include <string>

#include "../../include/bonsai_hip_batch.h"
#include "common.hpp"
#include "logits.hpp"
#include "paged.hpp"

namespace bh {
namespace {

constexpr int kMostFirsts = 1024;  // parts of a group
constexpr int kSelThreads = 1024, kSelWaves = kSelThreads / 64;  // of a group's block
constexpr int kDepths = 3;  // keys 1, 4, 16 of a part
constexpr int kMostCand = 1024;    // candidates that are ranked at once
constexpr int kAhead = 2;          // keys of a thread on their way

struct BeamArgs {
  const float *score;
  int32_t *parent;
  uint32_t *token;
  float *score_out;
  int width, n_best, n_parts;
  float inv_temp, k2;
  const Part *parts;
  const uint64_t *keys;
};

// A continuation: larger scores first, of equal ones the lower beam, of one beam's
// the larger logit and then the lower token, which is the larger key.
struct Cand {
  double score;  // -inf: none
  uint64_t key;
  int beam;
  __device__ __forceinline__ bool before(const Cand &o) const {
    if (score != o.score) return score > o.score;
    if (beam != o.beam) return beam < o.beam;
    return key > o.key;
  }
};

template <class T>
__device__ __forceinline__ T lane_xor(T x, int by) {
  return __shfl_xor(x, by);
}

// One block a group.
__global__ __launch_bounds__(kSelThreads) void beam_select_kernel(BeamArgs a) {
  __shared__ double base_s[BH_MAX_BEAMS];  // score - ln S; NaN: no continuations
  __shared__ float m_s[BH_MAX_BEAMS];
  __shared__ __attribute__((aligned(16))) double score_s[kMostCand];  // of the candidates
  __shared__ uint64_t key_s[kMostCand];
  __shared__ uint8_t beam_s[kMostCand];
  __shared__ Cand best_s[kSelWaves];
  __shared__ uint32_t bound_s[kSelWaves];
  __shared__ int count_s, n_live_s, best_at[kSelWaves];
  __shared__ uint16_t live_s[kMostFirsts];  // parts whose first reaches the bound
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int row0 = blockIdx.x * a.width, firsts = a.width * a.n_parts;
  const size_t part0 = static_cast<size_t>(row0) * a.n_parts;

  static_assert(kMostFirsts == kSelThreads, "a part a thread");
  uint64_t of_part[kDepths];  // its keys 1, 4, 16
#pragma unroll
  for (int i = 0; i < kDepths; ++i)
    of_part[i] = tid < firsts && 1 << 2 * i <= a.n_best
                     ? a.keys[(part0 + tid) * a.n_best + (1 << 2 * i) - 1] : 0;
  const uint64_t first = of_part[0];
  if (tid == 0) count_s = n_live_s = 0;
  for (int b = wave; b < a.width; b += kSelWaves) {
    const Part *parts = a.parts + part0 + static_cast<size_t>(b) * a.n_parts;
    Part p[2] = {{0.0, 0.0, -INFINITY}, {0.0, 0.0, -INFINITY}};
    static_assert(kMaxParts == 128, "two parts a lane");
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (lane + 64 * i < a.n_parts) p[i] = parts[lane + 64 * i];
    const float m = lane_group_reduce<64>(p[1].m > p[0].m ? p[1].m : p[0].m, MaxOp{});
    double s = 0.0;
#pragma unroll
    for (int i = 0; i < 2; ++i)  // (a part of -inf: 0, or NaN from a NaN logit)
      s += p[i].m == -INFINITY ? p[i].s
                               : p[i].s * static_cast<double>(__builtin_amdgcn_exp2f((p[i].m - m) * a.k2));
    s = lane_group_reduce<64>(s, SumOp{});
    const float score = a.score[row0 + b];
    const bool good = m > -INFINITY && m < INFINITY && fabsf(score) < INFINITY;
    if (lane == 0) {
      m_s[b] = m;
      base_s[b] = good ? static_cast<double>(score) - log(s) : NAN;
    }
  }
  __syncthreads();
  const auto of = [&](int beam, uint64_t key) {
    const double x = value_of(key);
    double score = base_s[beam] + (x - static_cast<double>(m_s[beam])) * static_cast<double>(a.inv_temp);
    if (key >> 32 == 0 || !(score > -INFINITY)) score = -INFINITY;  // none, NaN, banned
    return Cand{score, key, beam};
  };

  // The bound: where n_best / q parts' q-th keys reach one of 16 bits, n_best keys do.  The
  // highest of the waves' and of those of q = 1, 4 and 16 (where one beam has most of the
  // best, the first keys alone leave hundreds: 11 groups of 16 beams, best 26 59 us, so 10.2;
  // up to 8 they leave few enough: one of 4 4.6, so 5.3).
  uint32_t lanes_bound = 0;
#pragma unroll
  for (int i = 0; i < kDepths; ++i) {
    if (1 << 2 * i > a.n_best || (i > 0 && a.n_best <= 8)) break;
    float top = -INFINITY;
    if (tid < firsts) top = static_cast<float>(of(tid / a.n_parts, of_part[i]).score);
    const uint32_t at = bound_of_lanes(order_of(top), (a.n_best + (1 << 2 * i) - 1) >> 2 * i);
    lanes_bound = at > lanes_bound ? at : lanes_bound;
  }
  if (lane == 0) bound_s[wave] = lanes_bound;
  __syncthreads();
  uint32_t bound = 0;
#pragma unroll
  for (int w = 0; w < kSelWaves; ++w) bound = bound_s[w] > bound ? bound_s[w] : bound;
  const auto reaches = [&](const Cand &c) {
    return c.score > -INFINITY && order_of(static_cast<float>(c.score)) >= bound;
  };
  if (tid < firsts && reaches(of(tid / a.n_parts, first))) live_s[atomicAdd(&n_live_s, 1)] = tid;
  __syncthreads();
  const int n_keys = n_live_s * a.n_best;
  for (int i0 = tid; i0 < n_keys; i0 += kAhead * kSelThreads) {
    uint64_t key[kAhead];
    int of_part[kAhead];
#pragma unroll
    for (int x = 0; x < kAhead; ++x) {
      const int i = min(i0 + x * kSelThreads, n_keys - 1), at = i / a.n_best;
      of_part[x] = live_s[at];
      key[x] = a.keys[(part0 + of_part[x]) * a.n_best + (i - at * a.n_best)];
    }
#pragma unroll
    for (int x = 0; x < kAhead; ++x) {
      const Cand c = of(of_part[x] / a.n_parts, key[x]);
      if (i0 + x * kSelThreads >= n_keys || !reaches(c)) continue;
      const int at = atomicAdd(&count_s, 1);
      if (at < kMostCand) score_s[at] = c.score, key_s[at] = c.key, beam_s[at] = c.beam;
    }
  }
  __syncthreads();
  const int count = count_s;
  const size_t out = static_cast<size_t>(blockIdx.x) * a.n_best;
  const auto put = [&](int place, const Cand &c) {
    a.parent[out + place] = row0 + c.beam;
    a.token[out + place] = ~static_cast<uint32_t>(c.key);
    a.score_out[out + place] = static_cast<float>(c.score);
  };
  const auto none = [&](int place) {
    a.parent[out + place] = -1;
    a.token[out + place] = ~0u;
    a.score_out[out + place] = -INFINITY;
  };
  if (count <= kMostCand) {
    // four lanes a candidate, each against every fourth
    for (int i = count + tid; i < min((count + 31) & ~31, kMostCand); i += kSelThreads) score_s[i] = -INFINITY;
    __syncthreads();
    for (int i0 = 0; i0 < count; i0 += kSelThreads / 4) {
      const int i = min(i0 + tid / 4, count - 1);
      const Cand c{score_s[i], key_s[i], beam_s[i]};
      int rank = 0, same = 0;
      for (int k = tid & 3; k < count; k += 32) {
#pragma unroll
        for (int x = 0; x < 32; x += 4)
          rank += score_s[k + x] > c.score, same += score_s[k + x] == c.score;
      }
      if (__any(lane_group_sum<4>(static_cast<float>(same)) > 1.0f)) {  // (its own is one)
#pragma unroll 4
        for (int k = tid & 3; k < count; k += 4)
          rank += score_s[k] == c.score && Cand{score_s[k], key_s[k], beam_s[k]}.before(c);
      }
      rank = static_cast<int>(lane_group_sum<4>(static_cast<float>(rank)));
      if ((tid & 3) == 0 && i0 + tid / 4 < count && rank < a.n_best) put(rank, c);
    }
    for (int i = count + tid; i < a.n_best; i += kSelThreads) none(i);
    return;
  }
  // Too many equal ones: the parts' lists merged, one continuation a round.
  int next = 1;
  Cand head = tid < firsts ? of(tid / a.n_parts, first) : Cand{-INFINITY, 0, a.width};
  for (int place = 0; place < a.n_best; ++place) {
    Cand best = head;
    int at = tid;
#pragma unroll
    for (int by = 32; by > 0; by >>= 1) {
      const Cand o{lane_xor(best.score, by),
                   static_cast<uint64_t>(lane_xor(static_cast<unsigned long long>(best.key), by)),
                   lane_xor(best.beam, by)};
      const int o_at = lane_xor(at, by);
      if (o.before(best)) best = o, at = o_at;
    }
    __syncthreads();
    if (lane == 0) best_s[wave] = best, best_at[wave] = at;
    __syncthreads();
    best = best_s[0], at = best_at[0];
#pragma unroll
    for (int w = 1; w < kSelWaves; ++w)
      if (best_s[w].before(best)) best = best_s[w], at = best_at[w];
    if (tid == 0) {
      if (best.score > -INFINITY) put(place, best);
      else none(place);
    }
    if (tid == at && tid < firsts) {
      head.score = -INFINITY;
      if (next < a.n_best) head = of(tid / a.n_parts, a.keys[(part0 + tid) * a.n_best + next++]);
    }
  }
}

// ---- storage -----------------------------------------------------------------

constexpr int kColumns = 64;  // of a table, a block's at a time

struct ReorderArgs {
  const int32_t *parent;
  int32_t *table, *copy_from, *src, *dst, *spare;
  int width, parent_stride, table_width;
};

// Block (group, kColumns columns of its tables): each thread knows the whole
// permutation, the block its columns' old entries in LDS.  The group's first block
// has its slots too.
__global__ __launch_bounds__(256) void beam_reorder_kernel(ReorderArgs a, int parts) {
  __shared__ int32_t old[BH_MAX_BEAMS][kColumns];
  __shared__ int from_s[BH_MAX_BEAMS], copy_s[BH_MAX_BEAMS], parent_s[BH_MAX_BEAMS];
  const int g = blockIdx.x / parts, part = blockIdx.x - g * parts, tid = threadIdx.x;
  const int row0 = g * a.width, c0 = part * kColumns;
  const int columns = min(kColumns, a.table_width - c0);
  for (int i = tid; i < a.width * kColumns; i += 256) {
    const int b = i / kColumns, c = i % kColumns;
    if (c < columns) old[b][c] = a.table[static_cast<size_t>(row0 + b) * a.table_width + c0 + c];
  }
  if (tid < 64) {  // lane b: beam b
    const int lane = tid;
    int p = -1;
    if (lane < a.width) {
      const int of = a.parent[static_cast<size_t>(g) * a.parent_stride + lane];
      if (of >= row0 && of < row0 + a.width) p = of - row0;
    }
    int heir = lane;  // the first beam of the same parent
    uint64_t with_children = 0;
    for (int b = a.width - 1; b >= 0; --b) {
      const int of = __builtin_amdgcn_readlane(p, b);
      if (of < 0) continue;
      with_children |= uint64_t{1} << of;
      if (of == p) heir = b;
    }
    const uint64_t all = (uint64_t{1} << a.width) - 1;
    const bool takes = lane < a.width && (p < 0 || heir != lane);
    const uint64_t takers = __ballot(takes);
    int from = p;
    if (takes) {  // the n-th row without children, n = the takers before
      uint64_t free = all & ~with_children;
      for (int n = __popcll(takers & ((uint64_t{1} << lane) - 1)); n > 0; --n) free &= free - 1;
      from = __builtin_ffsll(free) - 1;
    }
    if (lane < a.width) {
      from_s[lane] = from;
      parent_s[lane] = p < 0 ? lane : p;
      copy_s[lane] = takes && p >= 0 ? row0 + heir : -1;
    }
  }
  __syncthreads();
  for (int i = tid; i < a.width * kColumns; i += 256) {
    const int b = i / kColumns, c = i % kColumns;
    if (c < columns)
      a.table[static_cast<size_t>(row0 + b) * a.table_width + c0 + c] = old[from_s[b]][c];
  }
  if (part == 0) {
    int written = 0, spare = 0, src = 0;
    if (tid < a.width) {
      a.copy_from[row0 + tid] = copy_s[tid];
      if (a.src) {
        written = a.dst[row0 + tid];
        spare = a.spare[row0 + tid];
        src = a.dst[row0 + parent_s[tid]];
      }
    }
    __syncthreads();
    if (tid < a.width && a.src) {
      a.src[row0 + tid] = src;
      a.dst[row0 + tid] = spare;
      a.spare[row0 + tid] = written;
    }
  }
}

struct CopyArgs {
  void *k, *v;
  const int32_t *table, *from, *begin, *end;
  size_t page_stride, pos_stride, head_stride;  // elements of T
  int n_req, width, n_pages, max_len, blocks;   // blocks a request
  int elems, hd;                                // of T, a position and a head
  FastDiv page, row, head;                      // row, head: pieces of T
};

constexpr int kCopyItems = 2;  // pieces a thread has on their way at once

// Block (request, share): the request's pieces of sizeof(T) bytes, position by
// position, kCopyItems a thread at a time.
template <class T>
__global__ __launch_bounds__(256) void kv_copy_paged_kernel(CopyArgs a) {
  const int r = blockIdx.x / a.blocks, share = blockIdx.x - r * a.blocks;
  const int of = a.from[r];
  if (of < 0 || of >= a.n_req) return;
  const int begin = a.begin ? min(max(a.begin[r], 0), a.max_len) : 0;
  const int end = min(max(a.end[r], 0), a.max_len);
  const int32_t *to_pages = a.table + static_cast<size_t>(r) * a.width;
  const int32_t *of_pages = a.table + static_cast<size_t>(of) * a.width;
  const int64_t pieces = static_cast<int64_t>(max(end - begin, 0)) * a.elems;
  const T *k_of = static_cast<const T *>(a.k), *v_of = static_cast<const T *>(a.v);
  T *k_to = static_cast<T *>(a.k), *v_to = static_cast<T *>(a.v);
  for (int64_t i0 = static_cast<int64_t>(share) * 256 * kCopyItems; i0 < pieces;
       i0 += static_cast<int64_t>(a.blocks) * 256 * kCopyItems) {
    const int p0 = static_cast<int>(i0 / a.elems);  // of the block's first piece
    const int rest = static_cast<int>(i0 - static_cast<int64_t>(p0) * a.elems);
    size_t to[kCopyItems];
    bool live[kCopyItems];
    T k[kCopyItems], v[kCopyItems];
#pragma unroll
    for (int x = 0; x < kCopyItems; ++x) {
      const int i = x * 256 + static_cast<int>(threadIdx.x);
      live[x] = i0 + i < pieces;
      const int at = rest + (live[x] ? i : 0), past = a.row.div(at), e = at - past * a.elems;
      const int p = begin + p0 + past, b = a.page.div(p), h = a.head.div(e);
      const int page_to = to_pages[b], page_of = of_pages[b];
      live[x] = live[x] && page_to >= 0 && page_to < a.n_pages && page_of >= 0 &&
                page_of < a.n_pages && page_to != page_of;
      const size_t in_page = static_cast<size_t>(p - b * a.page.d) * a.pos_stride +
                             h * a.head_stride + (e - h * a.head.d);
      to[x] = page_to * a.page_stride + in_page;
      if (live[x]) {
        k[x] = k_of[page_of * a.page_stride + in_page];
        v[x] = v_of[page_of * a.page_stride + in_page];
      }
    }
#pragma unroll
    for (int x = 0; x < kCopyItems; ++x)
      if (live[x]) k_to[to[x]] = k[x], v_to[to[x]] = v[x];
  }
}

constexpr size_t kMostBlocks = 0xffffff;

int check(const bh_beam_select_args &p) {
  if (p.width == 0 || p.width > BH_MAX_BEAMS)
    return fail(BH_ERR_SHAPE, "beam_select: width " + std::to_string(p.width) + " must be 1 .. " +
                                  std::to_string(BH_MAX_BEAMS));
  if (p.vocab == 0 || p.vocab > 0x7fffffffu)
    return fail(BH_ERR_SHAPE, "beam_select: vocab must be 1 .. 2^31 - 1");
  if (p.row_stride < p.vocab)
    return fail(BH_ERR_SHAPE, "beam_select: row_stride " + std::to_string(p.row_stride) +
                                  " below vocab " + std::to_string(p.vocab));
  if (p.n_best == 0 || p.n_best > BH_MAX_TOP || p.n_best > p.vocab)
    return fail(BH_ERR_SHAPE, "beam_select: n_best " + std::to_string(p.n_best) + " must be 1 .. " +
                                  std::to_string(BH_MAX_TOP) + " and up to vocab");
  size_t n;
  if (p.n_group > kMostBlocks / BH_MAX_BEAMS ||
      !mul_size(p.n_group * p.width, p.row_stride, sizeof(float), &n))
    return fail(BH_ERR_SHAPE, "beam_select: size overflow");
  if (!(p.inv_temp > 0.0f) || std::isinf(p.inv_temp * kExpL2E))
    return fail(BH_ERR_ARG, "beam_select: inv_temp must be finite and above 0");
  if (p.n_group != 0) {
    if (reinterpret_cast<uintptr_t>(p.x) % sizeof(float) != 0)
      return fail(BH_ERR_ARG, "beam_select: misaligned x");
    if (!p.x || !p.score || !p.parent || !p.token || !p.score_out)
      return fail(BH_ERR_ARG, "beam_select: null pointer");
    if (p.score_out == p.score && p.n_best != p.width)
      return fail(BH_ERR_ARG, "beam_select: score_out may be score only where n_best is width");
  }
  return BH_OK;
}

// Whether one of the groups' rows of `parent` shares memory with n words at `out`.
bool parents_meet(const bh_beam_reorder_args &p, const int32_t *out, size_t n) {
  const int64_t row = 4 * static_cast<int64_t>(p.width), stride = 4 * static_cast<int64_t>(p.parent_stride);
  const int64_t begin = static_cast<int64_t>(reinterpret_cast<uintptr_t>(out) - reinterpret_cast<uintptr_t>(p.parent));
  const int64_t end = begin + 4 * static_cast<int64_t>(n);
  if (end <= 0) return false;
  const int64_t g = begin < row ? 0 : (begin - row) / stride + 1;  // the first that ends behind `begin`
  return g < static_cast<int64_t>(p.n_group) && g * stride < end;
}

size_t parts_of(const bh_beam_select_args &p) {
  const size_t parts = parts_of_rows(p.n_group * p.width, p.vocab);
  const size_t most = kMostFirsts / p.width;  // (a group's parts have a thread each to look at them)
  return parts < most ? parts : most;
}

size_t workspace_of(const bh_beam_select_args &p) {
  return p.n_group * p.width * parts_of(p) * (sizeof(Part) + 8 * p.n_best);
}

}  // namespace
}  // namespace bh

using namespace bh;

extern "C" size_t bh_beam_select_workspace(const bh_beam_select_args *args) {
  if (!args || check(*args) != BH_OK || args->n_group == 0) return 0;
  return workspace_of(*args);
}

extern "C" int bh_beam_select(const bh_beam_select_args *args, bh_stream stream) {
  if (!args) return fail(BH_ERR_ARG, "beam_select: null args");
  const bh_beam_select_args &p = *args;
  if (int e = check(p)) return e;
  if (p.n_group == 0) return ok();
  hipStream_t st = as_stream(stream);
  const size_t need = workspace_of(p), parts = parts_of(p), rows = p.n_group * p.width;
  char *ws = static_cast<char *>(p.workspace);
  if (ws) {
    if (!aligned16(ws) || p.workspace_bytes < need)
      return fail(BH_ERR_SHAPE, "beam_select: workspace of " + std::to_string(p.workspace_bytes) +
                                    " bytes, " + std::to_string(need) +
                                    " needed on a 16-byte boundary");
  } else {
    ws = static_cast<char *>(device_scratch(need, kScratchLogprobs, st));
    if (!ws) return BH_ERR_HIP;
  }
  LogprobArgs l{};
  l.x = p.x, l.score = p.score, l.row_stride = p.row_stride;
  l.vocab = static_cast<int>(p.vocab), l.n_top = static_cast<int>(p.n_best);
  l.n_parts = static_cast<int>(parts);
  l.inv_temp = p.inv_temp, l.k2 = p.inv_temp * kExpL2E;
  l.parts = reinterpret_cast<Part *>(ws);
  l.keys = reinterpret_cast<uint64_t *>(ws + rows * parts * sizeof(Part));
  BH_LAUNCH((token_logprobs_kernel<true, true>), static_cast<unsigned>(rows * parts), kLpThreads, 0,
            st, l);
  BeamArgs a{};
  a.score = p.score, a.parent = p.parent, a.token = p.token, a.score_out = p.score_out;
  a.width = static_cast<int>(p.width), a.n_best = l.n_top, a.n_parts = l.n_parts;
  a.inv_temp = l.inv_temp, a.k2 = l.k2, a.parts = l.parts, a.keys = l.keys;
  BH_LAUNCH(beam_select_kernel, static_cast<unsigned>(p.n_group), kSelThreads, 0, st, a);
  return ok();
}

extern "C" int bh_beam_reorder(const bh_beam_reorder_args *args, bh_stream stream) {
  if (!args) return fail(BH_ERR_ARG, "beam_reorder: null args");
  const bh_beam_reorder_args &p = *args;
  if (p.width == 0 || p.width > BH_MAX_BEAMS)
    return fail(BH_ERR_SHAPE, "beam_reorder: width " + std::to_string(p.width) + " must be 1 .. " +
                                  std::to_string(BH_MAX_BEAMS));
  if (p.parent_stride < p.width)
    return fail(BH_ERR_SHAPE, "beam_reorder: parent_stride " + std::to_string(p.parent_stride) +
                                  " below width " + std::to_string(p.width));
  if (p.table_width == 0 || p.table_width > 0x7fff0000u)
    return fail(BH_ERR_SHAPE, "beam_reorder: table_width must be 1 .. 2^31 - 65536");
  const size_t parts = (p.table_width + kColumns - 1) / kColumns;
  size_t n;
  if (p.n_group > 0x7fffffffu / BH_MAX_BEAMS || p.parent_stride > 0x7fffffffu ||
      !mul_size(p.n_group, parts, &n) || n > kMostBlocks)
    return fail(BH_ERR_SHAPE, "beam_reorder: size overflow");
  if (p.n_group == 0) return ok();
  if (!p.parent || !p.block_table || !p.copy_from)
    return fail(BH_ERR_ARG, "beam_reorder: null pointer");
  if (!p.src_slot != !p.dst_slot || !p.src_slot != !p.spare_slot)
    return fail(BH_ERR_ARG, "beam_reorder: src_slot, dst_slot and spare_slot go together");
  if (p.src_slot && (p.src_slot == p.dst_slot || p.src_slot == p.spare_slot ||
                     p.dst_slot == p.spare_slot))
    return fail(BH_ERR_ARG, "beam_reorder: src_slot, dst_slot and spare_slot must differ");
  // (a group's blocks all read its parents while one of them writes)
  const size_t beams = p.n_group * p.width;
  if (parents_meet(p, p.block_table, beams * p.table_width) || parents_meet(p, p.copy_from, beams) ||
      (p.src_slot && (parents_meet(p, p.src_slot, beams) || parents_meet(p, p.dst_slot, beams) ||
                      parents_meet(p, p.spare_slot, beams))))
    return fail(BH_ERR_ARG, "beam_reorder: parent must not be an output");
  ReorderArgs a{p.parent, p.block_table, p.copy_from, p.src_slot, p.dst_slot, p.spare_slot,
                static_cast<int>(p.width), static_cast<int>(p.parent_stride),
                static_cast<int>(p.table_width)};
  BH_LAUNCH(beam_reorder_kernel, static_cast<unsigned>(n), 256, 0, as_stream(stream), a,
            static_cast<int>(parts));
  return ok();
}

namespace bh {
namespace {
template <class T>
int launch_copy(const bh_kv_copy_args &p, hipStream_t st) {
  const bh_paged_cache &c = p.cache;
  const size_t of = sizeof(T) / (c.kv_dtype == BH_KV_F16 ? 2 : 4);  // elements of a piece
  CopyArgs a{};
  a.k = c.k, a.v = c.v, a.table = p.block_table, a.from = p.copy_from;
  a.begin = p.begin, a.end = p.end;
  a.page_stride = c.page_stride / of, a.pos_stride = c.pos_stride / of;
  a.head_stride = c.head_stride / of;
  a.n_req = static_cast<int>(p.n_req), a.width = static_cast<int>(p.table_width);
  a.n_pages = static_cast<int>(c.n_pages);
  a.max_len = static_cast<int>(p.table_width * c.page_size);
  a.hd = static_cast<int>(c.hd / of), a.elems = static_cast<int>(c.n_kv * a.hd);
  a.page = FastDiv(static_cast<uint32_t>(c.page_size));
  a.row = FastDiv(static_cast<uint32_t>(a.elems));
  a.head = FastDiv(static_cast<uint32_t>(a.hd));
  // 64 blocks a compute unit, of which those of requests without a copy are gone at once, or
  // as many as the table's longest could need: blocks that go round twice wait twice.  54 of
  // 128 beams, 255 positions each (117 MB): 8 a unit, 4 pieces a thread 32.2 us; 16 26.3, 32
  // 23.2; 64 and 2 pieces 20.3, 128 and 1 21.2.
  size_t blocks = 64 * device_cu_count() / p.n_req;
  const size_t most = (static_cast<size_t>(a.max_len) * a.elems + 256 * kCopyItems - 1) / (256 * kCopyItems);
  if (blocks > most) blocks = most;
  if (blocks < 1) blocks = 1;
  a.blocks = static_cast<int>(blocks);
  BH_LAUNCH(kv_copy_paged_kernel<T>, static_cast<unsigned>(p.n_req * blocks), 256, 0, st, a);
  return ok();
}
}  // namespace
}  // namespace bh

extern "C" int bh_kv_copy_paged(const bh_kv_copy_args *args, bh_stream stream) {
  if (!args) return fail(BH_ERR_ARG, "kv_copy_paged: null args");
  const bh_kv_copy_args &p = *args;
  const bh_paged_cache &c = p.cache;
  if (int e = check_paged_cache(c, "kv_copy_paged")) return e;
  size_t n;
  if (p.table_width == 0 || !mul_size(p.table_width, c.page_size, &n) || n > 0x7fff0000u)
    return fail(BH_ERR_SHAPE, "kv_copy_paged: table_width * page_size must be 1 .. 2^31 - 65536");
  // (a piece's place from the position of the block's first: below 2^31)
  if (p.n_req > kMostBlocks || c.n_kv * c.hd > 0x7fff0000u)
    return fail(BH_ERR_SHAPE, "kv_copy_paged: size overflow");
  if (p.n_req == 0) return ok();
  if (!p.block_table || !p.copy_from || !p.end)
    return fail(BH_ERR_ARG, "kv_copy_paged: null pointer");
  const size_t esz = c.kv_dtype == BH_KV_F16 ? 2 : 4, of = 16 / esz;
  hipStream_t st = as_stream(stream);
  if (c.hd % of == 0 && (c.page_stride | c.pos_stride | c.head_stride) % of == 0 &&
      aligned16(c.k) && aligned16(c.v))
    return launch_copy<f32x4>(p, st);
  if (esz == 2) return launch_copy<uint16_t>(p, st);
  return launch_copy<float>(p, st);
}
