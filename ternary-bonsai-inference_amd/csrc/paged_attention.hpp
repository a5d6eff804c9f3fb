// Attention over a paged KV cache on the matrix cores: the walk over ragged requests,
// the kernels and their join, for bh_attention_paged and bh_attention_shared.
#pragma once

#include <hip/hip_runtime.h>

#include <string>
#include <type_traits>

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
  FastDiv page, grp;
  // of requests that share a prefix
  const int32_t *group_of, *group_start, *shared_len;
  int n_group;
  struct PrefixOf *prefix;  // [n_group]
  int launch;               // which of the call's
};

// Where the tiles of a group's prefix are: their launch and their first place in it, and
// the group's tokens.  Every call writes every group's: of a group without tiles `n` is 0,
// which only offsets that decrease can leave a request with tokens in.
struct PrefixOf {
  int launch, base, q0, n;
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

// ---- matrix-core path (hd 64, 128, 256) ---------------------------------------

typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef uint16_t u16x4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr float kPUnit = 16384.0f;  // probabilities in f16 stand in units of 2^-14
constexpr float kNoScore = -3.402823466e38f;  // the maximum of scores that are all -inf
// RUNS: units a worker below which a tile has whole runs, and how many workers the tiles'
// further units leave for one of them.
constexpr int kRunUnits = 8, kRunPads = 4;
constexpr int kJoinRows = 8;        // rows of a tile that the waves join at a time

// Where a call's work lies.  A request with n tokens has T = ceil(n group / R) row
// tiles a kv head, and a tile as many units of U positions as its last row sees.
// Tiles t and T - 1 - t together have about the same number for every t (what a
// tile sees grows evenly with t), so they stand side by side in a space of as many
// units as any such pair has, and where a unit lies is found by dividing.  The list
// of all (request, kv head, pair, unit) is cut into equal runs, one a worker.  Of
// the tiles in a run only the first and the last can be cut: their parts go to the
// worker's slots 0 and 1.
//
// SHARED: requests of a group see the same first positions.  The list then begins
// with the groups' prefixes: request g < n_group is the tokens of all requests of
// group g over those positions, every row seeing all of them; request n_group + r is
// the call's request r from where its group's prefix ends.  A row is in a tile of
// each, so no tile is done when its parts are: all leave them, a tile's part at its
// worker's number behind the tile's (along the line either grows from part to part).
// While runs are short, a run that goes on in a second tile, with its q, its table and its
// join, takes half as long again as the others: each tile then has whole runs.
struct Cut {  // a tile, written by the worker of its first part
  int rows;         // 0: it has one part, and its rows are done
  int first, last;  // workers of its parts
  int slot;         // of the first part; the others are in their workers' slots 0
  int row0;         // its first row: (token, head of the group) pairs of the request
  int q0, head;
};
struct SharedCut : Cut {
  int r, tile;  // request, place among the launch's tiles in the line's order
  int group;    // whose prefix its rows see, -1: none
};
template <bool SHARED>
using CutOf = std::conditional_t<SHARED, SharedCut, Cut>;
struct Split {
  int *n_tiles;    // one word
  Cut *cut;        // [most_cut], SHARED: of SharedCut
  uint32_t most_cut;  // tiles that a launch can have
  float *pm, *pl;  // [workers][2][R] running maximum (base 2) and sum
  float *pacc;     // [workers][2][R][hd]
  int workers;
  int over, most;  // requests of more than `over` and up to `most` rows a kv head
};

// x / d; by the 32-bit divide, a tenth of the 64-bit one, where that does.
__device__ __forceinline__ int64_t divide(int64_t x, int64_t d) {
  if ((x | d) >> 32 == 0) return static_cast<uint32_t>(x) / static_cast<uint32_t>(d);
  return x / d;
}
__device__ __forceinline__ int64_t run_begin(int64_t total, int workers, int w) {
  const int64_t base = divide(total, workers), rest = total - base * workers;
  return w * base + (w < rest ? w : rest);
}

// `units` rounded up to runs.
__device__ __forceinline__ int whole_runs(int units, int run) {
  return static_cast<int>(static_cast<uint32_t>(units + run - 1) / static_cast<uint32_t>(run)) * run;
}

// The worker whose run holds unit u.
__device__ __forceinline__ int worker_of(int64_t total, int workers, int64_t u) {
  const int64_t base = divide(total, workers), rest = total - base * workers;
  const int64_t big = rest * (base + 1);
  return static_cast<int>(u < big ? divide(u, base + 1) : rest + divide(u - big, base));
}

// Of SHARED work: its first position; its row of the table, below 0: ~row, and a
// group's prefix.
struct Part_of {
  int first, row, group;  // group: whose prefix ends at `first`, -1: none
};
struct All_of {
  static constexpr int first = 0, row = 0, group = -1;
};
template <bool SHARED>
using Extent = std::conditional_t<SHARED, Part_of, All_of>;

// A request's tiles and units.  COST: a tile's further units, for what it takes before and
// behind its steps.
template <int R, int U, bool SHARED, int COST>
struct Work : Extent<SHARED> {
  using Extent<SHARED>::first;
  using Extent<SHARED>::row;
  using Extent<SHARED>::group;
  int q0, n, len;  // first token, tokens (0: not this launch's), positions
  int tiles, pair, mid;  // units of a pair of tiles; of the one in the middle, or 0
  int64_t head;          // units of a kv head

  // Units of tile t; of a last tile that is not full also as if it were.
  __device__ __forceinline__ int units(const PagedArgs &a, int t, bool full = false) const {
    const int64_t last = (static_cast<int64_t>(t) + 1) * R - 1;
    const int tok = last > 0x7fffffff ? 0x7fffffff : a.grp.div(static_cast<int>(last));
    int64_t sees = static_cast<int64_t>(len) - n + tok + 1;
    if (SHARED && row < 0) sees = len;
    const int64_t seen = (full || sees < len ? sees : len) - first;
    return seen <= U ? 1 : static_cast<int>((seen + U - 1) / U);
  }
  __device__ __forceinline__ void load(const PagedArgs &a, const Split &sp, int r) {
    if constexpr (SHARED) {
      // A group's tokens are its requests'; a request has a prefix where its group names
      // it too and the prefix ends before its tokens.  What either kind reads goes side by
      // side: two loads after one another, not five.
      const bool prefix = r < a.n_group;
      const int own = prefix ? 0 : r - a.n_group;
      const int32_t *const bounds = prefix ? a.group_start + r : a.q_start + own;
      const int from = bounds[0], to = bounds[1], g = a.group_of[own];
      const int have = *(prefix ? a.shared_len + r : a.kv_len + own);
      const bool grouped = !prefix && g >= 0 && g < a.n_group;
      const int r0 = min(max(from, 0), a.n_req), r1 = min(max(to, r0), a.n_req);
      const int32_t *const start = prefix ? a.q_start + r0 : a.group_start + (grouped ? g : 0);
      const int s = start[0], e = start[prefix ? r1 - r0 : 1], of_group = a.shared_len[grouped ? g : 0];
      first = 0, group = -1;
      row = prefix ? ~r0 : own;
      q0 = min(max(prefix ? s : from, 0), a.n_tok);
      n = max(min(max(prefix ? e : to, 0), a.n_tok) - q0, 0);
      len = min(max(have, 0), a.max_len);
      const int shared = min(max(of_group, 0), a.max_len);
      if (grouped && own >= s && own < e && len - n >= shared && shared > 0) first = shared, group = g;
    } else {
      request(a, r, &q0, &n, &len);
    }
    const int64_t rows = static_cast<int64_t>(n) * a.group;
    if (rows <= sp.over || rows > sp.most) n = 0;
    tiles = n == 0 ? 0 : static_cast<int>((rows + R - 1) / R);
    pair = 1, mid = 0;
    // two tiles with as many positions in all, but for a token of rounding, have as
    // many units but for one
    if (tiles > 1) pair = units(a, 0) + units(a, tiles - 1, true) + 1;
    if (tiles & 1) mid = units(a, tiles / 2) + COST;
    pair += 2 * COST;
    head = static_cast<int64_t>(tiles / 2) * pair + mid;
  }
  __device__ __forceinline__ int64_t cost(const PagedArgs &a) const { return head * a.n_kv; }
  // Each tile in whole runs: its units from a multiple of `run` on.  A pair then takes up to
  // 3 (run - 1) units more.
  __device__ __forceinline__ int pads() const { return tiles / 2 * 3 + (tiles & 1); }
  __device__ __forceinline__ void pad(int run) {
    pair = whole_runs(pair - 2 * COST + 2 * (run - 1), run);
    if (mid != 0) mid = whole_runs(mid - COST, run);
    head = static_cast<int64_t>(tiles / 2) * pair + mid;
  }
  // From lane `l`.
  __device__ __forceinline__ void take(int l) {
    q0 = __builtin_amdgcn_readlane(q0, l), n = __builtin_amdgcn_readlane(n, l);
    len = __builtin_amdgcn_readlane(len, l), tiles = __builtin_amdgcn_readlane(tiles, l);
    pair = __builtin_amdgcn_readlane(pair, l), mid = __builtin_amdgcn_readlane(mid, l);
    if constexpr (SHARED)
      first = __builtin_amdgcn_readlane(first, l), row = __builtin_amdgcn_readlane(row, l),
      group = __builtin_amdgcn_readlane(group, l);
    head = static_cast<int64_t>(tiles / 2) * pair + mid;
  }
};

// f16 cache: SUB times 16 positions a step on v_mfma_f32_16x16x32_f16.
//
// S^T = K Q^T: a lane (g = lane / 16, c = lane % 16) loads 16 bytes of position c's
// row (dims 32 kk + 8 g ..) as its A operand, straight from memory; q stands in LDS
// as B operands, split into f16 hi + lo (22 bits) after an exact power of two
// that brings the row's largest to 2^14 .. 2^15.  Lane (g, c) gets the scores of
// row c at positions 16 s + 4 g + i.
// O^T = V^T P^T: with the k index of a lane's 4 SUB slots taken as those same
// positions, its scores are its B operand as they stand (hi + lo), and the A
// operand is what the lane has loaded: its positions by 8 dims, transposed by one
// v_perm a pair.  Row c's output and running state stay with the lanes of c.
// With hd 256 a step is 16 positions: at 32 the accumulators and both tiles take
// 192 of the 256 registers of two waves a SIMD and the rest spills (64 requests
// at 16384 positions: 1222 us, 715 with 16).  Two row tiles of hd 128 take 16 too (24
// caches of 3500, 24 rows: 80 us, 93 with 32).
template <int HD, int RT>
struct EngineF16 {
  using Elem = _Float16;
  static constexpr int SUB = HD >= 256 || (HD == 128 && RT == 2) ? 1 : 2;
  static constexpr int kBlocks = RT == 1 || HD <= 128 ? 2 : 1;  // a compute unit
  static constexpr int kAhead = kBlocks == 2 ? 1 : 3;  // steps of 32 dims whose q is read ahead
  static constexpr int kHd = HD, kRt = RT, kStep = 16 * SUB;
  static constexpr int KK = HD / 32, DV = HD >= 128 ? 8 : 4, NB = HD / (16 * DV);
  static constexpr int kQBytes = RT * KK * 2 * 64 * 16;
  static constexpr int kSlots = 4 * SUB;  // positions of a lane
  static constexpr float kAccUnit = 1.0f / kPUnit;
  typedef _Float16 VVec __attribute__((ext_vector_type(DV)));
  typedef _Float16 PVec __attribute__((ext_vector_type(kSlots)));

  h8 k[SUB][KK];
  VVec v[kSlots][NB];
  f32x4 acc[RT][NB][DV];
  float sc[RT][kSlots];
  PVec phi[RT], plo[RT];

  // Index of a lane's slot j among the positions of a step.
  static __device__ __forceinline__ int pos_of(int g, int j) { return (j & 4) * 4 + 4 * g + (j & 3); }
  static __device__ __forceinline__ f32x4 mma(PVec a, PVec b, f32x4 c) {
    if constexpr (SUB == 2) return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0);
  }

  static __device__ __forceinline__ void store_q(char *lds, int row, int d, float4 x, float up) {
    const int kk = d / 32, g = d % 32 / 8, e = d % 8;
    const f32x4 y = {x.x * up, x.y * up, x.z * up, x.w * up};
    const h4 hi = __builtin_convertvector(y, h4);
    const h4 lo = __builtin_convertvector(y - __builtin_convertvector(hi, f32x4), h4);
    h8 *base = reinterpret_cast<h8 *>(lds) + ((row / 16) * KK + kk) * 128 + g * 16 + row % 16;
    *reinterpret_cast<h4 *>(reinterpret_cast<_Float16 *>(base) + e) = hi;
    *reinterpret_cast<h4 *>(reinterpret_cast<_Float16 *>(base + 64) + e) = lo;
  }
  static constexpr bool kScaleQ = true;

  __device__ __forceinline__ void load_k(const Elem *kc, const int64_t *off, int lane) {
    const int g = lane >> 4, c = lane & 15;
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      const Elem *row = kc + off[16 * s + c] + 8 * g;
#pragma unroll
      for (int kk = 0; kk < KK; ++kk) k[s][kk] = *reinterpret_cast<const h8 *>(row + 32 * kk);
    }
  }
  __device__ __forceinline__ void load_v(const Elem *vc, const int64_t *off, int lane) {
    const int g = lane >> 4, c = lane & 15;
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      const Elem *row = vc + off[pos_of(g, j)] + DV * c;
#pragma unroll
      for (int b = 0; b < NB; ++b) v[j][b] = *reinterpret_cast<const VVec *>(row + 16 * DV * b);
    }
  }
  __device__ __forceinline__ void scores(const char *lds, int lane) {
    const h8 *q = reinterpret_cast<const h8 *>(lds) + lane;
    // one chain for each half of q, summed at the end: the small ones first
    f32x4 sh[RT][SUB], sl[RT][SUB];
    h8 hi[kAhead][RT], lo[kAhead][RT];
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int s = 0; s < SUB; ++s) sh[t][s] = sl[t][s] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int kk = 0; kk < kAhead && kk < KK; ++kk)
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        hi[kk][t] = q[(t * KK + kk) * 128];
        lo[kk][t] = q[(t * KK + kk) * 128 + 64];
      }
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) {
      // operands are read kAhead steps ahead and not earlier: registers are short
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const h8 h = hi[kk % kAhead][t], l = lo[kk % kAhead][t];
        if (kk + kAhead < KK) {
          hi[kk % kAhead][t] = q[(t * KK + kk + kAhead) * 128];
          lo[kk % kAhead][t] = q[(t * KK + kk + kAhead) * 128 + 64];
        }
#pragma unroll
        for (int s = 0; s < SUB; ++s) {
          sh[t][s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[s][kk], h, sh[t][s], 0, 0, 0);
          sl[t][s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[s][kk], l, sl[t][s], 0, 0, 0);
        }
      }
    }
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int s = 0; s < SUB; ++s)
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[t][4 * s + i] = sl[t][s][i] + sh[t][s][i];
  }
  // sc holds the probabilities: their halves.
  __device__ __forceinline__ void split_p(int t) {
#pragma unroll
    for (int j = 0; j < kSlots; ++j) {
      const float x = sc[t][j] * kPUnit;
      phi[t][j] = static_cast<_Float16>(x);
      plo[t][j] = static_cast<_Float16>(x - static_cast<float>(phi[t][j]));
    }
  }
  __device__ __forceinline__ void values() {
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < DV; ++e) {
        if (e % 2 == 0) __builtin_amdgcn_sched_barrier(0);
        PVec x;
#pragma unroll
        for (int j = 0; j < kSlots; ++j) x[j] = v[j][b][e];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          acc[t][b][e] = mma(x, phi[t], acc[t][b][e]);
          acc[t][b][e] = mma(x, plo[t], acc[t][b][e]);
        }
      }
  }
  __device__ __forceinline__ bool finite(int j) const {
    bool bad = false;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < DV; ++e)
        bad |= (__builtin_bit_cast(uint16_t, v[j][b][e]) & 0x7c00u) == 0x7c00u;
    return !bad;
  }
  // One position's values, from memory, with weight p in row c.
  __device__ __forceinline__ void add_value(int t, const Elem *row, float p, int lane) {
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const VVec x = *reinterpret_cast<const VVec *>(row + 16 * DV * b + DV * (4 * (lane >> 4) + i));
#pragma unroll
        for (int e = 0; e < DV; ++e) acc[t][b][e][i] += p * kPUnit * static_cast<float>(x[e]);
      }
  }
  // Lane (g, c) holds dims 16 DV b + DV (4 g + i) + e of row c.
  template <class F>
  __device__ __forceinline__ void each_piece(int t, int lane, F f) const {
    const int g = lane >> 4;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int e = 0; e < DV; e += 4)
          f(16 * DV * b + DV * (4 * g + i) + e,
            f32x4{acc[t][b][e][i], acc[t][b][e + 1][i], acc[t][b][e + 2][i], acc[t][b][e + 3][i]});
  }
  __device__ __forceinline__ void scale_acc(int t, float by) {
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < DV; ++e) acc[t][b][e] *= by;
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < DV; ++e) acc[t][b][e] = f32x4{0, 0, 0, 0};
  }
  __device__ __forceinline__ void drop_value(int j) {
#pragma unroll
    for (int b = 0; b < NB; ++b) v[j][b] = VVec{};
  }
};

// f32 cache: 16 positions a step on v_mfma_f32_16x16x4_f32, products and sums in
// f32, nothing split.  The same scheme: lane (g, c) loads 16 bytes of position
// c's row (dims 16 kk + 4 g ..), gets row c's scores at positions 4 g + i, and
// multiplies them by 4 dims of those positions' values.  Decoders are bound by the
// reads (64 at 8192: 6.2 TB/s, the matrix unit a quarter busy), many rows by that
// instruction and by each wave's wait for its own loads: 512 tokens at 4096 positions
// (24 / 4 heads of 256, 48.3 GFLOP) 493 us, 98 of the 154 TFLOP/s of a large product;
// at 8192 (99.9 GFLOP) 933 us.
template <int HD, int RT>
struct EngineF32 {
  using Elem = float;
  static constexpr int kHd = HD, kRt = RT, kStep = 16;
  static constexpr int kBlocks = RT == 1 || HD <= 128 ? 2 : 1;  // a compute unit
  static constexpr int KK = HD / 16, NB = HD / 64;
  static constexpr int kQBytes = RT * KK * 64 * 16;

  f32x4 k[KK], v[4][NB];
  f32x4 acc[RT][NB][4];
  float sc[RT][4];

  static __device__ __forceinline__ int pos_of(int g, int j) { return 4 * g + j; }
  static __device__ __forceinline__ void store_q(char *lds, int row, int d, float4 x, float) {
    reinterpret_cast<float4 *>(lds)[((row / 16) * KK + d / 16) * 64 + d % 16 / 4 * 16 + row % 16] = x;
  }
  static constexpr bool kScaleQ = false;

  __device__ __forceinline__ void load_k(const Elem *kc, const int64_t *off, int lane) {
    const Elem *row = kc + off[lane & 15] + 4 * (lane >> 4);
#pragma unroll
    for (int kk = 0; kk < KK; ++kk) k[kk] = *reinterpret_cast<const f32x4 *>(row + 16 * kk);
  }
  __device__ __forceinline__ void load_v(const Elem *vc, const int64_t *off, int lane) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const Elem *row = vc + off[pos_of(lane >> 4, j)] + 4 * (lane & 15);
#pragma unroll
      for (int b = 0; b < NB; ++b) v[j][b] = *reinterpret_cast<const f32x4 *>(row + 64 * b);
    }
  }
  __device__ __forceinline__ void scores(const char *lds, int lane) {
    const f32x4 *q = reinterpret_cast<const f32x4 *>(lds) + lane;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      f32x4 s0 = {0, 0, 0, 0}, s1 = {0, 0, 0, 0};  // two chains
      f32x4 an = q[t * KK * 64], bn = q[(t * KK + 1) * 64];
#pragma unroll
      for (int kk = 0; kk < KK; kk += 2) {
        __builtin_amdgcn_sched_barrier(0);
        const f32x4 a = an, b = bn;
        if (kk + 2 < KK) an = q[(t * KK + kk + 2) * 64], bn = q[(t * KK + kk + 3) * 64];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s0 = __builtin_amdgcn_mfma_f32_16x16x4f32(k[kk][e], a[e], s0, 0, 0, 0);
          s1 = __builtin_amdgcn_mfma_f32_16x16x4f32(k[kk + 1][e], b[e], s1, 0, 0, 0);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) sc[t][i] = s0[i] + s1[i];
    }
  }
  __device__ __forceinline__ void split_p(int) {}
  __device__ __forceinline__ void values() {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int t = 0; t < RT; ++t)
            acc[t][b][e] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[j][b][e], sc[t][j], acc[t][b][e],
                                                               0, 0, 0);
  }
  __device__ __forceinline__ bool finite(int j) const {
    bool bad = false;
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        bad |= (__float_as_uint(v[j][b][e]) & 0x7f800000u) == 0x7f800000u;
    return !bad;
  }
  __device__ __forceinline__ void add_value(int t, const Elem *row, float p, int lane) {
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const f32x4 x = *reinterpret_cast<const f32x4 *>(row + 64 * b + 4 * (4 * (lane >> 4) + i));
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][b][e][i] += p * x[e];
      }
  }
  // Lane (g, c) holds dims 64 b + 4 (4 g + i) + e of row c.
  template <class F>
  __device__ __forceinline__ void each_piece(int t, int lane, F f) const {
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < 4; ++i)
        f(64 * b + 4 * (4 * (lane >> 4) + i),
          f32x4{acc[t][b][0][i], acc[t][b][1][i], acc[t][b][2][i], acc[t][b][3][i]});
  }
  __device__ __forceinline__ void scale_acc(int t, float by) {
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[t][b][e] *= by;
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[t][b][e] = f32x4{0, 0, 0, 0};
  }
  static constexpr int kSlots = 4;
  static constexpr float kAccUnit = 1.0f;
  __device__ __forceinline__ void drop_value(int j) {
#pragma unroll
    for (int b = 0; b < NB; ++b) v[j][b] = f32x4{0, 0, 0, 0};
  }
};

// Over the four lanes of a row (lanes c, c + 16, c + 32, c + 48).
template <class Op>
__device__ __forceinline__ float row_lanes(float x, Op op) {
  float lo, hi;
  lane_swap<16>(x, lo, hi);
  x = op(lo, hi);
  lane_swap<32>(x, lo, hi);
  return op(lo, hi);
}

// The cache rows of a step's positions, a lane each: element offsets, and which
// of them the request has.
template <int STEP>
struct Rows {
  int page;  // table entry of the lane's position, -1 past the end
  __device__ __forceinline__ void fetch(const PagedArgs &a, const int32_t *table, int p, int end) {
    page = p < end ? table[a.page.div(p)] : -1;
  }
  // Writes the offsets, returns the mask of valid positions.
  __device__ __forceinline__ uint32_t place(const PagedArgs &a, int64_t *off, int p, int end,
                                            int lane) const {
    const bool in = page >= 0 && page < a.n_pages;
    if (p < end && !in && a.bad_page) *a.bad_page = page;
    const int64_t o = in ? static_cast<int64_t>(page) * static_cast<int64_t>(a.page_stride) +
                               static_cast<int64_t>(a.page.mod(p)) *
                                   static_cast<int64_t>(a.pos_stride)
                         : 0;
    if (lane < STEP) off[lane] = o;
    return static_cast<uint32_t>(__ballot(in)) & (~0u >> (32 - STEP));
  }
};

__device__ __forceinline__ int64_t wave_uniform(int64_t x) {
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(x));
  const uint32_t hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(x >> 32));
  return static_cast<int64_t>(static_cast<uint64_t>(hi) << 32 | lo);
}

// A worker's run, piece by piece.
struct PieceOf {
  int r, q0, n, len;             // request
  int head, tile, units;         // kv head, row tile and its units
  int unit, unit_end;            // those of this piece
  int rows;                      // rows of the tile
  int slot;                      // where a part of a tile goes: [workers][2]
  bool whole;                    // the piece is all of the tile
};
template <bool SHARED>
struct Piece : PieceOf, Extent<SHARED> {};

// RUNS, of SHARED: each tile in whole runs, where the call's sizes are such that it pays.
template <int R, int U, bool SHARED, bool RUNS, int COST>
struct Walk {
  int64_t total, end, at, base, begin;
  int tile_base, r, worker;
  int run;  // RUNS: units of a run that is one tile's; 0: runs are cut anywhere
  Work<R, U, SHARED, COST> work;

  // Every wave finds the run by itself: lane i adds up requests i per .. (i + 1)
  // per - 1, a scan over the lanes gives the total, and the lanes then go through
  // the one lane's requests that hold the run's beginning.
  // Requests that have more tokens together than the call overlap: what they ask for
  // may pass every count here and is bounded by nothing, so such a call does nothing.
  __device__ __forceinline__ void start(const PagedArgs &a, const Split &sp, int lane) {
    worker = blockIdx.x;
    const int n_req = SHARED ? a.n_group + a.n_req : a.n_req;
    const int per = (n_req + 63) / 64;
    int64_t mine = 0;
    int mine_tiles = 0, tokens = 0;  // (n_tok < 2^24: 64 lanes of n_tok + 1 stay below 2^31)
    int prefix_tokens = 0;           // a group's tokens count once more
    // the records of groups without tiles here (a later launch has them, or none)
    const bool records = SHARED && a.launch == 0 && worker == 0 && threadIdx.x < 64;
    for (int i = lane * per; i < min((lane + 1) * per, n_req) && tokens <= a.n_tok &&
                             (!SHARED || prefix_tokens <= a.n_tok); ++i) {
      work.load(a, sp, i);
      mine += work.cost(a);
      mine_tiles += work.tiles * a.n_kv;
      if (SHARED && records && work.row < 0 && work.n == 0) a.prefix[i] = PrefixOf{0, 0, 0, 0};
      if (SHARED && work.row < 0) prefix_tokens = min(prefix_tokens + work.n, a.n_tok + 1);
      else tokens = min(tokens + work.n, a.n_tok + 1);
    }
    int64_t upto = mine;
    int upto_tiles = mine_tiles;
    upto = lane_scan(upto, SumOp{});
    upto_tiles = lane_scan(upto_tiles, SumOp{});
    tokens = lane_scan(tokens, SumOp{});
    total = wave_uniform(__shfl(upto, 63));
    if constexpr (RUNS) {
      run = 0;
      // of n tiles and t units runs of (t - n) / (workers - n) units at most are enough
      const int units = static_cast<int>(min<int64_t>(
          total - static_cast<int64_t>(COST) * __builtin_amdgcn_readlane(upto_tiles, 63), 1 << 30));
      if (per == 1 && units < kRunUnits * sp.workers) {
        const int pads = __builtin_amdgcn_readlane(lane_scan(lane < n_req ? work.pads() * a.n_kv : 0, SumOp{}), 63);
        if (pads > 0 && pads <= sp.workers / kRunPads) {
          run = max((units - pads + sp.workers - pads - 1) / (sp.workers - pads), 1);
          // (a run that is longer by more than a second tile costs pays nothing)
          if (2 * run > 3 * ((units + sp.workers - 1) / sp.workers)) run = 0;
        }
        if (run != 0) {
          if (lane < n_req) {
            work.pad(run);
            mine = work.cost(a);
          }
          upto = lane_scan(mine, SumOp{});
          total = wave_uniform(__shfl(upto, 63));
        }
      }
    }
    if (__builtin_amdgcn_readlane(tokens, 63) > a.n_tok) total = 0, upto_tiles = 0;
    if constexpr (SHARED) {
      prefix_tokens = lane_scan(prefix_tokens, SumOp{});
      if (__builtin_amdgcn_readlane(prefix_tokens, 63) > a.n_tok) total = 0, upto_tiles = 0;
      if (records && total == 0)
        for (int i = lane; i < a.n_group; i += 64) a.prefix[i] = PrefixOf{0, 0, 0, 0};
    }
    if (RUNS && run != 0) {
      at = begin = min<int64_t>(static_cast<int64_t>(worker) * run, total);
      end = worker == sp.workers - 1 ? total : min<int64_t>(begin + run, total);
    } else {
      at = begin = wave_uniform(run_begin(total, sp.workers, worker));
      end = wave_uniform(run_begin(total, sp.workers, worker + 1));
    }
    if (worker == 0 && threadIdx.x == 63) *sp.n_tiles = upto_tiles;
    base = 0, tile_base = 0, r = 0;
    if (begin >= end) {
      work.take(0);
      return;
    }
    int owner = __builtin_ffsll(__ballot(begin < upto)) - 1;
    base = wave_uniform(__shfl(upto - mine, owner));
    tile_base = __builtin_amdgcn_readlane(upto_tiles - mine_tiles, owner);
    r = owner;
    if (per > 1) {
      for (int i = owner * per;; i += 64) {
        mine = 0;
        mine_tiles = 0;
        if (i + lane < min((owner + 1) * per, n_req)) {
          work.load(a, sp, i + lane);
          mine = work.cost(a);
          mine_tiles = work.tiles * a.n_kv;
        }
        upto = mine;
        upto_tiles = mine_tiles;
        upto = lane_scan(upto, SumOp{});
        upto_tiles = lane_scan(upto_tiles, SumOp{});
        upto += base;
        upto_tiles += tile_base;
        const uint64_t past = __ballot(begin < upto);
        if (past) {
          const int at_lane = __builtin_ffsll(past) - 1;
          r = i + at_lane;
          base = wave_uniform(__shfl(upto - mine, at_lane));
          tile_base = __builtin_amdgcn_readlane(upto_tiles - mine_tiles, at_lane);
          owner = at_lane;
          break;
        }
        base = wave_uniform(__shfl(upto, 63));
        tile_base = __builtin_amdgcn_readlane(upto_tiles, 63);
      }
    }
    r = __builtin_amdgcn_readfirstlane(r);
    work.take(owner);
  }

  // The next piece, or false at the run's end.
  __device__ __forceinline__ bool next(const PagedArgs &a, const Split &sp, Piece<SHARED> *p) {
    while (at < end) {
      if (at - base >= work.cost(a)) {  // on to the next request
        base += work.cost(a);
        tile_base += work.tiles * a.n_kv;
        work.load(a, sp, ++r);
        if (RUNS && run != 0) work.pad(run);
        continue;
      }
      const int head = static_cast<int>(divide(at - base, work.head));
      const int64_t in_head = at - base - head * work.head;
      const int pair = static_cast<int>(min<int64_t>(divide(in_head, work.pair), work.tiles / 2));
      int unit = static_cast<int>(in_head - static_cast<int64_t>(pair) * work.pair);
      int tile = work.tiles / 2, units = work.mid;
      if (pair < work.tiles / 2) {  // the longer tile first, then its partner
        tile = work.tiles - 1 - pair;
        units = work.units(a, tile);
        if (unit >= runs_of(units)) {
          unit -= runs_of(units);
          tile = pair;
          const int before = runs_of(units);
          units = work.units(a, tile);
          if (unit >= units) {  // the rest of the pair's space is empty
            at += work.pair - before - unit;
            continue;
          }
        }
      }
      if ((RUNS || COST != 0) && unit >= units) {  // the rest of the tile's part of the line
        at += runs_of(units) - unit;
        continue;
      }
      const int unit_end = static_cast<int>(min<int64_t>(units, unit + (end - at)));
      // all of it is the wave's, and stays in scalars
      *static_cast<PieceOf *>(p) = PieceOf{uni(r), uni(work.q0), uni(work.n), uni(work.len), uni(head), uni(tile), uni(units),
                 uni(unit), uni(unit_end), uni(min(R, work.n * a.group - tile * R)),
                 uni(worker * 2 + (at == begin ? 0 : 1)), uni(unit == 0 && unit_end == units) != 0};
      if constexpr (SHARED) {
        // its place in the line's order, in which a pair's longer tile stands first
        // (whatever the offsets on the device, a place that there is)
        const int nth = 2 * pair + (pair < work.tiles / 2 && tile == pair ? 1 : 0);
        const uint32_t i = static_cast<uint32_t>(tile_base + head * work.tiles + nth);
        p->slot = uni(static_cast<int>(min(i, sp.most_cut - 1)) + worker);
        p->whole = false;
        p->first = uni(work.first), p->row = uni(work.row), p->group = uni(work.group);
        work.first = p->first, work.row = p->row, work.group = p->group;
      }
      at = wave_uniform(at), base = wave_uniform(base), tile_base = uni(tile_base), r = p->r;
      work.q0 = p->q0, work.n = p->n, work.len = p->len, work.tiles = uni(work.tiles);
      work.pair = uni(work.pair), work.mid = uni(work.mid);
      work.head = static_cast<int64_t>(work.tiles / 2) * work.pair + work.mid;
      return true;
    }
    return false;
  }
  // Units of a tile's part of the line.
  __device__ __forceinline__ int runs_of(int units) const {
    return RUNS && run != 0 ? whole_runs(units, run) : units + COST;
  }
  static __device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }

  // The worker of a tile's first part says where its parts are; then past the piece.
  __device__ __forceinline__ void pass(const PagedArgs &a, const Split &sp, const Piece<SHARED> &p) {
    if (p.unit == 0 && threadIdx.x == 0) {
      Cut cut{p.whole ? 0 : p.rows, worker, worker, at == begin ? 0 : 1, p.tile * R, p.q0, p.head};
      if (!p.whole)
        cut.last = RUNS && run != 0
                       ? min(static_cast<int>(divide(at + p.units - 1, run)), sp.workers - 1)
                       : worker_of(total, sp.workers, at + p.units - 1);
      const uint32_t i = static_cast<uint32_t>(tile_base + p.head * work.tiles + p.tile);
      if constexpr (SHARED) {
        if (i < sp.most_cut)
          static_cast<SharedCut *>(sp.cut)[i] = SharedCut{cut, p.r, p.slot - worker, p.group};
        if (p.r < a.n_group && p.head == 0 && p.tile == 0)
          a.prefix[p.r] = PrefixOf{a.launch, tile_base, p.q0, p.n};
      } else {
        if (i < sp.most_cut) sp.cut[i] = cut;
      }
    }
    at += p.unit_end - p.unit;
  }
};

// Within a wave LDS operations are in order; this keeps the compiler to it.
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The waves of a block share its rows and take every fourth step of positions each;
// what they have is joined at the piece's end.  WIDE, for many rows over an f32 cache:
// the waves take rows of their own, 16 RT each, and go through all positions of a piece
// side by side, so that three of the four loads of a K or V row are served by the
// compute unit's own cache.  (Many rows over f16 have attn_paged_wide_kernel.)
template <class E, bool WIDE>
struct Shape {
  static_assert(!WIDE || sizeof(typename E::Elem) == 4, "many rows over f16 have a kernel of their own");
  static constexpr int kWaveRows = 16 * E::kRt, R = kWaveRows * (WIDE ? kWaves : 1);
  static constexpr int kStride = E::kStep * (WIDE ? 1 : kWaves);  // from a wave's step to its next
  static constexpr int U = WIDE ? 128 : kStride;
};

// Of SHARED, whose line holds tiles of hundreds of units and tiles of one or two: without a
// tile's cost the workers of the small ones, nine or so each, are the last to end.  In units,
// which over f16 take half as long.
template <class E>
constexpr int kTileCost = sizeof(typename E::Elem) == 2 ? 2 : 1;

template <class E, bool WIDE, bool SHARED, bool RUNS>
__global__ __launch_bounds__(kThreads, E::kBlocks) void attn_paged_kernel(PagedArgs a, Split sp) {
  using Elem = typename E::Elem;
  using S = Shape<E, WIDE>;
  constexpr int HD = E::kHd, RT = E::kRt, R = S::R, STEP = E::kStep, U = S::U;
  constexpr int kJoinStride = HD + 4, kJoinWave = kJoinRows * kJoinStride * 4;
  constexpr int kJoin = kWaves * kJoinWave, kQ = E::kQBytes * (WIDE ? kWaves : 1);
  constexpr int kLds = kJoin > kQ ? kJoin : kQ;
  static_assert(!WIDE || kJoinWave <= E::kQBytes, "a wave's rows leave through its own part");
  __shared__ __attribute__((aligned(16))) char lds[kLds];
  __shared__ int64_t off_s[kWaves][2][STEP];
  __shared__ float fac_s[R], m_s[kWaves][WIDE ? 1 : R], l_s[kWaves][WIDE ? 1 : R];
  // (read from a lane, so that what follows from the wave branches by scalars)
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, c = lane & 15;

  Walk<R, U, SHARED, RUNS, SHARED && !WIDE ? kTileCost<E> : 0> walk;
  walk.start(a, sp, lane);
  Piece<SHARED> piece;
  while (walk.next(a, sp, &piece)) {
    walk.pass(a, sp, piece);
    const int q0 = piece.q0, n = piece.n, len = piece.len, head = piece.head, tile = piece.tile;
    const bool all = SHARED && piece.row < 0;  // a prefix: every row sees all of it
    const int rows = piece.rows, r = piece.r;
    // this wave's rows
    const int row0 = WIDE ? wave * S::kWaveRows : 0;
    const int my_rows = WIDE ? min(S::kWaveRows, rows - row0) : rows;
    int min_vis = 0, max_vis = 0;
    if (my_rows > 0) {
      min_vis = max(SHARED && all ? len : len - n + a.grp.div(tile * R + row0) + 1, 0);
      max_vis =
          max(SHARED && all ? len : len - n + a.grp.div(tile * R + row0 + my_rows - 1) + 1, 0);
    }
    const int p_first = SHARED ? piece.first : 0;
    const int p_end = min(min(p_first + piece.unit_end * U, len), max_vis);
    const int32_t *table =
        a.table + static_cast<size_t>(SHARED ? max(piece.row, ~piece.row) : r) * a.width;
    const Elem *kc = static_cast<const Elem *>(a.kc) + head * a.head_stride;
    const Elem *vc = static_cast<const Elem *>(a.vc) + head * a.head_stride;

    // the table entries of this wave's first rows and the block's q rows on their
    // way together, then the cache rows, then q into LDS as matrix operands
    int p0 = p_first + piece.unit * U + (WIDE ? 0 : wave * STEP);
    Rows<STEP> rows_of;
    rows_of.fetch(a, table, p0 + lane % STEP, p_end);
    constexpr int kLanes = HD / 4, kAt = kThreads / kLanes;  // lanes of a row, rows at once
    constexpr int kRows = (R + kAt - 1) / kAt;
    const int qd = tid % kLanes * 4;
    E eng;
    uint32_t mask = 0;
    // four rows of a thread at a time: the registers of the cache rows are taken
    constexpr int kBatch = kRows < 4 ? kRows : 4;
#pragma unroll
    for (int x0 = 0; x0 < kRows; x0 += kBatch) {
      float4 qv[kBatch];
#pragma unroll
      for (int x = 0; x < kBatch; ++x) {
        const int i = tid / kLanes + (x0 + x) * kAt, row = tile * R + i, tok = a.grp.div(row);
        qv[x] = make_float4(0, 0, 0, 0);
        if (i < rows)
          qv[x] = *reinterpret_cast<const float4 *>(
              a.q + (static_cast<size_t>(q0 + tok) * a.n_head + head * a.group +
                     (row - tok * a.group)) * HD + qd);
      }
      if (x0 == 0) {
        if (p0 < p_end) {
          mask = rows_of.place(a, off_s[wave][0], p0 + lane % STEP, p_end, lane);
          eng.load_k(kc, off_s[wave][0], lane);
          eng.load_v(vc, off_s[wave][0], lane);
          rows_of.fetch(a, table, p0 + S::kStride + lane % STEP, p_end);
        }
        __syncthreads();  // the piece before has been read
      }
#pragma unroll
      for (int x = 0; x < kBatch; ++x) {
        const int i = tid / kLanes + (x0 + x) * kAt;
        float up = 1.0f, down = a.scale;
        if constexpr (E::kScaleQ) {
          float mx = fmaxf(fmaxf(fabsf(qv[x].x), fabsf(qv[x].y)),
                           fmaxf(fabsf(qv[x].z), fabsf(qv[x].w)));
          mx = lane_group_reduce<kLanes>(mx, MaxOp{});
          int ex = static_cast<int>(__float_as_uint(mx) >> 23) - 127;
          if (ex > -127 && ex < 128) {
            ex = max(ex, -100);
            up = ldexpf(1.0f, 14 - ex);
            down = ldexpf(a.scale, ex - 14);
          }
        }
        if (kRows * kAt == R || i < R) {
          E::store_q(lds + i / S::kWaveRows * E::kQBytes, i % S::kWaveRows, qd, qv[x], up);
          if (qd == 0) fac_s[i] = down * kExpL2E;
        }
      }
    }
    __syncthreads();

    float m[RT], l[RT], fac[RT];
    bool some[RT];  // of this lane's positions the row sees one
    int vis[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int i = row0 + 16 * t + c;
      m[t] = -INFINITY;
      l[t] = 0.0f;
      some[t] = false;
      fac[t] = fac_s[i];
      vis[t] = i < rows ? (SHARED && all ? len : len - n + a.grp.div(tile * R + i) + 1) : 0;
    }
    eng.clear();
    if (p0 < p_end) {
      for (int s = 1;; s ^= 1) {
        const int next = p0 + S::kStride;
        eng.scores(lds + (WIDE ? wave * E::kQBytes : 0), lane);
        uint32_t next_mask = 0;
        if (next < p_end) {
          next_mask = rows_of.place(a, off_s[wave][s], next + lane % STEP, p_end, lane);
          eng.load_k(kc, off_s[wave][s], lane);
          rows_of.fetch(a, table, next + S::kStride + lane % STEP, p_end);
        }
        constexpr uint32_t kAll = ~0u >> (32 - STEP);
        const bool edge = mask != kAll || p0 + STEP > min_vis;
#pragma unroll
        for (int t = 0; t < RT; ++t) {
#pragma unroll
          for (int j = 0; j < E::kSlots; ++j) eng.sc[t][j] *= fac[t];
          if (edge) {
#pragma unroll
            for (int j = 0; j < E::kSlots; ++j) {
              const int o = E::pos_of(g, j);
              const bool sees = p0 + o < vis[t] && (mask >> o & 1);
              if (!sees) eng.sc[t][j] = -INFINITY;
              some[t] |= sees;
            }
          } else {
            some[t] = true;
          }
          if constexpr (E::kScaleQ) {
            // an infinite key times the two halves of q may be inf - inf or 0 inf
            // where the whole product is infinite: such a score is formed again
            bool odd = false;
#pragma unroll
            for (int j = 0; j < E::kSlots; ++j) odd |= eng.sc[t][j] != eng.sc[t][j];
            if (__builtin_expect(__any(odd), false)) {
              const int row = tile * R + row0 + 16 * t + c, tok = a.grp.div(row);
              const float *q = a.q + (static_cast<size_t>(q0 + tok) * a.n_head + head * a.group +
                                      (row - tok * a.group)) * HD;
#pragma unroll
              for (int j = 0; j < E::kSlots; ++j) {
                if (eng.sc[t][j] == eng.sc[t][j] || 16 * t + c >= my_rows) continue;
                const Elem *key = kc + off_s[wave][s ^ 1][E::pos_of(g, j)];
                float dot = 0.0f;
                for (int d = 0; d < HD; ++d) dot += q[d] * static_cast<float>(key[d]);
                eng.sc[t][j] = dot * (a.scale * kExpL2E);
              }
            }
          }
          float top = eng.sc[t][0];
#pragma unroll
          for (int j = 1; j < E::kSlots; ++j) top = fmaxf(top, eng.sc[t][j]);
          top = row_lanes(top, MaxOp{});
          const float now = fmaxf(m[t], top);
          // What is kept moves only when a row's maximum has doubled its weights (512
          // tokens at 4096 over f32: 509 -> 490 us).  The difference of the two is exact where
          // they are near each other; m + 1 is not from 2^24 on, and may round up to m + 2.
          const bool grown = now - m[t] > 1.0f;
          if (__any(grown)) {  // (the other rows stay as they are, bit for bit)
            const float moved = m[t] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[t] - now);
            const float keep = grown ? moved : 1.0f;
            l[t] *= keep;
            eng.scale_acc(t, keep);
            m[t] = grown ? now : m[t];
          }
          // a row that has seen nothing above -inf is measured from 0
          const float ref = m[t] == -INFINITY ? 0.0f : m[t];
#pragma unroll
          for (int j = 0; j < E::kSlots; ++j) {
            eng.sc[t][j] = __builtin_amdgcn_exp2f(eng.sc[t][j] - ref);
            l[t] += eng.sc[t][j];
          }
          eng.split_p(t);
        }
        // A value that is not finite must not meet the zero weights of the rows that
        // do not see it: its position is left out of the product and added to the
        // rows that do.
        uint32_t apart = 0;
        if (edge) {
#pragma unroll
          for (int j = 0; j < E::kSlots; ++j) {
            const int o = E::pos_of(g, j);
            if (!(mask >> o & 1)) eng.drop_value(j);
            if (p0 + STEP > min_vis) {
              const uint64_t bad = __ballot(!eng.finite(j) && p0 + o >= min_vis);
              if (bad >> (16 * g) & 0xffff) eng.drop_value(j);
#pragma unroll
              for (int w = 0; w < 4; ++w)
                if (bad >> (16 * w) & 0xffff) apart |= 1u << E::pos_of(w, j);
            }
          }
        }
        eng.values();
        while (__builtin_expect(apart != 0, false)) {
          const int o = __ffs(apart) - 1;
          apart &= apart - 1;
#pragma unroll
          for (int t = 0; t < RT; ++t) {
            float p = 0.0f;
#pragma unroll
            for (int j = 0; j < E::kSlots; ++j)
              if (E::pos_of(o % 16 / 4, j) == o) p = eng.sc[t][j];
            p = __shfl(p, o % 16 / 4 * 16 + c);
            if (p0 + o < vis[t]) eng.add_value(t, vc + off_s[wave][s ^ 1][o], p, lane);
          }
        }
        if (next >= p_end) break;
        eng.load_v(vc, off_s[wave][s], lane);
        p0 = next;
        mask = next_mask;
      }
    }

#pragma unroll
    for (int t = 0; t < RT; ++t) {
      l[t] = row_lanes(l[t], SumOp{});
      // a row whose every score is -inf is 0 / 0; one that sees nothing keeps -inf
      // as its maximum and is 0
      const float seen = row_lanes(some[t] ? 1.0f : 0.0f, MaxOp{});
      if (m[t] == -INFINITY && seen != 0.0f) m[t] = kNoScore;
    }
    const bool whole = piece.whole;
    const size_t slot = piece.slot;
    if constexpr (WIDE) {
      // through the wave's part of LDS, so that rows leave in whole lines
      float *mine_s = reinterpret_cast<float *>(lds + wave * E::kQBytes);
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const float by = !whole ? 1.0f : m[t] == -INFINITY ? 0.0f : 1.0f / l[t];
        if (!whole && g == 0 && 16 * t + c < my_rows) {
          sp.pm[slot * R + row0 + 16 * t + c] = m[t];
          sp.pl[slot * R + row0 + 16 * t + c] = l[t];
        }
#pragma unroll
        for (int half = 0; half < 16; half += kJoinRows) {
          const int here = min(kJoinRows, my_rows - 16 * t - half);
          if (here <= 0) continue;
          wave_sync();
          if (c >= half && c < half + kJoinRows)
            eng.each_piece(t, lane, [&](int d, f32x4 o) {
              *reinterpret_cast<f32x4 *>(mine_s + (c - half) * kJoinStride + d) = o * by;
            });
          wave_sync();
          for (int i = lane; i < here * (HD / 4); i += 64) {
            const int rr = i / (HD / 4), d = i % (HD / 4) * 4, row = row0 + 16 * t + half + rr;
            const int tok = a.grp.div(tile * R + row);
            float *dst = whole ? a.out + (static_cast<size_t>(q0 + tok) * a.n_head + head * a.group +
                                          (tile * R + row - tok * a.group)) * HD
                               : sp.pacc + (slot * R + row) * HD;
            *reinterpret_cast<f32x4 *>(dst + d) =
                *reinterpret_cast<const f32x4 *>(mine_s + rr * kJoinStride + d);
          }
        }
      }
    } else {
      // the waves' states joined, kJoinRows rows at a time
#pragma unroll
      for (int t = 0; t < RT; ++t)
        if (g == 0) m_s[wave][16 * t + c] = m[t], l_s[wave][16 * t + c] = l[t];
      float *join = reinterpret_cast<float *>(lds);
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int half = 0; half < 16; half += kJoinRows) {
          const int r0 = 16 * t + half;
          if (r0 >= rows) continue;
          __syncthreads();
          if (c >= half && c < half + kJoinRows && 16 * t + c < rows)
            eng.each_piece(t, lane, [&](int d, f32x4 o) {
              *reinterpret_cast<f32x4 *>(join + (wave * kJoinRows + c - half) * kJoinStride + d) = o;
            });
          __syncthreads();
          const int here = min(kJoinRows, rows - r0);
          for (int i = tid; i < here * (HD / 4); i += kThreads) {
            const int rr = i / (HD / 4), d = i % (HD / 4) * 4, row = r0 + rr;
            float top = m_s[0][row];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) top = fmaxf(top, m_s[w][row]);
            const float ref = top == -INFINITY ? 0.0f : top;
            float sum = 0.0f;
            f32x4 o = {0, 0, 0, 0};
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
              const float keep = __builtin_amdgcn_exp2f(m_s[w][row] - ref);
              sum += keep * l_s[w][row];
              o += keep * *reinterpret_cast<const f32x4 *>(join + (w * kJoinRows + rr) * kJoinStride + d);
            }
            if (whole) {
              const int tok = a.grp.div(tile * R + row);
              const float inv = top == -INFINITY ? 0.0f : E::kAccUnit / sum;
              float *dst = a.out + (static_cast<size_t>(q0 + tok) * a.n_head + head * a.group +
                                    (tile * R + row - tok * a.group)) * HD + d;
              *reinterpret_cast<f32x4 *>(dst) = o * inv;
            } else {
              *reinterpret_cast<f32x4 *>(sp.pacc + (slot * R + row) * HD + d) = o * E::kAccUnit;
              if (d == 0) sp.pm[slot * R + row] = top, sp.pl[slot * R + row] = sum;
            }
          }
        }
    }
  }
}

// ---- f16 cache, requests of many rows --------------------------------------------
//
// A block of eight waves of 16 rows goes through the positions of a piece 32 at a
// time.  The block loads a K and a V tile once, into the order in which the waves
// read matrix operands (the same operands as EngineF16's), two buffers of each in
// LDS; a tile is on its way from memory while the one before it is multiplied, and
// is put into LDS beside the next.  q's operands stay in registers.
//
// An operand piece of 16 bytes lies at its lane's place within 1 KB, its place
// among 16 exchanged by an XOR so that the stores of a row's pieces, which are 1 KB
// or 256 bytes apart, fall into different banks.
//
// Measured (24 / 4 heads of 256, us of the call): 512 tokens at 8192 positions (99.9
// GFLOP) 258-288 by the box (347-387 TFLOP/s of useful products, twice that of issued
// ones), at 4096 (48.3) 152, 128 at 8192 103, 2048 from position 0 (51.6) 173-179.  Two waves a SIMD hide about half of the LDS reads and the
// softmax; half of the waves half a step behind the others, to run one's
// exponentials beside the other's products, took the registers past 256 and three
// times as long (at hd 128, where nothing spills, 319 for 265).
constexpr int kWideWaves = 8, kWideThreads = 64 * kWideWaves, kWideRows = 16 * kWideWaves;
constexpr int kWideUnit = 128;

template <int HD, bool SHARED>
__global__ __launch_bounds__(kWideThreads, 2) void attn_paged_wide_kernel(PagedArgs a, Split sp) {
  constexpr int KK = HD / 32, DT = HD / 16, STEP = 32, R = kWideRows, U = kWideUnit;
  constexpr int kTile = STEP * HD;                                   // halves
  constexpr int kPieces = STEP * HD / 8;                             // of K, 16 bytes each
  constexpr int kOwn = (kPieces + kWideThreads - 1) / kWideThreads;  // a thread's
  constexpr int kJoinStride = HD + 4, kOutRows = 4;                  // rows a wave lets out at once
  static_assert(kWideWaves * kOutRows * kJoinStride * 4 <= 4 * kTile * 2, "rows leave through the tiles");
  __shared__ __attribute__((aligned(16))) _Float16 tiles_s[4 * kTile];  // K, K, V, V
  __shared__ int64_t off_s[4][STEP];  // cache rows of a step's positions, four steps in turn
  __shared__ uint32_t mask_s[4];      // which of them the request has
  __shared__ uint32_t apart_s[4];     // those with values that are not finite
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int g = lane >> 4, c = lane & 15;

  Walk<R, U, SHARED, false, 0> walk;
  walk.start(a, sp, lane);
  Piece<SHARED> piece;
  while (walk.next(a, sp, &piece)) {
    walk.pass(a, sp, piece);
    const int q0 = piece.q0, n = piece.n, len = piece.len, head = piece.head, tile = piece.tile;
    const bool all = SHARED && piece.row < 0;  // a prefix: every row sees all of it
    const int rows = piece.rows, row0 = wave * 16, my_rows = min(16, rows - row0);
    // of the block's rows
    const int min_vis = max(SHARED && all ? len : len - n + a.grp.div(tile * R) + 1, 0);
    const int max_vis = max(SHARED && all ? len : len - n + a.grp.div(tile * R + rows - 1) + 1, 0);
    const int p_first = SHARED ? piece.first : 0;
    const int p_beg = p_first + piece.unit * U;
    const int p_end = min(min(p_first + piece.unit_end * U, len), max_vis);
    const int steps = p_beg < p_end ? (p_end - p_beg + STEP - 1) / STEP : 0;
    int my_end = 0;  // positions that a row of this wave sees
    if (my_rows > 0)
      my_end = min(p_end, SHARED && all ? len
                                        : len - n + a.grp.div(tile * R + row0 + my_rows - 1) + 1);
    const int32_t *table =
        a.table + static_cast<size_t>(SHARED ? max(piece.row, ~piece.row) : piece.r) * a.width;
    const _Float16 *kc = static_cast<const _Float16 *>(a.kc) + head * a.head_stride;
    const _Float16 *vc = static_cast<const _Float16 *>(a.vc) + head * a.head_stride;

    // the first three steps' rows; the table entry of the fourth's
    Rows<STEP> entry{-1};
    __syncthreads();  // the piece before is done with LDS
    if (wave == 0) {
      Rows<STEP> e0, e1, e2;
      const int p = p_beg + (lane & 31);
      e0.fetch(a, table, p, p_end);
      e1.fetch(a, table, p + STEP, p_end);
      e2.fetch(a, table, p + 2 * STEP, p_end);
      entry.fetch(a, table, p + 3 * STEP, p_end);
      const uint32_t m0 = e0.place(a, off_s[0], p, p_end, lane);
      const uint32_t m1 = e1.place(a, off_s[1], p + STEP, p_end, lane);
      const uint32_t m2 = e2.place(a, off_s[2], p + 2 * STEP, p_end, lane);
      if (lane < 4) {
        mask_s[lane] = lane == 0 ? m0 : lane == 1 ? m1 : m2;
        apart_s[lane] = 0;
      }
    }
    // q: row c's dims 32 kk + 8 g .. as B operands
    h8 qh[KK], ql[KK];
    float fac;
    int vis;
    {
      const int row = tile * R + row0 + c, tok = a.grp.div(row);
      const bool in = c < my_rows;
      const float *q = a.q + (static_cast<size_t>(q0 + (in ? tok : 0)) * a.n_head + head * a.group +
                              (in ? row - tok * a.group : 0)) * HD + 8 * g;
      f32x4 x[2 * KK];
      float mx = 0.0f;
#pragma unroll
      for (int k = 0; k < 2 * KK; ++k) {
        x[k] = in ? *reinterpret_cast<const f32x4 *>(q + 32 * (k >> 1) + 4 * (k & 1))
                  : f32x4{0, 0, 0, 0};
        mx = fmaxf(mx, fmaxf(fmaxf(fabsf(x[k].x), fabsf(x[k].y)), fmaxf(fabsf(x[k].z), fabsf(x[k].w))));
      }
      mx = row_lanes(mx, MaxOp{});
      float up = 1.0f;
      fac = a.scale * kExpL2E;
      int ex = static_cast<int>(__float_as_uint(mx) >> 23) - 127;
      if (ex > -127 && ex < 128) {
        ex = max(ex, -100);
        up = ldexpf(1.0f, 14 - ex);
        fac = ldexpf(fac, ex - 14);
      }
#pragma unroll
      for (int k = 0; k < KK; ++k)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float y = x[2 * k + (e >> 2)][e & 3] * up;
          qh[k][e] = static_cast<_Float16>(y);
          ql[k][e] = static_cast<_Float16>(y - static_cast<float>(qh[k][e]));
        }
      vis = in ? (SHARED && all ? len : len - n + tok + 1) : 0;
    }
    f32x4 acc[DT];
#pragma unroll
    for (int d = 0; d < DT; ++d) acc[d] = f32x4{0, 0, 0, 0};
    float m = -INFINITY, l = 0.0f;
    bool some = false;

    // a thread's share of a step: K pieces tid + 512 i; V dims 4 dq .. of positions
    // 4 pg .. 4 pg + 3
    const int dq = tid % (HD / 4), pg = tid / (HD / 4);
    h8 kr[kOwn];
    h4 vr[4];
    __syncthreads();
    for (int t = -2; t < steps; ++t) {
      // step t + 1 into LDS, beside step t's products
      if (t >= -1 && t + 1 < steps) {
        const int b = (t + 1) & 1, at = (t + 1) & 3;
        _Float16 *ks = tiles_s + b * kTile, *vs = tiles_s + (2 + b) * kTile;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
          const int x = tid + kWideThreads * i, pos = x / (HD / 8), pc = x % (HD / 8);
          if (kPieces % kWideThreads == 0 || x < kPieces)
            *reinterpret_cast<h8 *>(ks + ((pos / 16 * KK + pc / 4) * 64 + pc % 4 * 16 +
                                          ((pos & 15) ^ (pc & 15))) * 8) = kr[i];
        }
        if (tid < 2 * HD) {
          const uint32_t mask = mask_s[at];
          const int p = p_beg + (t + 1) * STEP;
          if (mask != ~0u || p + STEP > min_vis) {
            // no weight of 0 may meet a value that is not finite: what lies past the
            // end is 0, and where not every row sees a position such elements are
            // left out, to be added to the rows that do
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int o = 4 * pg + k;
              if (!(mask >> o & 1)) vr[k] = h4{0, 0, 0, 0};
              if (p + o >= min_vis) {
                // (on the bits: all ones in the exponent)
                const u16x4 bits = __builtin_bit_cast(u16x4, vr[k]);
                const u16x4 odd = __builtin_bit_cast(u16x4, (bits & uint16_t{0x7c00}) == uint16_t{0x7c00});
                vr[k] = __builtin_bit_cast(h4, bits & ~odd);
                if (odd[0] | odd[1] | odd[2] | odd[3]) atomicOr(&apart_s[at], 1u << o);
              }
            }
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const int d = 4 * dq + e;
            *reinterpret_cast<h4 *>(vs + (d / 16 * 64 + (pg & 3) * 16 + ((d & 15) ^ (d / 16 & 15))) * 8 +
                                    (pg >> 2) * 4) = h4{vr[0][e], vr[1][e], vr[2][e], vr[3][e]};
          }
        }
      }
      // step t + 2 on its way
      if (t + 2 < steps) {
        const int64_t *off = off_s[(t + 2) & 3];
#pragma unroll
        for (int i = 0; i < kOwn; ++i) {
          const int x = tid + kWideThreads * i, pos = x / (HD / 8), pc = x % (HD / 8);
          if (kPieces % kWideThreads == 0 || x < kPieces)
            kr[i] = *reinterpret_cast<const h8 *>(kc + off[pos] + 8 * pc);
        }
        if (tid < 2 * HD) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            vr[k] = *reinterpret_cast<const h4 *>(vc + off[4 * pg + k] + 4 * dq);
        }
      }
      // the rows of step t + 3
      if (t >= 0 && wave == 0 && t + 3 < steps) {
        const int p = p_beg + (t + 3) * STEP + (lane & 31), at = (t + 3) & 3;
        const uint32_t mk = entry.place(a, off_s[at], p, p_end, lane);
        if (lane == 0) mask_s[at] = mk, apart_s[at] = 0;
        entry.fetch(a, table, p + STEP, p_end);
      }
      const int p0 = p_beg + t * STEP;
      if (t >= 0 && p0 < my_end) {
        // places of this lane's pieces, formed from these by an XOR where they are read:
        // kept over the steps they would take 20 registers
        int at_k = (t & 1) * kTile + (g * 16 + (c ^ g)) * 8;
        int at_v = (2 + (t & 1)) * kTile + (g * 16 + c) * 8;
        asm volatile("" : "+v"(at_k), "+v"(at_v));
        const uint32_t mask = mask_s[t & 3];
        // operands are read a group of four ahead of the products, and not farther
        // (hd 128: 240 us for 258 with each group read beside its products)
        h8 ahead[2][4];
        const auto read_k = [&](int grp) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int kk = 2 * grp + (i >> 1);
            ahead[grp & 1][i] = *reinterpret_cast<const h8 *>(
                tiles_s + ((i & 1) * KK + kk) * 512 + (at_k ^ 32 * (kk & 3)));
          }
        };
        const auto read_v = [&](int grp) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int d = 4 * grp + i;
            ahead[grp & 1][i] = *reinterpret_cast<const h8 *>(tiles_s + d * 512 + (at_v ^ 8 * d));
          }
        };
        f32x4 sh[2], sl[2];
        sh[0] = sh[1] = sl[0] = sl[1] = f32x4{0, 0, 0, 0};
        read_k(0);
#pragma unroll
        for (int grp = 0; grp < KK / 2; ++grp) {
          if (grp + 1 < KK / 2) read_k(grp + 1);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int kk = 2 * grp + (i >> 1), s = i & 1;
            sh[s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ahead[grp & 1][i], qh[kk], sh[s], 0, 0, 0);
            sl[s] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ahead[grp & 1][i], ql[kk], sl[s], 0, 0, 0);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        read_v(0);
        float sc[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) sc[j] = (sl[j >> 2][j & 3] + sh[j >> 2][j & 3]) * fac;
        if (mask != ~0u || p0 + STEP > min_vis) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int o = (j >> 2) * 16 + 4 * g + (j & 3);
            const bool sees = p0 + o < vis && (mask >> o & 1);
            if (!sees) sc[j] = -INFINITY;
            some |= sees;
          }
        } else {
          some = true;
        }
        float sum = 0.0f, top = sc[0];
#pragma unroll
        for (int j = 0; j < 8; ++j) sum += sc[j], top = fmaxf(top, sc[j]);
        if (__builtin_expect(__any(sum != sum), false)) {
          // as in attn_paged_kernel: an infinite key against the halves of q (or
          // infinities of both signs, which are formed again to no harm)
          const int row = tile * R + row0 + c, tok = a.grp.div(row);
          const float *q = a.q + (static_cast<size_t>(q0 + tok) * a.n_head + head * a.group +
                                  (row - tok * a.group)) * HD;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (sc[j] == sc[j] || c >= my_rows) continue;
            const _Float16 *key = kc + off_s[t & 3][(j >> 2) * 16 + 4 * g + (j & 3)];
            float dot = 0.0f;
            for (int d = 0; d < HD; ++d) dot += q[d] * static_cast<float>(key[d]);
            sc[j] = dot * (a.scale * kExpL2E);
            top = fmaxf(top, sc[j]);
          }
        }
        top = row_lanes(top, MaxOp{});
        // As in attn_paged_kernel, what is kept moves only when a row's maximum has
        // doubled its weights: they stand in f16 up to 2 kPUnit, and most new maxima are
        // less above the last (512 tokens at 8192 321 -> 312 us).
        const float now = fmaxf(m, top);
        const bool grown = now - m > 1.0f;
        if (__any(grown)) {
          const float moved = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - now);
          const float keep = grown ? moved : 1.0f;
          l *= keep;
#pragma unroll
          for (int d = 0; d < DT; ++d) acc[d] *= keep;
          m = grown ? now : m;
        }
        const float ref = m == -INFINITY ? 0.0f : m;
        h8 ph, pl;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          sc[j] = __builtin_amdgcn_exp2f(sc[j] - ref);
          l += sc[j];
          const float x = sc[j] * kPUnit;
          ph[j] = static_cast<_Float16>(x);
          pl[j] = static_cast<_Float16>(x - static_cast<float>(ph[j]));
        }
#pragma unroll
        for (int grp = 0; grp < DT / 4; ++grp) {
          if (grp + 1 < DT / 4) read_v(grp + 1);
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int d = 4 * grp + i;
            acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ahead[grp & 1][i], ph, acc[d], 0, 0, 0);
            acc[d] = __builtin_amdgcn_mfma_f32_16x16x32_f16(ahead[grp & 1][i], pl, acc[d], 0, 0, 0);
          }
          __builtin_amdgcn_sched_barrier(0);
        }
        uint32_t apart = __builtin_amdgcn_readfirstlane(apart_s[t & 3]);
        while (__builtin_expect(apart != 0, false)) {
          const int o = __ffs(apart) - 1;
          apart &= apart - 1;
          float p = 0.0f;
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if ((j >> 2) * 16 + 4 * (o % 16 / 4) + (j & 3) == o) p = sc[j];
          p = __shfl(p, o % 16 / 4 * 16 + c) * kPUnit;
          const _Float16 *v = vc + off_s[t & 3][o] + 4 * g;
          if (p0 + o < vis) {
#pragma unroll
            for (int d = 0; d < DT; ++d) {
              __builtin_amdgcn_sched_barrier(0);  // (rare: it is not to cost the rest registers)
              const h4 x = *reinterpret_cast<const h4 *>(v + 16 * d);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float y = static_cast<float>(x[i]);
                if (!(fabsf(y) < INFINITY)) acc[d][i] += p * y;
              }
            }
          }
        }
      }
      __syncthreads();
    }

    l = row_lanes(l, SumOp{});
    const float seen = row_lanes(some ? 1.0f : 0.0f, MaxOp{});
    if (m == -INFINITY && seen != 0.0f) m = kNoScore;
    const float by = !piece.whole ? 1.0f / kPUnit : m == -INFINITY ? 0.0f : 1.0f / kPUnit / l;
    const size_t slot = piece.slot;
    if (!piece.whole && g == 0 && c < my_rows) {
      sp.pm[slot * R + row0 + c] = m;
      sp.pl[slot * R + row0 + c] = l;
    }
    // rows leave in whole lines through the wave's part of LDS
    float *mine = reinterpret_cast<float *>(tiles_s) + wave * kOutRows * kJoinStride;
#pragma unroll
    for (int r0 = 0; r0 < 16; r0 += kOutRows) {
      const int here = min(kOutRows, my_rows - r0);
      if (here <= 0) continue;
      wave_sync();
      if (c >= r0 && c < r0 + kOutRows)
#pragma unroll
        for (int d = 0; d < DT; ++d)
          *reinterpret_cast<f32x4 *>(mine + (c - r0) * kJoinStride + 16 * d + 4 * g) = acc[d] * by;
      wave_sync();
      for (int i = lane; i < here * (HD / 4); i += 64) {
        const int rr = i / (HD / 4), d = i % (HD / 4) * 4, row = row0 + r0 + rr;
        const int tok = a.grp.div(tile * R + row);
        float *dst = piece.whole ? a.out + (static_cast<size_t>(q0 + tok) * a.n_head + head * a.group +
                                            (tile * R + row - tok * a.group)) * HD
                                 : sp.pacc + (slot * R + row) * HD;
        *reinterpret_cast<f32x4 *>(dst + d) =
            *reinterpret_cast<const f32x4 *>(mine + rr * kJoinStride + d);
      }
    }
  }
}

// The join of a launch: `share` blocks a tile of `rows` rows.
struct Join {
  Split sp;
  int rows, share;
  unsigned blocks;
};

// Joins the parts of the tiles that more than one worker has, of both launches of a
// call.  16 lanes take 64 dims of a row; of the block's 16 such groups p share a
// row of more than 8 parts, each with every p-th, and the loads of up to 8 a group
// are all issued before the first is needed: one round trip for up to 128 parts,
// and no barrier for up to 8.  (Groups that share from 2 parts on: 21 us for the
// tiles of 128 rows of a chunk of 512 tokens, 12 so, 58 MB read and written.)
template <int HD>
__global__ __launch_bounds__(kThreads) void attn_paged_join_kernel(PagedArgs a, Join one, Join two) {
  constexpr int kAt = kThreads / 16, kSlices = HD / 64, kAhead = 8;
  __shared__ float part[kAt][64], sums[kAt], tops[kAt];
  const bool of_two = blockIdx.x >= one.blocks;
  const unsigned block = blockIdx.x - (of_two ? one.blocks : 0);
  const Split sp = of_two ? two.sp : one.sp;
  const int share = of_two ? two.share : one.share, R = of_two ? two.rows : one.rows;
  const int tile = block / share, tid = threadIdx.x;
  const Cut cut = sp.cut[tile];
  if (tile >= *sp.n_tiles || cut.rows == 0) return;  // (past n_tiles cut holds nothing)
  const int parts = cut.last - cut.first + 1;
  int p = 1;  // groups of a row
  while (kAhead * p < parts && p < kAt) p <<= 1;
  const int group = tid >> 4, mine = group & (p - 1), d = (tid & 15) * 4;
  const int items = cut.rows * kSlices, at_once = kAt / p;
  for (int i0 = (block - tile * share) * at_once; i0 < items; i0 += share * at_once) {
    const int item = i0 + group / p;
    const bool live = item < items;
    const int row = live ? item / kSlices : 0, dim = item % kSlices * 64 + d;
    const auto at = [&](int w) {
      return (static_cast<size_t>(w) * 2 + (w == cut.first ? cut.slot : 0)) * R + row;
    };
    f32x4 ahead[kAhead];
    float pm[kAhead], pl[kAhead];
#pragma unroll
    for (int x = 0; x < kAhead; ++x) {
      // past the last part: the last again, at no weight
      if (x * p >= parts) break;
      const size_t o = at(min(cut.first + mine + x * p, cut.last));
      ahead[x] = *reinterpret_cast<const f32x4 *>(sp.pacc + o * HD + dim);
      pm[x] = sp.pm[o];
      pl[x] = sp.pl[o];
    }
    float top = -INFINITY;
#pragma unroll
    for (int x = 0; x < kAhead; ++x) {
      if (x * p >= parts) break;
      top = fmaxf(top, pm[x]);
    }
    for (int w = cut.first + mine + kAhead * p; w <= cut.last; w += p)
      top = fmaxf(top, sp.pm[at(w)]);
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
      if (x * p >= parts) break;
      if (mine + x * p >= parts) continue;
      const float keep = __builtin_amdgcn_exp2f(pm[x] - ref);
      sum += keep * pl[x];
      o += keep * ahead[x];
    }
#pragma unroll 4
    for (int w = cut.first + mine + kAhead * p; w <= cut.last; w += p) {
      const size_t x = at(w);
      const float keep = __builtin_amdgcn_exp2f(sp.pm[x] - ref);
      sum += keep * sp.pl[x];
      o += keep * *reinterpret_cast<const f32x4 *>(sp.pacc + x * HD + dim);
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

// One launch of the kernel with RT row tiles a wave.
struct Form {
  int rt;
  bool wide;
  int over, most;  // the requests it takes, by rows a kv head
  int blocks;      // a compute unit
  bool runs = false;

  int rows() const { return 16 * rt * (wide ? kWaves : 1); }
  int workers() const { return static_cast<int>(device_cu_count()) * blocks; }
};

size_t align256(size_t n) { return (n + 255) & ~size_t{255}; }

// Tiles that a launch can have at most: requests of over `over` and up to `most`
// rows, n_tok group rows in all.
size_t most_tiles(const PagedArgs &a, const Form &f, size_t n_req) {
  const size_t R = f.rows(), rows = static_cast<size_t>(a.n_tok) * a.group;
  const size_t fit = f.over > a.group ? rows / f.over : static_cast<size_t>(a.n_tok);
  const size_t req = n_req < fit ? n_req : fit;
  const size_t of_one = (static_cast<size_t>(f.most) + R - 1) / R;
  const size_t all = rows / R + req;
  return static_cast<size_t>(a.n_kv) * (req < all / of_one ? req * of_one : all);
}

// SHARED: of the groups' prefixes and of the requests.
template <bool SHARED>
size_t most_tiles(const PagedArgs &a, const Form &f) {
  const size_t own = most_tiles(a, f, a.n_req);
  return SHARED ? own + most_tiles(a, f, a.n_group) : own;
}

// Rows of a launch's parts: two a worker, or one a tile and one a worker.
template <bool SHARED>
size_t part_rows(const PagedArgs &a, const Form &f) {
  return (f.workers() * size_t{2} + (SHARED ? most_tiles<SHARED>(a, f) - f.workers() : 0)) * f.rows();
}

// Workspace: tile count, tiles, maxima, sums, accumulators.
template <bool SHARED>
size_t workspace_of(const PagedArgs &a, const Form &f) {
  const size_t parts = part_rows<SHARED>(a, f);
  return 256 + align256(most_tiles<SHARED>(a, f) * sizeof(CutOf<SHARED>)) + 2 * align256(parts * 4) +
         align256(parts * a.hd * 4);
}

// Where a launch's parts lie in its workspace.
template <bool SHARED>
Split split_of(const PagedArgs &a, const Form &f, char *ws) {
  Split sp{};
  sp.workers = f.workers(), sp.over = f.over, sp.most = f.most;
  const size_t parts = part_rows<SHARED>(a, f);
  sp.n_tiles = reinterpret_cast<int *>(ws);
  ws += 256;
  sp.cut = reinterpret_cast<Cut *>(ws);
  sp.most_cut = static_cast<uint32_t>(most_tiles<SHARED>(a, f));
  ws += align256(sp.most_cut * sizeof(CutOf<SHARED>));
  sp.pm = reinterpret_cast<float *>(ws);
  ws += align256(parts * 4);
  sp.pl = reinterpret_cast<float *>(ws);
  ws += align256(parts * 4);
  sp.pacc = reinterpret_cast<float *>(ws);
  return sp;
}

template <bool SHARED>
Join join_of(const PagedArgs &a, const Form &f, const Split &sp, int unit) {
  Join j{sp, f.rows(), 1, 0};
  if (!SHARED && a.max_len <= unit) return j;  // with one unit a tile nothing is cut
  // a block a (row, 64 dims), as rows of many parts need, while they are not many
  // times what fits the card (4 / 8 / 16 a compute unit: draft 7.4 / 5.6 / 4.9 us,
  // batch 6.6 / 5.4 / 6.5, chunk 11.2 / 12.1 / 12.6)
  const size_t tiles = most_tiles<SHARED>(a, f), R = f.rows(), group = a.group;
  const size_t most = (a.n_tok > 1 ? R : group < R ? group : R) * (a.hd / 64);
  const size_t share = 8 * device_cu_count() / tiles;
  j.share = static_cast<int>(share < 1 ? 1 : share > most ? most : share);
  j.blocks = static_cast<unsigned>(tiles * j.share);
  return j;
}

[[maybe_unused]] int launch_join(const PagedArgs &a, const Join &one, const Join &two, hipStream_t st) {
  const unsigned blocks = one.blocks + two.blocks;
  if (blocks == 0) return BH_OK;
  if (a.hd == 64) BH_LAUNCH(attn_paged_join_kernel<64>, blocks, kThreads, 0, st, a, one, two);
  else if (a.hd == 128) BH_LAUNCH(attn_paged_join_kernel<128>, blocks, kThreads, 0, st, a, one, two);
  else BH_LAUNCH(attn_paged_join_kernel<256>, blocks, kThreads, 0, st, a, one, two);
  return BH_OK;
}

template <class E, bool WIDE, bool SHARED, bool RUNS = false>
int launch(const PagedArgs &a, const Form &f, char *ws, hipStream_t st, Join *join) {
  const Split sp = split_of<SHARED>(a, f, ws);
  BH_LAUNCH((attn_paged_kernel<E, WIDE, SHARED, RUNS>), static_cast<unsigned>(sp.workers), kThreads, 0, st, a, sp);
  *join = join_of<SHARED>(a, f, sp, Shape<E, WIDE>::U);
  return BH_OK;
}

template <int HD, bool SHARED>
int launch_wide(const PagedArgs &a, const Form &f, char *ws, hipStream_t st, Join *join) {
  const Split sp = split_of<SHARED>(a, f, ws);
  BH_LAUNCH((attn_paged_wide_kernel<HD, SHARED>), static_cast<unsigned>(sp.workers), kWideThreads, 0, st, a, sp);
  *join = join_of<SHARED>(a, f, sp, kWideUnit);
  return BH_OK;
}

template <int RT, bool SHARED, bool RUNS = false>
int launch_rt(const PagedArgs &a, bool f16, const Form &f, char *ws, hipStream_t st, Join *join) {
  if (f16) {
    if (a.hd == 64) return launch<EngineF16<64, RT>, false, SHARED, RUNS>(a, f, ws, st, join);
    if (a.hd == 128) return launch<EngineF16<128, RT>, false, SHARED, RUNS>(a, f, ws, st, join);
    return launch<EngineF16<256, RT>, false, SHARED, RUNS>(a, f, ws, st, join);
  }
  if (a.hd == 64) return launch<EngineF32<64, RT>, false, SHARED, RUNS>(a, f, ws, st, join);
  if (a.hd == 128) return launch<EngineF32<128, RT>, false, SHARED, RUNS>(a, f, ws, st, join);
  return launch<EngineF32<256, RT>, false, SHARED, RUNS>(a, f, ws, st, join);
}

template <bool SHARED>
int launch_form(const PagedArgs &a, bool f16, const Form &f, char *ws, hipStream_t st, Join *join) {
  if (f.wide && f16) {
    if (a.hd == 64) return launch_wide<64, SHARED>(a, f, ws, st, join);
    if (a.hd == 128) return launch_wide<128, SHARED>(a, f, ws, st, join);
    return launch_wide<256, SHARED>(a, f, ws, st, join);
  }
  if (f.wide) {
    if (a.hd == 64) return launch<EngineF32<64, 2>, true, SHARED>(a, f, ws, st, join);
    if (a.hd == 128) return launch<EngineF32<128, 2>, true, SHARED>(a, f, ws, st, join);
    return launch<EngineF32<256, 2>, true, SHARED>(a, f, ws, st, join);
  }
  if constexpr (SHARED) {
    if (f.runs && f.rt == 1) return launch_rt<1, SHARED, true>(a, f16, f, ws, st, join);
    if (f.runs) return launch_rt<2, SHARED, true>(a, f16, f, ws, st, join);
  }
  if (f.rt == 1) return launch_rt<1, SHARED>(a, f16, f, ws, st, join);
  return launch_rt<2, SHARED>(a, f16, f, ws, st, join);
}

// Whether a call runs on the matrix cores: rows of whole 16-byte pieces.
bool on_matrix_cores(const bh_attention_paged_args &p) {
  const bh_paged_cache &c = p.cache;
  const size_t piece = c.kv_dtype == BH_KV_F16 ? 8 : 4;
  return (c.hd == 64 || c.hd == 128 || c.hd == 256) && c.page_stride % piece == 0 &&
         c.pos_stride % piece == 0 && c.head_stride % piece == 0 && aligned16(c.k) &&
         aligned16(c.v) && aligned16(p.q) && aligned16(p.out);
}

// The launches of a call, by the most rows a kv head that a request may have.
// Rows past which a request goes to the wide form where there is one.  A prompt of 512 at
// 4096 beside 24 caches of 3500 (hd 256, us), line at 16 / 32 / 64 rows: with 18-30 rows
// each 246-260 / 283-294 / as 32 over f16, 902 / 756-762 over f32; with 48 rows 247 /
// 247 / 329 and 905 / 905 / 861.
constexpr int kWideOver = 32;
int forms_of(const bh_attention_paged_args &p, Form *f) {
  const size_t tokens = p.max_new == 0 || p.max_new > p.n_tok ? p.n_tok : p.max_new;
  const size_t rows = tokens * (p.n_head / p.cache.n_kv);
  constexpr int kAll = 0x7fffffff;
  const int two = p.cache.hd <= 128 ? 2 : 1;  // E::kBlocks of two row tiles
  const int wide = p.cache.kv_dtype == BH_KV_F16 ? 1 : two;
  // 24 caches of 3500, us, hd 256 / 128 / 64 over f16: one row tile and two for up to 16
  // rows 72, 76, 39 and 82, 76, 41; for 24 rows 120, 124, 75 and 87, 80, 42.  Narrow and
  // wide at 48 rows 135, 129, 68 and 135, 178, 137; at 72 rows 176, 169, 92 and 143, 186,
  // 139: the line is hd 256's.  Over f32 264, 256, 144 and 435, 404, 242 at 48; 353, 340,
  // 197 and 442, 411, 245 at 72.
  if (rows <= 64) {
    const int rt = rows <= 16 ? 1 : 2;
    f[0] = Form{rt, false, 0, kAll, rt == 1 ? 2 : two};
    return 1;
  }
  if (p.n_req == 1) {
    f[0] = Form{2, true, 0, kAll, wide};
    return 1;
  }
  f[0] = Form{2, true, kWideOver, kAll, wide};
  f[1] = Form{1, false, 0, kWideOver, 2};
  return 2;
}

// Blocks of a launch: a grid has fewer than 2^32 threads a dimension.
constexpr size_t kMostBlocks = 0xffffff;
static_assert(kMostBlocks * kThreads < (size_t{1} << 32), "");

// Checks the arguments and fills `a`.
int prepare(const bh_attention_paged_args &p, PagedArgs *a, const std::string &who) {
  const bh_paged_cache &c = p.cache;
  if (int e = check_paged_cache(c, who.c_str())) return e;
  if (p.n_head == 0 || p.n_head % c.n_kv != 0)
    return fail(BH_ERR_SHAPE, who + ": n_head " + std::to_string(p.n_head) +
                                  " is not a multiple of n_kv " + std::to_string(c.n_kv));
  if (c.hd > kAnyMaxHd)
    return fail(BH_ERR_SHAPE, who + ": hd " + std::to_string(c.hd) + " above " +
                                  std::to_string(kAnyMaxHd));
  size_t n;
  // (the threads that go through the requests step past the last by a round)
  if (p.n_head > 65535 || p.n_tok > kMostBlocks || p.n_req > 0x7fff0000u ||
      p.n_tok * p.n_head > 0x7fffffffu || !mul_size(p.n_tok, p.n_head * c.hd, sizeof(float), &n) ||
      n > SIZE_MAX / 2)
    return fail(BH_ERR_SHAPE, who + ": size overflow");
  if (p.table_width == 0 || !mul_size(p.table_width, c.page_size, &n) || n > 0x7fff0000u)
    return fail(BH_ERR_SHAPE, who + ": table_width * page_size must be 1 .. 2^31 - 65536");
  if (p.n_tok != 0 && p.n_req != 0) {
    if (!p.q || !p.out || !p.q_start || !p.kv_len || !p.block_table)
      return fail(BH_ERR_ARG, who + ": null pointer");
    if (p.q == p.out) return fail(BH_ERR_ARG, who + ": out must not be q");
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
  a->grp = FastDiv(static_cast<uint32_t>(a->group));
  return BH_OK;
}

}  // namespace
}  // namespace bh
