// The gated delta rule of many requests at once, each with its state in a slot.
//
// Per request, v-head h (q/k head h % h_k) and state row j, with m = M[j]:
//   m *= e^gate;  delta = (v[j] - m.k) beta;  m += k delta;  attn[j] = m.q / sqrt(s).
// A row only ever meets its own delta and the head's q and k, so rows are
// independent; with d_k = m.k and d_q = m.q of the row before the token
//   delta = (v - e^gate d_k) beta,  m' = e^gate m + delta k,
//   m'.q = e^gate d_q + delta (k.q),
// so that both dots come from the old row at once.  Decoding reads and writes the
// states, 2 x 4 h_v s^2 bytes a request, and is bound by that: 48 heads of 128, 64 requests
// 81.7 us, 4.96 TB/s; 8 10.2; one 3.7.
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
  int most;  // requests of more tokens are another launch's
  Ragged rag;
};

// Rows of S floats in registers, S / 8 lanes a row and RPG rows a lane, for as many
// tokens as the request has; the next token's inputs load under the present one.
template <int S, int RPG, int THREADS>
__device__ __forceinline__ void step_rows(const GdnArgs &a, int block) {
  constexpr int L = S / 8, kRows = THREADS / L * RPG, kTiles = S / kRows;
  static_assert(S % kRows == 0, "a block's rows are of one head");
  const int per = a.h_v * kTiles;
  const int r = block / per, rest = block - r * per;
  const int h = rest / kTiles, kh = h % a.h_k;
  const int sub = threadIdx.x % L, j = (rest - h * kTiles) * kRows + threadIdx.x / L * RPG;
  int t0, n, from, to;
  a.rag.tokens_of(r, &t0, &n);
  if (n == 0 || n > a.most) return;
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

template <int S, int RPG>
__global__ __launch_bounds__(kBlock) void gdn_ragged_step_kernel(GdnArgs a) {
  step_rows<S, RPG, kBlock>(a, blockIdx.x);
}

// Any s up to kAnyMaxS and any alignment: a wave a row, 16 of its floats a lane.
__global__ __launch_bounds__(kBlock) void gdn_ragged_any_kernel(GdnArgs a) {
  constexpr int kPer = kAnyMaxS / 64;
  const int rows = a.h_v * a.s, blocks = (rows + 3) / 4;
  const int r = blockIdx.x / blocks, lane = threadIdx.x & 63;
  const int row = (blockIdx.x - r * blocks) * 4 + (threadIdx.x >> 6);
  int t0, n, from, to;
  a.rag.tokens_of(r, &t0, &n);
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

// ---- prompts: chunks of 64 tokens on the matrix cores (s = 64, 128) ------------
//
// (The compact WY form of the product of the tokens' steps, which is published for such
// recurrences.)  Over a chunk with decays a_t = e^gate_t, A_t = a_0 .. a_t, D_ts = A_t / A_s and a
// state row m at its beginning, the tokens' steps unroll to
//   delta = T (v - A (K m)),  T = (I + L)^-1 diag(beta),  L_ts = beta_t D_ts (k_t.k_s), s < t,
//   attn = (A (Q m) + P delta) / sqrt(s),                 P_ts = D_ts (q_t.k_s), s <= t,
//   m' = A_63 m + sum_s e_s delta_s k_s,                  e_s = A_63 / A_s,
// where T, P, A and e are those of a (chunk, v-head), whatever the row.
// gdn_chunk_prep_kernel forms them, all chunks at once; gdn_chunk_walk_kernel takes
// the rows of a state through their chunks.
//
// Products are of f16 matrix instructions, each operand as hi + lo halves (hi hi + hi lo +
// lo hi, a third of the f32 instruction's time) in units of a power of two that brings
// the largest of what shares a unit to 2^14 .. 2^15: a token's row of K and of Q, a row of T
// and of P, a state row, its 64 right sides and deltas.  The halves keep 22 bits of each
// value down to 2^-17 of the largest, and 2^-40 of that one below: both round, by half a step
// of 11 bits each, or of f16's last place.
//
// Operands stand in memory as the instructions take them.  In 16x16x32 lane (lr =
// lane % 16, lg = lane / 16) holds row lr and the 8 of the 32 summed over that are
// 4 lg + i and 16 + 4 lg + i, i < 4.  Those are the places that a result's lane holds of
// its column, so results become operands as they stand.
//
// What that floor may cost: over the dims of a state row it is small beside |m| |k| and
// |m| |q|, as any sum's rounding (m the largest that it has been in the chunk: what a later
// token takes back of it leaves its rounding behind).  Over the tokens of a chunk it is not: a
// value far larger than the others would leave its error in the outputs of tokens before it, or
// in the state when it has decayed.  So the wave that has the rows looks whether each token's
// outputs reach 2^-18 of P's row times the largest delta (or T's largest row times the largest
// right side), and the chunk's part of the state the same; a chunk of which one does not it
// takes its rows through token by token.  64 products of two operands off by 2^-39 of their
// largest are then off by 4e-6 of the result at random.  (The look costs 1 to 4 per cent: a
// prompt of 1500 120.8 us for 116.5, three of 783 to 1172 beside 21 decoders 152.3 for 150.  A
// chunk token by token 55 us, all of them 1430.)  A product over tokens that are not before a
// row's has weights of 0 there, which a value that is not finite would make NaN: where an output
// is NaN the chunk goes token by token too, and where gates are above 0.
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef _Float16 h8 __attribute__((ext_vector_type(8)));

constexpr int kCk = 64;
// Tokens from which a request goes by chunks.  One request of 32 / 48 / 64 / 127 tokens, us:
// 24.3, 24.7, 25.1, 29.2, token by token 17.2, 24.3, 30.8, 63.3; 64 of 32 259 for 317.  (Before
// the look at a chunk's outputs, which adds 0.3.)
constexpr int kCkMin = 48;
constexpr int kCkPlace = 32;          // a chunk's place in the workspace every so many tokens
template <int S>
constexpr int kFragK = kCk * S * 4;              // bytes of K as halves; Q, K transposed
template <int S>
constexpr int kHeadK = 3 * kFragK<S>;            // of a (chunk, q/k head)
constexpr int kFragT = 12 * 64 * 16;             // of T's and P's 16 x 32 tiles to the diagonal
// floats: A k, A q, T's, P's units (0 of a row of 0), e k; A_63, the largest unit of T, that times
// the largest of K
constexpr int kVecs = 5 * kCk + kCk;
constexpr int kHeadV = 2 * kFragT + kVecs * 4;   // of a (chunk, v-head)
constexpr float kGateFloor = -200.0f;            // e^x below this is 0 in f32
constexpr float kUnits = 32768.0f;               // units that a unit's largest value has at most
constexpr float kLeast = 0x1p-18f;
constexpr size_t kMostStride = 0x7fffff;         // floats: a chunk's v within 2^31 bytes
constexpr int kPitch = 68;                       // floats of a row of a 64 x 64 matrix in LDS
constexpr int kVWaves = 3;                       // v-heads prepared side by side

struct GdnChunkArgs {
  GdnArgs g;
  char *ws;      // [slots][h_k kHeadK + h_v kHeadV]
  int slots;     // of chunks
  int walks;     // blocks of the walk
  int xcd;       // the blocks of a q/k head on one die
  int at_once;   // compute units / h_v
  int longs;     // requests of kCkMin tokens or more there can be
  int32_t *todo; // their number; they
};

// Where the chunks of a request begin whose first token is `begin`: from 32 tokens on n
// have ceil(n / 64) <= floor(n / 32), and a floor of a sum is no less than the floors'.
static_assert(kCkMin >= kCkPlace, "");
__device__ __forceinline__ int first_chunk(int begin) { return begin / kCkPlace; }

// The unit of values of which `most` is the largest: x up is its number of units.  (Of
// 0, an infinity or NaN the exponent is 0.)
__device__ __forceinline__ void unit_of(float most, float *up, float *down) {
  const int ex = max(__builtin_amdgcn_frexp_expf(most), -100);
  *up = __builtin_amdgcn_ldexpf(1.0f, 15 - ex);
  *down = __builtin_amdgcn_ldexpf(1.0f, ex - 15);
}
// c + a b
__device__ __forceinline__ f32x4 add_times(f32x4 c, float a, f32x4 b) {
  return f32x4{fmaf(a, b.x, c.x), fmaf(a, b.y, c.y), fmaf(a, b.z, c.z), fmaf(a, b.w, c.w)};
}
__device__ __forceinline__ float most_of(f32x4 x) {
  return fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
}
// Over lanes lr, lr + 16, lr + 32, lr + 48.
__device__ __forceinline__ float most_of_lanes(float x) {
  float lo, hi;
  lane_swap<16>(x, lo, hi);
  x = fmaxf(lo, hi);
  lane_swap<32>(x, lo, hi);
  return fmaxf(lo, hi);
}
// x up as hi + lo halves.
__device__ __forceinline__ void halves(f32x4 x, float up, h4 *hi, h4 *lo) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const _Float16 h = static_cast<_Float16>(x[e] * up);
    (*hi)[e] = h;
    (*lo)[e] = static_cast<_Float16>(fmaf(x[e], up, -static_cast<float>(h)));
  }
}
__device__ __forceinline__ h8 both(h4 a, h4 b) { return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7); }

__device__ __forceinline__ f32x4 mma(h8 a, h8 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma32(h8 ah, h8 al, h8 bh, h8 bl, f32x4 c) {
  c = __builtin_amdgcn_mfma_f32_16x16x32_f16(al, bh, c, 0, 0, 0);
  c = __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, bl, c, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(ah, bh, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma4(float a, float b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0);
}
struct AndOp {
  __device__ __forceinline__ uint32_t operator()(uint32_t a, uint32_t b) const { return a & b; }
};
// Orders the wave's LDS writes before its reads (the wave runs in step).
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}
// What lies at a base in scalars: a lane's place and an offset that all lanes share are 32
// bits each, which saves the vector arithmetic of 64-bit addresses.
struct Base {
  __amdgpu_buffer_rsrc_t of;
  // (what lies past `bytes` reads as 0 and is not written)
  __device__ explicit Base(const void *p, int bytes = 0x7fffffff)
      : of(__builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(p), 0, bytes, 0x00027000)) {}
  __device__ __forceinline__ h8 load(int lane_at, int at) const {
    return __builtin_bit_cast(h8, __builtin_amdgcn_raw_buffer_load_b128(of, lane_at, at, 0));
  }
  __device__ __forceinline__ float load1(int lane_at) const {
    return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(of, lane_at, 0, 0));
  }
  __device__ __forceinline__ void store1(float x, int lane_at) const {
    __builtin_amdgcn_raw_buffer_store_b32(__builtin_bit_cast(unsigned, x), of, lane_at, 0, 0);
  }
};
constexpr uint64_t kOnes = 0x0001000100010001;  // of 16 lanes each
constexpr int kTri[4] = {0, 1, 2, 4};  // 16 x 32 tiles to the diagonal before row i
// A row of up to four 16 x 16 tiles as operands of 32, hi and lo; 0 from tile n on.
__device__ __forceinline__ void store_row(char *out, const f32x4 *x, int n, float up, int lane) {
  h4 hi[4], lo[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    hi[j] = lo[j] = h4{0, 0, 0, 0};
    if (j < n) halves(x[j], up, &hi[j], &lo[j]);
  }
#pragma unroll
  for (int p = 0; 2 * p < n; ++p) {
    h8 *o = reinterpret_cast<h8 *>(out) + p * 128 + lane;
    o[0] = both(hi[2 * p], hi[2 * p + 1]), o[64] = both(lo[2 * p], lo[2 * p + 1]);
  }
}

// What a wave forms for a v-head: `kq` holds Q K^T on and below the diagonal and K K^T,
// transposed, above it; `l` is the wave's own matrix.  down: the units of K's and Q's rows.
__device__ __forceinline__ void prep_head(const GdnArgs &a, int h, int t0, int nt, const float *kq,
                                          float *l, double *G_s, float *w_s, float *b_s,
                                          const float *k_down, const float *q_down, float most_k,
                                          char *out) {
  const int lane = threadIdx.x & 63, lr = lane & 15, lg = lane >> 4;
  // decays: lane t = token t
  float g = 0.0f, beta = 0.0f;
  if (lane < nt) {
    const size_t at = static_cast<size_t>(t0 + lane) * a.h_v + h;
    g = a.gate[at], beta = a.beta[at];
  }
  g = g < kGateFloor ? kGateFloor : g;  // -inf too (a NaN stays)
  double G = g;
#pragma unroll
  for (int d = 1; d < kCk; d <<= 1) {
    const double o = __shfl_up(G, d, kCk);
    if (lane >= d) G += o;
  }
  G_s[lane] = G;
  b_s[lane] = beta;
  const double last = __shfl(G, kCk - 1);
  const double end = __shfl(G, lane | 15);  // of the lane's tile of 16 tokens
  w_s[lane] = exp_hw(static_cast<float>(end - G));
  // (A state that grows would share its units with one far larger: such a chunk's decays are
  // NaN, and it goes token by token.)
  const bool grows = __any(g > 0.0f);
  const float decay = grows ? NAN : expf(static_cast<float>(G)), left = expf(static_cast<float>(last - G));
  float *vec = reinterpret_cast<float *>(out + 2 * kFragT);
  vec[lane] = decay * k_down[lane];
  vec[kCk + lane] = decay * q_down[lane];
  vec[4 * kCk + lane] = left * k_down[lane];
  if (lane == kCk - 1) vec[5 * kCk] = decay;
  wave_sync();
  // P in its order, L into `l`: a tile's D_ts below the diagonal is e^(G_t - G_r)
  // e^(G_r - G_s), r the last token of s's tile: of decays neither factor passes 1.  (All of
  // LDS is read before the first is written: one wait instead of one a tile.)
  f32x4 qk[4][4], kk[4][4];
  double Gt[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = 16 * i + lr;
    Gt[i] = G_s[t];
#pragma unroll
    for (int j = 0; j <= i; ++j) {
      const int s = 16 * j + 4 * lg;
      qk[i][j] = *reinterpret_cast<const f32x4 *>(kq + t * kPitch + s);
#pragma unroll
      for (int e = 0; e < 4; ++e) kk[i][j][e] = kq[(s + e) * kPitch + t];
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int t = 16 * i + lr;
    const float bt = b_s[t];
    f32x4 p[4], lv[4];
    float most = 0.0f;
#pragma unroll
    for (int j = 0; j <= i; ++j) {
      const int s = 16 * j + 4 * lg;
      f32x4 d;
      if (j < i) {
        const float u = exp_hw(static_cast<float>(Gt[i] - G_s[16 * j + 15]));
#pragma unroll
        for (int e = 0; e < 4; ++e) d[e] = u * w_s[s + e];
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float arg = static_cast<float>(Gt[i] - G_s[s + e]);
          d[e] = s + e <= t ? exp_hw(arg) : 0.0f;
        }
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const bool in = j < i || s + e <= t, under = j < i || s + e < t;
        p[j][e] = in ? d[e] * qk[i][j][e] : 0.0f;
        lv[j][e] = under ? bt * d[e] * kk[i][j][e] : 0.0f;
      }
      most = fmaxf(most, most_of(p[j]));
    }
#pragma unroll
    for (int j = 0; j <= i; ++j) *reinterpret_cast<f32x4 *>(l + t * kPitch + 16 * j + 4 * lg) = lv[j];
    float up, down;
    most = most_of_lanes(most);
    unit_of(most, &up, &down);
    store_row(out + kFragT + kTri[i] * 2048, p, i + 1, up, lane);
    if (lg == 0) vec[3 * kCk + t] = most == 0.0f ? 0.0f : down;
  }
  wave_sync();
  // (I + L)^-1: its diagonal blocks by substitution, lane (lr, lg) column lr of block lg
  float x[16];
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    f32x4 row[4];
#pragma unroll
    for (int c = 0; c < 4; ++c)
      if (4 * c < r) row[c] = *reinterpret_cast<const f32x4 *>(l + (16 * lg + r) * kPitch + 16 * lg + 4 * c);
    float v = r == lr ? 1.0f : 0.0f;
#pragma unroll
    for (int c = 0; c < r; ++c) v = fmaf(-row[c / 4][c % 4], x[c], v);
    x[r] = v;
  }
  wave_sync();
#pragma unroll
  for (int r = 0; r < 16; ++r) l[(16 * lg + r) * kPitch + 16 * lg + lr] = x[r];
  wave_sync();
  // the blocks below by their distance: T_ij = -T_ii sum_(j <= m < i) L_im T_mj.  The k
  // index of step e in lane lg is 4 lg + e, which is what a result's lane holds.
  f32x4 inv[4][4], diag[4];  // results' lanes: row 4 lg + e, column lr; rows of T_ii
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    diag[i] = *reinterpret_cast<const f32x4 *>(l + (16 * i + lr) * kPitch + 16 * i + 4 * lg);
#pragma unroll
    for (int e = 0; e < 4; ++e) inv[i][i][e] = l[(16 * i + 4 * lg + e) * kPitch + 16 * i + lr];
  }
#pragma unroll
  for (int dist = 1; dist < 4; ++dist)
#pragma unroll
    for (int j = 0; j + dist < 4; ++j) {
      const int i = j + dist;
      f32x4 sum = {0, 0, 0, 0}, t = {0, 0, 0, 0};
#pragma unroll
      for (int m = j; m < i; ++m) {
        const f32x4 lm = *reinterpret_cast<const f32x4 *>(l + (16 * i + lr) * kPitch + 16 * m + 4 * lg);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum = mma4(lm[e], inv[m][j][e], sum);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) t = mma4(diag[i][e], sum[e], t);
      inv[i][j] = -t;
    }
  wave_sync();
  // T = (I + L)^-1 diag(beta), by rows through `l`
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j <= i; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        l[(16 * i + 4 * lg + e) * kPitch + 16 * j + lr] = inv[i][j][e] * b_s[16 * j + lr];
  wave_sync();
  float of_t = 0.0f;  // the largest unit
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f32x4 t[4];
    float most = 0.0f, up, down;
#pragma unroll
    for (int j = 0; j <= i; ++j) {
      t[j] = *reinterpret_cast<const f32x4 *>(l + (16 * i + lr) * kPitch + 16 * j + 4 * lg);
      most = fmaxf(most, most_of(t[j]));
    }
    most = most_of_lanes(most);
    unit_of(most, &up, &down);
    store_row(out + kTri[i] * 2048, t, i + 1, up, lane);
    if (most == 0.0f) down = 0.0f;
    if (lg == 0) vec[2 * kCk + 16 * i + lr] = down;
    of_t = fmaxf(of_t, down);
  }
  of_t = lane_group_reduce<16>(of_t, MaxOp{});
  if (lane == 0) vec[5 * kCk + 1] = of_t, vec[5 * kCk + 2] = of_t * most_k;
  wave_sync();
}

// The requests of kCkMin tokens or more, the longest first where a wave holds them all.
// (At most `longs`: of offsets that decrease there may be more.)
__device__ __forceinline__ void list_long(const Ragged &rag, int longs, int32_t *todo) {
  const int lane = threadIdx.x & 63;
  const auto tokens = [&](int r) {
    int begin, n;
    rag.tokens(r, &begin, &n);
    return n;
  };
  int count = 0, own = -1;  // own: the lane-th of them
  for (int i0 = 0; i0 < rag.n_req; i0 += 64) {
    const uint64_t is = __ballot(i0 + lane < rag.n_req && tokens(min(i0 + lane, rag.n_req - 1)) >= kCkMin);
    const int at = count + __popcll(is & ((uint64_t{1} << lane) - 1));
    if ((is >> lane & 1) && at < longs) todo[1 + at] = i0 + lane;
    uint64_t left = is;
    for (int k = count; k <= lane && left != 0; ++k, left &= left - 1)
      if (k == lane) own = i0 + __builtin_ffsll(left) - 1;
    count += __popcll(is);
  }
  count = min(count, longs);
  if (lane == 0) todo[0] = count;
  if (count > 64) return;
  if (lane >= count) own = -1;
  const int n = own >= 0 ? tokens(own) : 0;
  int rank = 0;
  for (int k = 0; k < count; ++k) {
    const int of = __builtin_amdgcn_readlane(n, k);
    rank += of > n || (of == n && k < lane);
  }
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");  // behind the first writes
  if (own >= 0) todo[1 + rank] = own;
}

// Block (chunk, q/k head): wave w has the tokens 16 w .. 16 w + 15.
// Bound by the chain of small products and LDS trips that a wave takes a v-head through,
// 16 us for a chunk, two blocks a compute unit by LDS: 47 chunks of 16 / 48 heads 48 us on
// inputs of the call before, 56 on others, of which writing 134 MB is 27.
template <int S>
__global__ __launch_bounds__(kBlock, 2) void gdn_chunk_prep_kernel(GdnChunkArgs c) {
  constexpr int kMat = kCk * kPitch, N = S / 32;  // N: of 32 dims
  // K's halves; then the v-heads' matrices.  Behind them Q K^T and K K^T.
  __shared__ __attribute__((aligned(16))) float lds[kVWaves * kMat + kMat];
  static_assert(kVWaves * kMat * 4 >= kFragK<S>, "K's halves fit");
  __shared__ double G_s[kVWaves][kCk];
  __shared__ float w_s[kVWaves][kCk], b_s[kVWaves][kCk], k_down[kCk], q_down[kCk];
  const GdnArgs &a = c.g;
  const int slot = blockIdx.x / a.h_k, kh = blockIdx.x - slot * a.h_k;
  if (blockIdx.x == gridDim.x - 1 && threadIdx.x < 64) list_long(a.rag, c.longs, c.todo);
  const int r = last_request(a.rag.n_req, [&](int i) {
    return first_chunk(min(max(a.rag.q_start[i], 0), a.rag.n_tok)) <= slot;
  });
  if (r < 0) return;
  int begin, n;
  a.rag.tokens_of(r, &begin, &n);
  const int at = (slot - first_chunk(begin)) * kCk;
  if (n < kCkMin || at >= n) return;
  const int t0 = begin + at, nt = min(kCk, n - at);
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int lr = lane & 15, lg = lane >> 4;
  char *of_slot = c.ws + static_cast<size_t>(slot) * (static_cast<size_t>(a.h_k) * kHeadK<S> + static_cast<size_t>(a.h_v) * kHeadV);
  char *out = of_slot + static_cast<size_t>(kh) * kHeadK<S>;
  float *kq = lds + kVWaves * kMat;
  h8 *k_lds = reinterpret_cast<h8 *>(lds);

  // K and Q of the wave's tokens as halves
  h8 qh[N], ql[N], kh_[N], kl[N];
  {
    const int t = 16 * w + lr;
    const bool in = t < nt;
    const size_t row = static_cast<size_t>(t0 + (in ? t : 0));
    const float *kp = a.k + row * a.k_stride + static_cast<size_t>(kh) * S + 4 * lg;
    const float *qp = a.q + row * a.q_stride + static_cast<size_t>(kh) * S + 4 * lg;
    f32x4 kv[2 * N], qv[2 * N];
    float km = 0.0f, qm = 0.0f;
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) {
      kv[i] = in ? *reinterpret_cast<const f32x4 *>(kp + 16 * i) : f32x4{0, 0, 0, 0};
      qv[i] = in ? *reinterpret_cast<const f32x4 *>(qp + 16 * i) : f32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) km = fmaxf(km, most_of(kv[i])), qm = fmaxf(qm, most_of(qv[i]));
    float ku, kd, qu, qd;
    unit_of(most_of_lanes(km), &ku, &kd);
    unit_of(most_of_lanes(qm), &qu, &qd);
    if (lg == 0) k_down[t] = kd, q_down[t] = qd;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      h4 h0, l0, h1, l1;
      halves(kv[2 * i], ku, &h0, &l0);
      halves(kv[2 * i + 1], ku, &h1, &l1);
      kh_[i] = both(h0, h1), kl[i] = both(l0, l1);
      halves(qv[2 * i], qu, &h0, &l0);
      halves(qv[2 * i + 1], qu, &h1, &l1);
      qh[i] = both(h0, h1), ql[i] = both(l0, l1);
      const int f = (w * N + i) * 128 + lane;  // of 16 bytes: hi, and lo 64 places on
      k_lds[f] = kh_[i], k_lds[f + 64] = kl[i];
      h8 *ko = reinterpret_cast<h8 *>(out) + f, *qo = reinterpret_cast<h8 *>(out + kFragK<S>) + f;
      ko[0] = kh_[i], ko[64] = kl[i];
      qo[0] = qh[i], qo[64] = ql[i];
    }
  }
  __syncthreads();
  // Q K^T and K K^T of the wave's tokens against those before: a row of one operand is a
  // column of the other, in the same lanes
  h8 of_j[2][2 * N];
  const auto read = [&](int j) {
#pragma unroll
    for (int i = 0; i < 2 * N; ++i) of_j[j & 1][i] = k_lds[(j * N + (i >> 1)) * 128 + 64 * (i & 1) + lane];
  };
  read(0);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (j > w) break;
    if (j + 1 < 4) read(j + 1);
    f32x4 kk[2], qk[2];  // two chains each
#pragma unroll
    for (int x = 0; x < 2; ++x) kk[x] = qk[x] = f32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      kk[i & 1] = mma32(kh_[i], kl[i], of_j[j & 1][2 * i], of_j[j & 1][2 * i + 1], kk[i & 1]);
      qk[i & 1] = mma32(qh[i], ql[i], of_j[j & 1][2 * i], of_j[j & 1][2 * i + 1], qk[i & 1]);
    }
    const int s = 16 * j + lr;  // column
    const float ds = k_down[s];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int t = 16 * w + 4 * lg + e;
      if (s <= t) kq[t * kPitch + s] = (qk[0][e] + qk[1][e]) * q_down[t] * ds;
      if (s < t) kq[s * kPitch + t] = (kk[0][e] + kk[1][e]) * k_down[t] * ds;
    }
  }
  // K transposed: tile (d, p) of 16 dims and 32 tokens, lane's dim 16 d + lr
  {
    const _Float16 *halves_of = reinterpret_cast<const _Float16 *>(lds);
#pragma unroll
    for (int x = 0; x < N; ++x) {
      const int d = N / 2 * w + (x >> 1), p = x & 1;  // wave w: dims 8 N w .. 8 N (w + 1) - 1
      const int dim = 16 * (d & 1) + lr;         // of 32
      const int in = (dim >> 4) * 4 + (dim & 3), group = (dim >> 2) & 3;
      h8 hi, lo;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int t = 2 * p + (e >> 2);
        const int f = ((t * N + (d >> 1)) * 128 + 4 * lg + (e & 3) + 16 * group) * 8 + in;
        hi[e] = halves_of[f], lo[e] = halves_of[f + 64 * 8];
      }
      h8 *o = reinterpret_cast<h8 *>(out + 2 * kFragK<S>) + (d * 2 + p) * 128 + lane;
      o[0] = hi, o[64] = lo;
    }
  }
  __syncthreads();
  if (w >= kVWaves) return;  // (no barrier follows)
  const float most_k = lane_group_reduce<64>(k_down[lane], MaxOp{});
  const int heads = (a.h_v - kh + a.h_k - 1) / a.h_k;  // v-heads kh + i h_k
  for (int i = w; i < heads; i += kVWaves) {
    const int h = kh + i * a.h_k;
    prep_head(a, h, t0, nt, kq, lds + w * kMat, G_s[w], w_s[w], b_s[w], k_down, q_down, most_k,
              of_slot + static_cast<size_t>(a.h_k) * kHeadK<S> + static_cast<size_t>(h) * kHeadV);
  }
}

// The walk.  A wave has 16 state rows to itself and takes them through the chunks in
// registers: every result is the next product's operand as it stands.  The operands that
// the waves share stand in LDS, K and Q apart from K transposed, T and P, so that each
// part of the next chunk comes in while the other is read: two barriers a chunk.
// Three prompts of 1536 tokens, 16 / 48 heads of 128: 183 us, one 100.

// Operands of a chunk in LDS: K, Q; K transposed, T, P; their vectors, of two chunks in
// turn.
template <int S>
constexpr int kA = 2 * kFragK<S> / 16;  // pieces of 16 bytes
template <int S>
constexpr int kB = (kFragK<S> + 2 * kFragT) / 16;
template <int S>
struct ChunkLds {
  h8 kq[kA<S>], u[kB<S>];
  float vec[2][kVecs];
};
struct WalkOf {
  int begin, n, from, to;  // a request's tokens and slots
  int h, row;              // v-head; a wave's first state row
  const char *ws_k, *ws_v;
  size_t slot_bytes;
};

// Pieces on their way to LDS: one is stored and the next chunk's loaded in its place.
// THREADS threads do it, of which this is number tid.
template <int S, int THREADS>
struct Stage {
  static constexpr int kAs = kA<S> / THREADS, kBk = kFragK<S> / 16 / THREADS, kBt = 2 * kFragT / 16 / THREADS;
  static_assert(kAs * THREADS == kA<S> && (kBk + kBt) * THREADS == kB<S>, "whole pieces a thread");
  h8 in_a[kAs], in_b[kBk + kBt];
  f32x4 in_vec;
  int tid, vec_i;
  __device__ __forceinline__ void load_a(const Base &k, int i) { in_a[i] = k.load(16 * tid, i * THREADS * 16); }
  __device__ __forceinline__ void load_b(const Base &k, const Base &v, int i) {
    in_b[i] = i < kBk ? k.load(16 * tid, 2 * kFragK<S> + i * THREADS * 16) : v.load(16 * tid, (i - kBk) * THREADS * 16);
  }
  __device__ __forceinline__ void load_vec(const Base &v) {
    in_vec = __builtin_bit_cast(f32x4, v.load(16 * vec_i, 2 * kFragT));
  }
  // The first chunk's, and the second's A on its way.
  __device__ __forceinline__ void begin(ChunkLds<S> &lds, const WalkOf &o, int chunks, int thread) {
    tid = thread, vec_i = min(tid, kVecs / 4 - 1);  // (the last ones the same)
    const Base k(o.ws_k), v(o.ws_v), k1(chunks > 1 ? o.ws_k + o.slot_bytes : o.ws_k);
#pragma unroll
    for (int i = 0; i < kAs; ++i) load_a(k, i);
#pragma unroll
    for (int i = 0; i < kBk + kBt; ++i) load_b(k, v, i);
    load_vec(v);
#pragma unroll
    for (int i = 0; i < kAs; ++i) {
      lds.kq[i * THREADS + tid] = in_a[i];
      load_a(k1, i);
    }
  }
  // A part of the next chunk's A (and the one's after it on its way), of this chunk's B.
  __device__ __forceinline__ void a(ChunkLds<S> &lds, const Base &after_k, int part, int parts) {
#pragma unroll
    for (int i = kAs * part / parts; i < kAs * (part + 1) / parts; ++i) {
      lds.kq[i * THREADS + tid] = in_a[i];
      load_a(after_k, i);
    }
  }
  __device__ __forceinline__ void b(ChunkLds<S> &lds, const Base &next_k, const Base &next_v, int part, int parts) {
#pragma unroll
    for (int i = (kBk + kBt) * part / parts; i < (kBk + kBt) * (part + 1) / parts; ++i) {
      lds.u[i * THREADS + tid] = in_b[i];
      load_b(next_k, next_v, i);
    }
  }
  __device__ __forceinline__ void vec(ChunkLds<S> &lds, const Base &next_v, int chunk) {
    reinterpret_cast<f32x4 *>(lds.vec[chunk & 1])[vec_i] = in_vec;
    load_vec(next_v);
  }
};

// Sum over lanes lr, lr + 16, lr + 32, lr + 48.
__device__ __forceinline__ float sum_of_lanes(float x) {
  float lo, hi;
  lane_swap<16>(x, lo, hi);
  x = lo + hi;
  lane_swap<32>(x, lo, hi);
  return lo + hi;
}

// n tokens of a request one by one; m as walk_rows has it.
template <int S>
__device__ __forceinline__ void walk_tokens(const GdnArgs &a, const WalkOf &of, int begin, int n,
                                            f32x4 (&m)[S / 16]) {
  const int lane = threadIdx.x & 63, lr = lane & 15, lg = lane >> 4;
  for (int t = begin; t < begin + n; ++t) {
    const size_t at = static_cast<size_t>(of.h % a.h_k) * S + 4 * lg;
    const float *kp = a.k + t * a.k_stride + at, *qp = a.q + t * a.q_stride + at;
    const size_t row = static_cast<size_t>(of.h) * S + of.row + lr, head = static_cast<size_t>(t) * a.h_v + of.h;
    const float eg = expf(a.gate[head]);
    float dk = 0.0f, dq = 0.0f, kq = 0.0f;
#pragma unroll
    for (int d = 0; d < S / 16; ++d) {
      const f32x4 k = *reinterpret_cast<const f32x4 *>(kp + 16 * d), q = *reinterpret_cast<const f32x4 *>(qp + 16 * d);
#pragma unroll
      for (int e = 0; e < 4; ++e)
        dk = fmaf(m[d][e], k[e], dk), dq = fmaf(m[d][e], q[e], dq), kq = fmaf(k[e], q[e], kq);
    }
    dk = sum_of_lanes(dk), dq = sum_of_lanes(dq), kq = sum_of_lanes(kq);
    const float delta = fmaf(-eg, dk, a.v[t * a.v_stride + row]) * a.beta[head];
#pragma unroll
    for (int d = 0; d < S / 16; ++d) {
      const f32x4 k = *reinterpret_cast<const f32x4 *>(kp + 16 * d);
#pragma unroll
      for (int e = 0; e < 4; ++e) m[d][e] = fmaf(k[e], delta, eg * m[d][e]);
    }
    if (lg == 0) a.attn[static_cast<size_t>(t) * a.h_v * S + row] = fmaf(eg, dq, delta * kq) * a.scale;
  }
}

// A wave's 16 rows through the chunks.  SHARES: it stages its part of the operands too.
template <int S, bool SHARES>
__device__ __forceinline__ void walk_rows(const GdnArgs &a, ChunkLds<S> &lds, const WalkOf &of) {
  const int begin = of.begin, n = of.n;
  const char *ws_k = of.ws_k, *ws_v = of.ws_v;
  const size_t slot_bytes = of.slot_bytes;
  const int lane = threadIdx.x & 63, lr = lane & 15, lg = lane >> 4;
  constexpr int N = S / 32;  // of 32 dims
  const int chunks = (n + kCk - 1) / kCk;
  Stage<S, 512> stage;
  if constexpr (SHARES) stage.begin(lds, of, chunks, threadIdx.x);
  // m[d]: state row lr of the wave's, dims 16 d + 4 lg ..
  const int row_w = of.h * S + of.row;
  const size_t m_at = (static_cast<size_t>(row_w) + lr) * S + 4 * lg;
  f32x4 m[2 * N];
#pragma unroll
  for (int d = 0; d < S / 16; ++d)
    m[d] = of.from >= 0 ? *reinterpret_cast<const f32x4 *>(a.state + of.from * a.rag.slot_stride + m_at + 16 * d)
                        : f32x4{0, 0, 0, 0};
  // v and outputs: tokens 16 t + 4 lg + e
  const int v_stride = 4 * static_cast<int>(a.v_stride), o_stride = 4 * a.h_v * S;
  const float *vp = a.v + static_cast<size_t>(begin) * a.v_stride + row_w;
  float *op = a.attn + static_cast<size_t>(begin) * a.h_v * S + row_w;
  const int v_at = 4 * lg * v_stride + 4 * lr, o_at = 4 * lg * o_stride + 4 * lr;
  f32x4 v[4];
  const auto load_v = [&](const Base &of, int t) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[t][e] = of.load1(v_at + (16 * t + e) * v_stride);
  };
  // 32 or 64 of a lane's values as operands, in units of a power of two
  const auto unit = [&](float most, float *up, float *down) { unit_of(most_of_lanes(most), up, down); };
  const auto pair = [](f32x4 x, f32x4 y, float up, h8 *hi, h8 *lo) {
    h4 h0, l0, h1, l1;
    halves(x, up, &h0, &l0);
    halves(y, up, &h1, &l1);
    *hi = both(h0, h1), *lo = both(l0, l1);
  };
  const auto most4 = [](const f32x4 *x) {
    return fmaxf(fmaxf(most_of(x[0]), most_of(x[1])), fmaxf(most_of(x[2]), most_of(x[3])));
  };
  const h8 *k_at = lds.kq + lane, *u_at = lds.u + lane;
  {
    const Base rows(vp, min(n, kCk) * v_stride);
#pragma unroll
    for (int t = 0; t < 4; ++t) load_v(rows, t);
  }
  for (int chunk = 0; chunk < chunks; ++chunk) {
    const int left = n - chunk * kCk;
    // the chunks whose pieces load now (past the last: the last again, read by nobody)
    const int ahead = min(chunks - 1 - chunk, 2);
    const Base next_k(ws_k + min(ahead, 1) * slot_bytes), next_v(ws_v + min(ahead, 1) * slot_bytes);
    const Base after_k(ws_k + ahead * slot_bytes);
    const float *vec = lds.vec[chunk & 1];
    const auto of_token = [&](int i, int t) {
      return *reinterpret_cast<const f32x4 *>(vec + i * kCk + 16 * t + 4 * lg);
    };
    const auto stage_a = [&](int part, int parts) {
      if constexpr (SHARES) stage.a(lds, after_k, part, parts);
    };
    const auto stage_b = [&](int part, int parts) {
      if constexpr (SHARES) stage.b(lds, next_k, next_v, part, parts);
    };
    float up, m_down;
    h8 mh[N], ml[N];
    unit(fmaxf(most4(m), most4(m + 2 * N - 4)), &up, &m_down);
#pragma unroll
    for (int i = 0; i < N; ++i) pair(m[2 * i], m[2 * i + 1], up, &mh[i], &ml[i]);
    __syncthreads();  // K and Q are there; K transposed, T and P of the chunk before are read
    // K m, then Q m, 32 dims a step; operands are read a step ahead
    h8 f[2][4][2];
    const auto read = [&](int step) {
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int p = 0; p < 2; ++p)
          f[step & 1][t][p] = k_at[step / N * (kA<S> / 2) + (t * N + step % N) * 128 + 64 * p];
    };
    f32x4 x[4], y[4];
    const auto times = [&](int step, f32x4 *z) {
      const int i = step % N;
#pragma unroll
      for (int p = 0; p < 3; ++p)  // lo hi, hi lo, hi hi
#pragma unroll
        for (int t = 0; t < 4; ++t)
          z[t] = mma(f[step & 1][t][p == 0], p == 1 ? ml[i] : mh[i], i == 0 && p == 0 ? f32x4{0, 0, 0, 0} : z[t]);
    };
    read(0);
    if constexpr (SHARES) stage.vec(lds, next_v, chunk);
#pragma unroll
    for (int step = 0; step < 2 * N; ++step) {
      __builtin_amdgcn_sched_barrier(0);
      if (step + 1 < 2 * N) read(step + 1);
      if (step + 1 < 2 * N) stage_b(step, 2 * N - 1);
      times(step, step < N ? x : y);
    }
    __syncthreads();  // K and Q are read; the others are there
    h8 tf[6][2];
#pragma unroll
    for (int i = 0; i < 12; ++i) tf[i >> 1][i & 1] = u_at[kFragK<S> / 16 + i * 64];
    const f32x4 of_chunk = *reinterpret_cast<const f32x4 *>(vec + 5 * kCk);
    // the right sides
    f32x4 s[4];
    h8 hi[2], lo[2];
    float down;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const f32x4 ak = of_token(0, t);
#pragma unroll
      for (int e = 0; e < 4; ++e) s[t][e] = fmaf(-ak[e], x[t][e] * m_down, v[t][e]);
    }
    const float most_s = most_of_lanes(most4(s));
    unit_of(most_s, &up, &down);
    pair(s[0], s[1], up, &hi[0], &lo[0]);
    pair(s[2], s[3], up, &hi[1], &lo[1]);
    __builtin_amdgcn_sched_barrier(0);
    // a row tile of T or P against the operand
    const auto lower = [&](f32x4 *d) {
#pragma unroll
      for (int p = 0; p < 2; ++p)
#pragma unroll
        for (int k = 0; k < 3; ++k)
#pragma unroll
          for (int t = 2 * p; t < 4; ++t)
            d[t] = mma(tf[kTri[t] + p][k == 0], k == 1 ? lo[p] : hi[p], p == 0 && k == 0 ? f32x4{0, 0, 0, 0} : d[t]);
    };
    // delta, and delta e with K's units
    f32x4 d[4];
    vp += kCk * a.v_stride;
    const Base rows(ahead ? vp : a.v, ahead ? min(left - kCk, kCk) * v_stride : 0);
    stage_a(0, 8);
    lower(d);
    load_v(rows, 0);
    load_v(rows, 1);
    __builtin_amdgcn_sched_barrier(0);
    stage_a(1, 8);
#pragma unroll
    for (int i = 0; i < 12; ++i) tf[i >> 1][i & 1] = u_at[(kFragK<S> + kFragT) / 16 + i * 64];
#pragma unroll
    for (int t = 0; t < 4; ++t) d[t] = d[t] * (of_token(2, t) * down);
#pragma unroll
    for (int t = 0; t < 4; ++t) s[t] = d[t] * of_token(4, t);
    const float most_d = most_of_lanes(most4(d));
    unit_of(most_d, &up, &down);
    // of the wave's rows
    const float most_ds = lane_group_reduce<16>(fmaxf(most_d, most_s * (of_chunk.y * kUnits)), MaxOp{});
    pair(d[0], d[1], up, &hi[0], &lo[0]);
    pair(d[2], d[3], up, &hi[1], &lo[1]);
    lower(d);
    stage_a(2, 8);
    load_v(rows, 2);
    load_v(rows, 3);
    h8 eh[2], el[2];
    float e_down;
    const float most_e = most_of_lanes(most4(s));
    unit_of(most_e, &up, &e_down);
    pair(s[0], s[1], up, &eh[0], &el[0]);
    pair(s[2], s[3], up, &eh[1], &el[1]);
    // outputs, and how far the row's are at least above kLeast of what their operands could give
    // (NaN where one is: a delta that is not finite makes its own output so)
    const float least = most_ds * (a.scale * (kUnits * kLeast));
    const auto above = [&](int t, int e, f32x4 p_unit) { return fmaf(-p_unit[e], least, fabsf(d[t][e])); };
    float lowest = INFINITY;
    {
      const float y_by = m_down * a.scale, d_by = down * a.scale;
#pragma unroll
      for (int t = 0; t < 4; ++t) {
        const f32x4 p_unit = of_token(3, t), of_q = of_token(1, t) * y_by, of_p = p_unit * d_by;
#pragma unroll
        for (int e = 0; e < 4; ++e) d[t][e] = fmaf(of_q[e], y[t][e], of_p[e] * d[t][e]);
#pragma unroll
        for (int e = 0; e < 4; e += 2)
          lowest = __builtin_elementwise_minimum(
              __builtin_elementwise_minimum(above(t, e, p_unit), above(t, e + 1, p_unit)), lowest);
      }
    }
    // One row whose outputs all are clears its 16 lanes' tokens; else each token needs one.
    const uint64_t clear = __ballot(lowest >= 0.0f);
    const uint64_t fine = __ballot(lowest == lowest && most_s * (of_chunk.z * (kUnits * kLeast)) <= most_e);
    bool odd = fine != ~uint64_t{0};
    if (__builtin_expect(((clear - kOnes) & ~clear & kOnes << 15) != 0, false)) {
      uint32_t below = 0;  // a bit a token
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) below = 2 * below + (above(t, e, of_token(3, t)) < 0.0f);
      odd = odd || __any(lane_group_reduce<16>(below, AndOp{}) != 0);
    }
    stage_a(3, 8);
    const Base to_rows(op, min(left, kCk) * o_stride);
    // the new state, 64 of its dims at a time
    const float all = of_chunk.x;
    h8 kt[2][4][2];
    const auto read_kt = [&](int step) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int k = 0; k < 2; ++k)
          kt[step & 1][i][k] = u_at[(2 * (4 * (step >> 1) + i) + (step & 1)) * 128 + 64 * k];
    };
    f32x4 u[4];
    read_kt(0);
#pragma unroll
    for (int step = 0; step < N; ++step) {
      __builtin_amdgcn_sched_barrier(0);
      if (step + 1 < N) read_kt(step + 1);
      stage_a(N + step, 2 * N);
#pragma unroll
      for (int t = 4 * step / N; t < 4 * (step + 1) / N; ++t)
#pragma unroll
        for (int e = 0; e < 4; ++e) to_rows.store1(d[t][e], o_at + (16 * t + e) * o_stride);
      const int p = step & 1;
#pragma unroll
      for (int k = 0; k < 3; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          u[i] = mma(kt[p][i][k == 0], k == 1 ? el[p] : eh[p], p == 0 && k == 0 ? f32x4{0, 0, 0, 0} : u[i]);
      if (p == 1 && !odd)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          f32x4 &to_m = m[4 * (step >> 1) + i];
          to_m = add_times(to_m * all, e_down, u[i]);
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    if (__builtin_expect(odd, false)) {
      __builtin_amdgcn_s_waitcnt(0x0f70);  // (vmcnt 0: the chunk's outputs are written, then again)
      walk_tokens<S>(a, of, begin + chunk * kCk, min(left, kCk), m);
    }
    op += static_cast<size_t>(kCk) * a.h_v * S;
    ws_k += slot_bytes, ws_v += slot_bytes;
  }
  if (of.to < 0) return;
#pragma unroll
  for (int d = 0; d < S / 16; ++d)
    *reinterpret_cast<f32x4 *>(a.state + of.to * a.rag.slot_stride + m_at + 16 * d) = m[d];
}

// Blocks of the walk.  All rows of a (request, v-head) are a block's, 16 a wave; or, of the
// longest requests, as far as blocks are fewer than compute units, half of them, and the
// other four waves stage the operands (as they do for heads of 64).  What bounds a block is its waves' reads of them
// from LDS (120 KB a wave and chunk), so half the rows are through sooner: 4.2 us a chunk
// for 7.6.
template <int S>
__global__ __launch_bounds__(512, 2) void gdn_chunk_walk_kernel(GdnChunkArgs c) {
  __shared__ __attribute__((aligned(16))) ChunkLds<S> lds;
  const GdnArgs &a = c.g;
  if (static_cast<int>(blockIdx.x) >= c.walks) {  // the requests of fewer tokens
    step_rows<S, S == 128 ? 4 : 1, 512>(a, blockIdx.x - c.walks);
    return;
  }
  const int count = __builtin_amdgcn_readfirstlane(c.todo[0]);
  // requests in halves
  const int halves = S == 64 || count > 64 ? 0 : min(count, max(c.at_once - count, 0));
  int nth = blockIdx.x / (2 * a.h_v), rest = blockIdx.x - nth * 2 * a.h_v;
  const bool half = nth < halves;
  if (!half) {
    rest = blockIdx.x - 2 * halves * a.h_v;
    nth = rest / a.h_v;
    rest -= nth * a.h_v;
    nth += halves;
  }
  if (nth >= count) return;
  const int r = __builtin_amdgcn_readfirstlane(c.todo[1 + nth]), slabs = half ? 2 : 1;
  WalkOf of;
  int slab;
  if (c.xcd) {  // block b runs on die b % 8: q/k heads x, x + 8, .. on die x
    const int of_head = a.h_v / a.h_k * slabs, x = rest & 7, y = rest >> 3;
    const int kh = y / of_head * 8 + x, z = y % of_head;
    of.h = kh + z / slabs * a.h_k, slab = z % slabs;
  } else {
    of.h = rest / slabs, slab = rest % slabs;
  }
  a.rag.tokens_of(r, &of.begin, &of.n);
  a.rag.slots(r, &of.from, &of.to);
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  of.slot_bytes = static_cast<size_t>(a.h_k) * kHeadK<S> + static_cast<size_t>(a.h_v) * kHeadV;
  of.ws_k = c.ws + static_cast<size_t>(first_chunk(of.begin)) * of.slot_bytes +
            static_cast<size_t>(of.h % a.h_k) * kHeadK<S>;
  of.ws_v = c.ws + static_cast<size_t>(first_chunk(of.begin)) * of.slot_bytes +
            static_cast<size_t>(a.h_k) * kHeadK<S> + static_cast<size_t>(of.h) * kHeadV;
  const int walkers = S / 16 / slabs;  // waves
  of.row = 16 * (slab * walkers + w % walkers);
  if (S == 128 && walkers == 8) {
    walk_rows<S, S == 128>(a, lds, of);
  } else if (w < walkers) {
    walk_rows<S, false>(a, lds, of);
  } else {  // the barriers are walk_rows'
    const int chunks = (of.n + kCk - 1) / kCk;
    Stage<S, 256> stage;
    stage.begin(lds, of, chunks, threadIdx.x - 256);
    for (int chunk = 0; chunk < chunks; ++chunk) {
      const int ahead = min(chunks - 1 - chunk, 2);
      const Base next_k(of.ws_k + min(ahead, 1) * of.slot_bytes), next_v(of.ws_v + min(ahead, 1) * of.slot_bytes);
      const Base after_k(of.ws_k + ahead * of.slot_bytes);
      __syncthreads();
      stage.vec(lds, next_v, chunk);
      stage.b(lds, next_k, next_v, 0, 1);
      __syncthreads();
      stage.a(lds, after_k, 0, 1);
      of.ws_k += of.slot_bytes, of.ws_v += of.slot_bytes;
    }
  }
}

// Blocks of a launch: a grid has fewer than 2^32 threads a dimension.
constexpr size_t kMostBlocks = 0xffffff;

// Bytes of a chunk in the workspace.
size_t slot_bytes(const bh_gdn_ragged_args &p) {
  return p.h_k * (p.s == 64 ? kHeadK<64> : kHeadK<128>) + p.h_v * kHeadV;
}

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
  // (a chunk's block a q/k head; a place every kCkPlace tokens)
  if (!mul_size(p.n_tok / kCkPlace + 1, p.h_k, &n) || n > kMostBlocks ||
      !mul_size(p.n_tok / kCkPlace + 1, slot_bytes(p), &n))
    return fail(BH_ERR_SHAPE, "gdn_ragged: size overflow");
  if (p.n_req != 0 && p.n_tok != 0) {
    if (!p.q || !p.k || !p.v || !p.gate || !p.beta || !p.attn || !p.q_start || !p.src_slot ||
        !p.dst_slot || (p.n_slots != 0 && !p.state))
      return fail(BH_ERR_ARG, "gdn_ragged: null pointer");
  }
  return BH_OK;
}

bool whole_rows(const bh_gdn_ragged_args &p) {
  return (p.q_stride | p.k_stride | p.slot_stride) % 4 == 0 && aligned16(p.q) && aligned16(p.k) &&
         aligned16(p.state);
}

// Slots of chunks of a call, 0: it has none.
size_t chunk_slots(const bh_gdn_ragged_args &p) {
  const size_t most = p.max_new == 0 || p.max_new > p.n_tok ? p.n_tok : p.max_new;
  if ((p.s != 64 && p.s != 128) || most < static_cast<size_t>(kCkMin) || !whole_rows(p) ||
      p.v_stride > kMostStride)
    return 0;
  return p.n_tok / kCkPlace + 1;
}

// Requests of kCkMin tokens or more that there can be.
size_t most_long(const bh_gdn_ragged_args &p) {
  return p.n_tok / kCkMin < p.n_req ? p.n_tok / kCkMin : p.n_req;
}

// The chunks' operands, and the list of the requests that go by chunks.
size_t workspace_of(const bh_gdn_ragged_args &p) {
  const size_t slots = chunk_slots(p);
  return slots == 0 ? 0 : slots * slot_bytes(p) + (1 + most_long(p)) * sizeof(int32_t);
}

}  // namespace
}  // namespace bh

using namespace bh;

extern "C" size_t bh_gdn_ragged_workspace(const bh_gdn_ragged_args *args) {
  if (!args || check(*args) != BH_OK || args->n_req == 0 || args->n_tok == 0) return 0;
  return workspace_of(*args);
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
  const bool whole = whole_rows(p);
  a.most = 0x7fffffff;
  if (const size_t slots = chunk_slots(p)) {
    const size_t need = workspace_of(p);
    char *ws = static_cast<char *>(p.workspace);
    if (ws) {
      if (!aligned16(ws) || p.workspace_bytes < need)
        return fail(BH_ERR_SHAPE, "gdn_ragged: workspace of " + std::to_string(p.workspace_bytes) +
                                      " bytes, " + std::to_string(need) +
                                      " needed on a 16-byte boundary");
    } else {
      ws = static_cast<char *>(device_scratch(need, kScratchGdnRagged, st));
      if (!ws) return BH_ERR_HIP;
    }
    a.most = kCkMin - 1;
    const size_t longs = most_long(p);
    const size_t at_once = device_cu_count() / p.h_v;
    size_t walks = 2 * longs;  // of h_v blocks
    if (walks > at_once) walks = longs > at_once ? longs : at_once;
    GdnChunkArgs c{a, ws, static_cast<int>(slots), static_cast<int>(walks * p.h_v),
                   p.h_k % 8 == 0 && p.h_v % p.h_k == 0, static_cast<int>(at_once), static_cast<int>(longs),
                   reinterpret_cast<int32_t *>(ws + slots * slot_bytes(p))};
    const unsigned preps = static_cast<unsigned>(slots * p.h_k), blocks = static_cast<unsigned>((walks + p.n_req) * p.h_v);
    if (p.s == 128) {
      BH_LAUNCH(gdn_chunk_prep_kernel<128>, preps, kBlock, 0, st, c);
      BH_LAUNCH(gdn_chunk_walk_kernel<128>, blocks, 512, 0, st, c);
    } else {
      BH_LAUNCH(gdn_chunk_prep_kernel<64>, preps, kBlock, 0, st, c);
      BH_LAUNCH(gdn_chunk_walk_kernel<64>, blocks, 512, 0, st, c);
    }
    return ok();
  }
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
