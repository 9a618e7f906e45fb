// Losses of one logit row and what they read of it: log probabilities of given tokens with entropy and
// top alternatives, and the divergence from a teacher's top logits.  With z = x / t over a row of V
// logits, m = max x, S = sum e^{(x - m) / t} and log p_v = (x_v - m) / t - log S:
//
//   logprob = log p_tok      entropy = log S - sum_v e^{(x_v - m) / t} (x_v - m) / t / S
//   top     = the n largest logits, value descending, ties to the lower column, NaN first
//   dx_v    = (g [v = tok] - p_v (g + g_H (log p_v + entropy))) / t
//
// and with a list of K columns c_j holding the teacher's t_j (first entry of a column counts, negative
// columns are none), R = the columns not listed, q = softmax(x / t):
//
//   tail 0: p = softmax_j(t_j / t)           L = t^2 sum_j p_j (log p_j - log q_{c_j})
//   tail 1: p_j = e^{t_j}, r = 1 - sum p_j   L = t^2 (sum_j p_j (log p_j - log q_{c_j}) + r (log r - log q(R)))
//   dx_v  = g t (n q_v - p_j) where v = c_j, else g t (n q_v - r q_v / q(R)) (tail 0: r = 0)
//
// with r never below 0, taken as 0 where it is rounding and q(R) is 0, and n = sum p_j + r: 1 but for lists whose
// exponentials (tail 1) sum to more.
#include "../../include/rte_hip.h"
#include "row_words.hpp"

#include <float.h>

namespace rte {

namespace {

constexpr int kMaxTop = 128;  // alternatives or list entries per row

// Order of the alternatives as unsigned keys: larger value first, -0 = +0, NaN above everything.
constexpr uint32_t kNanKey = 0xfffffffeu, kInfKey = 0xff800000u;
typedef unsigned long long u64;
__device__ __forceinline__ uint32_t value_key(float x) {
  const uint32_t b = __float_as_uint(x + 0.0f);
  return x != x ? kNanKey : b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k > kInfKey ? 0x7fc00000u : (k & 0x80000000u) ? k ^ 0x80000000u : ~k);
}

__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;  // without the canonical copies that fmaxf makes of operands it knows nothing of
  asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
  return r;
}
// Largest of a vector's columns and m (NaN loses).
template <class X>
__device__ __forceinline__ float words_max(const Words& v, float m) {
#pragma unroll
  for (int j = 0; j < Row<X>::VE; j += 2) m = max3(m, Row<X>::get(v, j), Row<X>::get(v, j + 1));
  return m;
}

// Keeps what was computed of these words from being kept too: each phase unpacks them again, for a row's bf16
// columns as floats take twice the registers of the row.
template <int N>
__device__ __forceinline__ void forget(Words (&w)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" : "+v"(w[i].w[0]), "+v"(w[i].w[1]), "+v"(w[i].w[2]), "+v"(w[i].w[3]));
}

struct RowArgs {
  int64_t ld;
  int T, V;
  int nparts, part;  // a row is computed in nparts ranges of `part` columns
  float c2, inv_t;   // log2(e) / t, 1 / t
  // log probabilities
  const int64_t* tokens;
  int n_top;
  float *logprob, *entropy, *top_lp;
  int32_t* top_ids;
  // divergence
  const int32_t* ids;
  const float* tl;
  int K, tail;
  double it, t2;
  double kept;  // half a step, and a sixteenth of it, of the type that the teacher's values were kept in (0: fp32)
  float* loss;
  int32_t* cols;
  float* coef;
  float* stats;       // kept for the backward (NULL: none)
  float4* part_stats; // [T, nparts] {max, sum, sum of e u}
  u64* part_keys;     // [T, nparts, n_top]
};

// One row's sums, relative to its maximum m: s = sum e^u, su = log2(e) sum e^u u with u = (x - m) / t.
struct Sums {
  float m, s, su;
};

// A row's token and its logit, asked for before the row is summed.
struct Token {
  int64_t tok;
  float x;
  Token() = default;
  template <class X>
  __device__ __forceinline__ Token(const RowArgs& a, const X* row, int64_t t) {
    tok = a.tokens[t];
    x = tok >= 0 && tok < a.V ? Row<X>::one(row, tok) : 0.0f;
  }
};

__device__ __forceinline__ void finish_logprobs(const RowArgs& a, const Token& k, int64_t t, const Sums& r) {
  const int64_t tok = k.tok;
  const float log_s = logf(r.s);
  const bool empty = r.s == 0.0f;  // no column above -inf
  float lp = 0.0f;
  if (tok >= a.V) lp = __builtin_nanf("");
  else if (tok >= 0) lp = empty ? -INFINITY : (k.x - r.m) * a.inv_t - log_s;
  a.logprob[t] = lp;
  a.entropy[t] = empty ? 0.0f : log_s - r.su * kLn2 / r.s;
  if (a.stats) {
    a.stats[2 * t] = r.m;
    a.stats[2 * t + 1] = log_s;
  }
}

__device__ __forceinline__ void put_top(const RowArgs& a, int64_t t, int rank, u64 key, const Sums& r, float log_s) {
  const float x = key_value((uint32_t)(key >> 32));
  a.top_ids[t * a.n_top + rank] = (int)~(uint32_t)key;
  a.top_lp[t * a.n_top + rank] = r.s == 0.0f ? -INFINITY : (x - r.m) * a.inv_t - log_s;
}

__device__ __forceinline__ double of_lane(double x, int lane) {
  return __hiloint2double(__builtin_amdgcn_readlane(__double2hiint(x), lane), __builtin_amdgcn_readlane(__double2loint(x), lane));
}

// The divergence of row t by one wave, from the sums of the columns not listed (rest.m = -inf: none).
// Lane i holds entries i and i + 64.  The list's part is computed in 64 bits: for a student near its teacher
// the terms p (log p - log q) cancel to the square of the difference, and q's total is put together from the
// same list and rest, so that an error of the rest's sum enters multiplied by that difference.  `unique`: no
// column is listed twice.
// Kept for the backward: dx_v = g t coef_j at column cols_j, g t c e^{(x_v - m) / t} elsewhere, with {m, c}
// in stats (c = 0: the row has no gradient).
template <class X>
__device__ void finish_distill(const RowArgs& a, const X* row, int64_t t, const Sums& rest, bool unique, int lane) {
  const int32_t* ids = a.ids + t * a.K;
  const float* tl = a.tl + t * a.K;
  int col[2];
  float y[2];
  double x[2];
  bool foreign = false;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int j = lane + 64 * i;
    col[i] = j < a.K ? ids[j] : -1;
    y[i] = j < a.K ? tl[j] : 0.0f;
    foreign |= col[i] >= a.V;
  }
  if (!unique) {
    bool again[2] = {false, false};
    for (int j = 0; j < a.K; ++j) {
      const int c = __shfl(col[j >> 6], j & 63, 64);
      again[0] |= c == col[0] && j < lane;
      again[1] |= c == col[1] && j < lane + 64;
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (again[i]) col[i] = -1;
  }
  foreign = __any(foreign);
  double top = rest.m, tmax = -INFINITY;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (col[i] >= a.V) col[i] = -1;
    x[i] = col[i] >= 0 ? (double)Row<X>::one(row, col[i]) : -INFINITY;
    if (col[i] >= 0) tmax = y[i] > tmax || tmax != tmax ? y[i] : tmax;
    top = x[i] > top || top != top ? x[i] : top;
  }
  bool some = __any(col[0] >= 0 || col[1] >= 0);
  top = wave_max(top);
  tmax = wave_max(tmax);
  // NaN entries reach the sums; a list of -inf alone holds no probability
  const bool teacher_nan = __any((col[0] >= 0 && y[0] != y[0]) || (col[1] >= 0 && y[1] != y[1]));
  if (!a.tail && tmax == -INFINITY && !teacher_nan) some = false;
  const double m = top == -INFINITY ? 0.0 : top;
  // Exponentials, logarithms and reciprocals in 64 bits are most of this function's time, so one of each kind serves
  // several values, in different lanes (8192 rows of 2048 columns, lists of 64: 26.1 us with each by itself, 24.3).
  const bool two = a.K > 64;
  const double to_rest = rest.m == -INFINITY ? -INFINITY : ((double)rest.m - m) * a.it;
  double scale = 0.0, e[2] = {0.0, 0.0}, p[2] = {0.0, 0.0}, lp[2] = {0.0, 0.0};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if (i == 1 && !two) break;
    const double ex = exp(col[i] >= 0 ? (x[i] - m) * a.it : to_rest);
    e[i] = col[i] >= 0 ? ex : 0.0;
    if (lane + 64 * i >= a.K) scale = ex;  // lanes without an entry, the last one if any
    lp[i] = a.tail ? (double)y[i] : ((double)y[i] - (tmax == -INFINITY ? 0.0 : tmax)) * a.it;
    p[i] = col[i] >= 0 ? exp(lp[i]) : 0.0;
  }
  scale = (a.K & 63) ? of_lane(scale, 63) : exp(to_rest);
  double rsum = rest.s == 0.0f ? 0.0 : rest.s * scale;  // a NaN sum stays
  if (rest.m == -INFINITY && rest.s != 0.0f) rsum = __builtin_nan("");
  const double total = wave_sum(e[0] + e[1]) + rsum, tsum = wave_sum(p[0] + p[1]);
  double r = a.tail ? (tsum > 1.0 ? 0.0 : 1.0 - tsum) : 0.0;
  // What roundings leave of 1 is no mass outside the list, which would make the loss infinite where the student can have
  // none there.  fp32 log probabilities of a row with K possible columns leave at most 2^-24 (K + 2 + 7 log K): K + 2 from
  // the exponentials and their sum, the rest from exponents, logarithm and results, each weighted by p; log K < 5.
  // Values kept in 16 bits are off by half a step of each, e^x - 1 < 17/16 x: so much of p_j |t_j| more.
  if (rest.s == 0.0f && r > 0.0) {
    double most = (a.K + 32) * 0x1p-23;
    if (a.kept != 0.0) most += a.kept * wave_sum((p[0] > 0.0 ? p[0] * -lp[0] : 0.0) + (p[1] > 0.0 ? p[1] * -lp[1] : 0.0));
    if (r <= most) r = 0.0;
  }
  // the rest's own sum: times its scale it may be below the least number, however finite its logarithm
  const double logs = log(lane == 0 ? total : lane == 1 ? tsum : lane == 2 ? r : (double)rest.s);
  const double inverses = 1.0 / (lane == 0 ? total : tsum);
  const double log_s = of_lane(logs, 0), inv = of_lane(inverses, 0);
  if (!a.tail) {
    const double tlog = of_lane(logs, 1), tinv = of_lane(inverses, 1);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      lp[i] -= tlog;
      p[i] *= tinv;
    }
  }
  const double mass = a.tail ? tsum + r : 1.0;
  const bool empty = total == 0.0;
  double l = 0.0;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const double lq = empty ? -INFINITY : (x[i] - m) * a.it - log_s;
    if (col[i] >= 0 && p[i] != 0.0) l += p[i] * (lp[i] - lq);
  }
  l = wave_sum(l);
  if (r > 0.0) l += r * (of_lane(logs, 2) - (rest.s == 0.0f ? -INFINITY : to_rest + of_lane(logs, 3) - log_s));
  if (lane == 0) a.loss[t] = foreign ? __builtin_nanf("") : some ? (float)(l * a.t2) : 0.0f;
  if (!a.stats) return;
  const bool none = foreign || !some || empty;
  if (lane == 0) {
    const bool out = none || rest.s == 0.0f;  // no column outside the list above -inf
    a.stats[2 * t] = out ? 0.0f : rest.m;
    // (mass q(R) - r) / (the rest's sum relative to its own maximum)
    a.stats[2 * t + 1] = out ? 0.0f : (float)((rsum * inv * mass - r) / rest.s);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int j = lane + 64 * i;
    if (j >= a.K) continue;
    a.cols[t * a.K + j] = none ? -1 : col[i];
    a.coef[t * a.K + j] = none ? 0.0f : (float)(e[i] * inv * mass - p[i]);
  }
}

__device__ __forceinline__ void wave_fence() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// Candidates: {value bits, column} words of LDS as they are found, keys once they are all there.
__device__ __forceinline__ u64 raw_cand(float x, int col) { return (u64)__float_as_uint(x) << 32 | (uint32_t)~col; }
__device__ __forceinline__ u64 cand_key(u64 raw) {
  return (u64)value_key(__uint_as_float((uint32_t)(raw >> 32))) << 32 | (uint32_t)raw;
}

// v of the lane whose number differs in the bit O.
template <int O>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
  const int x = (int)v;
  if constexpr (O == 1) return __builtin_amdgcn_update_dpp(x, x, 0xb1, 0xf, 0xf, false);
  else if constexpr (O == 2) return __builtin_amdgcn_update_dpp(x, x, 0x4e, 0xf, 0xf, false);
  else if constexpr (O == 4) {  // 7 - lane, then 3 - lane
    const int y = __builtin_amdgcn_update_dpp(x, x, 0x141, 0xf, 0xf, false);
    return __builtin_amdgcn_update_dpp(y, y, 0x1b, 0xf, 0xf, false);
  } else if constexpr (O == 8) return __builtin_amdgcn_update_dpp(x, x, 0x128, 0xf, 0xf, false);  // a rotation by half a row
  else return __shfl_xor(v, O, 64);
}

// Bitonic sort, largest first, of 64 R keys that lie R to a lane (key lane R + r): K the length of the runs being
// merged, J the distance compared.
template <int R, int K, int J>
__device__ __forceinline__ void sort_step(u64 (&v)[R], int lane) {
  if constexpr (J >= R) {
    const bool first = ((lane & (K / R)) == 0) == ((lane & (J / R)) == 0);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const u64 o = (u64)lane_xor<J / R>((uint32_t)(v[r] >> 32)) << 32 | lane_xor<J / R>((uint32_t)v[r]);
      v[r] = (v[r] > o) == first ? v[r] : o;
    }
  } else {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (r & J) continue;
      const bool down = K < R ? (r & K) == 0 : (lane & (K / R)) == 0;
      const u64 a = v[r], b = v[r | J];
      const bool keep = (a > b) == down;
      v[r] = keep ? a : b;
      v[r | J] = keep ? b : a;
    }
  }
  if constexpr (J > 1) sort_step<R, K, J / 2>(v, lane);
}
template <int R, int K = 2>
__device__ __forceinline__ void sort_keys(u64 (&v)[R], int lane) {
  sort_step<R, K, K / 2>(v, lane);
  if constexpr (K < 64 * R) sort_keys<R, K * 2>(v, lane);
}

// One wave sorts the n candidates in its registers and hands the first `want` to put(rank, key); ranks past the
// last candidate get key 0.
template <int R, class P>
__device__ __forceinline__ void sort_cands(const u64* cand, int n, int want, int lane, P put) {
  u64 v[R];
#pragma unroll
  for (int r = 0; r < R; ++r) v[r] = r * 64 + lane < n ? cand_key(cand[r * 64 + lane]) : 0;
  sort_keys<R>(v, lane);
#pragma unroll
  for (int r = 0; r < R; ++r)
    if (lane * R + r < want) put(lane * R + r, v[r]);
}

// The same for any n by one wave: from 17 to 256 sorted; few, or more (rows with many ties at the threshold),
// ranked by counting the larger keys.  (All ranked by counting, 8192 rows of 2048 fp32 took 32 us for 64
// alternatives and 51 for 128; 28 and 35 sorted.)
template <class P>
__device__ __forceinline__ void order_cands(u64* cand, int n, int want, int lane, P put) {
  if (n > 16) {
    if (n <= 64 && want <= 64) return sort_cands<1>(cand, n, want, lane, put);
    if (n <= 128) return sort_cands<2>(cand, n, want, lane, put);
    if (n <= 256) return sort_cands<4>(cand, n, want, lane, put);
  }
  for (int c = lane; c < n; c += 64) cand[c] = cand_key(cand[c]);
  wave_fence();
  for (int c = lane; c < n; c += 64) {
    const u64 mine = cand[c];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += cand[j] > mine;
    if (rank < want) put(rank, mine);
  }
  for (int c = n + lane; c < want; c += 64) put(c, 0ull);
}

// The want-th largest of 64 G keys (G per lane), to its bits from `low` up: at least `want` keys are not below
// the result.
template <int G>
__device__ __forceinline__ uint32_t nth_key(const uint32_t* k, int want, int low, bool exact) {
  uint32_t thr = 0;
  for (int b = 31; b >= low; --b) {
    const uint32_t c = thr | 1u << b;
    int n = 0;
#pragma unroll
    for (int g = 0; g < G; ++g) n += __popcll(__ballot(k[g] >= c));
    if (n >= want) thr = c;
    if (n == want && !exact) break;
  }
  return thr;
}

constexpr int kCandWave = 512, kCandGroup = 1024;

// A short row by one wave, held in registers: E columns per lane, read once.  The maximum comes first, so no
// sum is rescaled.  For the alternatives, the n-th largest of 256 maxima (of quarters of the lanes' columns) is
// a threshold that n columns reach at least; those that do go to LDS and each finds its rank there.  Rows whose
// ties bring more than LDS holds find the n-th value and the last of its columns by bits.
// 8192 x 2048 fp32: 64 alternatives 28 us, a list of 64 24, of which reading is 13: bound by instructions (threshold
// and sort; 64-bit exponentials).
template <class X, int E, bool DIST, bool TOP>
__global__ void __launch_bounds__(256, TOP ? (E == 64 ? 4 : 6) : 8) rows_wave_kernel(const X* __restrict__ logits, RowArgs a) {
  constexpr int VE = Row<X>::VE, NV = E / VE, COLS = 64 * VE;
  static_assert(NV * VE == E && NV >= 4 && NV % 4 == 0, "whole vectors, four groups of them");
  __shared__ uint32_t s_mask[DIST ? 4 : 1][DIST ? 2 * E : 1];
  __shared__ __align__(16) u64 s_cand[TOP ? 4 : 1][TOP ? kCandWave : 1];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int64_t t = (int64_t)blockIdx.x * 4 + wave;
  if (t >= a.T) return;
  const X* row = logits + t * a.ld;
  const int len = a.V;

  Words w[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int off = (i * 64 + lane) * VE;
    if ((i + 1) * COLS <= len) {
      w[i] = whole_words(row + off);
    } else if (i * COLS < len) {
      w[i] = load_words(row, off, len);
    } else {
#pragma unroll
      for (int j = 0; j < VE; ++j) Row<X>::set(w[i], j, -INFINITY);
    }
  }

  [[maybe_unused]] const Token token = [&] {
    if constexpr (DIST) return Token{};
    else return Token(a, row, t);
  }();
  bool unique = true;
  if constexpr (DIST) {
    uint32_t* mask = s_mask[wave];
    for (int i = lane; i < 2 * E; i += 64) mask[i] = 0;
    wave_fence();
    bool again = false;
    for (int j = lane; j < a.K; j += 64) {
      const int id = a.ids[t * a.K + j];
      if (id >= 0 && id < len) again |= (atomicOr(&mask[id >> 5], 1u << (id & 31)) >> (id & 31)) & 1;
    }
    unique = !__any(again);
    wave_fence();
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int off = (i * 64 + lane) * VE;
      const uint32_t bits = mask[off >> 5] >> (off & 31) & ((1u << VE) - 1);
      if (bits) {
#pragma unroll
        for (int j = 0; j < VE; ++j)
          if (bits >> j & 1) Row<X>::set(w[i], j, -INFINITY);
      }
    }
  }

  // maxima (a NaN column shows in the sums)
  // in four groups that short rows fill too: single vectors of fp32, halves of bf16 ones
  float gm[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (i * COLS >= len) continue;
#pragma unroll
    for (int j = 0; j < VE; j += 4) {
      float& g = gm[VE == 8 ? (i & 1) * 2 + j / 4 : i & 3];
      g = max3(max3(g, Row<X>::get(w[i], j), Row<X>::get(w[i], j + 1)), Row<X>::get(w[i], j + 2), Row<X>::get(w[i], j + 3));
    }
  }
  float m = fmaxf(fmaxf(gm[0], gm[1]), fmaxf(gm[2], gm[3]));
  m = wave_max(m);
  uint32_t thr = 0;
  const int want = a.n_top;
  if constexpr (TOP) {
    // as few maxima as bring few columns more than asked for: 32 of 64 about 44, 64 of 128 about 89, 128 of 256 about 177
    constexpr int kLow = VE == 8 ? 16 : 12;  // 16 bits are all of a bf16 value
    const uint32_t g4[4] = {value_key(gm[0]), value_key(gm[1]), value_key(gm[2]), value_key(gm[3])};
    const uint32_t g2[2] = {g4[0] > g4[2] ? g4[0] : g4[2], g4[1] > g4[3] ? g4[1] : g4[3]};
    const uint32_t g1 = g2[0] > g2[1] ? g2[0] : g2[1];
    thr = want <= 32 ? nth_key<1>(&g1, want, kLow, false) : want <= 64 ? nth_key<2>(g2, want, kLow, false)
                                                                       : nth_key<4>(g4, want, kLow, false);
  }

  forget(w);
  const float m0 = m == -INFINITY ? 0.0f : m;
  float s = 0.0f, su = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if (i * COLS >= len) continue;
#pragma unroll
    for (int j = 0; j < VE; ++j) {
      const float u = (Row<X>::get(w[i], j) - m0) * a.c2;
      const float e = exp2_(u);
      s += e;
      if constexpr (!DIST) su += e * fmaxf(u, -256.0f);  // -inf: e is 0 and the product has to be
    }
  }
  s = wave_sum(s);
  if constexpr (!DIST) su = wave_sum(su);
  const Sums r{m, s, su};
  if constexpr (DIST) {
    finish_distill(a, row, t, r, unique, lane);
  } else {
    if (lane == 0) finish_logprobs(a, token, t, r);
  }

  if constexpr (TOP) {
    u64* cand = s_cand[wave];
    const float least = key_value(thr);  // not less than it: in (NaN and, where it is NaN, everything in)
    int n = 0;
    auto collect = [&](auto any_of, auto in) {
      n = 0;
      forget(w);
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (i * COLS >= len || !__any(any_of(w[i]))) continue;
        const int off = (i * 64 + lane) * VE;
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          const float x = Row<X>::get(w[i], j);
          const bool here = in(x, off + j) && off + j < len;
          const u64 who = __ballot(here);
          if (who == 0) continue;
          const int pos = n + __builtin_amdgcn_mbcnt_hi((uint32_t)(who >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)who, 0));
          if (here && pos < kCandWave) cand[pos] = raw_cand(x, off + j);
          n += __popcll(who);
        }
      }
      wave_fence();
    };
    // a vector is looked into where its maximum passes, or where the row holds NaN (its sum is NaN then)
    const bool look = s != s;
    collect([&](const Words& v) { return look || !(words_max<X>(v, -INFINITY) < least); },
            [&](float x, int) { return !(x < least); });
    if (n > kCandWave) {
      // value of rank `want`, then the last of its columns that is in
      auto total = [&](auto in) {
        int c = 0;
        forget(w);
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
          for (int j = 0; j < VE; ++j) {
            const int at = (i * 64 + lane) * VE + j;
            c += __popcll(__ballot(at < len && in(value_key(Row<X>::get(w[i], j)), at)));
          }
        return c;
      };
      uint32_t kth = 0;
      for (int b = 31; b >= 0; --b) {
        const uint32_t c = kth | 1u << b;
        if (total([&](uint32_t k, int) { return k >= c; }) >= want) kth = c;
      }
      const int need = want - total([&](uint32_t k, int) { return k > kth; });
      int last = 0;
      for (int b = 11; b >= 0; --b) {
        const int c = last | 1 << b;
        if (total([&](uint32_t k, int at) { return k == kth && at < c; }) < need) last = c;
      }
      collect([](const Words&) { return true; }, [&](float x, int at) {
        const uint32_t k = value_key(x);
        return k > kth || (k == kth && at <= last);
      });
    }
    const float log_s = logf(s);
    order_cands(cand, n, want, lane, [&](int rank, u64 key) { put_top(a, t, rank, key, r, log_s); });
  }
}

// A range of a longer row in one pass of a workgroup: every lane keeps its own running maximum and sums over
// batches of four vectors, the next of them on its way, and nothing is exchanged before the end.  Columns listed
// (DIST) are left out by a bit mask in LDS.  For the alternatives (TOP) each lane leaves its maximum of every 32 of
// its columns in LDS; at the end the n-th largest of the 256 lanes' maxima is a threshold that n columns reach at
// least, and only the few 32s whose maximum reaches it are read again, a vector to a lane.
// Bound by reading: 4096 x 131072 with 20 alternatives 205 us in bf16 and 370 in fp32, 5.2 and 5.8 TB/s; 4099 x 32771
// bf16 87 us behind a backward pass, whose gradient is still being written back meanwhile, and 59 by itself.  Ranges of
// 65536 and their join, with room for the longest range's maxima in every workgroup, took 219 us for the first,
// 50 for 700 such rows (44 now) and 104 for 8000 x 9001 fp32 with 128 alternatives (88 now).
constexpr int kBatch = 4;
constexpr int kStreamCols = 131072;  // columns of a workgroup: 16 KB of bit mask, or of maxima, one for 32 columns of a lane
constexpr int kStreamMax = 32 * 256;  // columns to a row of those maxima
constexpr int kItems = 512;

template <class X, bool DIST, bool TOP>
__global__ void __launch_bounds__(256, 6) rows_stream_kernel(const X* __restrict__ logits, RowArgs a) {
  constexpr int VE = Row<X>::VE, COLS = kBatch * 256 * VE;
  constexpr int PER = 32 / (kBatch * VE);  // batches to a maximum
  extern __shared__ uint32_t s_range[];  // as much as the range needs: what is left lets more workgroups in
  uint32_t* s_mask = s_range;
  float (*s_bmax)[256] = reinterpret_cast<float (*)[256]>(s_range);
  __shared__ Sums s_sums[4];
  __shared__ uint32_t s_key[TOP ? 256 : 1];
  __shared__ __align__(16) u64 s_cand[TOP ? kCandGroup : 1];
  __shared__ int s_items[TOP ? kItems : 1];
  __shared__ int s_ctl[3];  // items, candidates, threshold
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int64_t t = blockIdx.x / (unsigned)a.nparts;
  const int p = blockIdx.x - (unsigned)t * (unsigned)a.nparts;
  const X* row = logits + t * a.ld;
  const int c0 = p * a.part;
  const int len = a.V - c0 < a.part ? a.V - c0 : a.part;
  const X* at = row + c0;
  auto load = [&](int b, Words* to) {
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int off = b + (i * 256 + tid) * VE;
      if (b + COLS <= len) to[i] = whole_words(at + off);
      else to[i] = load_words(at, off, len);
    }
  };
  Words next[kBatch];
  load(0, next);
  [[maybe_unused]] const Token token = [&] {
    if constexpr (DIST) return Token{};
    else return Token(a, row, t);
  }();
  bool unique = true;
  if constexpr (DIST) {
    for (int i = tid; i < (len + 31) / 32; i += 256) s_mask[i] = 0;
    __syncthreads();
    bool again = false;
    if (tid < a.K) {
      const int id = a.ids[t * a.K + tid], rel = id - c0;
      if (id >= c0 && rel < len) again = (atomicOr(&s_mask[rel >> 5], 1u << (rel & 31)) >> (rel & 31)) & 1;
    }
    unique = __syncthreads_or(again) == 0;
  }
  Sums r{-FLT_MAX, 0.0f, 0.0f};  // a lowest maximum: -inf columns add nothing, lowest ones count
  float most = -INFINITY;        // largest entry of s_bmax of this lane
  for (int b = 0; b < len; b += COLS) {
    Words w[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) w[i] = next[i];
    if (b + COLS < len) load(b + COLS, next);
    if constexpr (DIST) {
#pragma unroll
      for (int i = 0; i < kBatch; ++i) {
        const int off = b + (i * 256 + tid) * VE;
        const uint32_t bits = off < len ? s_mask[off >> 5] >> (off & 31) & ((1u << VE) - 1) : 0;
        if (bits) {
#pragma unroll
          for (int j = 0; j < VE; ++j)
            if (bits >> j & 1) Row<X>::set(w[i], j, -INFINITY);
        }
      }
    }
    float bm = -INFINITY;
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (b + i * 256 * VE < len) bm = words_max<X>(w[i], bm);
    const float m = fmaxf(r.m, bm), d = (r.m - m) * a.c2, scale = exp2_(d);
    if constexpr (!DIST) r.su = scale * (r.su + r.s * fmaxf(d, -256.0f));
    r.s *= scale;
    r.m = m;
    float s = 0.0f;
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      if (b + i * 256 * VE >= len) continue;
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        const float u = (Row<X>::get(w[i], j) - m) * a.c2, e = exp2_(u);
        s += e;
        if constexpr (!DIST) r.su += e * fmaxf(u, -256.0f);
      }
    }
    r.s += s;
    if constexpr (TOP) {
      bm = s != s ? INFINITY : bm;  // a batch with NaN is always looked into
      float& of = s_bmax[b / COLS / PER][tid];
      of = b / COLS % PER ? fmaxf(of, bm) : bm;
      most = fmaxf(most, bm);
    }
  }
  auto join = [&](const Sums& x, float top) {  // x relative to top
    const float d = (x.m - top) * a.c2, e = exp2_(d);
    return Sums{top, x.s != x.s ? x.s : x.s * e, e * (x.su + x.s * fmaxf(d, -256.0f))};
  };
  r = join(r, wave_max(r.m));
  r.s = wave_sum(r.s);
  r.su = wave_sum(r.su);
  if (lane == 0) s_sums[wave] = r;
  if constexpr (TOP) {
    s_key[tid] = value_key(most);
    if (tid < 2) s_ctl[tid] = 0;
  }
  __syncthreads();
  const int want = a.n_top;
  uint32_t keys[4];
  if constexpr (TOP) {
#pragma unroll
    for (int g = 0; g < 4; ++g) keys[g] = s_key[lane + 64 * g];
  }
  const float top = fmaxf(fmaxf(s_sums[0].m, s_sums[1].m), fmaxf(s_sums[2].m, s_sums[3].m));
  r = join(s_sums[0], top);
#pragma unroll
  for (int i = 1; i < 4; ++i) {
    const Sums o = join(s_sums[i], top);
    r.s += o.s;
    r.su += o.su;
  }
  if (wave == 0) {
    if constexpr (TOP) {
      const uint32_t thr = nth_key<4>(keys, want, VE == 8 ? 16 : 12, false);
      if (lane == 0) s_ctl[2] = (int)thr;
    }
    if (a.nparts > 1) {
      if (lane == 0) a.part_stats[t * a.nparts + p] = make_float4(r.m, r.s, r.su, 0.0f);
    } else if constexpr (DIST) {
      finish_distill(a, row, t, r, unique, lane);
    } else {
      if (lane == 0) finish_logprobs(a, token, t, r);
    }
  }
  if constexpr (TOP) {
    __syncthreads();
    const float least = key_value((uint32_t)s_ctl[2]);  // not less than it: in (NaN and, where it is NaN, everything in)
    auto add = [&](float x, int off) {
      const int pos = atomicAdd(&s_ctl[1], 1);
      if (pos < kCandGroup) s_cand[pos] = raw_cand(x, c0 + off);
    };
    if (!(most < least)) {
      for (int b = 0; b * PER * COLS < len; ++b)
        if (!(s_bmax[b][tid] < least)) {
          const int pos = atomicAdd(&s_ctl[0], 1);
          if (pos < kItems) s_items[pos] = b * 256 + tid;
        }
    }
    __syncthreads();
    const int items = s_ctl[0];
    if (items <= kItems) {
      for (int q = tid; q < items * PER * kBatch; q += 256) {
        const int it = s_items[q / (PER * kBatch)], v0 = q % (PER * kBatch);
        const int off = ((it >> 8) * PER + v0 / kBatch) * COLS + ((v0 % kBatch) * 256 + (it & 255)) * VE;
        const Words v = load_words(at, off, len);
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          const float x = Row<X>::get(v, j);
          if (!(x < least) && off + j < len) add(x, off + j);
        }
      }
      __syncthreads();
    }
    int n = s_ctl[1];
    if (items > kItems || n > kCandGroup) {  // ties, or a row whose large values sit in few lanes
      auto every = [&](auto f) {
        for (int off = tid * VE; off < len; off += 256 * VE) {
          const Words v = load_words(at, off, len);
#pragma unroll
          for (int j = 0; j < VE; ++j)
            if (off + j < len) f(Row<X>::get(v, j), off + j);
        }
      };
      auto total = [&](int c) {
        c = wave_sum(c);
        __syncthreads();
        if (lane == 0) s_items[wave] = c;
        __syncthreads();
        return (s_items[0] + s_items[1]) + (s_items[2] + s_items[3]);
      };
      auto above = [&](uint32_t k) {
        int c = 0;
        every([&](float x, int) { c += value_key(x) > k; });
        return total(c);
      };
      // the value of rank `want`: the lanes' own want-th maximum where fewer columns exceed it, else by bits above it
      uint32_t kth = nth_key<4>(keys, want, 0, true);
      int over = above(kth);
      if (over >= want) {
        const uint32_t floor = kth;
        kth = 0;
        for (int b = 31; b >= 0; --b) {
          const uint32_t c = kth | 1u << b;
          if (c <= floor || above(c - 1) >= want) kth = c;
        }
        over = above(kth);
      }
      __syncthreads();
      if (tid == 0) s_ctl[1] = 0;
      __syncthreads();
      every([&](float x, int off) {
        if (value_key(x) > kth) add(x, off);
      });
      // and the first columns that hold that value
      int left = want - over;
      for (int off = tid * VE, b = 0; b < len && left > 0; off += 256 * VE, b += 256 * VE) {
        const Words v = load_words(at, off, len);
        int c = 0;
#pragma unroll
        for (int j = 0; j < VE; ++j) c += off + j < len && value_key(Row<X>::get(v, j)) == kth;
        int before = c;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const int y = __shfl_up(before, o, 64);
          if (lane >= o) before += y;
        }
        __syncthreads();
        if (lane == 63) s_items[wave] = before;
        __syncthreads();
        before -= c;
        int all = 0;
        for (int i = 0; i < 4; ++i) {
          if (i < wave) before += s_items[i];
          all += s_items[i];
        }
#pragma unroll
        for (int j = 0; j < VE; ++j) {
          const float x = Row<X>::get(v, j);
          if (off + j < len && value_key(x) == kth && before++ < left) add(x, off + j);
        }
        left -= all;
      }
      __syncthreads();
      n = s_ctl[1];
    }
    if (wave != 0) return;
    u64* out = a.part_keys + (t * a.nparts + p) * want;
    const float log_s = logf(r.s);
    order_cands(s_cand, n, want, lane, [&](int rank, u64 key) {
      if (a.nparts > 1) out[rank] = key;
      else put_top(a, t, rank, key, r, log_s);
    });
  }
}

// Joins a row's ranges: sums rescaled to the common maximum, the alternatives merged by rank (a key's rank is
// the number of larger keys in every range's sorted list).  4096 rows of two ranges, 20 alternatives: 11 us, most of it the rows' dependent reads.
constexpr int kJoinKeys = 2048;
template <class X, bool DIST, bool TOP>
__global__ void __launch_bounds__(TOP ? 256 : 64) rows_join_kernel(const X* __restrict__ logits, RowArgs a) {
  __shared__ u64 s_keys[TOP ? kJoinKeys : 1];
  const int64_t t = blockIdx.x;
  const int lane = threadIdx.x & 63;
  const float4* part = a.part_stats + t * a.nparts;
  float m = -INFINITY;
  for (int i = lane; i < a.nparts; i += 64) m = fmaxf(m, part[i].x);
  m = wave_max(m);
  const float m0 = m == -INFINITY ? 0.0f : m;
  float s = 0.0f, su = 0.0f;
  for (int i = lane; i < a.nparts; i += 64) {
    const float4 q = part[i];
    const float u = (q.x - m0) * a.c2, e = exp2_(u);
    s += q.y != q.y ? q.y : q.y * e;
    su += e * (q.z + q.y * fmaxf(u, -256.0f));
  }
  const Sums r{m, wave_sum(s), wave_sum(su)};
  const X* row = logits + t * a.ld;
  if constexpr (DIST) {
    finish_distill(a, row, t, r, false, lane);
  } else {
    if (threadIdx.x == 0) finish_logprobs(a, Token(a, row, t), t, r);
  }
  if constexpr (TOP) {
    const int K = a.n_top, n = a.nparts * K;
    const u64* keys = a.part_keys + t * n;
    const bool fits = n <= kJoinKeys;
    const float log_s = logf(r.s);
    if (fits) {
      for (int i = threadIdx.x; i < n; i += 256) s_keys[i] = keys[i];
      __syncthreads();
    }
    for (int i = threadIdx.x; i < n; i += 256) {
      const u64 mine = fits ? s_keys[i] : keys[i];
      if (mine == 0) continue;
      int rank = 0;
      for (int q = 0; q < a.nparts && rank < K; ++q) {
        int lo = 0, hi = K;  // keys of list q above mine
        while (lo < hi) {
          const int mid = (lo + hi) >> 1;
          const u64 o = fits ? s_keys[q * K + mid] : keys[q * K + mid];
          if (o > mine) lo = mid + 1;
          else hi = mid;
        }
        rank += lo;
      }
      if (rank < K) put_top(a, t, rank, mine, r, log_s);
    }
  }
}

// Backward passes: a wave reads and writes 2048 columns once; bound by HBM (4099 x 32771 bf16, 537 MB: 85 us, 6.3 TB/s;
// with a list of 32 86).
constexpr int kSeg = 2048;

template <class X>
__global__ void __launch_bounds__(256)
    logprobs_bwd_kernel(const X* __restrict__ logits, int64_t ld, int64_t items, int V, int nseg,
                        const int64_t* __restrict__ tokens, float inv_t, const float* __restrict__ stats,
                        const float* __restrict__ entropy, const float* __restrict__ g_lp,
                        const float* __restrict__ g_ent, X* __restrict__ dlogits) {
  constexpr int VE = Row<X>::VE, NV = kSeg / 64 / VE;
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (item >= items) return;
  const int64_t t = item / nseg;
  const int c0 = (int)(item - t * nseg) * kSeg;
  const int len = V - c0 < kSeg ? V - c0 : kSeg;
  const X* x = logits + t * ld + c0;
  X* out = dlogits + t * V + c0;
  Words w[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if ((i * 64) * VE < len) w[i] = load_words(x, (i * 64 + lane) * VE, len);
  const float m = stats[2 * t], log_s = stats[2 * t + 1];
  const int64_t tok = tokens[t];
  const float g = g_lp && tok >= 0 && tok < V ? g_lp[t] : 0.0f, gh = g_ent ? g_ent[t] : 0.0f;
  const float gc = g + gh * entropy[t];
  const bool empty = log_s == -INFINITY;
  const bool none = empty || (gh == 0.0f && (tok < 0 || tok >= V));  // padding's logits may hold anything
  // the token's column is written again by the lane that holds it
  const int64_t rel = tok - c0;
  const bool mine = g != 0.0f && !empty && rel >= 0 && rel < len && (int)(rel / VE) % 64 == lane;
  const float at_tok = mine ? Row<X>::one(x, rel) : 0.0f;
  auto slope = [&](float v) {  // of every column: -p (g + g_H (log p + H)) / t
    const float lp = (v - m) * inv_t - log_s;
    return -exp2_(lp * kLog2e) * (gc + gh * fmaxf(lp, -200.0f)) * inv_t;
  };
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if ((i * 64) * VE >= len) continue;
    float d[VE];
#pragma unroll
    for (int j = 0; j < VE; ++j) d[j] = none ? 0.0f : slope(Row<X>::get(w[i], j));
    store_words(out, (i * 64 + lane) * VE, len, d);
  }
  if (mine) Row<X>::put(out, rel, slope(at_tok) + g * inv_t);
}

template <class X>
__global__ void __launch_bounds__(256)
    distill_bwd_kernel(const X* __restrict__ logits, int64_t ld, int64_t items, int V, int nseg, int K, float c2,
                       float temp, const float* __restrict__ stats, const int32_t* __restrict__ cols,
                       const float* __restrict__ coef, const float* __restrict__ g, X* __restrict__ dlogits) {
  constexpr int VE = Row<X>::VE, NV = kSeg / 64 / VE;
  const int lane = threadIdx.x & 63;
  const int64_t item = (int64_t)blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  if (item >= items) return;
  const int64_t t = item / nseg;
  const int c0 = (int)(item - t * nseg) * kSeg;
  const int len = V - c0 < kSeg ? V - c0 : kSeg;
  const X* x = logits + t * ld + c0;
  X* out = dlogits + t * V + c0;
  Words w[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if ((i * 64) * VE < len) w[i] = load_words(x, (i * 64 + lane) * VE, len);
  int col[2];
  float cf[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int j = lane + 64 * i;
    col[i] = j < K ? cols[t * K + j] - c0 : -1;
    cf[i] = j < K ? coef[t * K + j] : 0.0f;
  }
  const float m = stats[2 * t], gt = g[t] * temp, c = stats[2 * t + 1] * gt;
  const bool none = stats[2 * t + 1] == 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    if ((i * 64) * VE >= len) continue;
    float d[VE];
#pragma unroll
    for (int j = 0; j < VE; ++j) d[j] = none ? 0.0f : c * exp2_((Row<X>::get(w[i], j) - m) * c2);
    store_words(out, (i * 64 + lane) * VE, len, d);
  }
  // the listed columns, once every lane's stores are done
  const bool here[2] = {col[0] >= 0 && col[0] < len, col[1] >= 0 && col[1] < len};
  if (!__any(here[0] || here[1])) return;
  __builtin_amdgcn_fence(__ATOMIC_SEQ_CST, "workgroup");
#pragma unroll
  for (int i = 0; i < 2; ++i)
    if (here[i]) Row<X>::put(out, col[i], gt * cf[i]);
}

// Rows that one wave holds in 32 registers or fewer, where there are four waves of them for every CU; a row of its
// own workgroup otherwise.  (20 alternatives, wave / workgroup in us: 65536 rows of bf16 x 4096 245 / 289, x 3000
// 194 / 261, of fp32 x 2048 145 / 228; 8192 rows 34 / 37, -, 26 / 32; 1100 rows 12 / 11, -, 11 / 11; fp32 x 4096, in 64
// registers, 65536 rows 319 / 310; one bf16 row of 3000 8.8 / 6.3.)
bool by_wave(int T, int V, bool f32) { return T >= 1024 && V <= (f32 ? 2048 : 4096); }

// Ranges of a row: a workgroup takes up to kStreamCols columns, and rows too few to give every CU two workgroups
// are cut further, down to 8192 columns.
int part_len(int T, int V) {
  const int least = (V + kStreamCols - 1) / kStreamCols, most = (V + 8191) / 8192;
  const int wanted = (512 + T - 1) / T;
  const int n = wanted < least ? least : wanted > most ? most : wanted;
  return ((V + n - 1) / n + 2047) / 2048 * 2048;
}

template <class X, bool DIST, bool TOP>
int launch_rows(const void* logits, RowArgs a, void* ws, hipStream_t s) {
  const X* x = static_cast<const X*>(logits);
  if (by_wave(a.T, a.V, Row<X>::VE == 4)) {
    auto fn = rows_wave_kernel<X, 32, DIST, TOP>;
    if constexpr (Row<X>::VE == 8) {
      if (a.V > 2048) fn = rows_wave_kernel<X, 64, DIST, TOP>;
    }
    hipLaunchKernelGGL(fn, dim3((a.T + 3) / 4), dim3(256), 0, s, x, a);
    return check_launch("token_loss_rows");
  }
  a.part = part_len(a.T, a.V);
  a.nparts = (a.V + a.part - 1) / a.part;
  const int64_t grid = (int64_t)a.T * a.nparts;
  RTE_REQUIRE(grid < ((int64_t)1 << 31), "token_loss: too many rows");
  a.part_stats = static_cast<float4*>(ws);
  a.part_keys = reinterpret_cast<u64*>(a.part_stats + grid);
  const int words = DIST ? (a.part + 31) / 32 : TOP ? (a.part + kStreamMax - 1) / kStreamMax * 256 : 0;
  hipLaunchKernelGGL((rows_stream_kernel<X, DIST, TOP>), dim3((unsigned)grid), dim3(256), words * sizeof(uint32_t), s, x, a);
  RTE_TRY(check_launch("token_loss_stream"));
  if (a.nparts == 1) return 0;
  hipLaunchKernelGGL((rows_join_kernel<X, DIST, TOP>), dim3(a.T), dim3(TOP ? 256 : 64), 0, s, x, a);
  return check_launch("token_loss_join");
}

size_t rows_workspace(int T, int V, int n_top) {
  if (T <= 0) return 0;
  const int part = part_len(T, V), n = (V + part - 1) / part;
  return n > 1 ? (size_t)T * n * (sizeof(float4) + n_top * sizeof(u64)) : 0;
}

bool fits_grid(int T, int V) { return (int64_t)T * ((V + kSeg - 1) / kSeg) < ((int64_t)1 << 31); }

}  // namespace
}  // namespace rte

using namespace rte;

extern "C" {

size_t rte_token_logprobs_workspace_bytes(int T, int V, int n_top) { return rows_workspace(T, V, n_top); }

int rte_token_logprobs_fwd(const void* logits, int64_t ld, int f32, int T, int V, const int64_t* tokens, float temperature,
                           int n_top, float* logprob, float* entropy, float* top_logprobs, int32_t* top_ids, float* stats,
                           void* ws, size_t ws_bytes, void* stream) {
  RTE_REQUIRE(T >= 0 && V >= 1 && ld >= 0, "token_logprobs: bad sizes");
  RTE_REQUIRE(n_top >= 0 && n_top <= kMaxTop && n_top <= V, "token_logprobs: n_top must be in [0, min(%d, V)]", kMaxTop);
  RTE_REQUIRE(temperature > 0.0f && temperature < INFINITY, "token_logprobs: temperature must be positive and finite");
  if (T == 0) return 0;
  RTE_REQUIRE(logits && tokens && logprob && entropy && (!n_top || (top_logprobs && top_ids)),
              "token_logprobs: null argument");
  RTE_REQUIRE(fits_grid(T, V), "token_logprobs: too many rows");
  const size_t need = rows_workspace(T, V, n_top);
  RTE_REQUIRE(ws_bytes >= need && (ws || !need), "token_logprobs: workspace too small");
  RowArgs a{};
  a.ld = ld, a.T = T, a.V = V;
  a.inv_t = 1.0f / temperature, a.c2 = (float)(1.4426950408889634 / temperature);
  a.tokens = tokens, a.n_top = n_top, a.logprob = logprob, a.entropy = entropy, a.top_lp = top_logprobs;
  a.top_ids = top_ids, a.stats = stats;
  auto s = static_cast<hipStream_t>(stream);
  if (f32) return n_top ? launch_rows<float, false, true>(logits, a, ws, s) : launch_rows<float, false, false>(logits, a, ws, s);
  return n_top ? launch_rows<bf16, false, true>(logits, a, ws, s) : launch_rows<bf16, false, false>(logits, a, ws, s);
}

int rte_token_logprobs_bwd(const void* logits, int64_t ld, int f32, int T, int V, const int64_t* tokens, float temperature,
                           const float* stats, const float* entropy, const float* g_logprob, const float* g_entropy,
                           void* dlogits, void* stream) {
  RTE_REQUIRE(T >= 0 && V >= 1 && ld >= 0, "token_logprobs_bwd: bad sizes");
  RTE_REQUIRE(temperature > 0.0f && temperature < INFINITY, "token_logprobs_bwd: temperature must be positive and finite");
  if (T == 0) return 0;
  RTE_REQUIRE(logits && tokens && stats && entropy && dlogits, "token_logprobs_bwd: null argument");
  RTE_REQUIRE(fits_grid(T, V), "token_logprobs_bwd: too many rows");
  auto s = static_cast<hipStream_t>(stream);
  const int nseg = (V + kSeg - 1) / kSeg;
  const int64_t items = (int64_t)T * nseg;
  const dim3 grid((unsigned)((items + 3) / 4));
  if (f32)
    hipLaunchKernelGGL(logprobs_bwd_kernel<float>, grid, dim3(256), 0, s, static_cast<const float*>(logits), ld, items, V,
                       nseg, tokens, 1.0f / temperature, stats, entropy, g_logprob, g_entropy, static_cast<float*>(dlogits));
  else
    hipLaunchKernelGGL(logprobs_bwd_kernel<bf16>, grid, dim3(256), 0, s, static_cast<const bf16*>(logits), ld, items, V,
                       nseg, tokens, 1.0f / temperature, stats, entropy, g_logprob, g_entropy, static_cast<bf16*>(dlogits));
  return check_launch("token_logprobs_bwd");
}

size_t rte_topk_distill_workspace_bytes(int T, int V, int K) {
  (void)K;
  return rows_workspace(T, V, 0);
}

int rte_topk_distill_fwd(const void* logits, int64_t ld, int f32, int T, int V, const int32_t* ids,
                         const float* teacher, int K, float temperature, int tail, float* loss, float* stats,
                         int32_t* cols, float* coef, void* ws, size_t ws_bytes, void* stream) {
  RTE_REQUIRE(T >= 0 && V >= 1 && ld >= 0, "topk_distill: bad sizes");
  RTE_REQUIRE(K >= 1 && K <= kMaxTop, "topk_distill: list length must be in [1, %d]", kMaxTop);
  RTE_REQUIRE(tail >= 0 && tail <= 3, "topk_distill: tail must be in [0, 3]");
  RTE_REQUIRE(temperature > 0.0f && temperature < INFINITY, "topk_distill: temperature must be positive and finite");
  if (T == 0) return 0;
  RTE_REQUIRE(logits && ids && teacher && loss && (!stats || (cols && coef)), "topk_distill: null argument");
  RTE_REQUIRE(fits_grid(T, V), "topk_distill: too many rows");
  const size_t need = rows_workspace(T, V, 0);
  RTE_REQUIRE(ws_bytes >= need && (ws || !need), "topk_distill: workspace too small");
  RowArgs a{};
  a.ld = ld, a.T = T, a.V = V;
  a.inv_t = 1.0f / temperature, a.c2 = (float)(1.4426950408889634 / temperature);
  a.ids = ids, a.tl = teacher, a.K = K, a.tail = tail, a.it = 1.0 / temperature;
  a.kept = tail == 2 ? 0x1.1p-8 : tail == 3 ? 0x1.1p-11 : 0.0;
  a.t2 = (double)temperature * temperature, a.loss = loss, a.stats = stats, a.cols = cols, a.coef = coef;
  auto s = static_cast<hipStream_t>(stream);
  return f32 ? launch_rows<float, true, false>(logits, a, ws, s) : launch_rows<bf16, true, false>(logits, a, ws, s);
}

int rte_topk_distill_bwd(const void* logits, int64_t ld, int f32, int T, int V, int K, float temperature,
                         const float* stats, const int32_t* cols, const float* coef, const float* g, void* dlogits,
                         void* stream) {
  RTE_REQUIRE(T >= 0 && V >= 1 && ld >= 0 && K >= 1 && K <= kMaxTop, "topk_distill_bwd: bad sizes");
  RTE_REQUIRE(temperature > 0.0f && temperature < INFINITY, "topk_distill_bwd: temperature must be positive and finite");
  if (T == 0) return 0;
  RTE_REQUIRE(logits && stats && cols && coef && g && dlogits, "topk_distill_bwd: null argument");
  RTE_REQUIRE(fits_grid(T, V), "topk_distill_bwd: too many rows");
  auto s = static_cast<hipStream_t>(stream);
  const int nseg = (V + kSeg - 1) / kSeg;
  const int64_t items = (int64_t)T * nseg;
  const dim3 grid((unsigned)((items + 3) / 4));
  const float c2 = (float)(1.4426950408889634 / temperature);
  if (f32)
    hipLaunchKernelGGL(distill_bwd_kernel<float>, grid, dim3(256), 0, s, static_cast<const float*>(logits), ld, items, V,
                       nseg, K, c2, temperature, stats, cols, coef, g, static_cast<float*>(dlogits));
  else
    hipLaunchKernelGGL(distill_bwd_kernel<bf16>, grid, dim3(256), 0, s, static_cast<const bf16*>(logits), ld, items, V,
                       nseg, K, c2, temperature, stats, cols, coef, g, static_cast<bf16*>(dlogits));
  return check_launch("topk_distill_bwd");
}

}  // extern "C"
