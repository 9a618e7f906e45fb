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
//   dx_v  = g t (q_v - p_j) where v = c_j, else g t (q_v - r q_v / q(R)) (tail 0: r = 0)
#include "../../include/rte_hip.h"
#include "common.hpp"

namespace rte {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxTop = 128;  // alternatives or list entries per row

__device__ __forceinline__ float logit(const float* x, int64_t i) { return x[i]; }
__device__ __forceinline__ float logit(const bf16* x, int64_t i) { return bf2f(x[i]); }
__device__ __forceinline__ void put(float* x, int64_t i, float v) { x[i] = v; }
__device__ __forceinline__ void put(bf16* x, int64_t i, float v) { x[i] = f2bf(v); }

// Order of the alternatives as unsigned keys: larger value first, -0 = +0, NaN above everything.
__device__ __forceinline__ uint32_t value_key(float x) {
  if (x != x) return 0xfffffffeu;
  const uint32_t b = __float_as_uint(x + 0.0f);
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}

template <class F>
__device__ __forceinline__ float block_reduce(float v, F f, float* red) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = f(v, __shfl_xor(v, o, 64));
  __syncthreads();
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
  __syncthreads();
  v = red[0];
  for (int i = 1; i < kThreads / 64; ++i) v = f(v, red[i]);
  return v;
}
struct Max {
  __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
};
struct Sum {
  __device__ float operator()(float a, float b) const { return a + b; }
};

template <class X>
__global__ void __launch_bounds__(kThreads)
    logprobs_fwd_kernel(const X* __restrict__ logits, int64_t ld, int V, const int64_t* __restrict__ tokens,
                        float inv_t, int n_top, float* __restrict__ logprob, float* __restrict__ entropy,
                        float* __restrict__ top_lp, int32_t* __restrict__ top_ids, float* __restrict__ stats) {
  __shared__ float red[kThreads / 64];
  __shared__ unsigned long long best[kThreads / 64];
  const int64_t t = blockIdx.x;
  const X* row = logits + t * ld;
  float m = -INFINITY;
  for (int v = threadIdx.x; v < V; v += kThreads) m = fmaxf(m, logit(row, v));
  m = block_reduce(m, Max(), red);
  const bool none = m == -INFINITY;  // no column is possible (a row of NaN keeps its NaN through S)
  float s = 0.0f, su = 0.0f;
  for (int v = threadIdx.x; v < V; v += kThreads) {
    const float u = (logit(row, v) - (none ? 0.0f : m)) * inv_t;
    const float e = __expf(u);
    s += e;
    su += e * fmaxf(u, -200.0f);
  }
  s = block_reduce(s, Sum(), red);
  su = block_reduce(su, Sum(), red);
  const bool empty = none && s == 0.0f;
  const float log_s = logf(s);
  if (threadIdx.x == 0) {
    const int64_t tok = tokens[t];
    float lp = 0.0f;
    if (tok >= V) lp = __builtin_nanf("");
    else if (tok >= 0) lp = empty ? -INFINITY : (logit(row, tok) - m) * inv_t - log_s;
    logprob[t] = lp;
    entropy[t] = empty ? 0.0f : log_s - su / s;
    if (stats) {
      stats[2 * t] = m;
      stats[2 * t + 1] = log_s;
    }
  }
  unsigned long long last = ~0ull;
  for (int j = 0; j < n_top; ++j) {
    unsigned long long top = 0;
    for (int v = threadIdx.x; v < V; v += kThreads) {
      const unsigned long long key = (unsigned long long)value_key(logit(row, v)) << 32 | (uint32_t)~v;
      if (key < last && key > top) top = key;
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) {
      const unsigned long long other = __shfl_xor(top, o, 64);
      top = other > top ? other : top;
    }
    __syncthreads();
    if ((threadIdx.x & 63) == 0) best[threadIdx.x >> 6] = top;
    __syncthreads();
    for (int i = 0; i < kThreads / 64; ++i) top = best[i] > top ? best[i] : top;
    last = top;
    if (threadIdx.x == 0) {
      const int v = (int)~(uint32_t)top;
      top_ids[t * n_top + j] = v;
      top_lp[t * n_top + j] = empty ? -INFINITY : (logit(row, v) - m) * inv_t - log_s;
    }
  }
}

template <class X>
__global__ void __launch_bounds__(kThreads)
    logprobs_bwd_kernel(const X* __restrict__ logits, int64_t ld, int V, const int64_t* __restrict__ tokens,
                        float inv_t, const float* __restrict__ stats, const float* __restrict__ entropy,
                        const float* __restrict__ g_lp, const float* __restrict__ g_ent, X* __restrict__ dlogits) {
  const int64_t t = blockIdx.x;
  const X* row = logits + t * ld;
  X* out = dlogits + t * V;
  const float m = stats[2 * t], log_s = stats[2 * t + 1], h = entropy[t];
  const int64_t tok = tokens[t];
  const float g = g_lp && tok >= 0 && tok < V ? g_lp[t] : 0.0f, gh = g_ent ? g_ent[t] : 0.0f;
  const bool empty = log_s == -INFINITY;
  for (int v = threadIdx.x; v < V; v += kThreads) {
    const float lp = (logit(row, v) - m) * inv_t - log_s;
    const float d = (v == tok ? g : 0.0f) - __expf(lp) * (g + gh * (fmaxf(lp, -200.0f) + h));
    put(out, v, empty ? 0.0f : d * inv_t);
  }
}

// Row statistics of the divergence, kept for the backward: {max, log S of the whole row (relative to max),
// log of the teacher's normaliser (tail 0: of e^{(t_j - max t) / t}), the teacher's rest r}, then the
// rest's log sum relative to max.
constexpr int kDistillStats = 6;
enum { D_MAX, D_LOGS, D_TMAX, D_TLOG, D_REST, D_LOGR };

// Whether entry j is the first of its column and inside the vocabulary.
__device__ __forceinline__ bool counts(const int32_t* ids, int j, int V) {
  const int c = ids[j];
  if (c < 0 || c >= V) return false;
  for (int i = 0; i < j; ++i)
    if (ids[i] == c) return false;
  return true;
}

template <class X>
__global__ void __launch_bounds__(kThreads)
    distill_fwd_kernel(const X* __restrict__ logits, int64_t ld, int V, const int32_t* __restrict__ ids,
                       const float* __restrict__ tl, int K, float temp, int tail, float* __restrict__ loss,
                       float* __restrict__ stats) {
  __shared__ float red[kThreads / 64];
  __shared__ uint8_t first[kMaxTop];
  const int64_t t = blockIdx.x;
  const X* row = logits + t * ld;
  ids += t * K;
  tl += t * K;
  const float inv_t = 1.0f / temp;
  if (threadIdx.x < K) first[threadIdx.x] = counts(ids, threadIdx.x, V);
  __syncthreads();
  float m = -INFINITY;
  for (int v = threadIdx.x; v < V; v += kThreads) m = fmaxf(m, logit(row, v));
  m = block_reduce(m, Max(), red);
  const bool none = m == -INFINITY;
  const float m0 = none ? 0.0f : m;
  float s = 0.0f;
  for (int v = threadIdx.x; v < V; v += kThreads) {
    bool listed = false;
    for (int j = 0; j < K; ++j) listed |= ids[j] == v;
    s += listed ? 0.0f : __expf((logit(row, v) - m0) * inv_t);
  }
  s = block_reduce(s, Sum(), red);
  if (threadIdx.x != 0) return;
  bool bad = false, some = false;
  double tmax = -INFINITY;
  for (int j = 0; j < K; ++j) {
    bad |= ids[j] >= V;
    if (!first[j]) continue;
    some = true;
    tmax = fmax(tmax, (double)tl[j]);
  }
  if (!tail && tmax == -INFINITY) some = false;  // the list holds no probability
  const double it = 1.0 / (double)temp;
  double rest = s, total = rest, tsum = 0.0, psum = 0.0;
  for (int j = 0; j < K; ++j) {
    if (!first[j]) continue;
    total += exp(((double)logit(row, ids[j]) - m0) * it);
    tsum += exp(((double)tl[j] - tmax) * it);
  }
  const double log_s = log(total), tlog = log(tsum);
  const bool empty = total == 0.0;
  double l = 0.0;
  for (int j = 0; j < K; ++j) {
    if (!first[j]) continue;
    const double lp = tail ? (double)tl[j] : ((double)tl[j] - tmax) * it - tlog;
    const double lq = empty ? -INFINITY : ((double)logit(row, ids[j]) - m0) * it - log_s;
    const double p = exp(lp);
    psum += p;
    if (p > 0.0 || lp != lp) l += p * (lp - lq);
  }
  double r = tail ? fmax(1.0 - psum, 0.0) : 0.0;
  if (r > 0.0) l += r * (log(r) - (empty ? -INFINITY : log(rest) - log_s));
  if (bad) l = __builtin_nan("");
  loss[t] = some || bad ? (float)(l * temp * temp) : 0.0f;
  if (stats) {
    stats += t * kDistillStats;
    stats[D_MAX] = m0;
    stats[D_LOGS] = (float)log_s;
    stats[D_TMAX] = some && !bad ? (float)tmax : __builtin_nanf("");
    stats[D_TLOG] = (float)tlog;
    stats[D_REST] = (float)r;
    stats[D_LOGR] = (float)log(rest);
  }
}

template <class X>
__global__ void __launch_bounds__(kThreads)
    distill_bwd_kernel(const X* __restrict__ logits, int64_t ld, int V, const int32_t* __restrict__ ids,
                       const float* __restrict__ tl, int K, float temp, int tail, const float* __restrict__ stats,
                       const float* __restrict__ g, X* __restrict__ dlogits) {
  const int64_t t = blockIdx.x;
  const X* row = logits + t * ld;
  X* out = dlogits + t * V;
  ids += t * K;
  tl += t * K;
  stats += t * kDistillStats;
  const float inv_t = 1.0f / temp, gt = g[t] * temp;
  const float m = stats[D_MAX], log_s = stats[D_LOGS], r = stats[D_REST], log_r = stats[D_LOGR];
  const float tmax = stats[D_TMAX], tlog = stats[D_TLOG];
  const bool skip = tmax != tmax || log_s == -INFINITY;
  for (int v = threadIdx.x; v < V; v += kThreads) {
    int at = -1;
    for (int j = K - 1; j >= 0; --j)
      if (ids[j] == v) at = j;
    const float u = (logit(row, v) - m) * inv_t;
    float d = __expf(u - log_s);
    if (at >= 0) d -= __expf(tail ? tl[at] : (tl[at] - tmax) * inv_t - tlog);
    else if (r > 0.0f) d -= r * __expf(u - log_r);
    put(out, v, skip ? 0.0f : gt * d);
  }
}

}  // namespace
}  // namespace rte

using namespace rte;

extern "C" {

size_t rte_token_logprobs_workspace_bytes(int T, int V, int n_top) { return 0; }

int rte_token_logprobs_fwd(const void* logits, int64_t ld, int f32, int T, int V, const int64_t* tokens, float temperature,
                           int n_top, float* logprob, float* entropy, float* top_logprobs, int32_t* top_ids, float* stats,
                           void* ws, size_t ws_bytes, void* stream) {
  RTE_REQUIRE(T >= 0 && V >= 1 && ld >= 0, "token_logprobs: bad sizes");
  RTE_REQUIRE(n_top >= 0 && n_top <= kMaxTop && n_top <= V, "token_logprobs: n_top must be in [0, min(%d, V)]", kMaxTop);
  RTE_REQUIRE(temperature > 0.0f && temperature < INFINITY, "token_logprobs: temperature must be positive and finite");
  if (T == 0) return 0;
  RTE_REQUIRE(logits && tokens && logprob && entropy && (!n_top || (top_logprobs && top_ids)),
              "token_logprobs: null argument");
  auto s = static_cast<hipStream_t>(stream);
  if (f32)
    hipLaunchKernelGGL(logprobs_fwd_kernel<float>, dim3(T), dim3(kThreads), 0, s, static_cast<const float*>(logits), ld,
                       V, tokens, 1.0f / temperature, n_top, logprob, entropy, top_logprobs, top_ids, stats);
  else
    hipLaunchKernelGGL(logprobs_fwd_kernel<bf16>, dim3(T), dim3(kThreads), 0, s, static_cast<const bf16*>(logits), ld, V,
                       tokens, 1.0f / temperature, n_top, logprob, entropy, top_logprobs, top_ids, stats);
  return check_launch("token_logprobs_fwd");
}

int rte_token_logprobs_bwd(const void* logits, int64_t ld, int f32, int T, int V, const int64_t* tokens, float temperature,
                           const float* stats, const float* entropy, const float* g_logprob, const float* g_entropy,
                           void* dlogits, void* stream) {
  RTE_REQUIRE(T >= 0 && V >= 1 && ld >= 0, "token_logprobs_bwd: bad sizes");
  RTE_REQUIRE(temperature > 0.0f && temperature < INFINITY, "token_logprobs_bwd: temperature must be positive and finite");
  if (T == 0) return 0;
  RTE_REQUIRE(logits && tokens && stats && entropy && dlogits, "token_logprobs_bwd: null argument");
  auto s = static_cast<hipStream_t>(stream);
  if (f32)
    hipLaunchKernelGGL(logprobs_bwd_kernel<float>, dim3(T), dim3(kThreads), 0, s, static_cast<const float*>(logits), ld,
                       V, tokens, 1.0f / temperature, stats, entropy, g_logprob, g_entropy, static_cast<float*>(dlogits));
  else
    hipLaunchKernelGGL(logprobs_bwd_kernel<bf16>, dim3(T), dim3(kThreads), 0, s, static_cast<const bf16*>(logits), ld, V,
                       tokens, 1.0f / temperature, stats, entropy, g_logprob, g_entropy, static_cast<bf16*>(dlogits));
  return check_launch("token_logprobs_bwd");
}

size_t rte_topk_distill_workspace_bytes(int T, int V, int K) { return 0; }

int rte_topk_distill_fwd(const void* logits, int64_t ld, int f32, int T, int V, const int32_t* ids,
                         const float* teacher, int K, float temperature, int tail, float* loss, float* stats, void* ws,
                         size_t ws_bytes, void* stream) {
  RTE_REQUIRE(T >= 0 && V >= 1 && ld >= 0, "topk_distill: bad sizes");
  RTE_REQUIRE(K >= 1 && K <= kMaxTop, "topk_distill: list length must be in [1, %d]", kMaxTop);
  RTE_REQUIRE(temperature > 0.0f && temperature < INFINITY, "topk_distill: temperature must be positive and finite");
  if (T == 0) return 0;
  RTE_REQUIRE(logits && ids && teacher && loss, "topk_distill: null argument");
  auto s = static_cast<hipStream_t>(stream);
  if (f32)
    hipLaunchKernelGGL(distill_fwd_kernel<float>, dim3(T), dim3(kThreads), 0, s, static_cast<const float*>(logits), ld, V,
                       ids, teacher, K, temperature, tail, loss, stats);
  else
    hipLaunchKernelGGL(distill_fwd_kernel<bf16>, dim3(T), dim3(kThreads), 0, s, static_cast<const bf16*>(logits), ld, V,
                       ids, teacher, K, temperature, tail, loss, stats);
  return check_launch("topk_distill_fwd");
}

int rte_topk_distill_bwd(const void* logits, int64_t ld, int f32, int T, int V, const int32_t* ids,
                         const float* teacher, int K, float temperature, int tail, const float* stats, const float* g,
                         void* dlogits, void* stream) {
  RTE_REQUIRE(T >= 0 && V >= 1 && ld >= 0 && K >= 1 && K <= kMaxTop, "topk_distill_bwd: bad sizes");
  RTE_REQUIRE(temperature > 0.0f && temperature < INFINITY, "topk_distill_bwd: temperature must be positive and finite");
  if (T == 0) return 0;
  RTE_REQUIRE(logits && ids && teacher && stats && g && dlogits, "topk_distill_bwd: null argument");
  auto s = static_cast<hipStream_t>(stream);
  if (f32)
    hipLaunchKernelGGL(distill_bwd_kernel<float>, dim3(T), dim3(kThreads), 0, s, static_cast<const float*>(logits), ld, V,
                       ids, teacher, K, temperature, tail, stats, g, static_cast<float*>(dlogits));
  else
    hipLaunchKernelGGL(distill_bwd_kernel<bf16>, dim3(T), dim3(kThreads), 0, s, static_cast<const bf16*>(logits), ld, V,
                       ids, teacher, K, temperature, tail, stats, g, static_cast<bf16*>(dlogits));
  return check_launch("topk_distill_bwd");
}

}  // extern "C"
