// Log probabilities of tokens and entropies straight from hidden states h [T, d] and the vocabulary matrix
// w [V, d]: the logits x = h w^T live in the product's accumulators only (the formulas are those of
// token_loss.hip).
//
// Forward: the tile product w h^T leaves, for every row of h and 64 or 128 tokens of the vocabulary, {max, sum,
// sum of e u}: a 32nd of the fp32 logits; a second launch joins a row's blocks.  Sums and logarithms are in
// units of log 2, relative to the rounded maximum itself.  Backward: the product again, whose epilogue writes the
// logits' gradient in bf16 for the two products that follow (dh = dx w, dw = dx^T h).
#include "../../include/rte_hip.h"
#include "gemm_tile.hpp"
#include "row_words.hpp"

namespace rte {

namespace {

constexpr int kRows = 16, kSlices = 16;  // of a join workgroup: sixteen rows' blocks are read 256 bytes at a time

struct Sum3 {  // relative to m, in units of log 2
  float m, s, su;
  __device__ void add(const Sum3& o) {
    const float top = fmaxf(m, o.m), ua = fmaxf(m - top, -256.0f), ub = fmaxf(o.m - top, -256.0f);
    const float a = exp2_(ua), b = exp2_(ub);
    su = a * (su + s * ua) + b * (o.su + o.s * ub);
    s = s * a + o.s * b;
    m = top;
  }
};

constexpr float kLowest = -3.0e38f;  // of a block that holds nothing

__global__ void __launch_bounds__(kRows* kSlices)
    head_join_kernel(const float4* __restrict__ part, int np, int T, int V, const float* __restrict__ tok_logit,
                     const int64_t* __restrict__ tokens, float c2, float* __restrict__ logprob,
                     float* __restrict__ entropy, float* __restrict__ stats) {
  __shared__ Sum3 slices[kSlices][kRows];
  const int r = threadIdx.x % kRows, q = threadIdx.x / kRows;
  const int64_t t = (int64_t)blockIdx.x * kRows + r;
  Sum3 a{kLowest, 0.0f, 0.0f};
  if (t < T) {
    for (int p0 = q; p0 < np; p0 += 8 * kSlices) {
      float4 x[8];
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int p = p0 + u * kSlices;
        x[u] = p < np ? part[(int64_t)p * T + t] : make_float4(kLowest, 0.0f, 0.0f, 0.0f);
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) a.add(Sum3{x[u].x, x[u].y, x[u].z});
    }
  }
  slices[q][r] = a;
  __syncthreads();
  if (q != 0 || t >= T) return;
  for (int i = 1; i < kSlices; ++i) a.add(slices[i][r]);
  const int64_t tok = tokens[t];
  const float log_s = log2f(a.s);
  const bool empty = a.s == 0.0f;
  logprob[t] = tok >= V   ? __builtin_nanf("")
               : tok < 0 ? 0.0f
               : empty   ? -INFINITY
                         : (__builtin_fmaf(tok_logit[t], c2, -a.m) - log_s) * kLn2;
  entropy[t] = empty ? 0.0f : (log_s - a.su / a.s) * kLn2;
  stats[t] = a.m + log_s;
}

// What the backward's epilogue needs of a row: with l = log2 p, dx_v = p_v (a + b l) + [v = token] g / t,
// a = -(g + g_H entropy) / t, b = -g_H ln 2 / t.
__global__ void head_rows_kernel(int T, int V, const int64_t* __restrict__ tokens, const float* __restrict__ stats,
                                 const float* __restrict__ entropy, const float* __restrict__ g_lp,
                                 const float* __restrict__ g_ent, float inv_t, float4* __restrict__ rows) {
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= T) return;
  const int64_t tok = tokens[t];
  const float g = g_lp && tok >= 0 && tok < V ? g_lp[t] * inv_t : 0.0f, gh = g_ent ? g_ent[t] * inv_t : 0.0f;
  rows[t] = make_float4(stats[t], -(g + gh * entropy[t]), -gh * kLn2, g);
}

// The product w h^T over n rows of w on the tile kernels.
int tiles(const void* w, const void* h, int n, int T, int d, const Epilogue& e, int kind, hipStream_t s) {
  GemmArgs p;
  p.a.ptr = static_cast<const bf16*>(w);
  p.b.ptr = static_cast<const bf16*>(h);
  p.a.ld = p.b.ld = d;
  p.M = n, p.N = T, p.K = d;
  p.a_bytes = (uint32_t)((int64_t)n * d * 2);
  p.b_bytes = (uint32_t)((int64_t)T * d * 2);
  p.epi = e;
  int splits = 1;
  return gemm_tile_launch(p, kind, s, 1, nullptr, 0, &splits);
}

bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace
}  // namespace rte

using namespace rte;

extern "C" {

int rte_lm_head_logprobs_ok(int T, int d, int V) {
  const int64_t lim = (int64_t)1 << 30;  // elements of an operand: the tile kernels address 2^31 bytes
  return T >= 1 && V >= 1 && d % 64 == 0 && d >= kTileMinK && (int64_t)T * d < lim && (int64_t)V * d < lim;
}

size_t rte_lm_head_logprobs_workspace_bytes(int T, int V) {
  if (T <= 0 || V <= 0) return 0;
  return (size_t)T * ((V + 63) / 64) * sizeof(float4) + (size_t)T * sizeof(float);
}

int rte_lm_head_logprobs_fwd(const void* hidden, const void* w, int T, int d, int V, const int64_t* tokens,
                             float temperature, float* logprob, float* entropy, float* stats, void* ws, size_t ws_bytes,
                             void* stream) {
  RTE_REQUIRE(rte_lm_head_logprobs_ok(T, d, V), "lm_head_logprobs: size not taken (T %d, d %d, V %d)", T, d, V);
  RTE_REQUIRE(temperature > 0.0f && temperature < INFINITY, "lm_head_logprobs: temperature must be positive and finite");
  RTE_REQUIRE(hidden && w && tokens && logprob && entropy && stats, "lm_head_logprobs: null argument");
  RTE_REQUIRE(aligned(hidden) && aligned(w) && aligned(ws), "lm_head_logprobs: operands must be 16-byte aligned");
  RTE_REQUIRE(ws && ws_bytes >= rte_lm_head_logprobs_workspace_bytes(T, V), "lm_head_logprobs: workspace too small");
  auto s = static_cast<hipStream_t>(stream);
  const int np = gemm_tile_row_blocks(V, T, d);
  Epilogue e;
  e.c2 = (float)(1.4426950408889634 / temperature);
  e.tokens = tokens;
  e.row_part = static_cast<float4*>(ws);
  e.tok_logit = reinterpret_cast<float*>(e.row_part + (int64_t)T * np);
  RTE_TRY(tiles(w, hidden, V, T, d, e, EPI_ROW_SUMS, s));
  hipLaunchKernelGGL(head_join_kernel, dim3((T + kRows - 1) / kRows), dim3(kRows * kSlices), 0, s, e.row_part, np, T, V,
                     e.tok_logit, tokens, e.c2, logprob, entropy, stats);
  return check_launch("lm_head_logprobs_join");
}

size_t rte_lm_head_dlogits_workspace_bytes(int T) { return T > 0 ? (size_t)T * sizeof(float4) : 0; }

int rte_lm_head_dlogits(const void* hidden, const void* w_rows, int T, int d, int V, int col0, int n, const int64_t* tokens,
                        float temperature, const float* stats, const float* entropy, const float* g_logprob,
                        const float* g_entropy, void* dlogits, void* ws, size_t ws_bytes, void* stream) {
  RTE_REQUIRE(rte_lm_head_logprobs_ok(T, d, V), "lm_head_dlogits: size not taken (T %d, d %d, V %d)", T, d, V);
  RTE_REQUIRE(n >= 8 && n % 8 == 0 && col0 >= 0 && col0 < V && n - 8 < V - col0,
              "lm_head_dlogits: need a multiple of 8 columns that starts inside V and covers it at most");
  RTE_REQUIRE(temperature > 0.0f && temperature < INFINITY, "lm_head_dlogits: temperature must be positive and finite");
  RTE_REQUIRE(hidden && w_rows && tokens && stats && entropy && dlogits, "lm_head_dlogits: null argument");
  RTE_REQUIRE(aligned(hidden) && aligned(w_rows) && aligned(dlogits) && aligned(ws),
              "lm_head_dlogits: operands must be 16-byte aligned");
  RTE_REQUIRE(ws && ws_bytes >= rte_lm_head_dlogits_workspace_bytes(T), "lm_head_dlogits: workspace too small");
  auto s = static_cast<hipStream_t>(stream);
  Epilogue e;
  e.c = dlogits;
  e.ldc = n;
  e.c2 = (float)(1.4426950408889634 / temperature);
  e.col0 = col0;
  e.tokens = tokens;
  float4* rows = static_cast<float4*>(ws);
  e.row_in = rows;
  hipLaunchKernelGGL(head_rows_kernel, dim3((T + 255) / 256), dim3(256), 0, s, T, V, tokens, stats, entropy, g_logprob,
                     g_entropy, 1.0f / temperature, rows);
  RTE_TRY(check_launch("lm_head_rows"));
  return tiles(w_rows, hidden, n, T, d, e, EPI_DLOGITS, s);
}

}  // extern "C"
