// Log probabilities of tokens and entropies straight from hidden states h [T, d] and the vocabulary matrix
// w [V, d]: the logits x = h w^T live in the product's accumulators only (the formulas are those of
// token_loss.hip).
//
// Forward: the tile product w h^T leaves, for every row of h and 64 or 128 tokens of the vocabulary, {max, sum,
// sum of e u}: a 16th or 32nd of the fp32 logits; a second launch joins a row's blocks.  Sums and logarithms are in
// units of log 2, relative to the rounded maximum itself.  Backward: the product again, whose epilogue writes the
// logits' gradient in bf16 for the two products that follow (dh = dx w, dw = dx^T h).  Bound by the matrix units: 8192
// tokens of d 1024, vocabulary 32768, 537 + 9 us forward, 558 + 446 + 18 + 433 backward.  Keeping the logits instead of
// the second product would hold them from forward to backward: in bf16 0.54 GB, written and read in 165 us at 6.5 TB/s,
// but a logit of 10 would be off by up to 2^-5 there and so would its probability; in fp32 1.07 GB and 330 us.
// The logits' gradient is rounded to bf16 for the products with h and w, which take no more on the matrix units: over
// these sizes dh and dw in bf16 are 0.0024 of their norm off the exact ones, 0.0017 by their own rounding.
#include "../../include/rte_hip.h"
#include "gemm_tile.hpp"
#include "row_words.hpp"

namespace rte {

int cast_f32_bf16(const float* x, int64_t n, bf16* y, hipStream_t s);

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
  stats[2 * t] = a.m;
  stats[2 * t + 1] = log_s;
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

// Rows lo .. lo + n of w [V, d] with zeros past V (their logits' gradients add nothing to dh).
__global__ void head_pad_kernel(const bf16* __restrict__ w, int lo, int V, int64_t d, int64_t n, bf16* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i < n * d) out[i] = lo + i / d < V ? w[lo * d + i] : 0;
}

__global__ void head_rows_out_kernel(const float* __restrict__ x, int64_t n, int f32, void* __restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  if (f32) static_cast<float*>(out)[i] = x[i];
  else static_cast<bf16*>(out)[i] = f2bf(x[i]);
}

// out [M, N] (+)= the product of two operands given as in memory, on the library's dense GEMM.
int product(const void* a, int64_t lda, int a_t, const void* b, int64_t ldb, int b_t, void* out, int f32, int M, int N, int K,
            float beta, void* ws, size_t ws_bytes, hipStream_t s) {
  GemmArgs p;
  p.a.ptr = static_cast<const bf16*>(a);
  p.a.ld = lda;
  p.b.ptr = static_cast<const bf16*>(b);
  p.b.ld = ldb;
  p.a_t = a_t, p.b_t = b_t;
  p.M = M, p.N = N, p.K = K;
  p.epi.c = out;
  p.epi.ldc = N;
  p.epi.c_f32 = f32;
  p.epi.beta = beta;
  return gemm_launch(p, EPI_STORE, s, ws, ws_bytes);
}

size_t up(size_t n) { return (n + 255) / 256 * 256; }

// The backward's vocabulary ranges: `width` columns each (a multiple of 64) over the whole 64s, then the rest.
struct Ranges {
  int width, whole, rest, rest8;
  Ranges(int V, int w) : width(w), whole(V / 64 * 64), rest(V % 64), rest8((V % 64 + 7) / 8 * 8) {
    if (width > whole) width = whole;
  }
  int most() const { return width > rest8 ? width : rest8; }
  bool one() const { return whole == 0 || (rest == 0 && width == whole); }
};

struct BwdSpace {
  size_t grad, dh, pad, tail, gemm, total;
  BwdSpace(int T, int d, int V, const Ranges& r, bool h, bool h_f32, bool w) {
    grad = 0;
    dh = grad + up((size_t)T * r.most() * sizeof(bf16));  // fp32 sums of several ranges on their way to bf16
    pad = dh + (h && !h_f32 && !r.one() ? up((size_t)T * d * sizeof(float)) : 0);
    const bool ragged = r.rest8 != r.rest;
    tail = pad + (ragged ? up((size_t)r.rest8 * d * sizeof(bf16)) : 0);
    gemm = tail + (ragged && w ? up((size_t)r.rest8 * d * sizeof(float)) : 0);
    size_t g = 0;
    for (int n : {r.width, r.whole ? (r.whole - 1) % (r.width ? r.width : 1) + 1 : 0, r.rest8}) {
      if (n <= 0) continue;
      if (h && gemm_splitk_bytes(T, d, n) > g) g = gemm_splitk_bytes(T, d, n);
      if (w && gemm_splitk_bytes(n, d, T) > g) g = gemm_splitk_bytes(n, d, T);
    }
    total = gemm + up(g);
  }
};

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

size_t rte_lm_head_logprobs_bwd_workspace_bytes(int T, int d, int V, int width, int need_dh, int need_dw) {
  if (!rte_lm_head_logprobs_ok(T, d, V) || width < 64 || width % 64 != 0) return 0;
  return BwdSpace(T, d, V, Ranges(V, width), need_dh, need_dh == 2, need_dw).total;
}

int rte_lm_head_logprobs_bwd(const void* hidden, const void* w, int T, int d, int V, const int64_t* tokens,
                             float temperature, const float* stats, const float* entropy, const float* g_logprob,
                             const float* g_entropy, int width, void* dhidden, void* dw, int grads_f32, void* ws,
                             size_t ws_bytes, void* stream) {
  RTE_REQUIRE(rte_lm_head_logprobs_ok(T, d, V), "lm_head_logprobs_bwd: size not taken (T %d, d %d, V %d)", T, d, V);
  RTE_REQUIRE(width >= 64 && width % 64 == 0, "lm_head_logprobs_bwd: width must be a positive multiple of 64");
  RTE_REQUIRE(temperature > 0.0f && temperature < INFINITY, "lm_head_logprobs_bwd: temperature must be positive and finite");
  RTE_REQUIRE(hidden && w && tokens && stats && entropy, "lm_head_logprobs_bwd: null argument");
  RTE_REQUIRE(aligned(hidden) && aligned(w) && aligned(dhidden) && aligned(dw) && aligned(ws),
              "lm_head_logprobs_bwd: operands must be 16-byte aligned");
  RTE_REQUIRE(grads_f32 >= 0 && grads_f32 <= 3, "lm_head_logprobs_bwd: grads_f32 must be in [0, 3]");
  if (!dhidden && !dw) return 0;
  const bool dw_f32 = grads_f32 & 1, dh_f32 = grads_f32 & 2;
  const Ranges r(V, width);
  const BwdSpace at(T, d, V, r, dhidden != nullptr, dh_f32, dw != nullptr);
  RTE_REQUIRE((int64_t)T * r.most() < (int64_t)1 << 30, "lm_head_logprobs_bwd: width too large for %d rows", T);
  RTE_REQUIRE(ws && ws_bytes >= at.total, "lm_head_logprobs_bwd: workspace too small");
  auto s = static_cast<hipStream_t>(stream);
  char* base = static_cast<char*>(ws);
  void* grad = base + at.grad;
  void* gemm_ws = base + at.gemm;
  const size_t gemm_bytes = at.total - at.gemm;
  // sums of several ranges are kept in fp32
  const bool dh_sum = !dh_f32 && !r.one();
  float* dh32 = reinterpret_cast<float*>(base + at.dh);
  for (int lo = 0; lo < V;) {
    const bool last = lo == r.whole;  // the columns past the whole 64s
    int n = last ? r.rest8 : r.whole - lo < r.width ? r.whole - lo : r.width;
    const int real = last ? r.rest : n;
    const bf16* wr = static_cast<const bf16*>(w) + (int64_t)lo * d;
    if (n != real) {
      bf16* pad = reinterpret_cast<bf16*>(base + at.pad);
      hipLaunchKernelGGL(head_pad_kernel, dim3((unsigned)(((int64_t)n * d + 255) / 256)), dim3(256), 0, s,
                         static_cast<const bf16*>(w), lo, V, (int64_t)d, (int64_t)n, pad);
      RTE_TRY(check_launch("lm_head_pad"));
      wr = pad;
    }
    Epilogue e;
    e.c = grad;
    e.ldc = n;
    e.c2 = (float)(1.4426950408889634 / temperature);
    e.col0 = lo;
    e.cols = real;
    e.tokens = tokens;
    e.row_stats = stats;
    e.row_entropy = entropy;
    e.g_lp = g_logprob;
    e.g_ent = g_entropy;
    e.inv_t = 1.0f / temperature;
    e.vocab = V;
    RTE_TRY(tiles(wr, hidden, n, T, d, e, EPI_DLOGITS, s));
    if (dhidden)  // [T, n] [n, d]
      RTE_TRY(product(grad, n, 0, wr, d, 1, dh_sum ? dh32 : dhidden, dh_f32 || dh_sum, T, d, n, lo > 0 ? 1.0f : 0.0f, gemm_ws,
                      gemm_bytes, s));
    if (dw) {     // [n, T] [T, d]
      void* out = static_cast<char*>(dw) + (int64_t)lo * d * (dw_f32 ? 4 : 2);
      float* tail = reinterpret_cast<float*>(base + at.tail);
      const bool direct = n == real;
      RTE_TRY(product(grad, n, 1, hidden, d, 1, direct ? out : tail, direct ? dw_f32 : 1, n, d, T, 0.0f, gemm_ws, gemm_bytes,
                      s));
      if (!direct) {
        const int64_t k = (int64_t)real * d;
        hipLaunchKernelGGL(head_rows_out_kernel, dim3((unsigned)((k + 255) / 256)), dim3(256), 0, s, tail, k, dw_f32, out);
        RTE_TRY(check_launch("lm_head_rows_out"));
      }
    }
    lo += real;
  }
  return dhidden && dh_sum ? cast_f32_bf16(dh32, (int64_t)T * d, static_cast<bf16*>(dhidden), s) : 0;
}

}  // extern "C"
