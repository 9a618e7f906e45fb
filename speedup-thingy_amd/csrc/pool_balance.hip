// Load balance of routed pools.  For T rows of C router logits with the k pools each row was sent to:
//
//   p_t = softmax(x_t)     P_c = mean_t p_tc     counts_c = rows sent to c     f_c = counts_c / sum counts
//   balance = C sum_c f_c P_c     z = mean_t (log sum_c e^{x_tc})^2
//   dx_tc = p_tc (g_b C (f_c - sum_c' f_c' p_tc') + 2 g_z lse_t) / n
//
// over the n rows that the mask keeps and whose logits are not all -inf; other rows take no part and
// their logits may hold anything.  Pools outside [0, C) are none; a pool named twice counts twice.
#include "../../include/rte_hip.h"
#include "common.hpp"

namespace rte {

namespace {

constexpr int kMaxPools = 1024;
constexpr int kRows = 128;  // rows of a workgroup of four waves

__device__ __forceinline__ float logit(const float* x, int64_t i) { return x[i]; }
__device__ __forceinline__ float logit(const bf16* x, int64_t i) { return bf2f(x[i]); }
__device__ __forceinline__ void put(float* x, int64_t i, float v) { x[i] = v; }
__device__ __forceinline__ void put(bf16* x, int64_t i, float v) { x[i] = f2bf(v); }

__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int o = 32; o >= 1; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

constexpr int kPer = kMaxPools / 64;  // columns of a lane, lane + 64 i

// Logits of row t in v, its maximum and sum; false for a row that takes no part.
template <class X>
__device__ __forceinline__ bool load_row(const X* logits, int64_t ld, int64_t t, int C, const uint8_t* mask, int lane,
                                         float* v, float& m, float& s) {
  if (mask && !mask[t]) return false;
  m = -INFINITY;
  bool nan = false;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    v[i] = lane + 64 * i < C ? logit(logits + t * ld, lane + 64 * i) : -INFINITY;
    m = fmaxf(m, v[i]);
    nan |= v[i] != v[i];
  }
  m = wave_max(m);
  if (m == -INFINITY && !__any(nan)) return false;
  s = 0.0f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) s += __expf(v[i] - m);
  s = wave_sum(s);
  return true;
}

// Partials of a workgroup: [C] sums of p, [C] counts, sum of lse^2, rows.
template <class X>
__global__ void __launch_bounds__(256) balance_fwd_kernel(const X* __restrict__ logits, int64_t ld, int T, int C,
                                                          const int32_t* __restrict__ ids, int k,
                                                          const uint8_t* __restrict__ mask, float* __restrict__ part) {
  __shared__ float sum[4][kMaxPools];
  __shared__ int cnt[kMaxPools];
  __shared__ float zs[4];
  __shared__ int ns[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int c = threadIdx.x; c < C; c += 256) cnt[c] = 0;
  __syncthreads();
  float acc[kPer], v[kPer], z = 0.0f;
  int n = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) acc[i] = 0.0f;
  const int64_t t0 = (int64_t)blockIdx.x * kRows;
  const int64_t t1 = t0 + kRows < T ? t0 + kRows : T;
  for (int64_t t = t0 + wave; t < t1; t += 4) {
    float m, s;
    if (!load_row(logits, ld, t, C, mask, lane, v, m, s)) continue;
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc[i] += __expf(v[i] - m) / s;
    const float lse = m + logf(s);
    z += lse * lse;
    ++n;
    for (int j = lane; j < k; j += 64) {
      const int c = ids[t * k + j];
      if (c >= 0 && c < C) atomicAdd(&cnt[c], 1);
    }
  }
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (lane + 64 * i < C) sum[wave][lane + 64 * i] = acc[i];
  if (lane == 0) {
    zs[wave] = z;
    ns[wave] = n;
  }
  __syncthreads();
  float* out = part + (int64_t)blockIdx.x * (2 * C + 2);
  for (int c = threadIdx.x; c < C; c += 256) {
    out[c] = ((sum[0][c] + sum[1][c]) + sum[2][c]) + sum[3][c];
    reinterpret_cast<int*>(out)[C + c] = cnt[c];
  }
  if (threadIdx.x == 0) {
    out[2 * C] = ((zs[0] + zs[1]) + zs[2]) + zs[3];
    reinterpret_cast<int*>(out)[2 * C + 1] = ns[0] + ns[1] + ns[2] + ns[3];
  }
}

__global__ void __launch_bounds__(1024) balance_join_kernel(const float* __restrict__ part, int nblk, int C,
                                                            float* __restrict__ out, int32_t* __restrict__ counts,
                                                            float* __restrict__ frac) {
  __shared__ double red[1024];
  const int c = threadIdx.x;
  const int w = 2 * C + 2;
  double p = 0.0;
  long long n = 0;
  if (c < C)
    for (int b = 0; b < nblk; ++b) {
      p += part[(int64_t)b * w + c];
      n += reinterpret_cast<const int*>(part)[(int64_t)b * w + C + c];
    }
  auto total = [&](double v) {
    __syncthreads();
    red[c] = v;
    for (int o = 512; o >= 1; o >>= 1) {
      __syncthreads();
      if (c < o) red[c] += red[c + o];
    }
    __syncthreads();
    return red[0];
  };
  double z = 0.0, rows = 0.0;
  for (int b = c; b < nblk; b += 1024) {
    z += part[(int64_t)b * w + 2 * C];
    rows += reinterpret_cast<const int*>(part)[(int64_t)b * w + 2 * C + 1];
  }
  z = total(z);
  rows = total(rows);
  const double all = total((double)n);
  const double f = all > 0.0 ? (double)n / all : 0.0;
  const double bal = total(f * p);
  if (c < C) {
    counts[c] = (int32_t)n;
    frac[c] = (float)f;
  }
  if (c == 0) {
    const double inv = rows > 0.0 ? 1.0 / rows : 0.0;
    out[0] = (float)(C * bal * inv);
    out[1] = (float)(z * inv);
    frac[C] = (float)inv;
  }
}

template <class X>
__global__ void __launch_bounds__(256) balance_bwd_kernel(const X* __restrict__ logits, int64_t ld, int T, int C,
                                                          const uint8_t* __restrict__ mask,
                                                          const float* __restrict__ frac, const float* __restrict__ g_bal,
                                                          const float* __restrict__ g_z, X* __restrict__ dx) {
  const int lane = threadIdx.x & 63;
  const float inv_n = frac[C];
  const float gb = g_bal ? *g_bal * C * inv_n : 0.0f, gz = g_z ? *g_z * 2.0f * inv_n : 0.0f;
  const int64_t t = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (t >= T) return;
  float v[kPer], m, s;
  const bool here = load_row(logits, ld, t, C, mask, lane, v, m, s);
  float dot = 0.0f;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    if (lane + 64 * i >= C) continue;
    v[i] = here ? __expf(v[i] - m) / s : 0.0f;
    dot += v[i] * frac[lane + 64 * i];
  }
  dot = wave_sum(dot);
  const float lz = gz * (here ? m + logf(s) : 0.0f);
#pragma unroll
  for (int i = 0; i < kPer; ++i)
    if (lane + 64 * i < C)
      put(dx + t * C, lane + 64 * i, here ? v[i] * (gb * (frac[lane + 64 * i] - dot) + lz) : 0.0f);
}

int blocks(int T) { return (T + kRows - 1) / kRows; }

}  // namespace
}  // namespace rte

using namespace rte;

extern "C" {

size_t rte_pool_balance_workspace_bytes(int T, int C) {
  return T > 0 && C > 0 ? (size_t)blocks(T) * (2 * C + 2) * sizeof(float) : 0;
}

int rte_pool_balance_fwd(const void* logits, int64_t ld, int f32, int T, int C, const int32_t* ids, int k,
                         const uint8_t* mask, float* out, int32_t* counts, float* frac, void* ws, size_t ws_bytes,
                         void* stream) {
  RTE_REQUIRE(T >= 0 && C >= 1 && C <= kMaxPools && k >= 1 && ld >= 0, "pool_balance: need 1 <= pools <= %d and k >= 1",
              kMaxPools);
  RTE_REQUIRE((T == 0 || (logits && ids)) && out && counts && frac, "pool_balance: null argument");
  RTE_REQUIRE(ws_bytes >= rte_pool_balance_workspace_bytes(T, C) && (T == 0 || ws), "pool_balance: workspace too small");
  auto s = static_cast<hipStream_t>(stream);
  float* part = static_cast<float*>(ws);
  if (T > 0) {
    if (f32)
      hipLaunchKernelGGL(balance_fwd_kernel<float>, dim3(blocks(T)), dim3(256), 0, s, static_cast<const float*>(logits),
                         ld, T, C, ids, k, mask, part);
    else
      hipLaunchKernelGGL(balance_fwd_kernel<bf16>, dim3(blocks(T)), dim3(256), 0, s, static_cast<const bf16*>(logits), ld,
                         T, C, ids, k, mask, part);
    RTE_TRY(check_launch("pool_balance_fwd"));
  }
  hipLaunchKernelGGL(balance_join_kernel, dim3(1), dim3(1024), 0, s, part, T > 0 ? blocks(T) : 0, C, out, counts, frac);
  return check_launch("pool_balance_join");
}

int rte_pool_balance_bwd(const void* logits, int64_t ld, int f32, int T, int C, const uint8_t* mask, const float* frac,
                         const float* g_balance, const float* g_z, void* dlogits, void* stream) {
  RTE_REQUIRE(T >= 0 && C >= 1 && C <= kMaxPools && ld >= 0, "pool_balance_bwd: bad sizes");
  if (T == 0) return 0;
  RTE_REQUIRE(logits && frac && dlogits, "pool_balance_bwd: null argument");
  auto s = static_cast<hipStream_t>(stream);
  if (f32)
    hipLaunchKernelGGL(balance_bwd_kernel<float>, dim3((T + 3) / 4), dim3(256), 0, s, static_cast<const float*>(logits),
                       ld, T, C, mask, frac, g_balance, g_z, static_cast<float*>(dlogits));
  else
    hipLaunchKernelGGL(balance_bwd_kernel<bf16>, dim3((T + 3) / 4), dim3(256), 0, s, static_cast<const bf16*>(logits), ld,
                       T, C, mask, frac, g_balance, g_z, static_cast<bf16*>(dlogits));
  return check_launch("pool_balance_bwd");
}

}  // extern "C"
