// Load balance of routed pools.  For T rows of C router logits with the k pools each row was sent to:
//
//   p_t = softmax(x_t)     P_c = mean_t p_tc     counts_c = rows sent to c     f_c = counts_c / sum counts
//   balance = C sum_c f_c P_c     z = mean_t (log sum_c e^{x_tc})^2
//   dx_tc = p_tc (g_b C (f_c - sum_c' f_c' p_tc') + 2 g_z lse_t) / n
//
// over the n rows that the mask keeps and whose logits are not all -inf; other rows take no part and
// their logits may hold anything.  Pools outside [0, C) are none; a pool named twice counts twice.
#include "../../include/rte_hip.h"
#include "row_words.hpp"

namespace rte {

namespace {

constexpr int kMaxPools = 1024;
constexpr int kWaves = 16;       // of a forward workgroup
constexpr int kMaxBlocks = 256;  // forward workgroups, one per CU: each leaves 2 C + 2 numbers to be joined by one

// LPR lanes hold a row, NV vectors each: column (i LPR + lane) VE + j.  False for a row that takes no part.
// On return v holds e^(x - m) (0 past the end) and s its sum.
template <class X, int LPR, int NV>
__device__ __forceinline__ bool soft_row(const Words* w, float (*v)[Row<X>::VE], float& m, float& s) {
  constexpr int VE = Row<X>::VE;
  m = -INFINITY;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VE; ++j) m = fmaxf(m, Row<X>::get(w[i], j));
  m = wave_max<LPR>(m);
  const float m0 = m == -INFINITY ? 0.0f : m;
  s = 0.0f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VE; ++j) {
      v[i][j] = exp2_((Row<X>::get(w[i], j) - m0) * kLog2e);
      s += v[i][j];
    }
  s = wave_sum<LPR>(s);
  return s != 0.0f;  // NaN rows take part
}

// Partials of a workgroup: [C] sums of p, [C] counts (both filled up to fours), sum of lse^2, rows.  Bound by
// reading the logits: a wave keeps its columns' sums in registers over all its rows, 64 / LPR at a time, and the waves' sums
// meet in LDS at the end.  131071 x 256 fp32, top 16: 31 us, 4.6 TB/s (45 behind a backward pass, whose gradient is
// still being written back); 8192 x 64, top 8: 4.8.
template <class X, int LPR, int NV>
__global__ void __launch_bounds__(kWaves * 64)
    balance_fwd_kernel(const X* __restrict__ logits, int64_t ld, int64_t T, int C, const int32_t* __restrict__ ids, int k,
                       const uint8_t* __restrict__ mask, int64_t rows, float* __restrict__ part) {
  constexpr int VE = Row<X>::VE, RPW = 64 / LPR, CW = LPR * NV * VE;
  constexpr int kFlags = 2048;
  __shared__ float sum[kWaves / 2][CW];
  __shared__ int cnt[CW];
  __shared__ float zs[kWaves];
  __shared__ int ns[kWaves];
  __shared__ uint8_t in[kFlags];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane & (LPR - 1), rl = lane / LPR;
  for (int c = threadIdx.x; c < CW; c += kWaves * 64) cnt[c] = 0;
  float acc[NV][VE], z = 0.0f;
  int n = 0;
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VE; ++j) acc[i][j] = 0.0f;
  const int64_t t0 = blockIdx.x * rows, t1 = t0 + rows < T ? t0 + rows : T;
  for (int64_t base = t0; base < t1; base += kFlags) {  // flags of 2048 rows at a time
    const int nr = (int)(t1 - base < kFlags ? t1 - base : kFlags);
    __syncthreads();
    // the next row is on its way while one is computed: alone, a row's latency is what a wave sees
    auto fetch = [&](int r, Words* to) {
      const int rr = r + rl;
      const bool want = rr < nr && (!mask || mask[base + rr]);
      const X* row = logits + (base + (rr < nr ? rr : 0)) * ld;
#pragma unroll
      for (int i = 0; i < NV; ++i) to[i] = load_words(row, (i * LPR + sub) * VE, want ? C : 0);
      return want;
    };
    Words next[NV];
    bool next_here = false;
    if (wave * RPW < nr) next_here = fetch(wave * RPW, next);
    for (int r = wave * RPW; r < nr; r += kWaves * RPW) {
      Words w[NV];
      float v[NV][VE], m, s;
#pragma unroll
      for (int i = 0; i < NV; ++i) w[i] = next[i];
      const bool here = next_here;
      if (r + kWaves * RPW < nr) next_here = fetch(r + kWaves * RPW, next);
      const bool part_of = soft_row<X, LPR, NV>(w, v, m, s) && here;
      if (r + rl < nr && sub == 0) in[r + rl] = part_of;
      const float inv = part_of ? 1.0f / s : 0.0f;
#pragma unroll
      for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int j = 0; j < VE; ++j) acc[i][j] += part_of ? v[i][j] * inv : 0.0f;
      if (part_of && sub == 0) {
        const float lse = m + logf(s);
        z += lse * lse;
        ++n;
      }
    }
    __syncthreads();
    const int32_t* list = ids + base * k;
    const float inv_k = 1.0f / k;
    for (int i0 = threadIdx.x; i0 < nr * k; i0 += 8 * kWaves * 64) {
      int c[8];  // loads of eight pairs on their way together
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int i = i0 + u * kWaves * 64;
        c[u] = i < nr * k ? list[i] : -1;
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const int i = i0 + u * kWaves * 64;
        if (c[u] < 0 || c[u] >= C) continue;
        int r = (int)((i + 0.5f) * inv_k);  // i / k within one, put right below
        r -= r * k > i;
        r += (r + 1) * k <= i;
        if (in[r]) atomicAdd(&cnt[c[u]], 1);
      }
    }
  }
  // the wave's rows, then the waves, in a fixed order
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VE; ++j)
#pragma unroll
      for (int o = LPR; o < 64; o <<= 1) acc[i][j] += __shfl_xor(acc[i][j], o, 64);
  z = wave_sum(z);
  n = wave_sum(n);
  if (lane == 0) {
    zs[wave] = z;
    ns[wave] = n;
  }
  auto put_sums = [&](int at, bool add) {
    if (rl != 0) return;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        float* to = &sum[at][(i * LPR + sub) * VE + j];
        *to = add ? *to + acc[i][j] : acc[i][j];
      }
  };
  if (wave >= kWaves / 2) put_sums(wave - kWaves / 2, false);
  __syncthreads();
  if (wave < kWaves / 2) put_sums(wave, true);
  __syncthreads();
  const int c4 = (C + 3) / 4 * 4;
  float* out = part + (int64_t)blockIdx.x * (2 * c4 + 4);
  for (int c = threadIdx.x; c < c4; c += kWaves * 64) {
    float p = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves / 2; ++w) p += sum[w][c];
    out[c] = p;
    reinterpret_cast<int*>(out)[c4 + c] = cnt[c];
  }
  if (threadIdx.x == 0) {
    float zt = 0.0f;
    int nt = 0;
    for (int w = 0; w < kWaves; ++w) {
      zt += zs[w];
      nt += ns[w];
    }
    out[2 * c4] = zt;
    reinterpret_cast<int*>(out)[2 * c4 + 1] = nt;
  }
}

// One workgroup adds the partials: four columns by every threads / vecs-th thread, each over its share of
// the blocks with sixteen loads on their way (256 blocks of 256: 9.5 us, column by column 12.5; of 64: 8, nearly
// all of it dependent memory round trips).
__global__ void __launch_bounds__(1024) balance_join_kernel(const float* __restrict__ part, int nblk, int C, int vecs,
                                                            float* __restrict__ out, int32_t* __restrict__ counts,
                                                            float* __restrict__ frac) {
  __shared__ double red[4][16];
  __shared__ double s_p[4][1024];
  __shared__ int s_n[4][1024];
  const int c4 = (C + 3) / 4 * 4;
  const int64_t w = 2 * c4 + 4;
  const int gs = 1024 / vecs, q = threadIdx.x & (vecs - 1), g = threadIdx.x / vecs;
  double p4[4] = {0.0, 0.0, 0.0, 0.0};
  int n4[4] = {0, 0, 0, 0};
  if (4 * q < C) {
#pragma unroll 8
    for (int b = g; b < nblk; b += gs) {
      const float4 x = *reinterpret_cast<const float4*>(part + b * w + 4 * q);
      const int4 y = *reinterpret_cast<const int4*>(part + b * w + c4 + 4 * q);
      p4[0] += x.x, p4[1] += x.y, p4[2] += x.z, p4[3] += x.w;
      n4[0] += y.x, n4[1] += y.y, n4[2] += y.z, n4[3] += y.w;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    s_p[i][threadIdx.x] = p4[i];
    s_n[i][threadIdx.x] = n4[i];
  }
  double z = 0.0;
  int rows = 0;
  for (int b = threadIdx.x; b < nblk; b += 1024) {
    z += part[b * w + 2 * c4];
    rows += reinterpret_cast<const int*>(part)[b * w + 2 * c4 + 1];
  }
  const int wave = threadIdx.x >> 6;
  z = wave_sum(z);
  rows = wave_sum(rows);
  const int pairs = wave_sum((n4[0] + n4[1]) + (n4[2] + n4[3]));
  if ((threadIdx.x & 63) == 0) {
    red[0][wave] = z;
    red[1][wave] = rows;
    red[2][wave] = pairs;
  }
  __syncthreads();
  const int c = threadIdx.x;
  const bool mine = c < C;
  double p = 0.0, all = 0.0;
  int n = 0;
  for (int i = 0; i < 16; ++i) all += red[2][i];
  if (mine) {
#pragma unroll 4
    for (int i = 0; i < gs; ++i) {
      p += s_p[c & 3][i * vecs + (c >> 2)];
      n += s_n[c & 3][i * vecs + (c >> 2)];
    }
  }
  const double f = all > 0.0 ? n / all : 0.0;
  const double term = wave_sum(f != 0.0 ? f * p : p != p ? p : 0.0);
  if ((threadIdx.x & 63) == 0) red[3][wave] = term;
  __syncthreads();
  if (mine) {
    counts[c] = n;
    frac[c] = (float)f;
  }
  if (threadIdx.x == 0) {
    double total = 0.0, bal = 0.0;
    z = 0.0;
    for (int i = 0; i < 16; ++i) {
      z += red[0][i];
      total += red[1][i];
      bal += red[3][i];
    }
    const double inv = total > 0.0 ? 1.0 / total : 0.0;
    out[0] = (float)(C * bal * inv);
    out[1] = (float)(z * inv);
    frac[C] = (float)inv;
  }
}

// Bound by reading the logits and writing their gradient (131071 x 256 fp32, an eighth of the rows masked: 51 us,
// 4.9 TB/s).
template <class X, int LPR, int NV>
__global__ void __launch_bounds__(256)
    balance_bwd_kernel(const X* __restrict__ logits, int64_t ld, int64_t T, int C, const uint8_t* __restrict__ mask,
                       int64_t rows, const float* __restrict__ frac, const float* __restrict__ g_bal,
                       const float* __restrict__ g_z, X* __restrict__ dx) {
  constexpr int VE = Row<X>::VE, RPW = 64 / LPR;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, sub = lane & (LPR - 1), rl = lane / LPR;
  const float inv_n = frac[C];
  const float gb = g_bal ? *g_bal * C * inv_n : 0.0f, gz = g_z ? *g_z * 2.0f * inv_n : 0.0f;
  float f[NV][VE];
#pragma unroll
  for (int i = 0; i < NV; ++i)
#pragma unroll
    for (int j = 0; j < VE; ++j) {
      const int c = (i * LPR + sub) * VE + j;
      f[i][j] = c < C ? frac[c] : 0.0f;
    }
  const int64_t t0 = blockIdx.x * rows, t1 = t0 + rows < T ? t0 + rows : T;
  for (int64_t r = t0 + wave * RPW; r < t1; r += 4 * RPW) {
    const int64_t t = r + rl < t1 ? r + rl : t1 - 1;  // lanes past the end repeat the last row and store nothing
    const bool here = !mask || mask[t];
    Words w[NV];
    float v[NV][VE], m, s;
#pragma unroll
    for (int i = 0; i < NV; ++i) w[i] = load_words(logits + t * ld, (i * LPR + sub) * VE, here ? C : 0);
    const bool part_of = soft_row<X, LPR, NV>(w, v, m, s) && here;
    const float inv = part_of ? 1.0f / s : 0.0f;
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
      for (int j = 0; j < VE; ++j) {
        v[i][j] *= inv;
        dot += v[i][j] * f[i][j];
      }
    dot = wave_sum<LPR>(dot);
    const float lz = gz * (m + logf(s));
#pragma unroll
    for (int i = 0; i < NV; ++i) {
#pragma unroll
      for (int j = 0; j < VE; ++j) v[i][j] = part_of ? v[i][j] * (gb * (f[i][j] - dot) + lz) : 0.0f;
      if (r + rl < t1) store_words(dx + t * C, (i * LPR + sub) * VE, C, v[i]);
    }
  }
}

// Rows of a forward workgroup: the fewest that keep the workgroups at one per CU.
int64_t fwd_rows(int T) {
  const int64_t rows = ((int64_t)T + kMaxBlocks - 1) / kMaxBlocks;
  return rows < 16 ? 16 : rows;
}
int blocks(int T) { return (int)((T + fwd_rows(T) - 1) / fwd_rows(T)); }

struct Call {
  const void* logits;
  int64_t ld;
  int T, C;
  const int32_t* ids;
  int k;
  const uint8_t* mask;
  float* part;
  const float *frac, *g_bal, *g_z;
  void* dx;
};

template <class X, int LPR, int NV>
int run(const Call& c, hipStream_t s) {
  const X* x = static_cast<const X*>(c.logits);
  if (!c.dx) {
    hipLaunchKernelGGL((balance_fwd_kernel<X, LPR, NV>), dim3(blocks(c.T)), dim3(kWaves * 64), 0, s, x, c.ld, (int64_t)c.T,
                       c.C, c.ids, c.k, c.mask, fwd_rows(c.T), c.part);
    return check_launch("pool_balance_fwd");
  }
  // four passes of a workgroup's waves, or one where that leaves fewer than four workgroups per CU
  int64_t rows = 4 * 4 * (64 / LPR);
  if (c.T / rows < 1024) rows /= 4;
  hipLaunchKernelGGL((balance_bwd_kernel<X, LPR, NV>), dim3((unsigned)((c.T + rows - 1) / rows)), dim3(256), 0, s, x, c.ld,
                     (int64_t)c.T, c.C, c.mask, rows, c.frac, c.g_bal, c.g_z, static_cast<X*>(c.dx));
  return check_launch("pool_balance_bwd");
}

// A row on the fewest lanes (a power of two, 4 at least) that hold it in one vector each, or in sixteen
// columns each once every wave of the chip has two rounds of such rows: fewer exchanges per row.
template <class X>
int pick(const Call& c, hipStream_t s) {
  constexpr int NV = 16 / Row<X>::VE;
  const int lanes = (c.C + 15) / 16;
  const int wide = lanes <= 4 ? 4 : lanes <= 8 ? 8 : lanes <= 16 ? 16 : lanes <= 32 ? 32 : 64;
  if (wide == 64 || (int64_t)c.T * wide >= 2 * 64 * kMaxBlocks * kWaves) {
    if (wide == 4) return run<X, 4, NV>(c, s);
    if (wide == 8) return run<X, 8, NV>(c, s);
    if (wide == 16) return run<X, 16, NV>(c, s);
    if (wide == 32) return run<X, 32, NV>(c, s);
    return run<X, 64, NV>(c, s);
  }
  const int vecs = (c.C + Row<X>::VE - 1) / Row<X>::VE;
  if (vecs <= 4) return run<X, 4, 1>(c, s);
  if (vecs <= 8) return run<X, 8, 1>(c, s);
  if (vecs <= 16) return run<X, 16, 1>(c, s);
  if (vecs <= 32) return run<X, 32, 1>(c, s);
  if (Row<X>::VE == 8 || vecs <= 64) return run<X, 64, 1>(c, s);
  return run<X, 64, 16 / Row<X>::VE / 2>(c, s);
}

}  // namespace
}  // namespace rte

using namespace rte;

extern "C" {

size_t rte_pool_balance_workspace_bytes(int T, int C) {
  return T > 0 && C > 0 ? (size_t)blocks(T) * (2 * ((C + 3) / 4 * 4) + 4) * sizeof(float) : 0;
}

int rte_pool_balance_fwd(const void* logits, int64_t ld, int f32, int T, int C, const int32_t* ids, int k,
                         const uint8_t* mask, float* out, int32_t* counts, float* frac, void* ws, size_t ws_bytes,
                         void* stream) {
  RTE_REQUIRE(T >= 0 && C >= 1 && C <= kMaxPools && k >= 1 && k <= kMaxPools && ld >= 0,
              "pool_balance: need 1 to %d pools and as many per row at most", kMaxPools);
  RTE_REQUIRE((int64_t)T * k < ((int64_t)1 << 31), "pool_balance: fewer than 2^31 (row, pool) pairs expected");
  RTE_REQUIRE((T == 0 || (logits && ids)) && out && counts && frac, "pool_balance: null argument");
  RTE_REQUIRE(ws_bytes >= rte_pool_balance_workspace_bytes(T, C) && (T == 0 || ws), "pool_balance: workspace too small");
  auto s = static_cast<hipStream_t>(stream);
  Call c{};
  c.logits = logits, c.ld = ld, c.T = T, c.C = C, c.ids = ids, c.k = k, c.mask = mask, c.part = static_cast<float*>(ws);
  if (T > 0) RTE_TRY(f32 ? pick<float>(c, s) : pick<bf16>(c, s));
  int vecs = 16;  // a power of two of four columns each
  while (4 * vecs < C) vecs *= 2;
  hipLaunchKernelGGL(balance_join_kernel, dim3(1), dim3(1024), 0, s, c.part, T > 0 ? blocks(T) : 0, C, vecs, out, counts,
                     frac);
  return check_launch("pool_balance_join");
}

int rte_pool_balance_bwd(const void* logits, int64_t ld, int f32, int T, int C, const uint8_t* mask, const float* frac,
                         const float* g_balance, const float* g_z, void* dlogits, void* stream) {
  RTE_REQUIRE(T >= 0 && C >= 1 && C <= kMaxPools && ld >= 0, "pool_balance_bwd: bad sizes");
  if (T == 0) return 0;
  RTE_REQUIRE(logits && frac && dlogits, "pool_balance_bwd: null argument");
  Call c{};
  c.logits = logits, c.ld = ld, c.T = T, c.C = C, c.mask = mask, c.frac = frac, c.g_bal = g_balance, c.g_z = g_z;
  c.dx = dlogits;
  auto s = static_cast<hipStream_t>(stream);
  return f32 ? pick<float>(c, s) : pick<bf16>(c, s);
}

}  // extern "C"
