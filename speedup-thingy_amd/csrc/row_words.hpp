// Rows of fp32 or bf16 numbers read and written sixteen bytes at a time, and sums over lanes.
#pragma once

#include "common.hpp"

namespace rte {

namespace {

constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.69314718055994530942f;

__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }

// Sixteen bytes of a row at any alignment of its element type: rows of odd length start anywhere, and a
// global load or store of four words asks for no more.
typedef uint32_t words_v __attribute__((ext_vector_type(4), aligned(2), may_alias));
struct Words {
  uint32_t w[4];
};

template <class X>
struct Row;
template <>
struct Row<float> {
  static constexpr int VE = 4;
  __device__ static float one(const float* x, int64_t i) { return x[i]; }
  __device__ static void put(float* x, int64_t i, float v) { x[i] = v; }
  __device__ static float get(const Words& v, int j) { return __uint_as_float(v.w[j]); }
  __device__ static void set(Words& v, int j, float f) { v.w[j] = __float_as_uint(f); }
  __device__ static Words pack(const float* f) {
    return {{__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3])}};
  }
};
template <>
struct Row<bf16> {
  static constexpr int VE = 8;
  __device__ static float one(const bf16* x, int64_t i) { return bf2f(x[i]); }
  __device__ static void put(bf16* x, int64_t i, float v) { x[i] = f2bf(v); }
  __device__ static float get(const Words& v, int j) {
    return __uint_as_float(j & 1 ? v.w[j >> 1] & 0xffff0000u : v.w[j >> 1] << 16);
  }
  __device__ static void set(Words& v, int j, float f) {
    const uint32_t h = __float_as_uint(f) >> 16;
    v.w[j >> 1] = j & 1 ? (v.w[j >> 1] & 0xffffu) | h << 16 : (v.w[j >> 1] & 0xffff0000u) | h;
  }
  __device__ static Words pack(const float* f) {
    return {{pack_bf2(f[0], f[1]), pack_bf2(f[2], f[3]), pack_bf2(f[4], f[5]), pack_bf2(f[6], f[7])}};
  }
};

template <class X>
__device__ __forceinline__ Words whole_words(const X* at) {
  const words_v v = *reinterpret_cast<const words_v*>(at);
  return {{v.x, v.y, v.z, v.w}};
}

// Elements at .. at + VE of a row that ends at `end`; what lies past the end is -inf.
template <class X>
__device__ __forceinline__ Words load_words(const X* row, int at, int end) {
  constexpr int VE = Row<X>::VE;
  if (at + VE <= end) return whole_words(row + at);
  Words r;
#pragma unroll
  for (int j = 0; j < VE; ++j) Row<X>::set(r, j, -INFINITY);
  if (at < end) {
#pragma unroll
    for (int j = 0; j < VE - 1; ++j)
      if (at + j < end) Row<X>::set(r, j, Row<X>::one(row, at + j));
  }
  return r;
}

template <class X>
__device__ __forceinline__ void store_words(X* row, int at, int end, const float* f) {
  constexpr int VE = Row<X>::VE;
  if (at + VE <= end) {
    const Words p = Row<X>::pack(f);
    *reinterpret_cast<words_v*>(row + at) = words_v{p.w[0], p.w[1], p.w[2], p.w[3]};
  } else {
#pragma unroll
    for (int j = 0; j < VE; ++j)
      if (at + j < end) Row<X>::put(row, at + j, f[j]);
  }
}

// v of the lane at xor distance O.  Up to 8 the exchange is a register move: 4 and 8 mirror half a row of
// sixteen and a whole one, which after the smaller distances is the same sum.
template <int O, class V>
__device__ __forceinline__ V across(V v) {
  if constexpr (O <= 8 && sizeof(V) == 4) {
    constexpr int ctrl = O == 1 ? 0xb1 : O == 2 ? 0x4e : O == 4 ? 0x141 : 0x140;
    const int x = __builtin_bit_cast(int, v);
    return __builtin_bit_cast(V, __builtin_amdgcn_update_dpp(x, x, ctrl, 0xf, 0xf, false));
  } else {
    return __shfl_xor(v, O, 64);
  }
}

// Sum and maximum (NaN loses) over every aligned group of N lanes; whole waves only.
template <int N = 64, class V>
__device__ __forceinline__ V wave_sum(V v) {
  if constexpr (N > 1) v += across<1>(v);
  if constexpr (N > 2) v += across<2>(v);
  if constexpr (N > 4) v += across<4>(v);
  if constexpr (N > 8) v += across<8>(v);
  if constexpr (N > 16) v += across<16>(v);
  if constexpr (N > 32) v += across<32>(v);
  return v;
}
template <int N = 64, class V>
__device__ __forceinline__ V wave_max(V v) {
  auto more = [](V a, V b) { return b > a || a != a ? b : a; };
  if constexpr (N > 1) v = more(v, across<1>(v));
  if constexpr (N > 2) v = more(v, across<2>(v));
  if constexpr (N > 4) v = more(v, across<4>(v));
  if constexpr (N > 8) v = more(v, across<8>(v));
  if constexpr (N > 16) v = more(v, across<16>(v));
  if constexpr (N > 32) v = more(v, across<32>(v));
  return v;
}

}  // namespace
}  // namespace rte
