// Small device helpers of the row and sequence kernels (norm.hip, scan.hip, gemm_i8.hip): values of
// float or bfloat16 rows as float, and reductions over neighbouring lanes.
#pragma once

#include <type_traits>

#include "common.h"

namespace spmi {

using bf16 = __bf16;

// Four neighbouring values as float, from any address that is a multiple of the value's own size:
// global memory accesses need no more alignment than that on gfx950 (the compiler emits one 16-
// or 8-byte access), so rows of an odd width or stride take the same code as aligned ones.
//
// STREAM: the access is marked as one that is not repeated soon (nontemporal).  The kernels that pass
// over tall matrices use it for what they read or write once: layer norm of 10^6 x 128 values goes
// from 212 to 171 us forward and from 310 to 265 us backward with it.
using f32x4 = float __attribute__((ext_vector_type(4)));
using f32x4_any = float __attribute__((ext_vector_type(4), aligned(4)));
using u16x4_any = unsigned short __attribute__((ext_vector_type(4), aligned(2)));

template <bool STREAM = false>
__device__ __forceinline__ void load4(const float* p, float (&v)[4]) {
  const auto* q = reinterpret_cast<const f32x4_any*>(p);
  const f32x4 t = STREAM ? __builtin_nontemporal_load(q) : *q;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = t[i];
}
template <bool STREAM = false>
__device__ __forceinline__ void load4(const bf16* p, float (&v)[4]) {
  const auto* q = reinterpret_cast<const u16x4_any*>(p);
  const u16x4_any t = STREAM ? __builtin_nontemporal_load(q) : *q;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __builtin_bit_cast(float, static_cast<unsigned>(t[i]) << 16);
}
template <bool STREAM = false>
__device__ __forceinline__ void store4(float* p, const float (&v)[4]) {
  auto* q = reinterpret_cast<f32x4_any*>(p);
  const f32x4_any t = {v[0], v[1], v[2], v[3]};
  if constexpr (STREAM) __builtin_nontemporal_store(t, q);
  else *q = t;
}
template <bool STREAM = false>
__device__ __forceinline__ void store4(bf16* p, const float (&v)[4]) {
  auto* q = reinterpret_cast<u16x4_any*>(p);
  u16x4_any t;
#pragma unroll
  for (int i = 0; i < 4; ++i) t[i] = __builtin_bit_cast(unsigned short, static_cast<bf16>(v[i]));  // to nearest even
  if constexpr (STREAM) __builtin_nontemporal_store(t, q);
  else *q = t;
}

// Four values as they are stored.  Loads that should be in flight together are issued as these, without a
// branch or a conversion between them, and widened where they are used: with either in between, each
// load is waited for before the next is sent.
template <typename T> struct Held;
template <> struct Held<float> { using type = f32x4; using any = f32x4_any; };
template <> struct Held<bf16> {
  using type = unsigned short __attribute__((ext_vector_type(4)));
  using any = u16x4_any;
};
template <typename T>
using held = typename Held<T>::type;

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(unsigned short v) {
  return __builtin_bit_cast(float, static_cast<unsigned>(v) << 16);
}
template <bool STREAM, typename T>
__device__ __forceinline__ held<T> hold4(const T* p) {
  const auto* q = reinterpret_cast<const typename Held<T>::any*>(p);
  return STREAM ? __builtin_nontemporal_load(q) : *q;
}
// Values c .. c + 3 of a row of D, c a multiple of four that may lie past its end.  Where the row ends
// first, its last four are loaded; widen_row moves them into place and gives zero for what is not there.
// (Rows of fewer than four values are read one by one.)
template <bool STREAM, typename T>
__device__ __forceinline__ held<T> hold_row(const T* row, int c, int D) {
  if (D >= 4) return hold4<STREAM>(row + (c <= D - 4 ? c : D - 4));
  using U = std::conditional_t<sizeof(T) == 4, float, unsigned short>;
  held<T> v;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = c + i < D ? reinterpret_cast<const U*>(row)[c + i] : U(0);
  return v;
}
template <typename T>
__device__ __forceinline__ void widen_row(held<T> t, int c, int D, float (&v)[4]) {
  const int by = D < 4 || c <= D - 4 ? 0 : c - (D - 4);
  if constexpr (sizeof(T) == 2) {
    const uint64_t w = by < 4 ? __builtin_bit_cast(uint64_t, t) >> (16 * by) : 0;
    t = __builtin_bit_cast(held<T>, w);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = widen(t[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = t[i];
    if (D % 4) {
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = (by & 2) ? (i < 2 ? v[i + 2] : 0.0f) : v[i];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = (by & 1) ? (i < 3 ? v[i + 1] : 0.0f) : v[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = by < 4 ? v[i] : 0.0f;
  }
}

// Loads and stores of the last values of a row: `left` >= 1 of them exist, the others read as `fill`.
template <typename T>
__device__ __forceinline__ void load4_upto(const T* p, int left, float fill, float (&v)[4]) {
  if (left >= 4) {
    load4(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = i < left ? static_cast<float>(p[i]) : fill;
  }
}
template <bool STREAM = false, typename T>
__device__ __forceinline__ void store4_upto(T* p, int left, const float (&v)[4]) {
  if (left >= 4) {
    store4<STREAM>(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 3; ++i)
      if (i < left) p[i] = static_cast<T>(v[i]);
  }
}

template <int CTRL>
__device__ __forceinline__ float dpp(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}

// The sum (maximum) over groups of G neighbouring lanes, in every lane of the group.  Inside 16
// lanes the partner's value comes with the instruction itself (data-parallel primitives: swaps
// within four lanes, mirrors of 8 and of 16); only the last two steps go through LDS hardware.
// Every lane adds the same pairs, so all lanes hold the same bits.
template <int G, typename Op>
__device__ __forceinline__ float group_reduce(float v, Op op) {
  if constexpr (G >= 2) v = op(v, dpp<0xB1>(v));   // lanes 1 0 3 2
  if constexpr (G >= 4) v = op(v, dpp<0x4E>(v));   // lanes 2 3 0 1
  if constexpr (G >= 8) v = op(v, dpp<0x141>(v));  // mirror of 8 lanes
  if constexpr (G >= 16) v = op(v, dpp<0x140>(v)); // mirror of 16 lanes
  if constexpr (G >= 32) v = op(v, __shfl_xor(v, 16, 64));
  if constexpr (G >= 64) v = op(v, __shfl_xor(v, 32, 64));
  return v;
}
template <int G>
__device__ __forceinline__ float group_sum(float v) {
  return group_reduce<G>(v, [](float a, float b) { return a + b; });
}

}  // namespace spmi
