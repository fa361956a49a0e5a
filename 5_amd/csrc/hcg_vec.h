// hcg_vec.h -- 16-byte vectors of row elements for the row-wise operators
// (device code), and their launch checks (host).
//
// A row is handled in vectors of 16 bytes (8 f16 / bf16 or 4 f32 elements).
// Global loads and stores need no alignment beyond the element on gfx950, so
// one form serves every row stride; the vector that reaches past a row's end
// is taken element by element, and nothing past the row is touched.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>
#include <string.h>

#include "hcg_lm.h"
#include "hcg_runtime.h"

namespace hcg {

template <int DT>
struct ElemOf;
template <>
struct ElemOf<HCG_F16> {
  typedef _Float16 type;
};
template <>
struct ElemOf<HCG_BF16> {
  typedef __bf16 type;
};
template <>
struct ElemOf<HCG_F32> {
  typedef float type;
};

// Elements in 16 bytes.
template <class T>
constexpr int kVec = 16 / (int)sizeof(T);

typedef uint32_t raw4 __attribute__((ext_vector_type(4)));
// The same at an address aligned to an element only.
template <int BYTES>
struct RawAt;
template <>
struct RawAt<2> {
  typedef uint32_t type __attribute__((ext_vector_type(4), aligned(2)));
};
template <>
struct RawAt<4> {
  typedef uint32_t type __attribute__((ext_vector_type(4), aligned(4)));
};

// 16 bytes at an element-aligned address, of which the first `valid` elements
// are in the row (the rest zero, not read).
template <class T>
__device__ __forceinline__ raw4 load_raw(const T* p, int valid) {
  if (valid >= kVec<T>) {
    typedef typename RawAt<sizeof(T)>::type raw4a;
    return *reinterpret_cast<const raw4a*>(p);
  }
  raw4 r{0, 0, 0, 0};
  if constexpr (sizeof(T) == 4) {
    const uint32_t* q = reinterpret_cast<const uint32_t*>(p);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < valid) r[e] = q[e];
  } else {
    const uint16_t* q = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < valid) r[e >> 1] |= (uint32_t)q[e] << (16 * (e & 1));
  }
  return r;
}

// NT: non-temporal, for outputs much larger than the caches (they leave no
// dirty lines for the launch's end to write back).
template <bool NT = false, class T>
__device__ __forceinline__ void store_raw(T* p, raw4 v, int valid) {
  if (valid >= kVec<T>) {
    typedef typename RawAt<sizeof(T)>::type raw4a;
    if constexpr (NT)
      __builtin_nontemporal_store((raw4a)v, reinterpret_cast<raw4a*>(p));
    else
      *reinterpret_cast<raw4a*>(p) = v;
    return;
  }
  if constexpr (sizeof(T) == 4) {
    uint32_t* q = reinterpret_cast<uint32_t*>(p);
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < valid) q[e] = v[e];
  } else {
    uint16_t* q = reinterpret_cast<uint16_t*>(p);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < valid) q[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
  }
}

template <class T>
__device__ __forceinline__ void unpack(raw4 r, float (&f)[kVec<T>]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const uint32_t w = r[e];  // (a bit cast of a vector's element itself reads element 0)
      f[e] = __builtin_bit_cast(float, w);
    }
  } else {
    typedef T vec __attribute__((ext_vector_type(8)));
    const vec v = __builtin_bit_cast(vec, r);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = (float)v[e];
  }
}

// Rounded to T, to nearest with ties to even.
template <class T>
__device__ __forceinline__ raw4 pack(const float (&f)[kVec<T>]) {
  if constexpr (sizeof(T) == 4) {
    raw4 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = __builtin_bit_cast(uint32_t, f[e]);
    return r;
  } else {
    typedef T vec __attribute__((ext_vector_type(8)));
    vec v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = (T)f[e];
    return __builtin_bit_cast(raw4, v);
  }
}

// N consecutive elements as float, the first `valid` of them in the row.
template <class T, int N>
__device__ __forceinline__ void load_floats(const T* p, int valid, float (&f)[N]) {
  static_assert(N % kVec<T> == 0, "whole vectors");
#pragma unroll
  for (int i = 0; i < N / kVec<T>; ++i) {
    float part[kVec<T>];
    unpack<T>(load_raw(p + i * kVec<T>, valid - i * kVec<T>), part);
#pragma unroll
    for (int e = 0; e < kVec<T>; ++e) f[i * kVec<T> + e] = part[e];
  }
}

__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v += __shfl_xor(v, m);
  return v;
}
__device__ __forceinline__ float wave_max(float v) {
#pragma unroll
  for (int m = 32; m >= 1; m >>= 1) v = fmaxf(v, __shfl_xor(v, m));
  return v;
}

// The grid of n workgroups, in two dimensions past 2^20 of them (a launch's
// threads along one are fewer than 2^32), and a workgroup's number in it, which
// may be n or more.
constexpr int kGridShift = 20;
inline dim3 grid_of(int64_t n) {
  const int64_t x = n < (1 << kGridShift) ? n : 1 << kGridShift;
  return dim3((unsigned)x, (unsigned)((n + x - 1) / x));
}
__device__ __forceinline__ int64_t workgroup() { return (int64_t)blockIdx.y * gridDim.x + blockIdx.x; }
// The same for a kernel so short that gridDim, a load, shows.
__device__ __forceinline__ int64_t workgroup_short() { return ((int64_t)blockIdx.y << kGridShift) + blockIdx.x; }

// Host: the shape and pointer rules that every row-wise entry point has.
inline int elem_bytes(int dtype) { return dtype == HCG_F32 ? 4 : 2; }
inline bool elem_ok(int dtype) { return dtype == HCG_F16 || dtype == HCG_BF16 || dtype == HCG_F32; }
inline bool elem_aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) % (unsigned)bytes) == 0; }

}  // namespace hcg

#define HCG_LM_HIP_CHECK(expr)                                                                              \
  do {                                                                                                      \
    hipError_t _e = (expr);                                                                                 \
    if (_e != hipSuccess) return hcg::set_error(HCG_EHIP, "%s failed: %s", #expr, hipGetErrorString(_e)); \
  } while (0)
#define HCG_LM_REQUIRE(cond, ...)                                      \
  do {                                                                 \
    if (!(cond)) return hcg::set_error(HCG_EINVAL, __VA_ARGS__);       \
  } while (0)
