// hcg_scale8.h -- 8-bit floating point on gfx950: scales and conversions (device
// code), and the launch checks of quantised matrices (host).
//
// e4m3 and e5m2 are the open formats, which gfx950's conversions and MFMAs
// take: e4m3 without infinities.  A block's largest magnitude is compared as
// the integer that its bits are, so that infinities and NaNs win.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "hcg_fp8.h"
#include "hcg_vec.h"

namespace hcg {
namespace fp8 {

constexpr int kBlock = HCG_FP8_BLOCK;

// Where and in which types a quantised matrix is written.
struct Out {
  unsigned char* q;
  void* scale;
  int64_t ldq, scale_row, scale_block;
  bool e5m2, e8m0;
};

struct Scale {
  float inverse;  // q = x * inverse, rounded
  uint32_t held;  // the scale: a float's bits, or (e8m0) an exponent byte
};

__device__ __forceinline__ uint32_t magnitude(float v) { return __builtin_bit_cast(uint32_t, v) & 0x7fffffffu; }

// top: the largest magnitude() of a block.
__device__ __forceinline__ Scale scale_of(uint32_t top, bool e5m2, bool e8m0) {
  top = max(top, 0x0d800000u);  // 2^-100: neither quotient below overflows
  Scale s;
  if (e8m0) {
    // 448 and 57344 are 1.75 times 2^8 and 2^15.
    const uint32_t byte = (top >> 23) - (e5m2 ? 15 : 8) + ((top & 0x7fffff) > 0x600000);
    const bool finite = top < 0x7f800000u;
    s.held = finite ? byte : 255;
    s.inverse = __builtin_bit_cast(float, finite ? (254 - byte) << 23 : 0x7fc00000u);
  } else {
    const float largest = e5m2 ? 57344.f : 448.f, t = __builtin_bit_cast(float, top);
    s.held = __builtin_bit_cast(uint32_t, t / largest);
    s.inverse = largest / t;
  }
  return s;
}

__device__ __forceinline__ void put_scale(const Out& o, int64_t row, int64_t block, uint32_t held) {
  const int64_t at = row * o.scale_row + block * o.scale_block;
  if (o.e8m0)
    static_cast<unsigned char*>(o.scale)[at] = (unsigned char)held;
  else
    static_cast<uint32_t*>(o.scale)[at] = held;
}

// Four values rounded to nearest (ties to even), packed.
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d, bool e5m2) {
  int r;
  if (e5m2) {
    r = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, 0, false);
    r = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, r, true);
  } else {
    r = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, r, true);
  }
  return (uint32_t)r;
}

// E (4 or 8) values times `inverse` as 8-bit elements at p, the first `valid` of
// them in the row.
template <int E>
__device__ __forceinline__ void store_q(unsigned char* p, const float (&v)[E], float inverse, int valid, bool e5m2) {
  uint32_t w[E / 4];
#pragma unroll
  for (int i = 0; i < E / 4; ++i)
    w[i] = pack4(v[4 * i] * inverse, v[4 * i + 1] * inverse, v[4 * i + 2] * inverse, v[4 * i + 3] * inverse, e5m2);
  if (valid >= E) {
    if constexpr (E == 4) {
      typedef uint32_t u32a __attribute__((aligned(1)));
      *reinterpret_cast<u32a*>(p) = w[0];
    } else {
      typedef uint32_t u32x2a __attribute__((ext_vector_type(2), aligned(1)));
      *reinterpret_cast<u32x2a*>(p) = u32x2a{w[0], w[1]};
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < E; ++e)
    if (e < valid) p[e] = (unsigned char)(w[e / 4] >> (8 * (e % 4)));
}

// Host: a quantised matrix's types and strides.
inline bool type_ok(int dtype) { return dtype == HCG_E4M3 || dtype == HCG_E5M2; }
inline bool scale_ok(int dtype) { return dtype == HCG_F32 || dtype == HCG_E8M0; }
inline int scale_bytes(int dtype) { return dtype == HCG_F32 ? 4 : 1; }

}  // namespace fp8
}  // namespace hcg
