// layer.cuh -- what the MLP layer's kernels share: 16-bit types, activations and
// their slopes, and dropout from a counter-based generator.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "kernels.h"

namespace mlpg {

// ---- 16-bit types ----------------------------------------------------------------
// The type is a template parameter (kTypeF16, kTypeBF16): a branch per conversion cost
// the epilogues more than the conversion.

// Two values of a 32-bit word, low half first.
template <int TYPE>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if constexpr (TYPE == kTypeF16) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  else return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}

// Round to nearest even, both types; f16 overflows to infinity.
template <int TYPE>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  if constexpr (TYPE == kTypeF16) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&b);
  }
}

template <int TYPE>
__device__ __forceinline__ float load1(const void* base, size_t i) {
  return unpack2<TYPE>(static_cast<const uint16_t*>(base)[i]).x;
}

template <int TYPE>
__device__ __forceinline__ void store1(void* base, size_t i, float v) {
  static_cast<uint16_t*>(base)[i] = (uint16_t)(pack2<TYPE>(v, 0.f) & 0xFFFFu);
}

// Eight neighbours in 16 bytes.
template <int TYPE>
__device__ __forceinline__ void unpack8(float (&v)[8], uint4 w) {
  const uint32_t q[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack2<TYPE>(q[i]);
    v[2 * i] = f.x;
    v[2 * i + 1] = f.y;
  }
}

template <int TYPE>
__device__ __forceinline__ uint4 pack8(const float (&v)[8]) {
  return make_uint4(pack2<TYPE>(v[0], v[1]), pack2<TYPE>(v[2], v[3]), pack2<TYPE>(v[4], v[5]),
                    pack2<TYPE>(v[6], v[7]));
}

// W (4 or 8) elements of a row of `cols` from column c on, element `at` of base: one
// access where the rows allow it (vec); elements past the row read as 0 and are not written.
template <int TYPE, int W>
__device__ __forceinline__ void loadn(float (&v)[W], const void* base, size_t at, int c, int cols, bool vec) {
  const uint16_t* p = static_cast<const uint16_t*>(base) + at;
  if (vec && c + W <= cols) {
    if constexpr (W == 8) {
      unpack8<TYPE>(v, *reinterpret_cast<const uint4*>(p));
    } else {
      const uint2 w = *reinterpret_cast<const uint2*>(p);
      const float2 a = unpack2<TYPE>(w.x), b = unpack2<TYPE>(w.y);
      v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
    }
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i) v[i] = c + i < cols ? load1<TYPE>(p, i) : 0.f;
  }
}

template <int TYPE, int W>
__device__ __forceinline__ void storen(const float (&v)[W], void* base, size_t at, int c, int cols, bool vec) {
  uint16_t* p = static_cast<uint16_t*>(base) + at;
  if (vec && c + W <= cols) {
    if constexpr (W == 8) *reinterpret_cast<uint4*>(p) = pack8<TYPE>(v);
    else *reinterpret_cast<uint2*>(p) = make_uint2(pack2<TYPE>(v[0], v[1]), pack2<TYPE>(v[2], v[3]));
  } else {
#pragma unroll
    for (int i = 0; i < W; ++i)
      if (c + i < cols) store1<TYPE>(p, i, v[i]);
  }
}

// ---- activations ------------------------------------------------------------------
// gelu_tanh is written as z * sigmoid(2u), u = sqrt(2/pi) (z + 0.044715 z^3), which
// equals 0.5 z (1 + tanh u) without the cancellation at large negative z.
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// z between -m and m; NaN stays NaN
__device__ __forceinline__ float clampf(float z, float m) {
  float y;
  asm("{\n\t.reg .f32 t;\n\tmin.NaN.f32 t, %1, %2;\n\tmax.NaN.f32 %0, t, %3;\n\t}" : "=f"(y) : "f"(z), "f"(m), "f"(-m));
  return y;
}

// 1 / (1 + exp(-t))
__device__ __forceinline__ float sigmoidf_(float t) { return rcp_approx(1.f + ex2_approx(-1.4426950408889634f * t)); }

__device__ __forceinline__ float gelu_u2(float z) { return 1.5957691216057308f * (z + 0.044715f * z * z * z); }

// e = exp(-a^2/2) and Phi(-a), the normal distribution's tail, for a >= 0 by Abramowitz
// and Stegun 7.1.26: erfc(x) = (a1 t + ... + a5 t^5) exp(-x^2), t = 1 / (1 + 0.3275911 x),
// off by at most 1.5e-7: far below a 16-bit result's rounding, no branch, and the slope
// reuses e.  The coefficients here are halved (Phi(-a) = erfc(x) / 2), x = a / sqrt(2);
// the tail comes without its factor e.
__device__ __forceinline__ float normal_tail(float a, float& e) {
  const float t = rcp_approx(fmaf(0.23164189f, a, 1.f));
  e = ex2_approx(-0.72134752044448170f * a * a);
  float q = fmaf(t, 0.5307027145f, -0.7265760135f);
  q = fmaf(t, q, 0.7107068705f);
  q = fmaf(t, q, -0.142248368f);
  q = fmaf(t, q, 0.127414796f);
  return q * t;
}

template <int ACT>
__device__ __forceinline__ float act_fwd(float z) {
  if constexpr (ACT == kActRelu) return z < 0.f ? 0.f : z;   // NaN stays NaN
  if constexpr (ACT == kActGelu) {
    float e;
    const float tail = normal_tail(fabsf(z), e) * e;
    return z * (z < 0.f ? tail : 1.f - tail);
  }
  if constexpr (ACT == kActGeluTanh) return z * sigmoidf_(gelu_u2(z));
  if constexpr (ACT == kActSilu) return z * sigmoidf_(z);
  return z;
}

// The same for neighbours and an activation known at run time: one branch for all.
template <int W>
__device__ __forceinline__ void act_fwd_n(float (&v)[W], int act) {
  switch (act) {
    case kActRelu:
#pragma unroll
      for (int i = 0; i < W; ++i) v[i] = act_fwd<kActRelu>(v[i]);
      break;
    case kActGelu:
#pragma unroll
      for (int i = 0; i < W; ++i) v[i] = act_fwd<kActGelu>(v[i]);
      break;
    case kActGeluTanh:
#pragma unroll
      for (int i = 0; i < W; ++i) v[i] = act_fwd<kActGeluTanh>(v[i]);
      break;
    case kActSilu:
#pragma unroll
      for (int i = 0; i < W; ++i) v[i] = act_fwd<kActSilu>(v[i]);
      break;
    default: break;
  }
}

// act'(z).  z is a stored pre-activation, which f16 may have rounded to an
// infinity: beyond the clamps every slope is 0 or 1 to f32 precision, so an
// infinite z gets its limit instead of inf * 0.  NaN passes the comparisons.
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  if constexpr (ACT == kActRelu) return z > 0.f ? 1.f : (z <= 0.f ? 0.f : z);
  if constexpr (ACT == kActGelu) {
    // slope(-a) = 1 - slope(a)
    float a, e;
    asm("min.NaN.f32 %0, %1, 0f41F00000;" : "=f"(a) : "f"(fabsf(z)));   // 30
    const float tail = normal_tail(a, e);
    const float h = e * fmaf(0.3989422804014327f, a, -tail);
    return z < 0.f ? -h : 1.f + h;
  }
  if constexpr (ACT == kActGeluTanh) {
    z = clampf(z, 30.f);
    const float q = sigmoidf_(gelu_u2(z));
    return q + z * q * (1.f - q) * (1.5957691216057308f * (1.f + 0.134145f * z * z));
  }
  if constexpr (ACT == kActSilu) {
    z = clampf(z, 80.f);
    const float q = sigmoidf_(z);
    return q * (1.f + z * (1.f - q));
  }
  return 1.f;
}

// ---- dropout ------------------------------------------------------------------------
// Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy
// as 1, 2, 3", SC 2011).  The counter is (column / 8, row, offset), the key the
// seed, so any tile shape computes the same mask; eight neighbours of a row share
// one evaluation, 16 bits each, low half-words first.  16 bits per element halve the
// integer work, which shows in the elementwise kernels; p is rounded to a multiple of
// 2^-16 and the scale is that of the rounded p, so the expectation is exact.  The ten
// round keys come ready-made in the kernel's arguments.
__device__ __forceinline__ uint4 drop_bits(const DropArgs& d, uint64_t off, int row, int g) {
  uint32_t c0 = (uint32_t)g, c1 = (uint32_t)row, c2 = (uint32_t)off, c3 = (uint32_t)(off >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
    c0 = (uint32_t)(p1 >> 32) ^ c1 ^ d.key[r][0];
    c2 = (uint32_t)(p0 >> 32) ^ c3 ^ d.key[r][1];
    c1 = (uint32_t)p1;
    c3 = (uint32_t)p0;
  }
  return make_uint4(c0, c1, c2, c3);
}

__device__ __forceinline__ uint64_t drop_offset(const DropArgs& d) {
  return d.offset + ((d.on && d.offset_ptr) ? *d.offset_ptr : 0ull);
}

// Two neighbours and their word of 16-bit numbers u.  u < t is u * 2^16 <= t * 2^16 - 1
// = d.last, which the upper half-word's compare needs no shift for.  A dropped element is
// 0 whatever it held, infinities and NaN included.
__device__ __forceinline__ void drop2(float& lo, float& hi, const DropArgs& d, uint32_t w) {
  lo = (w << 16) <= d.last ? 0.f : lo * d.scale;
  hi = w <= d.last ? 0.f : hi * d.scale;
}

__device__ __forceinline__ void drop8(float (&v)[8], const DropArgs& d, uint4 b) {
  drop2(v[0], v[1], d, b.x);
  drop2(v[2], v[3], d, b.y);
  drop2(v[4], v[5], d, b.z);
  drop2(v[6], v[7], d, b.w);
}

// Columns c .. c+3 (c a multiple of 4).
__device__ __forceinline__ void drop4(float (&v)[4], const DropArgs& d, uint64_t off, int row, int c) {
  const uint4 b = drop_bits(d, off, row, c >> 3);
  drop2(v[0], v[1], d, c & 4 ? b.z : b.x);
  drop2(v[2], v[3], d, c & 4 ? b.w : b.y);
}

}  // namespace mlpg
