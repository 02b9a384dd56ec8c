// layer.cuh -- what the MLP layer's kernels share: 16-bit types, activations and
// their slopes, and dropout from a counter-based generator.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cstdint>

#include "kernels.h"

namespace mlpg {

// ---- 16-bit types ----------------------------------------------------------------
// Two values of a 32-bit word, low half first.
__device__ __forceinline__ float2 unpack2(uint32_t w, int type) {
  if (type == kTypeF16) return __half22float2(*reinterpret_cast<const __half2*>(&w));
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u));
}

// Round to nearest even, both types; f16 overflows to infinity.
__device__ __forceinline__ uint32_t pack2(float lo, float hi, int type) {
  if (type == kTypeF16) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&b);
}

__device__ __forceinline__ float load1(const void* base, size_t i, int type) {
  if (type == kTypeF32) return static_cast<const float*>(base)[i];
  const uint32_t w = static_cast<const uint16_t*>(base)[i];
  return unpack2(w, type).x;
}

__device__ __forceinline__ void store1(void* base, size_t i, float v, int type) {
  if (type == kTypeF32) static_cast<float*>(base)[i] = v;
  else static_cast<uint16_t*>(base)[i] = (uint16_t)(pack2(v, 0.f, type) & 0xFFFFu);
}

// ---- activations ------------------------------------------------------------------
// gelu_tanh is written as z * sigmoid(2u), u = sqrt(2/pi) (z + 0.044715 z^3), which
// equals 0.5 z (1 + tanh u) without the cancellation at large negative z.
__device__ __forceinline__ float sigmoidf_(float t) { return __fdividef(1.f, 1.f + __expf(-t)); }

__device__ __forceinline__ float gelu_u2(float z) { return 1.5957691216057308f * (z + 0.044715f * z * z * z); }

__device__ __forceinline__ float act_fwd(float z, int act) {
  switch (act) {
    case kActRelu: return z < 0.f ? 0.f : z;   // NaN stays NaN
    case kActGelu: return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
    case kActGeluTanh: return z * sigmoidf_(gelu_u2(z));
    case kActSilu: return z * sigmoidf_(z);
    default: return z;
  }
}

// The same for eight values: one branch on the activation, not eight.
__device__ __forceinline__ void act_fwd8(float (&v)[8], int act) {
  switch (act) {
    case kActRelu:
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = act_fwd(v[i], kActRelu);
      break;
    case kActGelu:
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = act_fwd(v[i], kActGelu);
      break;
    case kActGeluTanh:
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = act_fwd(v[i], kActGeluTanh);
      break;
    case kActSilu:
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = act_fwd(v[i], kActSilu);
      break;
    default: break;
  }
}

// act'(z).  z is a stored pre-activation, which f16 may have rounded to an
// infinity: beyond the clamps every slope is 0 or 1 to f32 precision, so an
// infinite z gets its limit instead of inf * 0.  NaN passes the comparisons.
__device__ __forceinline__ float act_slope(float z, int act) {
  switch (act) {
    case kActRelu: return z > 0.f ? 1.f : (z <= 0.f ? 0.f : z);
    case kActGelu: {
      z = z > 30.f ? 30.f : (z < -30.f ? -30.f : z);
      return 0.5f * (1.f + erff(z * 0.70710678118654752f)) + z * __expf(-0.5f * z * z) * 0.3989422804014327f;
    }
    case kActGeluTanh: {
      z = z > 30.f ? 30.f : (z < -30.f ? -30.f : z);
      const float q = sigmoidf_(gelu_u2(z));
      return q + z * q * (1.f - q) * (1.5957691216057308f * (1.f + 0.134145f * z * z));
    }
    case kActSilu: {
      z = z > 80.f ? 80.f : (z < -80.f ? -80.f : z);
      const float q = sigmoidf_(z);
      return q * (1.f + z * (1.f - q));
    }
    default: return 1.f;
  }
}

// ---- dropout ------------------------------------------------------------------------
// Philox4x32-10 (Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as easy
// as 1, 2, 3", SC 2011).  The counter is (column / 8, row, offset), the key the
// seed, so any tile shape computes the same mask; eight neighbours of a row share
// one evaluation, 16 bits each, low half-words first.  16 bits per element halve the
// integer work that would otherwise bound the elementwise kernels (about 80
// instructions per evaluation); p is rounded to a multiple of 2^-16 and the scale is
// that of the rounded p, so the expectation is exact.
__device__ __forceinline__ uint4 philox4x32_10(uint32_t c0, uint32_t c1, uint32_t c2, uint32_t c3, uint32_t k0,
                                               uint32_t k1) {
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const uint64_t p0 = (uint64_t)0xD2511F53u * c0, p1 = (uint64_t)0xCD9E8D57u * c2;
    const uint32_t n0 = (uint32_t)(p1 >> 32) ^ c1 ^ k0, n2 = (uint32_t)(p0 >> 32) ^ c3 ^ k1;
    c1 = (uint32_t)p1;
    c3 = (uint32_t)p0;
    c0 = n0;
    c2 = n2;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(c0, c1, c2, c3);
}

__device__ __forceinline__ uint64_t drop_offset(const DropArgs& d) {
  return d.offset + ((d.thr && d.offset_ptr) ? *d.offset_ptr : 0ull);
}

// The eight 16-bit numbers of columns 8 g .. 8 g + 7 of `row`.
__device__ __forceinline__ uint4 drop_bits(const DropArgs& d, uint64_t off, int row, int g) {
  return philox4x32_10((uint32_t)g, (uint32_t)row, (uint32_t)off, (uint32_t)(off >> 32), (uint32_t)d.seed,
                       (uint32_t)(d.seed >> 32));
}

// A dropped element is 0 whatever it held, infinities and NaN included.
__device__ __forceinline__ void drop8(float (&v)[8], const DropArgs& d, uint64_t off, int row, int g) {
  const uint4 b = drop_bits(d, off, row, g);
  const uint32_t w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    v[2 * i] = (w[i] & 0xFFFFu) >= d.thr ? v[2 * i] * d.scale : 0.f;
    v[2 * i + 1] = (w[i] >> 16) >= d.thr ? v[2 * i + 1] * d.scale : 0.f;
  }
}

__device__ __forceinline__ float drop1(float v, const DropArgs& d, uint64_t off, int row, int col) {
  const uint4 b = drop_bits(d, off, row, col >> 3);
  const uint32_t w[4] = {b.x, b.y, b.z, b.w};
  const int i = col & 7;
  const uint32_t u = (w[i >> 1] >> (16 * (i & 1))) & 0xFFFFu;
  return u >= d.thr ? v * d.scale : 0.f;
}

}  // namespace mlpg
