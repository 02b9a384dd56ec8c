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
// access where the rows allow it (vec); elements past the row read as 0.
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

// Four elements the same way; none past the row is written.
template <int TYPE>
__device__ __forceinline__ void store4(const float (&v)[4], void* base, size_t at, int c, int cols, bool vec) {
  uint16_t* p = static_cast<uint16_t*>(base) + at;
  if (vec && c + 4 <= cols) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack2<TYPE>(v[0], v[1]), pack2<TYPE>(v[2], v[3]));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + i < cols) store1<TYPE>(p, i, v[i]);
  }
}

// ---- pairs of f32 -------------------------------------------------------------------
// sm_100 multiplies, adds and fuses two f32 per instruction; the epilogues are bound by
// instructions issued, so their arithmetic goes in pairs.
struct f32x2 {
  unsigned long long v;
};
__device__ __forceinline__ f32x2 pair2(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ f32x2 pair2(float x) { return pair2(x, x); }
__device__ __forceinline__ void split2(f32x2 a, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(a.v));
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
template <typename F>
__device__ __forceinline__ f32x2 each2(f32x2 a, F f) {
  float lo, hi;
  split2(a, lo, hi);
  return pair2(f(lo), f(hi));
}

// ---- activations ------------------------------------------------------------------
__device__ __forceinline__ f32x2 rcp2(f32x2 a) {
  return each2(a, [](float x) {
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
  });
}
__device__ __forceinline__ f32x2 ex2_2(f32x2 a) {   // 2^a
  return each2(a, [](float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
  });
}
__device__ __forceinline__ f32x2 abs2(f32x2 a) {
  return each2(a, [](float x) { return fabsf(x); });
}
// between -m and m; NaN stays NaN
__device__ __forceinline__ f32x2 clamp2(f32x2 a, float m) {
  return each2(a, [m](float x) {
    float y;
    asm("{\n\t.reg .f32 t;\n\tmin.NaN.f32 t, %1, %2;\n\tmax.NaN.f32 %0, t, %3;\n\t}"
        : "=f"(y)
        : "f"(x), "f"(m), "f"(-m));
    return y;
  });
}

// 1 / (1 + 2^x): the sigmoid of -x / log2(e)
__device__ __forceinline__ f32x2 sigmoid2(f32x2 x) { return rcp2(add2(ex2_2(x), pair2(1.f))); }

// gelu_tanh is z * sigmoid(2u), u = sqrt(2/pi) (z + 0.044715 z^3), which equals
// 0.5 z (1 + tanh u) without the cancellation at large negative z; -2u log2(e) here.
__device__ __forceinline__ f32x2 gelu_2u(f32x2 z) {
  return mul2(z, fma2(mul2(z, z), pair2(-0.10294324f), pair2(-2.3022082f)));
}

// e = exp(-a^2/2) and -Phi(-a), the normal distribution's tail, for a >= 0.  Phi(-a) / e
// falls from 1/2 like 1 / (sqrt(2 pi) a), so it is t P(t) with t = 1 / (1 + 0.3 a) and a
// polynomial P.  A 16-bit float resolves the tail as finely as the middle, so P is fitted to a
// small relative error for a <= 13.4, where e underflows, with the absolute one of e t P(t)
// held down beside it: 1.3e-5 and 3.7e-7 as evaluated here, in f32, 1/40 of f16's half step.
// (One degree more: 1.3e-6, and 3 % of act_grad's time; one less: 1.2e-4 and 2.3e-6.)  No
// branch, and the slope reuses e.  The tail comes negated and without its factor e.
__device__ __forceinline__ f32x2 normal_tail2(f32x2 a, f32x2& e) {
  const f32x2 t = rcp2(fma2(pair2(0.3f), a, pair2(1.f)));
  e = ex2_2(mul2(mul2(a, a), pair2(-0.72134752044448170f)));
  f32x2 q = fma2(t, pair2(0.07940985262f), pair2(-0.2223330438f));
  q = fma2(t, q, pair2(0.02329958044f));
  q = fma2(t, q, pair2(-0.1471278965f));
  q = fma2(t, q, pair2(-0.1131272018f));
  q = fma2(t, q, pair2(-0.1201210469f));
  return mul2(q, t);
}

// z < 0 ? neg : pos, element by element (NaN takes pos)
__device__ __forceinline__ f32x2 by_sign2(f32x2 z, f32x2 neg, f32x2 pos) {
  float zl, zh, nl, nh, pl, ph;
  split2(z, zl, zh);
  split2(neg, nl, nh);
  split2(pos, pl, ph);
  return pair2(zl < 0.f ? nl : pl, zh < 0.f ? nh : ph);
}

template <int ACT>
__device__ __forceinline__ f32x2 act_fwd2(f32x2 z) {
  if constexpr (ACT == kActRelu) return by_sign2(z, pair2(0.f), z);   // NaN stays NaN
  if constexpr (ACT == kActGelu) {
    f32x2 e;
    const f32x2 tail = normal_tail2(abs2(z), e), p = mul2(tail, e);
    return mul2(z, by_sign2(z, mul2(p, pair2(-1.f)), add2(p, pair2(1.f))));
  }
  if constexpr (ACT == kActGeluTanh) return mul2(z, sigmoid2(gelu_2u(z)));
  if constexpr (ACT == kActSilu) return mul2(z, sigmoid2(mul2(z, pair2(-1.4426950408889634f))));
  return z;
}

template <int ACT, int W>
__device__ __forceinline__ void act_fwd_n(float (&v)[W]) {
#pragma unroll
  for (int i = 0; i < W; i += 2) split2(act_fwd2<ACT>(pair2(v[i], v[i + 1])), v[i], v[i + 1]);
}

// The same for an activation known at run time: one branch for all.
template <int W>
__device__ __forceinline__ void act_fwd_n(float (&v)[W], int act) {
  switch (act) {
    case kActRelu: act_fwd_n<kActRelu, W>(v); break;
    case kActGelu: act_fwd_n<kActGelu, W>(v); break;
    case kActGeluTanh: act_fwd_n<kActGeluTanh, W>(v); break;
    case kActSilu: act_fwd_n<kActSilu, W>(v); break;
    default: break;
  }
}

// act'(z).  z is a stored pre-activation, which f16 may have rounded to an
// infinity: beyond the clamps the exps are 0 or infinite in f32 and every slope is 0 or 1,
// so an infinite z gets its limit instead of inf * 0.  NaN stays NaN.
template <int ACT>
__device__ __forceinline__ f32x2 act_slope2(f32x2 z) {
  const f32x2 one = pair2(1.f), minus = pair2(-1.f);
  if constexpr (ACT == kActRelu) return each2(z, [](float x) { return x > 0.f ? 1.f : (x <= 0.f ? 0.f : x); });
  if constexpr (ACT == kActGelu) {
    // slope(-a) = Phi(-a) - a phi(a), slope(a) = 1 - slope(-a): each from the small side, so
    // that the negative tail keeps its digits
    f32x2 e;
    const f32x2 a = each2(z, [](float x) {
      float y;
      asm("min.NaN.f32 %0, %1, 0f41F00000;" : "=f"(y) : "f"(fabsf(x)));   // 30
      return y;
    });
    const f32x2 tail = normal_tail2(a, e);
    const f32x2 h = mul2(e, fma2(a, pair2(0.3989422804014327f), tail));   // -slope(-a)
    const f32x2 sign = each2(z, [](float x) { return copysignf(1.f, x); });
    return fma2(sign, h, fma2(sign, pair2(0.5f), pair2(0.5f)));
  }
  if constexpr (ACT == kActGeluTanh) {
    // q + z q (1 - q) (2u)'
    z = clamp2(z, 30.f);
    const f32x2 q = sigmoid2(gelu_2u(z));
    const f32x2 d = mul2(z, fma2(mul2(z, z), pair2(0.21406445f), pair2(1.5957691216057308f)));
    return mul2(q, fma2(d, fma2(q, minus, one), one));
  }
  if constexpr (ACT == kActSilu) {
    z = clamp2(z, 90.f);   // e^-80 = 2e-35 is a bf16 number still
    const f32x2 q = sigmoid2(mul2(z, pair2(-1.4426950408889634f)));
    return mul2(q, fma2(z, fma2(q, minus, one), one));
  }
  return one;
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
  float a, b;
  split2(mul2(pair2(lo, hi), pair2(d.scale)), a, b);
  lo = (w << 16) <= d.last ? 0.f : a;
  hi = w <= d.last ? 0.f : b;
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
