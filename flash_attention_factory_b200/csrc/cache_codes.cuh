// Conversion of fp32 values to what a KV cache stores, shared by the cache writers: fp16, FP8
// (round to nearest even, saturating to the largest finite code) and 8-bit integers.
#pragma once

#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "paged_attention_policy_v2.hpp"
#include "paged_attention_utils.hpp"

namespace pa {

// Where the scale of an element comes from.
enum ScaleKind : int { SCALE_SCALAR = 0, SCALE_PER_HEAD = 1, SCALE_PER_BLOCK = 2 };

// One value over its scale -> the nearest integer of -127 .. 127 (ties to even; NaN -> 0).  -128 stays
// unused so that the codes are symmetric.
__device__ __forceinline__ uint32_t int8_code(float x) {
  return static_cast<uint32_t>(max(-127, min(127, __float2int_rn(x)))) & 0xffu;
}

// Four values, already divided by their scale, -> four 8-bit codes
template <int KV>
__device__ __forceinline__ uint32_t pack_codes(float a, float b, float c, float d) {
  static_assert(KV != KV_F16, "8-bit caches only");
  if constexpr (KV == KV_I8) {
    return int8_code(a) | (int8_code(b) << 8) | (int8_code(c) << 16) | (int8_code(d) << 24);
  } else {
    constexpr __nv_fp8_interpretation_t fmt = (KV == KV_E5M2) ? __NV_E5M2 : __NV_E4M3;
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, fmt);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(c, d), __NV_SATFINITE, fmt);
    return lo | (hi << 16);
  }
}

// Four codes -> their values (exact)
template <int KV>
__device__ __forceinline__ void unpack_codes(uint32_t v, float (&x)[4]) {
  uint32_t lo, hi;
  fp8x4_to_half2x2<KV>(v, lo, hi);
  const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&lo));
  const float2 b = __half22float2(*reinterpret_cast<const __half2 *>(&hi));
  x[0] = a.x;
  x[1] = a.y;
  x[2] = b.x;
  x[3] = b.y;
}

// Division of many values by one scale.  q = x r with r the rounded reciprocal is off by at most two units in
// the last place; one residual step (Markstein, "Computation of elementary functions on the IBM RISC System/6000
// processor", 1990), q + (x - q s) r, gives the correctly rounded quotient but for rare cases of one unit,
// so a code can differ from that of the rounded quotient only where the quotient lies within 2^-23 of
// itself from a rounding border.  Three operations instead of a full division.  The residual needs s and 1 / s away from the ends
// of the exponent range; other scales take the division.  So do infinities, whose residual is a NaN.
struct Divider {
  float s, r;
  bool plain;
  __device__ __forceinline__ explicit Divider(float scale) {
    s = scale;
    r = __frcp_rn(scale);
    plain = !(scale >= 0x1p-60f && scale <= 0x1p60f);
  }
  __device__ __forceinline__ float operator()(float x) const {
    const float q = __fmul_rn(x, r);
    return __fmaf_rn(__fmaf_rn(-q, s, x), r, q);
  }
};

// Eight values over their scale
__device__ __forceinline__ void divide8(float (&x)[8], const Divider &by) {
  float largest = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) largest = fmaxf(largest, fabsf(x[j])); // passes over NaNs, which stay NaNs either way
  if (by.plain || largest > 3.0e38f) {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = __fdiv_rn(x[j], by.s);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = by(x[j]);
  }
}

// Four finite values of at most 127.5 in size -> four codes.  Adding 1.5 * 2^23 leaves the nearest integer (ties to
// even) in the low bits of the sum, whose low byte is the code: full-rate additions and byte
// placements instead of float-to-integer conversions, which run at an eighth of that rate.
template <int KV>
__device__ __forceinline__ uint32_t pack_small_codes(float a, float b, float c, float d) {
  if constexpr (KV == KV_I8) {
    constexpr float kShift = 12582912.f;
    const uint32_t ab = __byte_perm(__float_as_uint(__fadd_rn(a, kShift)), __float_as_uint(__fadd_rn(b, kShift)), 0x0040);
    const uint32_t cd = __byte_perm(__float_as_uint(__fadd_rn(c, kShift)), __float_as_uint(__fadd_rn(d, kShift)), 0x0040);
    return __byte_perm(ab, cd, 0x5410);
  } else {
    return pack_codes<KV>(a, b, c, d);
  }
}

// Eight fp16 values of one 16-byte load as fp32
__device__ __forceinline__ void unpack_half8(uint4 v, float (&x)[8]) {
  const __half2 *h = reinterpret_cast<const __half2 *>(&v);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(h[i]);
    x[2 * i] = f.x;
    x[2 * i + 1] = f.y;
  }
}

__device__ __forceinline__ uint4 pack_half8(const float (&x)[8]) {
  return make_uint4(pack_half2(x[0], x[1]), pack_half2(x[2], x[3]), pack_half2(x[4], x[5]), pack_half2(x[6], x[7]));
}

// ------------------------------------------------------------------- position rotation
// A head is dealt to lanes in items of 16 elements.  Inside the rotated part (the first
// `rotary_dim` dims) item i holds the eight pairs 8 i .. 8 i + 7: elements [8 i, 8 i + 8) and the
// same eight behind rotary_dim / 2 (halves), or the 16 elements from 16 i on (interleaved).  Behind it
// item i is the 16 elements from 16 i on.  Either way an item is two 16-byte pieces of fp16.
struct RotaryItem {
  uint32_t first, second; // element offsets of the two pieces of eight
  bool rotated;
};

__device__ __forceinline__ RotaryItem rotary_item(uint32_t item, uint32_t rotary_dim, bool interleaved) {
  RotaryItem r;
  r.rotated = item * 16u < rotary_dim;
  if (r.rotated && !interleaved) {
    r.first = item * 8u;
    r.second = rotary_dim / 2u + item * 8u;
  } else {
    r.first = item * 16u;
    r.second = r.first + 8u;
  }
  return r;
}

// Cosines and sines of an item's eight pairs from the table row of a position
// (rotary_dim / 2 cosines, then the sines).
__device__ __forceinline__ void load_cos_sin(const float *__restrict__ row, uint32_t item, uint32_t rotary_dim,
                                             float (&c)[8], float (&s)[8]) {
  const float4 *pc = reinterpret_cast<const float4 *>(row + item * 8u);
  const float4 *ps = reinterpret_cast<const float4 *>(row + rotary_dim / 2u + item * 8u);
  const float4 c0 = __ldg(pc), c1 = __ldg(pc + 1), s0 = __ldg(ps), s1 = __ldg(ps + 1);
  c[0] = c0.x; c[1] = c0.y; c[2] = c0.z; c[3] = c0.w; c[4] = c1.x; c[5] = c1.y; c[6] = c1.z; c[7] = c1.w;
  s[0] = s0.x; s[1] = s0.y; s[2] = s0.z; s[3] = s0.w; s[4] = s1.x; s[5] = s1.y; s[6] = s1.z; s[7] = s1.w;
}

// a' = a c - b s, b' = b c + a s for an item's eight pairs, in place.  The products and the sum are
// rounded one by one (no fused multiply-add), so that the fp32 values are those of the formula
// evaluated operation by operation in any order-preserving implementation.
__device__ __forceinline__ void rotate_item(float (&x)[8], float (&y)[8], const float (&c)[8], const float (&s)[8],
                                            bool interleaved) {
  auto turn = [](float &a, float &b, float co, float si) {
    const float na = __fsub_rn(__fmul_rn(a, co), __fmul_rn(b, si));
    const float nb = __fadd_rn(__fmul_rn(b, co), __fmul_rn(a, si));
    a = na;
    b = nb;
  };
  if (interleaved) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      turn(x[2 * j], x[2 * j + 1], c[j], s[j]);
      turn(y[2 * j], y[2 * j + 1], c[4 + j], s[4 + j]);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) turn(x[j], y[j], c[j], s[j]);
  }
}

// ------------------------------------------------ the same on pairs of values (one instruction for two)
__device__ __forceinline__ unsigned long long pair_bits(float2 v) {
  return static_cast<unsigned long long>(__float_as_uint(v.x)) | (static_cast<unsigned long long>(__float_as_uint(v.y)) << 32);
}
__device__ __forceinline__ float2 bits_pair(unsigned long long v) {
  return make_float2(__uint_as_float(static_cast<uint32_t>(v)), __uint_as_float(static_cast<uint32_t>(v >> 32)));
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  unsigned long long r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(pair_bits(a)), "l"(pair_bits(b)));
  return bits_pair(r);
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  unsigned long long r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(pair_bits(a)), "l"(pair_bits(b)), "l"(pair_bits(c)));
  return bits_pair(r);
}

struct Item2 {
  float2 x[4], y[4]; // the item's two pieces of eight
};

__device__ __forceinline__ void unpack_item(const uint4 &first, const uint4 &second, Item2 &v) {
  const __half2 *a = reinterpret_cast<const __half2 *>(&first);
  const __half2 *b = reinterpret_cast<const __half2 *>(&second);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v.x[j] = __half22float2(a[j]);
    v.y[j] = __half22float2(b[j]);
  }
}

// rotate_item with the table row's pieces read on the way; every product and sum is rounded as there
__device__ __forceinline__ void rotate_item2(Item2 &v, const float *__restrict__ cosines, const float *__restrict__ sines,
                                             bool interleaved) {
  // u - v as fma(v, -1, u): a plain addition of two packed products is contracted into a fused multiply-add by
  // the compiler, rounding modifiers or not
  const float2 minus = make_float2(-1.f, -1.f), alternate = make_float2(-1.f, 1.f);
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float4 c4 = __ldg(reinterpret_cast<const float4 *>(cosines) + k);
    const float4 s4 = __ldg(reinterpret_cast<const float4 *>(sines) + k);
    if (!interleaved) {
      const float2 c[2] = {make_float2(c4.x, c4.y), make_float2(c4.z, c4.w)};
      const float2 s[2] = {make_float2(s4.x, s4.y), make_float2(s4.z, s4.w)};
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float2 a = v.x[2 * k + j], b = v.y[2 * k + j];
        v.x[2 * k + j] = fma2(mul2(b, s[j]), minus, mul2(a, c[j]));
        v.y[2 * k + j] = fma2(mul2(a, make_float2(-s[j].x, -s[j].y)), minus, mul2(b, c[j]));
      }
    } else {
      const float c[4] = {c4.x, c4.y, c4.z, c4.w}, s[4] = {s4.x, s4.y, s4.z, s4.w};
      float2 *p = (k == 0) ? v.x : v.y;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        p[j] = fma2(mul2(make_float2(p[j].y, p[j].x), make_float2(s[j], s[j])), alternate,
                    mul2(p[j], make_float2(c[j], c[j])));
    }
  }
}

// Divider on a pair
__device__ __forceinline__ float2 divide2(float2 x, float2 minus_s, float2 r) {
  const float2 q = mul2(x, r);
  return fma2(fma2(q, minus_s, x), r, q);
}

} // namespace pa
