// Codes of 8 bits and the numbers they stand for (the formats stand in g16.h, at g16_cache_write).
#pragma once

#include "g16_common.hpp"

namespace g16 {

typedef float float2v __attribute__((ext_vector_type(2)));

// n / by without a division: (2 n magic >> 32) >> shift, for n below 2^31.
struct Divide {
  uint32_t by, magic, shift;
  __device__ uint32_t operator()(uint32_t n) const { return __umulhi(2 * n, magic) >> shift; }
};
inline Divide divide_by(uint32_t by) {
  uint32_t shift = 0;
  while ((1ull << shift) < by) ++shift;
  return Divide{by, static_cast<uint32_t>((1ull << (31 + shift)) / by + 1), shift};
}

// The eight numbers of two dwords of codes, exactly.
template <int CODE>
__device__ inline void decode8(u32x2 codes, float (&x)[8]) {
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    if constexpr (CODE == G16_CODE_INT8) {
#pragma unroll
      for (int j = 0; j < 4; ++j) x[4 * w + j] = static_cast<float>(static_cast<int8_t>(codes[w] >> (8 * j)));
    } else {
      const float2v lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(codes[w]), false);
      const float2v hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(codes[w]), true);
      x[4 * w] = lo[0];
      x[4 * w + 1] = lo[1];
      x[4 * w + 2] = hi[0];
      x[4 * w + 3] = hi[1];
    }
  }
}

// Scale of a run of values and what they are multiplied by for their codes; 0 for a run that is written as zeros
// (`keeps` false).
struct Scaling {
  float scale, inverse;
  bool keeps;
};
template <int CODE>
__device__ inline Scaling scaling_of(float top) {  // top: the largest magnitude; not finite where one of them is not
  Scaling s;
  const uint32_t bits = __float_as_uint(top);
  const bool lost = bits >= 0x7f800000u;
  s.keeps = !lost && top >= G16_CODE_LEAST;
  if constexpr (CODE == G16_CODE_INT8) {
    s.scale = top / 127.f;
    s.inverse = 127.f / top;
  } else {
    // 448 = 1.75 * 2^8: the exponent of top less 8, one more where its digits are past 1.75
    const uint32_t e = (bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1u : 0u);
    s.scale = __uint_as_float(e << 23);
    s.inverse = __uint_as_float((254u - e) << 23);
  }
  if (!s.keeps) s.scale = lost ? __uint_as_float(0x7fc00000u) : 0.f;
  return s;
}

// Codes of eight values.
template <int CODE>
__device__ inline u32x2 encode8(const float (&x)[8], const Scaling& s) {
  u32x2 codes;
#pragma unroll
  for (int w = 0; w < 2; ++w) {
    if constexpr (CODE == G16_CODE_INT8) {
      // The sum with 1.5 * 2^23 is rounded once, to a whole number, whose last byte is the code.
      uint32_t n[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) n[j] = __float_as_uint(fmaf(x[4 * w + j], s.inverse, 12582912.f));
      const uint32_t lo = __builtin_amdgcn_perm(n[1], n[0], 0x0c0c0400u), hi = __builtin_amdgcn_perm(n[3], n[2], 0x04000c0cu);
      codes[w] = lo | hi;
    } else {
      int c = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * w] * s.inverse, x[4 * w + 1] * s.inverse, 0, false);
      c = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * w + 2] * s.inverse, x[4 * w + 3] * s.inverse, c, true);
      codes[w] = static_cast<uint32_t>(c);
    }
    if (!s.keeps) codes[w] = 0;
  }
  return codes;
}

}  // namespace g16
