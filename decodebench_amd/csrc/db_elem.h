// db_elem.h -- the 16-bit element types of activations, their vectors and the
// matrix instructions on them.
#pragma once

#include "db_device.h"

namespace dbk {

typedef __bf16 b2 __attribute__((ext_vector_type(2)));
typedef __bf16 b4 __attribute__((ext_vector_type(4)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef unsigned u2 __attribute__((ext_vector_type(2)));

// Element types of the activations (and of a cache or weights of that type).
struct ElemF16 {
  typedef _Float16 type;
  typedef h8 vec8;
  typedef h4 vec4;
  static constexpr unsigned kExp = 0x7C00u;  // exponent bits: all set in Inf and NaN
  __device__ static f4 mfma16(vec8 a, vec8 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  __device__ static f4 mfma16k16(vec4 a, vec4 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(a, b, c, 0, 0, 0);
  }
  __device__ static f16v mfma32(vec8 a, vec8 b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
  // four e4m3 values to two pairs (exact: all of them are fp16 numbers)
  __device__ static u2 widen(unsigned w) {
    u2 r;
    r[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, false));
    r[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.0f, true));
    return r;
  }
};
struct ElemBF16 {
  typedef __bf16 type;
  typedef b8 vec8;
  typedef b4 vec4;
  static constexpr unsigned kExp = 0x7F80u;
  __device__ static f4 mfma16(vec8 a, vec8 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  __device__ static f4 mfma16k16(vec4 a, vec4 b, f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s4, a),
                                                     __builtin_bit_cast(s4, b), c, 0, 0, 0);
  }
  __device__ static f16v mfma32(vec8 a, vec8 b, f16v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  __device__ static u2 widen(unsigned w) {  // exact as well: three mantissa bits
    u2 r;
    r[0] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, false));
    r[1] = __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.0f, true));
    return r;
  }
};

// NaN stays NaN, everything else is clamped to the largest finite e4m3.
__device__ __forceinline__ float clamp448(float x) {
  return x > 448.0f ? 448.0f : x < -448.0f ? -448.0f : x;
}

}  // namespace dbk
