// quant_blocks.h -- 128 elements to e4m3 and their scale, by the 16 lanes of a DPP row:
//   scale = max |x| * fp32(1 / 448) (1 where that is 0), q = e4m3(clamp(x / scale, -448, 448)).
// The product, not the quotient: it is what a tensor divided by a number gives on the
// GPU in torch, so a plain form there has the same codes.
#pragma once

#include "db_elem.h"

namespace dbk {

template <int CTRL>
__device__ __forceinline__ unsigned dpp_max(unsigned v) {
  return max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true));
}

// The largest magnitude's bits of the 128 elements that a DPP row holds: their
// order is that of the numbers, with Inf and NaN on top.
__device__ __forceinline__ unsigned row_magnitude(u4 w) {
  unsigned m = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) m = max(m, max(w[i] & 0x7FFFu, (w[i] >> 16) & 0x7FFFu));
  m = dpp_max<kQuadSwap1>(m);
  m = dpp_max<kQuadSwap2>(m);
  m = dpp_max<kRowHalfMirror>(m);
  return dpp_max<kRowMirror>(m);
}

template <class E>
__device__ __forceinline__ float float_of(unsigned bits) {
  return (float)__builtin_bit_cast(typename E::type, (unsigned short)bits);
}

// Eight elements of the lane; every lane of the row gets the scale.
//
// The quotients are those of an fp32 division, from the scale's reciprocal r:
// p = x r is at most two steps off, p + (x - p scale) r rounds the exact quotient
// but for errors of 2^-46 of it (Markstein's correction of a quotient), and one that fp32
// holds exactly, as a tie between two codes is, comes out as it is.  Three
// operations an element instead of ten: 8191 x 14336 elements 67.7 us, 76.5 with the
// division.
// Scales near the ends of fp32's range, Inf and NaN among them, take the division.
template <class E>
__device__ __forceinline__ u2 quantize128(u4 w, float& scale) {
  scale = float_of<E>(row_magnitude(w)) * (1.0f / 448.0f);
  if (scale == 0.0f) scale = 1.0f;
  float v[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = float_of<E>(w[j / 2] >> (16 * (j & 1)));
  if (__all(scale > 0x1p-100f && scale < 0x1p100f)) {
    const float r = 1.0f / scale;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float p = v[j] * r;
      v[j] = __builtin_fmaf(__builtin_fmaf(-p, scale, v[j]), r, p);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = v[j] / scale;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) v[j] = clamp448(v[j]);
  u2 q;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int p = __builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h], v[4 * h + 1], 0, false);
    q[h] = (unsigned)__builtin_amdgcn_cvt_pk_fp8_f32(v[4 * h + 2], v[4 * h + 3], p, true);
  }
  return q;
}

}  // namespace dbk
