// quant_blocks.hip -- activations to OCP e4m3 with one fp32 scale for each 128
// elements of a row.
//
//   scale[t, b] = max |x[t, 128 b ..]| / 448  (1 where that is 0)
//   q[t, k]     = e4m3(clamp(x[t, k] / scale[t, k / 128], -448, 448))
//
// Bound by HBM: three bytes an element.  Sixteen lanes have a block, eight
// elements each, so its maximum is taken within a DPP row: on the magnitudes'
// bits, whose order is that of the numbers with Inf and NaN on top, which so
// stay visible in the scale.  A workgroup has 16 tokens and four blocks of each:
// the scales of a block's tokens lie side by side in memory (the product's
// lanes read them so), and each row is read 1 KB at a time.
#include "db_elem.h"
#include "db_kernels.h"

namespace dbk {

namespace {

constexpr int kThreads = 256;
constexpr int kTokens = kThreads / 16;  // of a workgroup
constexpr int kBlocks = 4;              // of each of its tokens

template <int CTRL>
__device__ __forceinline__ unsigned dpp_max(unsigned v) {
  return max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true));
}

// The largest magnitude's bits of the 128 elements that a DPP row holds.
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
__device__ __forceinline__ float to_float(unsigned bits) {
  return (float)__builtin_bit_cast(typename E::type, (unsigned short)bits);
}

template <class E>
__global__ __launch_bounds__(kThreads) void quantize_blocks_kernel(QuantCall c) {
  typedef typename E::type elem;
  const int t = blockIdx.x * kTokens + threadIdx.x / 16, lane = threadIdx.x & 15;
  if (t >= c.T) return;
  const int KB = (c.K + 127) / 128;
  const elem* const row = static_cast<const elem*>(c.x) + t * c.x_row;
  unsigned char* const out = static_cast<unsigned char*>(c.q) + (size_t)t * c.K;
  u4 w[kBlocks];
#pragma unroll
  for (int i = 0; i < kBlocks; ++i) {
    const int k = (blockIdx.y * kBlocks + i) * 128 + lane * 8;
    w[i] = k < c.K ? ld_stream(row + k) : u4{0, 0, 0, 0};
  }
#pragma unroll
  for (int i = 0; i < kBlocks; ++i) {
    const int b = blockIdx.y * kBlocks + i, k = b * 128 + lane * 8;
    float scale = to_float<E>(row_magnitude(w[i])) / 448.0f;
    if (scale == 0.0f) scale = 1.0f;
    u2 r;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float v[4];
#pragma unroll
      for (int j = 0; j < 4; ++j)
        v[j] = clamp448(to_float<E>(w[i][2 * h + j / 2] >> (16 * (j & 1))) / scale);
      int p = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
      p = __builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], p, true);
      r[h] = (unsigned)p;
    }
    if (k < c.K) *reinterpret_cast<u2*>(out + k) = r;
    if (lane == 0 && b < KB) c.scale[t * c.scale_t + b * c.scale_b] = scale;
  }
}

}  // namespace

hipError_t launch_quantize_blocks(const QuantCall& c, hipStream_t stream) {
  const dim3 grid((c.T + kTokens - 1) / kTokens, ((c.K + 127) / 128 + kBlocks - 1) / kBlocks);
  if (c.bf16)
    quantize_blocks_kernel<ElemBF16><<<grid, kThreads, 0, stream>>>(c);
  else
    quantize_blocks_kernel<ElemF16><<<grid, kThreads, 0, stream>>>(c);
  return hipGetLastError();
}

}  // namespace dbk
