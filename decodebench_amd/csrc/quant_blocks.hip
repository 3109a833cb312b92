// quant_blocks.hip -- activations to OCP e4m3 with one fp32 scale for each 128
// elements of a row.
//
//   scale[t, b] = max |x[t, 128 b ..]| * fp32(1 / 448)  (1 where that is 0)
//   q[t, k]     = e4m3(clamp(x[t, k] / scale[t, k / 128], -448, 448))
//
// Bound by HBM: three bytes an element.  Sixteen lanes have a block, eight
// elements each, so its maximum is taken within a DPP row: on the magnitudes'
// bits, whose order is that of the numbers with Inf and NaN on top, which so
// stay visible in the scale.  A workgroup has 16 tokens and four blocks of each:
// the scales of a block's tokens lie side by side in memory (the product's
// lanes read them so), and each row is read 1 KB at a time.
// 8191 x 14336: 67.2 us, 5.3 TB/s, which is a large copy's rate; 5 x 4096: 5.9 us, the call.
#include "db_kernels.h"
#include "quant_blocks.h"

namespace dbk {

namespace {

constexpr int kThreads = 256;
constexpr int kTokens = kThreads / 16;  // of a workgroup
constexpr int kBlocks = 4;              // of each of its tokens

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
    float scale;
    const u2 r = quantize128<E>(w[i], scale);
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
