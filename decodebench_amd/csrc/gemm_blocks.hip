// gemm_blocks.hip -- products of e4m3 activations with one scale for each 128
// elements of a row and e4m3 weights with one scale for each block of 128 x 128:
//
//   y[t, n] = sum_b xs[t, b] ws[n / 128, b] sum_{k in b} x[t, k] W[n, k]
//
// v_mfma_f32_16x16x128_f8f6f4 sums a whole block of k at once: its result is
// scaled and added to the fp32 sum with one multiply-add for each of the four
// outputs of a lane.  Weights are the A operand and tokens the B operand, so a
// lane's outputs belong to one token and share one scale.
#include "db_elem.h"
#include "db_kernels.h"

namespace dbk {

namespace {

typedef int i8v __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kOut = 1 << 30;  // an offset behind every buffer: loads give zero

__device__ __forceinline__ i8v join(u4 lo, u4 hi) {
  i8v r;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    r[i] = (int)lo[i];
    r[4 + i] = (int)hi[i];
  }
  return r;
}

__device__ __forceinline__ u4 ld_buf(__amdgpu_buffer_rsrc_t r, int offset) {
  return __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(r, offset, 0, 0));
}

__device__ __forceinline__ f4 product(i8v w, i8v x) {
  const f4 zero = {0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(w, x, zero, 0, 0, 0, 0, 0, 0);
}

// Four outputs n .. n + 3 of one token.
template <class E>
__device__ __forceinline__ void store4(void* y, size_t at, int left, bool vec, f4 v) {
  typename E::vec4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = (typename E::type)v[i];
  typename E::type* p = static_cast<typename E::type*>(y) + at;
  if (vec && left >= 4) {
    *reinterpret_cast<typename E::vec4*>(p) = r;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) p[i] = r[i];
  }
}

// 16 outputs and 16 TT tokens a workgroup, its waves taking blocks of K in turn.
template <class E, int TT>
__global__ __launch_bounds__(kThreads) void gemm_blocks_rows(GemmBlocksCall c) {
  __shared__ f4 s_part[kWaves][TT][kWave];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int r16 = lane & 15, q = lane >> 4;
  const int n0 = blockIdx.x * 16, t0 = blockIdx.y * 16 * TT;
  const int KB = (c.K + 127) / 128;
  const __amdgpu_buffer_rsrc_t rw = make_rsrc(
      static_cast<const char*>(c.W) + (size_t)n0 * c.K, min(16, c.N - n0) * c.K);
  const __amdgpu_buffer_rsrc_t rx =
      make_rsrc(static_cast<const char*>(c.x) + t0 * c.x_row,
                (int)((min(16 * TT, c.T - t0) - 1) * c.x_row) + c.K);
  const float* const ws = c.w_scale + (size_t)(n0 / 128) * KB;
  f4 acc[TT] = {};
  for (int b = wave; b < KB; b += kWaves) {
    const int k0 = b * 128 + q * 16, k1 = k0 + 64;
    const int wr = r16 * c.K;
    const i8v w = join(ld_buf(rw, k0 < c.K ? wr + k0 : kOut), ld_buf(rw, k1 < c.K ? wr + k1 : kOut));
    const float wscale = ws[b];
#pragma unroll
    for (int i = 0; i < TT; ++i) {
      const int t = i * 16 + r16;
      const int xr = t0 + t < c.T ? t * (int)c.x_row : kOut;
      const i8v x = join(ld_buf(rx, k0 < c.K ? xr + k0 : kOut), ld_buf(rx, k1 < c.K ? xr + k1 : kOut));
      const float s = c.x_scale[min(t0 + t, c.T - 1) * c.xs_t + b * c.xs_b] * wscale;
      const f4 p = product(w, x);
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] += p[j] * s;
    }
  }
#pragma unroll
  for (int i = 0; i < TT; ++i) s_part[wave][i][lane] = acc[i];
  __syncthreads();
  for (int i = wave; i < TT; i += kWaves) {
    f4 sum = s_part[0][i][lane];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) sum += s_part[w][i][lane];
    const int t = t0 + i * 16 + r16, n = n0 + 4 * q;
    if (t < c.T && n < c.N) store4<E>(c.y, (size_t)t * c.N + n, c.N - n, c.N % 4 == 0, sum);
  }
}

template <class E>
void launch(const GemmBlocksCall& c, hipStream_t stream) {
  const int TT = c.T <= 16 ? 1 : c.T <= 32 ? 2 : 4;
  const dim3 grid((c.N + 15) / 16, (c.T + 16 * TT - 1) / (16 * TT));
  auto* const fn = TT == 1 ? gemm_blocks_rows<E, 1> : TT == 2 ? gemm_blocks_rows<E, 2>
                                                              : gemm_blocks_rows<E, 4>;
  fn<<<grid, kThreads, 0, stream>>>(c);
}

}  // namespace

hipError_t launch_gemm_blocks(const GemmBlocksCall& c, hipStream_t stream) {
  if (c.bf16)
    launch<ElemBF16>(c, stream);
  else
    launch<ElemF16>(c, stream);
  return hipGetLastError();
}

}  // namespace dbk
