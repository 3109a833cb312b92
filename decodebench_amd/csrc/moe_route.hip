// moe_route.hip -- the router of a mixture-of-experts layer: which experts a
// token takes, and with what weight.
//
//   l[t, e] = sum_h x[t, h] Wr[e, h]
//   experts[t] = the k largest l[t], ties to the lower index (NaN above all)
//   weights[t, j] = exp(l_j - max) / sum of the same over the k, or over all E
//
// The choice is a comparison of sums that may be nearly alike, so the logits are
// summed in 64 bits (v_mfma_f64_16x16x4, products of 16-bit numbers are exact):
// they do not depend on the order of the sum where that could be seen, and a
// token's experts not on the batch it comes in.
#include "db_elem.h"
#include "db_kernels.h"

namespace dbk {

namespace {

typedef double d4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 16;  // of a logits workgroup: each has a part of H

// Logits of 16 tokens and 16 experts: experts are the rows of A, tokens the
// columns of B.  A lane loads eight elements of a row at a time, the elements
// 32 s + 8 (lane / 16) + 0..7 of step s, and instruction j of the step takes the
// j-th of each lane.
template <class E>
__global__ __launch_bounds__(kWaves* kWave) void moe_logits(MoeRouteCall c) {
  typedef typename E::type elem;
  typedef typename E::vec8 vec8;
  __shared__ double s_part[kWaves][4][kWave];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int r16 = lane & 15, q = lane >> 4;
  const int e0 = blockIdx.x * 16, t0 = blockIdx.y * 16;
  const elem* const wr = static_cast<const elem*>(c.router) +
                         (size_t)min(e0 + r16, c.E - 1) * c.H;
  const elem* const xr = static_cast<const elem*>(c.x) + min(t0 + r16, c.T - 1) * c.x_row;
  d4 acc = {0, 0, 0, 0};
  for (int s = wave; 32 * s < c.H; s += kWaves) {
    const int h = 32 * s + 8 * q;
    u4 w = {0, 0, 0, 0}, x = {0, 0, 0, 0};
    if (h < c.H) {
      w = ld16(wr + h);
      x = ld16(xr + h);
    }
    const vec8 wv = __builtin_bit_cast(vec8, w), xv = __builtin_bit_cast(vec8, x);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)(float)wv[j], (double)(float)xv[j], acc,
                                                 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) s_part[wave][i][lane] = acc[i];
  __syncthreads();
  if (threadIdx.x < 256) {
    const int i = threadIdx.x >> 6;
    double sum = s_part[0][i][lane];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) sum += s_part[w][i][lane];
    // register i of a lane is row 4 i + lane / 16, column lane % 16
    const int e = e0 + 4 * i + q, t = t0 + r16;
    if (e < c.E && t < c.T) c.logits[(size_t)t * c.E + e] = sum;
  }
}

__device__ __forceinline__ double shfl_xor(double v, int mask) {
  return __shfl_xor(v, mask, kWave);
}

// Whether logit a of expert i comes before logit b of expert j.
__device__ __forceinline__ bool before(double a, int i, double b, int j) {
  const bool an = a != a, bn = b != b;
  if (an != bn) return an;
  if (an || a == b) return i < j;
  return a > b;
}

// A wave has a token; lane l its experts l, l + 64, ...
template <int N>
__global__ __launch_bounds__(kWave) void moe_select(MoeRouteCall c) {
  const int t = blockIdx.x, lane = threadIdx.x;
  double l[N];
  bool left[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int e = lane + 64 * i;
    left[i] = e < c.E;
    l[i] = left[i] ? c.logits[(size_t)t * c.E + e] : 0.0;
  }
  double top = 0.0;
  float total = 0.0f, mine = 0.0f;  // mine: exp of choice `lane`
  int chosen = 0;
  for (int j = 0; j < c.k; ++j) {
    double best = 0.0;
    int at = 1 << 30;  // none left in this lane
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (left[i] && (at == 1 << 30 || before(l[i], lane + 64 * i, best, at))) {
        best = l[i];
        at = lane + 64 * i;
      }
#pragma unroll
    for (int m = 1; m < kWave; m *= 2) {
      const double ob = shfl_xor(best, m);
      const int oa = __shfl_xor(at, m, kWave);
      if (oa != 1 << 30 && (at == 1 << 30 || before(ob, oa, best, at))) {
        best = ob;
        at = oa;
      }
    }
    if (j == 0) top = best;
    const float p = expf((float)(best - top));
    total += p;
    if (lane == j) {
      mine = p;
      chosen = at;
    }
#pragma unroll
    for (int i = 0; i < N; ++i) left[i] = left[i] && lane + 64 * i != at;
  }
  if (!c.renormalize) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (lane + 64 * i < c.E) sum += expf((float)(l[i] - top));
#pragma unroll
    for (int m = 1; m < kWave; m *= 2) sum += __shfl_xor(sum, m, kWave);
    total = sum;
  }
  if (lane < c.k) {
    c.experts[(size_t)t * c.k + lane] = chosen;
    c.weights[(size_t)t * c.k + lane] = mine / total;
  }
}

}  // namespace

hipError_t launch_moe_route(const MoeRouteCall& c, hipStream_t stream) {
  const dim3 grid((c.E + 15) / 16, (c.T + 15) / 16);
  if (c.bf16)
    moe_logits<ElemBF16><<<grid, kWaves * kWave, 0, stream>>>(c);
  else
    moe_logits<ElemF16><<<grid, kWaves * kWave, 0, stream>>>(c);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  auto* const fn = c.E <= 64 ? moe_select<1> : c.E <= 128 ? moe_select<2> : c.E <= 256
                   ? moe_select<4> : moe_select<16>;
  fn<<<c.T, kWave, 0, stream>>>(c);
  return hipGetLastError();
}

}  // namespace dbk
