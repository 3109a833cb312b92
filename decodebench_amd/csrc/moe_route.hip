// moe_route.hip -- the router of a mixture-of-experts layer: which experts a
// token takes, and with what weight.
//
//   l[t, e] = sum_h x[t, h] Wr[e, h]
//   experts[t] = the k largest l[t], ties to the lower index (NaN above all)
//   weights[t, j] = exp(l_j - max) / sum of the same over the k, or over all E
//
// The choice is a comparison of sums that may be nearly alike, so the logits are
// multiplied and summed in 64 bits (v_mfma_f64_16x16x4, products of 16-bit numbers
// are exact).  The order of a sum goes by the number of tokens: where the 64-bit sums
// are exact, a token's experts do not depend on the batch it comes in; elsewhere two
// logits that are as near to each other as the roundings of 64 bits may change places.
//
// Bound by latency: two launches, each a few dependent reads long.  One token, 128
// experts of 4096: 8.5 to 8.8 us; 509 tokens, 64 experts of 2048: 10.1 (the matrix cores would
// need 1.7 at their 64-bit rate).
#include "db_kernels.h"
#include "moe_select.h"

namespace dbk {

namespace {

typedef double d4 __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;       // of a logits workgroup: each has a part of its columns
constexpr int kMostParts = 16;  // of H

// Workgroups of the logits: 16 tokens, 16 experts and one of the parts of H that make
// enough of them (201 tokens, 8 experts of 4096: the router 15.7 us in one part, 8 so).
int logit_parts(int T, int H, int E) {
  const long long tiles = (long long)((T + 15) / 16) * ((E + 15) / 16);
  const long long want = (1024 + tiles - 1) / tiles;
  return (int)max(1ll, min(want, (long long)min(kMostParts, H / 256)));
}

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
  const int e0 = blockIdx.y * 16, t0 = blockIdx.x * 16;
  const int steps = (c.H + 31) / 32, each = (steps + c.parts - 1) / c.parts;
  const int begin = blockIdx.z * each, end = min(steps, begin + each);
  const elem* const wr = static_cast<const elem*>(c.router) +
                         (size_t)min(e0 + r16, c.E - 1) * c.H;
  const elem* const xr = static_cast<const elem*>(c.x) + min(t0 + r16, c.T - 1) * c.x_row;
  d4 acc = {0, 0, 0, 0};
  // four steps' loads at once
  constexpr int kSteps = 4;
  for (int s0 = begin + wave; s0 < end; s0 += kWaves * kSteps) {
    u4 w[kSteps], x[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int s = s0 + i * kWaves, h = 32 * s + 8 * q;
      const bool in = s < end && h < c.H;
      w[i] = in ? ld16(wr + h) : u4{0, 0, 0, 0};
      x[i] = in ? ld16(xr + h) : u4{0, 0, 0, 0};
    }
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      if (s0 + i * kWaves >= end) break;
      const vec8 wv = __builtin_bit_cast(vec8, w[i]), xv = __builtin_bit_cast(vec8, x[i]);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        acc = __builtin_amdgcn_mfma_f64_16x16x4f64((double)(float)wv[j], (double)(float)xv[j], acc,
                                                   0, 0, 0);
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) s_part[wave][i][lane] = acc[i];
  __syncthreads();
  const int i = wave;
  double sum = s_part[0][i][lane];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) sum += s_part[w][i][lane];
  // register i of a lane is row 4 i + lane / 16, column lane % 16
  const int e = e0 + 4 * i + q, t = t0 + r16;
  if (e < c.E && t < c.T) c.logits[((size_t)blockIdx.z * c.T + t) * c.E + e] = sum;
}

// Few tokens: a wave has an expert and all of them.  Eight elements of a row a
// lane and step, multiplied and added up in 64 bits: bf16 products leave the range
// of 32 at both ends.
constexpr int kFewTokens = 4;

template <class E>
__global__ __launch_bounds__(4 * kWave) void moe_logits_few(MoeRouteCall c) {
  typedef typename E::type elem;
  typedef typename E::vec8 vec8;
  const int lane = threadIdx.x & (kWave - 1);
  const int e = blockIdx.x * 4 + threadIdx.x / kWave;
  if (e >= c.E) return;
  const elem* const wr = static_cast<const elem*>(c.router) + (size_t)e * c.H;
  double acc[kFewTokens] = {};
  // four steps' loads at once
  constexpr int kSteps = 4;
  for (int h0 = lane * 8; h0 < c.H; h0 += kWave * 8 * kSteps) {
    u4 w[kSteps];
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
      const int h = h0 + i * kWave * 8;
      w[i] = h < c.H ? ld16(wr + h) : u4{0, 0, 0, 0};
    }
#pragma unroll
    for (int t = 0; t < kFewTokens; ++t) {
      if (t >= c.T) break;
      const elem* const row = static_cast<const elem*>(c.x) + t * c.x_row;
      u4 x[kSteps];
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const int h = h0 + i * kWave * 8;
        x[i] = h < c.H ? ld16(row + h) : u4{0, 0, 0, 0};
      }
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const vec8 wv = __builtin_bit_cast(vec8, w[i]), xv = __builtin_bit_cast(vec8, x[i]);
#pragma unroll
        for (int j = 0; j < 8; ++j)
          acc[t] = __builtin_fma((double)(float)wv[j], (double)(float)xv[j], acc[t]);
      }
    }
  }
#pragma unroll
  for (int t = 0; t < kFewTokens; ++t) {
    if (t >= c.T) break;
#pragma unroll
    for (int m = 1; m < kWave; m *= 2) acc[t] += __shfl_xor(acc[t], m, kWave);
    if (lane == 0) c.logits[(size_t)t * c.E + e] = acc[t];
  }
}

// A workgroup has a token.
__global__ __launch_bounds__(256) void moe_select(MoeRouteCall c) {
  __shared__ MoeChoice s;
  const size_t t = blockIdx.x;
  MoeLogits<256> logits;
  logits.load(c.logits + t * c.E, c.parts, (size_t)c.T * c.E, c.E);
  moe_rank(s, logits, c.E, c.k);
  moe_weigh(s, c.E, c.k, c.renormalize);
  if (threadIdx.x < c.k) {
    c.experts[t * c.k + threadIdx.x] = s.expert[threadIdx.x];
    c.weights[t * c.k + threadIdx.x] = s.p[threadIdx.x] / s.total;
  }
}

}  // namespace

int moe_logit_parts(int T, int H, int E) {
  return T <= kFewTokens ? 1 : logit_parts(T, H, E);
}

hipError_t launch_moe_logits(const MoeRouteCall& c, hipStream_t stream) {
  if (c.T <= kFewTokens) {
    const int grid = (c.E + 3) / 4;
    if (c.bf16)
      moe_logits_few<ElemBF16><<<grid, 4 * kWave, 0, stream>>>(c);
    else
      moe_logits_few<ElemF16><<<grid, 4 * kWave, 0, stream>>>(c);
    return hipGetLastError();
  }
  const dim3 grid((c.T + 15) / 16, (c.E + 15) / 16, c.parts);
  if (c.bf16)
    moe_logits<ElemBF16><<<grid, kWaves * kWave, 0, stream>>>(c);
  else
    moe_logits<ElemF16><<<grid, kWaves * kWave, 0, stream>>>(c);
  return hipGetLastError();
}

hipError_t launch_moe_route(const MoeRouteCall& c, hipStream_t stream) {
  const hipError_t e = launch_moe_logits(c, stream);
  if (e != hipSuccess) return e;
  moe_select<<<c.T, 256, 0, stream>>>(c);
  return hipGetLastError();
}

}  // namespace dbk
