// moe_select.h -- the k experts of one token and their weights, from its E logits,
// by the threads of a workgroup.  Shared by the router's own kernel and by the
// expert kernel of few tokens, which chooses for itself: both give the same bits.
#pragma once

#include "db_elem.h"

namespace dbk {

constexpr int kMostExperts = 1024;
constexpr int kMostChoices = 64;

struct MoeChoice {
  double logit[kMostExperts];
  __align__(16) double key[kMostExperts + 2];
  int rank[kMostExperts];
  int expert[kMostChoices];
  float p[kMostChoices];
  float total;
};

// A logit's place in the order: NaN above Inf above all numbers (sums of products of
// 16-bit numbers stay far below the largest double).
__device__ __forceinline__ double logit_key(double l) {
  return l != l ? __builtin_huge_val() : l == __builtin_huge_val() ? 0x1.fffffffffffffp1023 : l;
}

// A token's logits as the threads of a workgroup load them: expert tid + i NT's is l[i],
// the sum of `sums` parts, each `apart` from the one before.
template <int NT>
struct MoeLogits {
  double l[kMostExperts / NT];
  __device__ __forceinline__ void load(const double* logits, int sums, size_t apart, int E) {
#pragma unroll
    for (int i = 0; i < kMostExperts / NT; ++i) {
      const int e = threadIdx.x + i * NT;
      if (i * NT >= E) break;
      l[i] = e < E ? logits[e] : 0.0;
      // four parts' loads at once
      for (int j0 = 1; j0 < sums; j0 += 4) {
        double v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
          v[j] = e < E && j0 + j < sums ? logits[(j0 + j) * apart + e] : 0.0;
#pragma unroll
        for (int j = 0; j < 4; ++j) l[i] += v[j];
      }
    }
  }
};

// Fills s.logit and s.expert, the k largest in order.  Ranks are counted: an expert
// comes after those of larger logits, and of equal ones with a lower index.  NT
// threads, barriers within (the last one behind all of it); E and k are uniform.
template <int NT>
__device__ __forceinline__ void moe_rank(MoeChoice& s, const MoeLogits<NT>& in, int E, int k) {
  const int tid = threadIdx.x;
#pragma unroll
  for (int i = 0; i < kMostExperts / NT; ++i) {
    const int e = tid + i * NT;
    if (i * NT >= E) break;
    if (e < E) {
      s.logit[e] = in.l[i];
      s.key[e] = logit_key(in.l[i]);
      s.rank[e] = 0;
    }
  }
  // (behind the last one stands what comes before nothing)
  if (tid < 2) s.key[E + tid] = -__builtin_huge_val();
  __syncthreads();
  // experts by the threads, what they are compared with in `parts` parts
  int lanes = 64;
  while (lanes < E && lanes < NT) lanes *= 2;
  const int parts = NT / lanes, mine = tid & (lanes - 1), part = tid / lanes;
  const int each = ((E + parts - 1) / parts + 1) & ~1, begin = part * each;
  const int end = min(E, begin + each);
  for (int e = mine; e < E; e += lanes) {
    const double l = s.key[e];
    int before = 0;
#pragma unroll 8
    for (int o = begin; o < end; o += 2) {
      const double a = s.key[o], b = s.key[o + 1];
      before += (a > l) | ((a == l) & (o < e)) ? 1 : 0;
      before += (b > l) | ((b == l) & (o + 1 < e)) ? 1 : 0;
    }
    atomicAdd(&s.rank[e], before);
  }
  __syncthreads();
  for (int e = tid; e < E; e += NT)
    if (s.rank[e] < k) s.expert[s.rank[e]] = e;
  __syncthreads();
}

// After moe_rank: s.p (exp of each choice against the largest) and s.total (of the
// choices, or of all experts).
__device__ __forceinline__ void moe_weigh(MoeChoice& s, int E, int k, bool renormalize) {
  const int tid = threadIdx.x;
  const double top = s.logit[s.expert[0]];
  if (tid < k) s.p[tid] = expf((float)(s.logit[s.expert[tid]] - top));
  if (!renormalize && tid < kWave) {
    float sum = 0.0f;
    for (int e = tid; e < E; e += kWave) sum += expf((float)(s.logit[e] - top));
#pragma unroll
    for (int m = 1; m < kWave; m *= 2) sum += __shfl_xor(sum, m, kWave);
    if (tid == 0) s.total = sum;
  }
  __syncthreads();
  if (renormalize && tid == 0) {
    float sum = 0.0f;
    for (int j = 0; j < k; ++j) sum += s.p[j];
    s.total = sum;
  }
  __syncthreads();
}

}  // namespace dbk
