// rope_append.hip -- rotary positions on queries and keys, keys and values into
// the pages of the cache.
//
// A row of qkv is Hq query heads, Hkv key heads and Hkv value heads of D
// elements.  Pair i of a query or key head turns by pos[axis(i)] * freq[i]:
//   (a, b) -> (a cos - b sin, b cos + a sin),
// a and b being elements i and i + rot/2 of the head, or 2 i and 2 i + 1;
// elements past `rot` stay.  The angle is taken in 64 bits (positions of 1e5
// leave an fp32 product 5e-3 off) and reduced to a part of a turn before the
// fp32 sine and cosine; the rotation is fp32 with one rounding at the end.
// An e4m3 cache holds round(clamp(x / scale[head], -448, 448)).
//
// Bound by HBM: each element is read once and written once.  A workgroup has a
// few tokens: its threads take the sines and cosines of all their pairs once
// into LDS, then 8 pairs (or 8 values) at a time in 16-byte loads and stores.
#include "db_device.h"
#include "db_kernels.h"
#include "paged_attn.h"

namespace dbk {

namespace {

constexpr int kThreads = 256;
constexpr int kTokens = 4;  // tokens of a workgroup at most

struct RopeArgs {
  RopeCall c;
  int tokens;      // of a workgroup
  int pairs;       // rot / 2
  int vecs;        // work items of one query or key head: rot / 16 + (D - rot) / 8
  int items;       // of one token
};

// Eight fp32 values to the cache's or the output's type.
template <class E>
__device__ __forceinline__ u4 pack8(const float (&x)[8]) {
  typename E::vec8 r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = (typename E::type)x[i];
  return __builtin_bit_cast(u4, r);
}

// NaN stays NaN, everything else is clamped to the largest finite e4m3.
__device__ __forceinline__ float clamp448(float x) {
  return x > 448.0f ? 448.0f : x < -448.0f ? -448.0f : x;
}

__device__ __forceinline__ u2 pack8_e4m3(const float (&x)[8], float scale) {
  u2 r;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    int w = 0;
    w = __builtin_amdgcn_cvt_pk_fp8_f32(clamp448(x[4 * h] / scale), clamp448(x[4 * h + 1] / scale),
                                        w, false);
    w = __builtin_amdgcn_cvt_pk_fp8_f32(clamp448(x[4 * h + 2] / scale),
                                        clamp448(x[4 * h + 3] / scale), w, true);
    r[h] = (unsigned)w;
  }
  return r;
}

template <class E, bool FP8>
__global__ __launch_bounds__(kThreads) void rope_append_kernel(RopeArgs a) {
  typedef typename E::type elem;
  typedef typename E::vec8 vec8;
  const RopeCall& c = a.c;
  const db_paged_cache& kv = c.cache;
  const int D = kv.D, Hq = c.Hq, Hkv = kv.Hkv;
  __shared__ __align__(16) float s_cos[kTokens][128], s_sin[kTokens][128];

  const int t0 = blockIdx.x * a.tokens;
  const int here = min(a.tokens, c.T - t0);
  for (int i = threadIdx.x; i < here * a.pairs; i += kThreads) {
    const int t = i / a.pairs, pair = i % a.pairs;
    const int axis = (c.axes[pair >> 4] >> (2 * (pair & 15))) & 3;
    const int pos = c.position[(size_t)axis * c.T + t0 + t];
    // turns, less the whole ones; 1 / (2 pi) in 64 bits
    double turn = (double)pos * (double)c.freq[pair] * 0.15915494309189535;
    turn -= rint(turn);
    float s, co;
    sincospif(2.0f * (float)turn, &s, &co);
    s_cos[t][pair] = co;
    s_sin[t][pair] = s;
  }
  __syncthreads();
  const int rot = 2 * a.pairs;
  for (int i = threadIdx.x; i < here * a.items; i += kThreads) {
    const int t = i / a.items, item = i % a.items;
    const int turned = (Hq + Hkv) * a.vecs;
    const elem* row = static_cast<const elem*>(c.qkv) + (t0 + t) * c.qkv_row;
    // head of the row, element of the head, and what is written of it
    const int head = item < turned ? item / a.vecs : Hq + Hkv + (item - turned) / (D / 8);
    const int j = item < turned ? item % a.vecs : (item - turned) % (D / 8);
    const bool rotates = item < turned && j < a.pairs / 8;
    const int e0 = !rotates ? (item < turned ? rot + 8 * (j - a.pairs / 8) : 8 * j)
                            : c.interleaved ? 16 * j : 8 * j;
    const int e1 = c.interleaved ? e0 + 8 : e0 + a.pairs;
    char* out;
    long long slot = 0;
    if (head >= Hq) {
      slot = c.slot[t0 + t];
      if (slot < 0 || slot >= (long long)kv.pages * kv.page_size) continue;
    }
    const elem* from = row + (size_t)head * D;
    const vec8 x0 = __builtin_bit_cast(vec8, ld16(from + e0));
    float y0[8], y1[8];
    if (rotates) {
      const vec8 x1 = __builtin_bit_cast(vec8, ld16(from + e1));
      const float* co = &s_cos[t][8 * j];
      const float* si = &s_sin[t][8 * j];
      if (c.interleaved) {
        float z[16];
#pragma unroll
        for (int p = 0; p < 8; ++p) {
          const float u = (float)(p < 4 ? x0[2 * p] : x1[2 * p - 8]);
          const float v = (float)(p < 4 ? x0[2 * p + 1] : x1[2 * p - 7]);
          z[2 * p] = u * co[p] - v * si[p];
          z[2 * p + 1] = v * co[p] + u * si[p];
        }
#pragma unroll
        for (int p = 0; p < 8; ++p) {
          y0[p] = z[p];
          y1[p] = z[8 + p];
        }
      } else {
#pragma unroll
        for (int p = 0; p < 8; ++p) {
          const float u = (float)x0[p], v = (float)x1[p];
          y0[p] = u * co[p] - v * si[p];
          y1[p] = v * co[p] + u * si[p];
        }
      }
    } else {
#pragma unroll
      for (int p = 0; p < 8; ++p) y0[p] = (float)x0[p];
    }
    if (head < Hq) {
      elem* q = static_cast<elem*>(c.q) + ((size_t)(t0 + t) * Hq + head) * D;
      *reinterpret_cast<u4*>(q + e0) = pack8<E>(y0);
      if (rotates) *reinterpret_cast<u4*>(q + e1) = pack8<E>(y1);
      continue;
    }
    const bool value = head >= Hq + Hkv;
    const int h = head - Hq - (value ? Hkv : 0);
    const long long page = slot / kv.page_size, off = slot % kv.page_size;
    const long long at = value ? page * kv.v_page_stride + h * kv.v_head_stride +
                                     off * kv.v_token_stride
                               : page * kv.k_page_stride + h * kv.k_head_stride +
                                     off * kv.k_token_stride;
    out = static_cast<char*>(value ? kv.v : kv.k) + at * (FP8 ? 1 : 2);
    if constexpr (FP8) {
      const float scale = value ? kv.v_scale[h] : kv.k_scale[h];
      *reinterpret_cast<u2*>(out + e0) = pack8_e4m3(y0, scale);
      if (rotates) *reinterpret_cast<u2*>(out + e1) = pack8_e4m3(y1, scale);
    } else {
      *reinterpret_cast<u4*>(out + 2 * e0) = pack8<E>(y0);
      if (rotates) *reinterpret_cast<u4*>(out + 2 * e1) = pack8<E>(y1);
    }
  }
}

}  // namespace

hipError_t launch_rope_append(const RopeCall& c, int cu_count, hipStream_t stream) {
  RopeArgs a;
  a.c = c;
  a.pairs = c.rot / 2;
  a.vecs = c.rot / 16 + (c.cache.D - c.rot) / 8;
  a.items = (c.Hq + c.cache.Hkv) * a.vecs + c.cache.Hkv * (c.cache.D / 8);
  a.tokens = c.T >= kTokens * cu_count ? kTokens : 1;
  const bool fp8 = c.cache.dtype == DB_DTYPE_FP8_E4M3;
  const auto fn = c.bf16 ? (fp8 ? rope_append_kernel<ElemBF16, true> : rope_append_kernel<ElemBF16, false>)
                         : (fp8 ? rope_append_kernel<ElemF16, true> : rope_append_kernel<ElemF16, false>);
  hipLaunchKernelGGL(fn, dim3((c.T + a.tokens - 1) / a.tokens), dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace dbk
