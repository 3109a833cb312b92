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
// Bound by HBM: each element is read once and written once.  A workgroup has
// up to four tokens: its threads take the sines and cosines of all their pairs
// into LDS, and where their slots lie; then a thread takes one place of a token
// (8 pairs of a head, or 8 values) for all the tokens, so that what it has to
// work out about the place is shared and four tokens' loads are in flight.
// Measured on MI355X, 8192 tokens of 32 + 2 x 8 heads of 128 in bf16 (201 MB):
// 35.5 us, 5.7 TB/s, where a copy of as many bytes reaches 4.8; with a place worked
// out anew for each token and one token's loads in flight 45 us.
#include "paged_attn.h"

namespace dbk {

namespace {

constexpr int kThreads = 256;
constexpr int kTokens = 4;  // of a workgroup at most

struct RopeArgs {
  RopeCall c;
  int pairs;       // rot / 2
  int vecs;        // places of a query or key head: rot / 16 + (D - rot) / 8
  int places;      // of a token
};

// Eight fp32 values to the cache's or the output's type.
template <class E>
__device__ __forceinline__ u4 pack8(const float (&x)[8]) {
  typename E::vec8 r;
#pragma unroll
  for (int i = 0; i < 8; ++i) r[i] = (typename E::type)x[i];
  return __builtin_bit_cast(u4, r);
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

template <class E, bool FP8, int TOKENS>
__global__ __launch_bounds__(kThreads) void rope_append_kernel(RopeArgs a) {
  typedef typename E::type elem;
  typedef typename E::vec8 vec8;
  constexpr int CB = FP8 ? 1 : 2;  // bytes of a cache element
  const RopeCall& c = a.c;
  const db_paged_cache& kv = c.cache;
  const int D = kv.D, Hq = c.Hq, Hkv = kv.Hkv;
  __shared__ __align__(16) float s_cos[TOKENS][128], s_sin[TOKENS][128];
  __shared__ long long s_k[TOKENS], s_v[TOKENS];  // byte offsets of the tokens' rows, -1: none

  const int t0 = blockIdx.x * TOKENS;
  const int here = min(TOKENS, c.T - t0);
  if (threadIdx.x < here) {
    const long long slot = c.slot[t0 + threadIdx.x];
    const bool ok = slot >= 0 && slot < (long long)kv.pages * kv.page_size;
    const long long page = ok ? slot / kv.page_size : 0, off = slot - page * kv.page_size;
    s_k[threadIdx.x] = ok ? (page * kv.k_page_stride + off * kv.k_token_stride) * CB : -1;
    s_v[threadIdx.x] = ok ? (page * kv.v_page_stride + off * kv.v_token_stride) * CB : -1;
  }
  for (int i = threadIdx.x; i < here * a.pairs; i += kThreads) {
    const int t = TOKENS == 1 ? 0 : i / a.pairs, pair = i - t * a.pairs;
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
  const int turned = (Hq + Hkv) * a.vecs;
  for (int place = blockIdx.y * kThreads + threadIdx.x; place < a.places;
       place += gridDim.y * kThreads) {
    // head of the row, elements of the head, and what they become
    const bool value = place >= turned;
    const int head = value ? Hq + Hkv + (place - turned) / (D / 8) : place / a.vecs;
    const int j = value ? (place - turned) % (D / 8) : place - head * a.vecs;
    const bool rotates = !value && j < a.pairs / 8;
    const int e0 = value      ? 8 * j
                   : !rotates ? 2 * a.pairs + 8 * (j - a.pairs / 8)
                              : (c.interleaved ? 16 : 8) * j;
    const int e1 = !rotates ? e0 : c.interleaved ? e0 + 8 : e0 + a.pairs;
    const elem* from = static_cast<const elem*>(c.qkv) + t0 * c.qkv_row + (size_t)head * D;
    u4 w0[TOKENS], w1[TOKENS];
#pragma unroll
    for (int t = 0; t < TOKENS; ++t) {
      const elem* row = from + min(t, here - 1) * c.qkv_row;
      w0[t] = ld_stream(row + e0);
      w1[t] = ld_stream(row + e1);
    }
    char* const base = static_cast<char*>(value ? kv.v : kv.k) +
                       (head < Hq ? 0
                                  : (value ? (head - Hq - Hkv) * kv.v_head_stride
                                           : (head - Hq) * kv.k_head_stride) *
                                        CB);
    const float scale = !FP8 || head < Hq ? 1.0f
                        : value           ? kv.v_scale[head - Hq - Hkv]
                                          : kv.k_scale[head - Hq];
#pragma unroll
    for (int t = 0; t < TOKENS; ++t) {
      if (t >= here) break;
      const vec8 x0 = __builtin_bit_cast(vec8, w0[t]), x1 = __builtin_bit_cast(vec8, w1[t]);
      float y0[8], y1[8];
      if (rotates) {
        const float* co = &s_cos[t][8 * j];
        const float* si = &s_sin[t][8 * j];
        if (c.interleaved) {
#pragma unroll
          for (int p = 0; p < 4; ++p) {
            const float u = (float)x0[2 * p], v = (float)x0[2 * p + 1];
            y0[2 * p] = u * co[p] - v * si[p];
            y0[2 * p + 1] = v * co[p] + u * si[p];
            const float m = (float)x1[2 * p], n = (float)x1[2 * p + 1];
            y1[2 * p] = m * co[4 + p] - n * si[4 + p];
            y1[2 * p + 1] = n * co[4 + p] + m * si[4 + p];
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
        *reinterpret_cast<u4*>(q + e0) = rotates ? pack8<E>(y0) : w0[t];
        if (rotates) *reinterpret_cast<u4*>(q + e1) = pack8<E>(y1);
        continue;
      }
      const long long off = value ? s_v[t] : s_k[t];
      if (off < 0) continue;
      char* out = base + off;
      if constexpr (FP8) {
        *reinterpret_cast<u2*>(out + e0) = pack8_e4m3(y0, scale);
        if (rotates) *reinterpret_cast<u2*>(out + e1) = pack8_e4m3(y1, scale);
      } else {
        *reinterpret_cast<u4*>(out + 2 * e0) = rotates ? pack8<E>(y0) : w0[t];
        if (rotates) *reinterpret_cast<u4*>(out + 2 * e1) = pack8<E>(y1);
      }
    }
  }
}

template <class E, bool FP8>
void (*pick_tokens(bool four))(RopeArgs) {
  return four ? rope_append_kernel<E, FP8, kTokens> : rope_append_kernel<E, FP8, 1>;
}

}  // namespace

hipError_t launch_rope_append(const RopeCall& c, int cu_count, hipStream_t stream) {
  RopeArgs a;
  a.c = c;
  a.pairs = c.rot / 2;
  a.vecs = c.rot / 16 + (c.cache.D - c.rot) / 8;
  a.places = (c.Hq + c.cache.Hkv) * a.vecs + c.cache.Hkv * (c.cache.D / 8);
  // Four tokens a workgroup once that fills the chip; a workgroup for each 256
  // places of a token where even one a token does not.
  const bool four = c.T >= kTokens * cu_count;
  const int parts = c.T >= cu_count ? 1 : min((a.places + kThreads - 1) / kThreads, 8);
  const int tokens = four ? kTokens : 1;
  const bool fp8 = c.cache.dtype == DB_DTYPE_FP8_E4M3;
  const auto fn = c.bf16 ? (fp8 ? pick_tokens<ElemBF16, true>(four) : pick_tokens<ElemBF16, false>(four))
                         : (fp8 ? pick_tokens<ElemF16, true>(four) : pick_tokens<ElemF16, false>(four));
  hipLaunchKernelGGL(fn, dim3((c.T + tokens - 1) / tokens, parts), dim3(kThreads), 0, stream, a);
  return hipGetLastError();
}

}  // namespace dbk
