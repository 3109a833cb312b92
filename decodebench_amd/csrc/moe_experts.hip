// moe_experts.hip -- the experts of a mixture-of-experts layer on a few tokens:
//
//   h_p = silu(Wg[e] x[t]) * (Wu[e] x[t])     for each pair p = (t, j), e = experts[t, j]
//   y[t] = sum_j weights[t, j] Wd[e] h_p
//
// The weights of the experts that are asked are read once for all their tokens,
// and are what bounds the call: a batch of few tokens reads megabytes for each
// of them.  Pairs are sorted by expert, 16 TT of one expert make a tile, and
// each product is 16 rows of the weights (A) by the tile's tokens (B) on
// v_mfma_f32_16x16x32, the waves of a workgroup taking blocks of 128 columns in
// turn.  e4m3 weights are widened to the activations' type (exact), each block's
// sum scaled in fp32; the activations keep their 16 bits.
//
// g, u, silu and the product are fp32; h is rounded once to the activations'
// type, which the second product takes; what the pairs of a token add up to is
// fp32 again, in the order of its experts, and rounded once.
#include "db_kernels.h"
#include "moe_select.h"

namespace dbk {

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kOut = 1 << 30;  // an offset behind every buffer: loads give zero

// Sorts the pairs by expert and cuts them into tiles of `most`.
//   order[slot]   = pair
//   tiles[0]      = number of tiles, then (expert, first slot, pairs) for each
__global__ __launch_bounds__(1024) void moe_sort(MoeExpertsCall c, int most) {
  __shared__ int s_count[kMostExperts], s_first[kMostExperts], s_tile[kMostExperts];
  __shared__ int s_sum[2][16];
  const int e = threadIdx.x, P = c.T * c.k;
  s_count[e] = 0;
  __syncthreads();
  for (int p = e; p < P; p += 1024) {
    const int x = c.experts[p];
    if ((unsigned)x < (unsigned)c.w.E) atomicAdd(&s_count[x], 1);
  }
  __syncthreads();
  // running sums of the counts and of their tiles
  const int lane = e & 63, wave = e >> 6;
  const int mine = s_count[e], tiles = (mine + most - 1) / most;
  int a = mine, b = tiles;
  for (int d = 1; d < 64; d *= 2) {
    const int oa = __shfl_up(a, d, 64), ob = __shfl_up(b, d, 64);
    if (lane >= d) {
      a += oa;
      b += ob;
    }
  }
  if (lane == 63) {
    s_sum[0][wave] = a;
    s_sum[1][wave] = b;
  }
  __syncthreads();
  for (int w = 0; w < wave; ++w) {
    a += s_sum[0][w];
    b += s_sum[1][w];
  }
  s_first[e] = a - mine;
  s_tile[e] = b - tiles;
  for (int i = 0; i < tiles; ++i) {
    int* const d = c.tiles + 1 + 3 * (b - tiles + i);
    d[0] = e;
    d[1] = a - mine + i * most;
    d[2] = min(most, mine - i * most);
  }
  if (e == 1023) c.tiles[0] = b;
  __syncthreads();
  for (int p = e; p < P; p += 1024) {
    const int x = c.experts[p];
    if ((unsigned)x < (unsigned)c.w.E) c.order[atomicAdd(&s_first[x], 1)] = p;
  }
}

__device__ __forceinline__ u4 ld_buf(__amdgpu_buffer_rsrc_t r, int offset) {
  return __builtin_bit_cast(u4, __builtin_amdgcn_raw_buffer_load_b128(r, offset, 0, 0));
}

// A block of 128 columns of 16 weight rows, as a lane (row r16, quarter q) holds
// it: 16-bit load j has columns 32 j + 8 q .. + 7, e4m3 load j columns
// 64 j + 16 q .. + 15.
template <bool FP8>
struct Weights {
  static constexpr int kLoads = FP8 ? 2 : 4;
  u4 w[kLoads];
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, int row, int b, int q, int K) {
    constexpr int CB = FP8 ? 1 : 2, VE = 16 / CB;
#pragma unroll
    for (int j = 0; j < kLoads; ++j) {
      const int k = b * 128 + j * (128 / kLoads) + q * VE;
      w[j] = ld_buf(r, k < K ? (row * K + k) * CB : kOut);
    }
  }
  // Operand s of four: columns col(s, q) .. + 7.
  template <class E>
  __device__ __forceinline__ typename E::vec8 operand(int s) const {
    if constexpr (!FP8) {
      return __builtin_bit_cast(typename E::vec8, w[s]);
    } else {
      const u2 lo = E::widen(w[s / 2][2 * (s % 2)]), hi = E::widen(w[s / 2][2 * (s % 2) + 1]);
      return __builtin_bit_cast(typename E::vec8, u4{lo[0], lo[1], hi[0], hi[1]});
    }
  }
  __device__ __forceinline__ static int col(int s, int q) {
    return FP8 ? 64 * (s / 2) + 16 * q + 8 * (s % 2) : 32 * s + 8 * q;
  }
};

// GATED: gate and up rows of the experts on the tokens, h to the workspace;
// otherwise the down rows on h, each pair's sums to the workspace in fp32.
template <class E, bool FP8, int TT, bool GATED>
__global__ __launch_bounds__(kThreads) void moe_product(MoeExpertsCall c) {
  typedef typename E::type elem;
  typedef typename E::vec8 vec8;
  constexpr int NW = GATED ? 2 : 1, CB = FP8 ? 1 : 2;
  __shared__ f4 s_part[kWaves][NW * TT][kWave];
  const int slices = ((GATED ? c.w.I : c.w.H) + 15) / 16;
  const int tile = blockIdx.x / slices, slice = blockIdx.x - tile * slices;
  if (tile >= c.tiles[0]) return;
  const int expert = c.tiles[1 + 3 * tile], first = c.tiles[2 + 3 * tile],
            pairs = c.tiles[3 + 3 * tile];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int r16 = lane & 15, q = lane >> 4;
  const int K = GATED ? c.w.H : c.w.I, N = GATED ? c.w.I : c.w.H;
  const int n0 = slice * 16, KB = (K + 127) / 128, NB = (N + 127) / 128;
  const size_t w_at = ((size_t)expert * N + n0) * K * CB;
  const int w_bytes = min(16, N - n0) * K * CB;
  __amdgpu_buffer_rsrc_t rw[NW];
  const float* ws[NW] = {};
#pragma unroll
  for (int m = 0; m < NW; ++m) {
    const void* base = GATED ? (m ? c.w.wu : c.w.wg) : c.w.wd;
    rw[m] = make_rsrc(static_cast<const char*>(base) + w_at, w_bytes);
    if constexpr (FP8)
      ws[m] = (GATED ? (m ? c.w.su : c.w.sg) : c.w.sd) + ((size_t)expert * NB + n0 / 128) * KB;
  }
  // rows of the other operand: tokens of x, or slots of h
  const __amdgpu_buffer_rsrc_t rx = GATED ? make_rsrc(c.x, (c.T - 1) * (int)c.x_row * 2 + K * 2)
                                          : make_rsrc(c.h, c.T * c.k * K * 2);
  int xr[TT];
#pragma unroll
  for (int i = 0; i < TT; ++i) {
    const int p = i * 16 + r16;
    xr[i] = p >= pairs ? kOut
            : GATED    ? c.order[first + p] / c.k * (int)c.x_row * 2
                       : (first + p) * K * 2;
  }
  f4 acc[NW][TT] = {};
  for (int b = wave; b < KB; b += kWaves) {
    Weights<FP8> w[NW];
#pragma unroll
    for (int m = 0; m < NW; ++m) w[m].load(rw[m], r16, b, q, K);
    f4 part[NW][TT] = {};
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      vec8 a[NW];
#pragma unroll
      for (int m = 0; m < NW; ++m) a[m] = w[m].template operand<E>(s);
      const int k = b * 128 + Weights<FP8>::col(s, q);
#pragma unroll
      for (int i = 0; i < TT; ++i) {
        const vec8 x = __builtin_bit_cast(vec8, ld_buf(rx, k < K ? xr[i] + k * 2 : kOut));
#pragma unroll
        for (int m = 0; m < NW; ++m) {
          if constexpr (FP8)
            part[m][i] = E::mfma16(a[m], x, part[m][i]);
          else
            acc[m][i] = E::mfma16(a[m], x, acc[m][i]);
        }
      }
    }
    if constexpr (FP8) {
#pragma unroll
      for (int m = 0; m < NW; ++m) {
        const float scale = ws[m][b];
#pragma unroll
        for (int i = 0; i < TT; ++i)
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[m][i][j] += part[m][i][j] * scale;
      }
    }
  }
#pragma unroll
  for (int m = 0; m < NW; ++m)
#pragma unroll
    for (int i = 0; i < TT; ++i) s_part[wave][m * TT + i][lane] = acc[m][i];
  __syncthreads();
  for (int i = wave; i < TT; i += kWaves) {
    f4 sum[NW];
#pragma unroll
    for (int m = 0; m < NW; ++m) {
      sum[m] = s_part[0][m * TT + i][lane];
#pragma unroll
      for (int w = 1; w < kWaves; ++w) sum[m] += s_part[w][m * TT + i][lane];
    }
    // register j of a lane is row 4 q + j, column r16
    const int p = i * 16 + r16, n = n0 + 4 * q;
    if (p >= pairs || n >= N) continue;
    if constexpr (GATED) {
      typename E::vec4 h;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float g = sum[0][j];
        h[j] = (elem)(g / (1.0f + expf(-g)) * sum[1][j]);
      }
      *reinterpret_cast<typename E::vec4*>(static_cast<elem*>(c.h) + (size_t)(first + p) * N + n) =
          h;
    } else {
      *reinterpret_cast<f4*>(c.parts + (size_t)c.order[first + p] * N + n) = sum[0];
    }
  }
}

template <class E>
__global__ __launch_bounds__(kThreads) void moe_combine(MoeExpertsCall c) {
  typedef typename E::type elem;
  const size_t at = ((size_t)blockIdx.x * kThreads + threadIdx.x) * 4;
  const int t = at / c.w.H, n = at - (size_t)t * c.w.H;
  if (t >= c.T) return;
  f4 sum = {0, 0, 0, 0};
  for (int j = 0; j < c.k; ++j) {
    const int p = t * c.k + j;
    if ((unsigned)c.experts[p] >= (unsigned)c.w.E) continue;
    const f4 v = *reinterpret_cast<const f4*>(c.parts + (size_t)p * c.w.H + n);
    const float w = c.weights[p];
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] += w * v[i];
  }
  typename E::vec4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = (elem)sum[i];
  *reinterpret_cast<typename E::vec4*>(static_cast<elem*>(c.y) + (size_t)t * c.w.H + n) = r;
}

template <class E, bool FP8, int TT>
void launch(const MoeExpertsCall& c, hipStream_t stream) {
  const int P = c.T * c.k;
  const int tiles = min(P, c.w.E) + P / (16 * TT);  // at most
  moe_sort<<<1, 1024, 0, stream>>>(c, 16 * TT);
  moe_product<E, FP8, TT, true><<<(c.w.I + 15) / 16 * tiles, kThreads, 0, stream>>>(c);
  moe_product<E, FP8, TT, false><<<(c.w.H + 15) / 16 * tiles, kThreads, 0, stream>>>(c);
  const size_t quads = (size_t)c.T * c.w.H / 4;
  moe_combine<E><<<(quads + kThreads - 1) / kThreads, kThreads, 0, stream>>>(c);
}

template <class E, bool FP8>
void pick(const MoeExpertsCall& c, hipStream_t stream) {
  // tokens that an expert has on average
  const int mean = c.T * c.k / c.w.E;
  if (mean <= 8)
    launch<E, FP8, 1>(c, stream);
  else if (mean <= 24)
    launch<E, FP8, 2>(c, stream);
  else
    launch<E, FP8, 4>(c, stream);
}

size_t round256(size_t n) { return (n + 255) & ~(size_t)255; }

}  // namespace

size_t moe_experts_workspace(MoeExpertsCall& c, void* ws) {
  const size_t P = (size_t)c.T * c.k;
  char* p = static_cast<char*>(ws);
  auto take = [&](size_t bytes) {
    char* const at = p;
    p += round256(bytes);
    return at;
  };
  c.order = reinterpret_cast<int*>(take(P * 4));
  c.tiles = reinterpret_cast<int*>(take((1 + 3 * (P + (size_t)c.w.E)) * 4));
  c.h = take(P * c.w.I * 2);
  c.parts = reinterpret_cast<float*>(take(P * c.w.H * 4));
  return p - static_cast<char*>(ws);
}

hipError_t launch_moe_experts(const MoeExpertsCall& c, hipStream_t stream) {
  const bool fp8 = c.w.w_dtype == DB_DTYPE_FP8_E4M3;
  if (c.bf16)
    fp8 ? pick<ElemBF16, true>(c, stream) : pick<ElemBF16, false>(c, stream);
  else
    fp8 ? pick<ElemF16, true>(c, stream) : pick<ElemF16, false>(c, stream);
  return hipGetLastError();
}

}  // namespace dbk
