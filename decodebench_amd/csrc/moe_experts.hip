// moe_experts.hip -- the experts of a mixture-of-experts layer on a few tokens:
//
//   h_p = silu(Wg[e] x[t]) * (Wu[e] x[t])     for each pair p = (t, j), e = experts[t, j]
//   y[t] = sum_j weights[t, j] Wd[e] h_p
//
// The weights of the experts that are asked are read once for all their tokens,
// and are what bounds the call: a batch of few tokens reads megabytes for each
// of them.  Pairs are sorted by expert and cut into tiles of 16 to 128 of one expert;
// a workgroup has 64 or 128 gate rows and the up rows beside them (or twice as many
// down rows) of a tile, a wave 32 of the weight rows (A) by all of the tile's tokens (B)
// on v_mfma_f32_16x16x32.  Both operands come straight into the LDS, several stages
// ahead.  e4m3 weights are widened to the activations' type (exact), each block's
// sum scaled in fp32; the activations keep their 16 bits.
//
// 201 tokens, 2 of 8 experts of 14336 x 4096, fp16 (2.8 GB): 504 to 593 us by
// card, 4.8 to 5.6 TB/s (traced on one: gate and up 363 us, 5.2 TB/s; down 231, 4.1, in
// 290 workgroups on 256 CUs);
// 33 tokens, 6 of 64 of 1392 x 2048, e4m3 (about 54 of the experts asked, 465 MB): 103
// us, of which the gate takes 48 (6.5 TB/s) and the down product 40 (3.9), whose rows are
// 11 steps long and mostly start.
//
// g, u, silu and the product are fp32; h is rounded once to the activations'
// type, which the second product's matrix instructions take (two 16-bit parts of it
// would double that product and the LDS that its operand fills), so that in fp16 an h
// above 65504 becomes Inf; what the pairs of a token add up to is fp32 again, in the
// order of its experts, and rounded once.
#include "db_kernels.h"
#include "lds_dma.h"
#include "moe_select.h"

namespace dbk {

namespace {

constexpr int kThreads = 256;
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

// GATED: 16 NW gate rows and the up rows of the same channels on the tokens of a
// tile, h to the workspace; otherwise 32 NW down rows on h, each pair's sums to the
// workspace in fp32.  K goes in steps of 128 bytes of a weight row; S stages lie in
// the LDS, S - 1 of them on their way while one is multiplied.  A row's 16-byte
// chunk c lies at place c ^ row % 8, set by which chunk a lane fetches: the rows
// that a quarter of a wave reads then lie in different banks.
template <class E, bool FP8, int BT, bool GATED, int S, int NW>
__global__ __launch_bounds__(NW* kWave, 2) void moe_product(MoeExpertsCall c) {
  typedef typename E::type elem;
  typedef typename E::vec8 vec8;
  constexpr int CB = FP8 ? 1 : 2, KE = 128 / CB, XB = KE * 2;  // XB: bytes of a token's step
  constexpr int TT = BT / 16;
  constexpr int BN = 32 * NW;  // weight rows: 32 a wave
  constexpr int kLoadsW = 4, kLoadsX = BT * XB / 1024 / NW;
  static_assert(kLoadsX >= 1 && BT * XB % (1024 * NW) == 0, "whole loads");
  constexpr int kLoads = kLoadsW + kLoadsX;
  constexpr int kRowsX = 1024 / XB;  // tokens of a load instruction
  constexpr int kStage = BN * 128 + BT * XB;
  constexpr int kOutputs = GATED ? BN / 2 : BN;
  __shared__ __align__(16) char s_stage[S * kStage];
  const int slices = ((GATED ? c.w.I : c.w.H) + kOutputs - 1) / kOutputs;
  const int tile = blockIdx.x / slices, slice = blockIdx.x - tile * slices;
  if (tile >= scalar_load(c.tiles)) return;
  const int expert = scalar_load(c.tiles + 1 + 3 * tile),
            first = scalar_load(c.tiles + 2 + 3 * tile),
            pairs = scalar_load(c.tiles + 3 + 3 * tile);
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int r16 = lane & 15, q = lane >> 4;
  const int K = GATED ? c.w.H : c.w.I, N = GATED ? c.w.I : c.w.H;
  const int n0 = slice * kOutputs, KB = (K + 127) / 128, NB = (N + 127) / 128;
  const int rows = min(kOutputs, N - n0);
  const size_t w_at = ((size_t)expert * N + n0) * K * CB;

  // Load i of a wave has weight rows 8 (NW i + wave) .. + 7: of gate (or down) in the
  // first half of the loads, of up in the second.
  const u4 rw[2] = {
      dma_rsrc(static_cast<const char*>(GATED ? c.w.wg : c.w.wd) + w_at, rows * K * CB),
      dma_rsrc(static_cast<const char*>(GATED ? c.w.wu : c.w.wd) + w_at, rows * K * CB)};
  const int w_row = (8 * wave + (lane >> 3)) * K * CB;
  const int w_chunk = ((lane & 7) ^ (lane >> 3)) * 16;
  // The tokens of x (or slots of h): kRowsX of a load, 1024 / kRowsX bytes of each.
  const u4 rx = GATED ? dma_rsrc(c.x, ((c.T - 1) * (int)c.x_row + K) * 2)
                      : dma_rsrc(c.h, c.T * c.k * K * 2);
  constexpr int kLanesX = 64 / kRowsX;
  int x_row[kLoadsX];
#pragma unroll
  for (int i = 0; i < kLoadsX; ++i) {
    const int p = (i * NW + wave) * kRowsX + lane / kLanesX;
    x_row[i] = p >= pairs ? kOut
               : GATED    ? c.order[first + p] / c.k * (int)c.x_row * 2
                          : (first + p) * K * 2;
  }
  const int x_place = lane % kLanesX;
  const unsigned lds = lds_address(s_stage);
  auto fetch = [&](int stage, int step) {
    const unsigned to = lds + stage * kStage;
    // behind the row's end, and behind the last step, come zeros
    const int kw = step * 128 + w_chunk;
    const int ow = kw < K * CB ? kw : kOut;
#pragma unroll
    for (int i = 0; i < kLoadsW; ++i) {
      const int half = GATED && i >= kLoadsW / 2 ? 1 : 0, group = i - half * (kLoadsW / 2);
      dma16_stream(to + (i * NW + wave) * 1024, rw[half], ow + w_row + group * NW * 8 * K * CB);
    }
#pragma unroll
    for (int i = 0; i < kLoadsX; ++i) {
      const int row = (i * NW + wave) * kRowsX + lane / kLanesX;
      const int kx = step * XB + (x_place ^ (row & 7)) * 16;
      dma16(to + BN * 128 + (i * NW + wave) * 1024, rx,
            kx < K * 2 ? x_row[i] + kx : kOut);
    }
  };

  // Two row tiles of a wave: gate and up of the same channels, or two of down.
  const int tile_row[2] = {GATED ? 16 * wave : 32 * wave, GATED ? BN / 2 + 16 * wave : 32 * wave + 16};
  const float* ws[2] = {};
  if constexpr (FP8) {
    constexpr int kRows = kOutputs / NW;  // of a wave, of each matrix
    static_assert(kOutputs % NW == 0 && 128 % kRows == 0, "a wave's rows lie in one block");
    const size_t at = ((size_t)expert * NB + min((n0 + tile_row[0] % kOutputs) / 128, NB - 1)) * KB;
    ws[0] = (GATED ? c.w.sg : c.w.sd) + at;
    ws[1] = (GATED ? c.w.su : c.w.sd) + at;
  }
  f4 acc[2][TT] = {};
  auto multiply = [&](int stage, int step) {
    const char* const pw = s_stage + stage * kStage;
    const char* const px = pw + BN * 128;
    const int sw = r16 & 7;
    f4 part[2][TT] = {};
    vec8 a[2][4];
    constexpr int kOps = FP8 ? 4 : 2;  // products of 32 columns a step
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      const char* const row = pw + (tile_row[m] + r16) * 128;
      if constexpr (FP8) {
        // 16-byte chunks q and 4 + q: columns 16 q .. + 15 of each half, two operands each
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const u4 v = ld16(row + ((4 * h + q) ^ sw) * 16);
          const u2 b0 = E::widen(v[0]), b1 = E::widen(v[1]), b2 = E::widen(v[2]),
                   b3 = E::widen(v[3]);
          a[m][2 * h] = __builtin_bit_cast(vec8, u4{b0[0], b0[1], b1[0], b1[1]});
          a[m][2 * h + 1] = __builtin_bit_cast(vec8, u4{b2[0], b2[1], b3[0], b3[1]});
        }
      } else {
#pragma unroll
        for (int h = 0; h < 2; ++h)
          a[m][h] = __builtin_bit_cast(vec8, ld16(row + ((4 * h + q) ^ sw) * 16));
      }
    }
#pragma unroll
    for (int j = 0; j < TT; ++j) {
      if (16 * j >= pairs) break;
      const char* const row = px + (16 * j + r16) * XB;
#pragma unroll
      for (int s = 0; s < kOps; ++s) {
        // the same columns: e4m3 64 (s / 2) + 16 q + 8 (s % 2), 16-bit 32 s + 8 q
        const int place = FP8 ? 8 * (s / 2) + 2 * q + s % 2 : 4 * s + q;
        const vec8 x = __builtin_bit_cast(vec8, ld16(row + (place ^ sw) * 16));
#pragma unroll
        for (int m = 0; m < 2; ++m) {
          if constexpr (FP8)
            part[m][j] = E::mfma16(a[m][s], x, part[m][j]);
          else
            acc[m][j] = E::mfma16(a[m][s], x, acc[m][j]);
        }
      }
    }
    if constexpr (FP8) {
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const float scale = scalar_load(ws[m] + step);
#pragma unroll
        for (int j = 0; j < TT; ++j) {
          if (16 * j >= pairs) break;
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[m][j][e] += part[m][j][e] * scale;
        }
      }
    }
  };
  const int steps = (K + KE - 1) / KE;
#pragma unroll
  for (int s = 0; s < S - 1; ++s) fetch(s, s);
  int stage = 0, free_stage = S - 1;
  for (int s = 0; s < steps; ++s) {
    dma_barrier<(S - 2) * kLoads>();
    fetch(free_stage, s + S - 1);
    multiply(stage, s);
    stage = stage + 1 == S ? 0 : stage + 1;
    free_stage = free_stage + 1 == S ? 0 : free_stage + 1;
  }
  // register i of a lane is row 4 q + i of a row tile, column r16: a pair
#pragma unroll
  for (int j = 0; j < TT; ++j) {
    const int p = 16 * j + r16;
    if (p >= pairs) continue;
    if constexpr (GATED) {
      const int n = n0 + 16 * wave + 4 * q;
      if (n < N) {
        typename E::vec4 h;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float g = acc[0][j][e];
          h[e] = (elem)(g / (1.0f + expf(-g)) * acc[1][j][e]);
        }
        *reinterpret_cast<typename E::vec4*>(static_cast<elem*>(c.h) + (size_t)(first + p) * N +
                                             n) = h;
      }
    } else {
      float* const to = c.parts + (size_t)c.order[first + p] * N;
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const int n = n0 + tile_row[m] + 4 * q;
        if (n < N) *reinterpret_cast<f4*>(to + n) = acc[m][j];
      }
    }
  }
  dma_drain();  // what is still on its way into the LDS (zeros), before that is given back
}

template <class E>
__global__ __launch_bounds__(kThreads) void moe_combine(MoeExpertsCall c) {
  typedef typename E::type elem;
  const size_t at = ((size_t)blockIdx.x * kThreads + threadIdx.x) * 4;
  const int t = at / c.w.H, n = at - (size_t)t * c.w.H;
  if (t >= c.T) return;
  f4 sum = {0, 0, 0, 0};
  // eight pairs' loads at once, added in order; what lies there for a pair without
  // an expert does not count
  for (int j0 = 0; j0 < c.k; j0 += 8) {
    f4 v[8];
    float w[8];
    bool exists[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int p = t * c.k + min(j0 + i, c.k - 1);
      exists[i] = j0 + i < c.k && (unsigned)c.experts[p] < (unsigned)c.w.E;
      v[i] = *reinterpret_cast<const f4*>(c.parts + (size_t)p * c.w.H + n);
      w[i] = c.weights[p];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (exists[i])
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] += w[i] * v[i][e];
  }
  typename E::vec4 r;
#pragma unroll
  for (int i = 0; i < 4; ++i) r[i] = (elem)sum[i];
  *reinterpret_cast<typename E::vec4*>(static_cast<elem*>(c.y) + (size_t)t * c.w.H + n) = r;
}

template <class E, bool FP8, int BT, int S, int NW>
void launch(const MoeExpertsCall& c, hipStream_t stream) {
  const int P = c.T * c.k;
  const int tiles = min(P, c.w.E) + P / BT;  // at most
  const int gate = (c.w.I + 16 * NW - 1) / (16 * NW), down = (c.w.H + 32 * NW - 1) / (32 * NW);
  moe_sort<<<1, 1024, 0, stream>>>(c, BT);
  moe_product<E, FP8, BT, true, S, NW><<<gate * tiles, NW * kWave, 0, stream>>>(c);
  moe_product<E, FP8, BT, false, S, NW><<<down * tiles, NW * kWave, 0, stream>>>(c);
  const size_t quads = (size_t)c.T * c.w.H / 4;
  moe_combine<E><<<(quads + kThreads - 1) / kThreads, kThreads, 0, stream>>>(c);
}

// The tile's tokens go by how many an expert has on average (the fullest has more), the
// stages by what two workgroups a CU leave room for.  us of a layer with tiles of, in
// brackets the tokens an expert has:
//   e4m3                                     16   32   64   64 and eight waves
//     33 tokens, 6 of 64 of 1392 x 2048 (3)  100  102  115  113
//     32 tokens, 2 of 8 of 14336 x 4096 (8)  235  235  288  277
//     64 of these (16)                       328  234  278  284
//     128 (32)                               501  358  315  343
//     256 (64)                               872  583  454  446
//     512 (128)                                   993  769  756
//   16-bit                                   32   64   128 and eight waves
//     33 tokens, 6 of 64 of 1392 x 2048 (3)  177  180  194
//     32 tokens, 2 of 8 of 14336 x 4096 (8)  467  464  526
//     64 of these (16)                       467  468  514
//     128 (32)                               673  485  552
//     201 (50)                               884  604  606
//     256 (64)                              1129  752  627
//     512 (128)                             1882 1193  818
// With other stages or waves: e4m3 16 tokens in four stages the same, 64 in four (one
// workgroup a CU) 331 at 128 tokens, 128 tokens and eight waves 708 at 512.
template <class E, bool FP8>
void pick(const MoeExpertsCall& c, hipStream_t stream) {
  const int mean = c.T * c.k / c.w.E;
  if constexpr (FP8) {
    if (mean <= 5)
      launch<E, FP8, 16, 3, 4>(c, stream);
    else if (mean <= 20)
      launch<E, FP8, 32, 3, 4>(c, stream);
    else if (mean <= 64)
      launch<E, FP8, 64, 2, 4>(c, stream);
    else
      launch<E, FP8, 64, 3, 8>(c, stream);
  } else {
    if (mean <= 12)
      launch<E, FP8, 32, 4, 4>(c, stream);
    else if (mean <= 50)
      launch<E, FP8, 64, 3, 4>(c, stream);
    else
      launch<E, FP8, 128, 3, 8>(c, stream);
  }
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
  c.h = take(P * c.w.I * (moe_few(c.w, c.T, c.k) ? 4 : 2));
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
