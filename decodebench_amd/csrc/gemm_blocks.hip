// gemm_blocks.hip -- products of e4m3 activations with one scale for each 128
// elements of a row and e4m3 weights with one scale for each block of 128 x 128:
//
//   y[t, n] = sum_b xs[t, b] ws[n / 128, b] sum_{k in b} x[t, k] W[n, k]
//
// v_mfma_f32_16x16x128_f8f6f4 sums a whole block of k at once: its result is
// scaled and added to the fp32 sum with one multiply-add for each of the four
// outputs of a lane.  Weights are the A operand and tokens the B operand, so a
// lane's outputs belong to one token and share one scale.
//
// Within the instruction the products of eight consecutive k are cut off, towards
// zero, 13 binary places below the largest one's leading place (so found with
// products of powers of two, and alike in the 16x16x32 form); the sixteen sums of
// eight meet in fp32.  Eight products so lose less than 7 * 2^-13 of the largest of
// them, where rounding x to e4m3 has cost each up to 2^-4.  Sums that keep all places
// would take the 16-bit instructions, at half the rate.
#include <algorithm>
#include <atomic>

#include "db_kernels.h"
#include "lds_dma.h"
#include "quant_blocks.h"

namespace dbk {

namespace {

typedef int i8v __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256;
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

// ------------------------------------------------------------- few tokens
// A workgroup has plan.each outputs (a multiple of 4: even shares of any N) of all
// T <= 16 tokens, 16 at a time; its waves take blocks of K in turn, and their sums
// meet in the LDS.  x lies there whole, its scales behind it, copied or quantised
// by every workgroup for itself while the first weights are on their way.
//
// Bound by the weights' bytes: one token of [14336, 4096] 12.2 us, 4.8 TB/s, where a
// kernel that only reads them takes 9.7; the difference is the start, x before weights.
//
// A load instruction has 8 rows of one 128-byte line each, consecutive lanes
// consecutive chunks (operand order, rows on consecutive lanes, takes the L1 four
// times as long); a wave's block passes through an LDS tile of its own into operand
// order, chunk c of row r at place c ^ r % 8.  No barrier: a wave's LDS accesses
// execute in order.
constexpr int kAhead = 8;     // blocks of a wave on their way
constexpr int kFewRounds = 4;  // of 4 blocks of x a wave, asked for before the weights
constexpr int kFewTiles = 4;  // of 16 outputs, at most, of a workgroup

template <class E, bool QUANT, int NW>
__global__ __launch_bounds__(NW* kWave) void gemm_blocks_few(GemmBlocksCall c,
                                                             GemmBlocksPlan plan) {
  extern __shared__ __align__(16) char s_x[];
  __shared__ __align__(16) char s_tile[NW][2048];
  __shared__ f4 s_part[kFewTiles][NW][kWave];
  constexpr int kThreadsHere = NW * kWave;
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int r16 = lane & 15, q = lane >> 4;
  const int KB = (c.K + 127) / 128, KP = (c.K + 1023) / 1024 * 1024;
  const int n_first = blockIdx.x * plan.each, n_last = min(c.N, n_first + plan.each);
  const int nb0 = n_first / 128, nbs = (n_last - 1) / 128 - nb0 + 1;
  float* const s_scale = reinterpret_cast<float*>(s_x + c.T * KP);  // [T, KB]
  float* const s_w = s_scale + c.T * KB;                            // [nbs, KB]

  // x and all scales are asked for before the first weights, which come in order
  // behind them; without branches, which would make the waits for them whole.
  const int items = c.T * KB, w_items = nbs * KB;
  // i / KB (which of 1 is beyond what the product with 2^32 / KB can give)
  auto row_of = [&](int i) { return KB == 1 ? i : (int)__umulhi(i, plan.magic); };
  u4 x_raw[kFewRounds];
  float xs_first = 0.0f;
  int x_at = threadIdx.x / 16;  // this row of lanes' block of x: every (4 NW)th of them
  auto ask = [&](int i) {
    const int in = min(i, items - 1), t = row_of(in), b = in - t * KB;
    const typename E::type* const row = static_cast<const typename E::type*>(c.x) + t * c.x_row;
    return ld16(row + min(b * 128 + r16 * 8, c.K - 8));
  };
  auto put_x = [&](int i, u4 raw) {
    const int t = row_of(i), b = i - t * KB;
    float scale;
    const u2 v = quantize128<E>(b * 128 + r16 * 8 < c.K ? raw : u4{0, 0, 0, 0}, scale);
    *reinterpret_cast<u2*>(s_x + t * KP + b * 128 + (((r16 >> 1) ^ (t & 7)) * 16) +
                           (r16 & 1) * 8) = v;
    if (r16 == 0) s_scale[i] = scale;
  };
  if constexpr (QUANT) {
    // all but the last rounds go into the LDS at once
    while (x_at - (int)threadIdx.x / 16 + kFewRounds * NW * 4 < items) {
#pragma unroll
      for (int r = 0; r < kFewRounds; ++r) x_raw[r] = ask(x_at + r * NW * 4);
#pragma unroll
      for (int r = 0; r < kFewRounds; ++r) put_x(x_at + r * NW * 4, x_raw[r]);
      x_at += kFewRounds * NW * 4;
    }
#pragma unroll
    for (int r = 0; r < kFewRounds; ++r) x_raw[r] = ask(x_at + r * NW * 4);
  } else {
    const u4 rx = dma_rsrc(c.x, (int)((c.T - 1) * c.x_row) + c.K);
    for (int t = 0; t < c.T; ++t)
      for (int at = ((wave + t) & (NW - 1)) * 1024; at < KP; at += NW * 1024) {
        const int k = at + (lane >> 3) * 128 + ((lane & 7) ^ (t & 7)) * 16;
        dma16(lds_address(s_x) + t * KP + at, rx, k < c.K ? t * (int)c.x_row + k : kOut);
      }
    const int i = min((int)threadIdx.x, items - 1), t = row_of(i);
    xs_first = c.x_scale[t * c.xs_t + (i - t * KB) * c.xs_b];
  }
  const float w_first = c.w_scale[(size_t)nb0 * KB + min((int)threadIdx.x, w_items - 1)];
  asm volatile("" ::: "memory");

  const __amdgpu_buffer_rsrc_t rw = make_rsrc(
      static_cast<const char*>(c.W) + (size_t)n_first * c.K, (n_last - n_first) * c.K);
  const int turns = (KB - wave + NW - 1) / NW;  // blocks of this wave, of each 16 outputs
  const int tiles = (n_last - n_first + 15) / 16;
  const int line = (lane >> 3) * c.K, chunk = (lane & 7) * 16;
  int at_tile = 0, at_turn = 0;  // the next block to load
  u4 w[kAhead][2];
  auto load = [&](int u) {
    const int k = (wave + at_turn * NW) * 128 + chunk;
    const int off = at_tile < tiles && k < c.K ? at_tile * 16 * c.K + line + k : kOut;
    w[u][0] = ld_buf_stream(rw, off);
    w[u][1] = ld_buf_stream(rw, off + 8 * c.K);
    const bool wrap = ++at_turn >= turns;
    at_turn = wrap ? 0 : at_turn;
    at_tile += wrap ? 1 : 0;
  };
#pragma unroll
  for (int u = 0; u < kAhead; ++u) load(u);

  if constexpr (QUANT) {
#pragma unroll
    for (int r = 0; r < kFewRounds; ++r)
      if (x_at + r * NW * 4 < items) put_x(x_at + r * NW * 4, x_raw[r]);
  } else {
    if (threadIdx.x < items) s_scale[threadIdx.x] = xs_first;
    for (int i = threadIdx.x + kThreadsHere; i < items; i += kThreadsHere) {
      const int t = row_of(i);
      s_scale[i] = c.x_scale[t * c.xs_t + (i - t * KB) * c.xs_b];
    }
    // what went straight to the LDS came before the 2 kAhead loads of weights
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * kAhead) : "memory");
  }
  if (threadIdx.x < w_items) s_w[threadIdx.x] = w_first;
  for (int i = threadIdx.x + kThreadsHere; i < w_items; i += kThreadsHere)
    s_w[i] = c.w_scale[(size_t)nb0 * KB + i];
  __syncthreads();

  const int t = min(r16, c.T - 1);
  char* const tile = s_tile[wave];
  char* const put = tile + (lane >> 3) * 128 + (((lane & 7) ^ (lane >> 3)) * 16);
  const char* const get = tile + r16 * 128;
  const char* const px = s_x + t * KP;
  const int g0 = (q ^ (r16 & 7)) * 16, g1 = g0 ^ 64;
  const int x0 = (q ^ (t & 7)) * 16, x1 = x0 ^ 64;
  int turn = 0, n_tile = 0;
  f4 acc = {0, 0, 0, 0};
  const int steps = tiles * turns;
  for (int s = 0; s < steps; s += kAhead) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (s + u >= steps) break;
      *reinterpret_cast<u4*>(put) = w[u][0];
      *reinterpret_cast<u4*>(put + 1024) = w[u][1];
      load(u);
      wave_lds_order();
      const int b = wave + turn * NW;
      const i8v a = join(ld16(get + g0), ld16(get + g1));
      const i8v x = join(ld16(px + b * 128 + x0), ld16(px + b * 128 + x1));
      const int n = min(n_first + 16 * n_tile + 4 * q, n_last - 1);
      const float scale = s_scale[t * KB + b] * s_w[(n / 128 - nb0) * KB + b];
      wave_lds_order();
      const f4 p = product(a, x);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] += p[e] * scale;
      if (++turn == turns) {
        s_part[n_tile++][wave][lane] = acc;
        acc = f4{0, 0, 0, 0};
        turn = 0;
      }
    }
  }
  __syncthreads();
  const int parts = min(NW, KB);
  for (int i = wave; i < tiles; i += NW) {
    f4 sum = s_part[i][0][lane];
    for (int p = 1; p < parts; ++p) sum += s_part[i][p][lane];
    const int n = n_first + 16 * i + 4 * q;
    if (r16 < c.T && n < n_last)
      store4<E>(c.y, (size_t)r16 * c.N + n, n_last - n, c.N % 4 == 0, sum);
  }
}

// ------------------------------------------------------------- full tiles
// A workgroup has tiles of BN outputs by BT tokens, its waves WN by WT of them, and
// goes through K a block at a time: S stages lie in the LDS, S - 1 of them on their
// way (behind a tile's last blocks, the first ones of the workgroup's next tile)
// while one is multiplied.  Rows of 128 bytes lie 16 bytes at a time in the order
// (chunk ^ row % 8), set by which global chunk a lane fetches: the 16 rows that a
// quarter of a wave reads then lie in different banks.  Each wave fetches the scales
// of its own tokens along with them.
//
// Small tiles, of few tokens, have G groups of waves that take the blocks of K in turn,
// each with stages of its own: a barrier then has G blocks, and a step of small tiles
// is the latency of barrier, reads and products (0.3 us), whatever they are.  The
// groups' sums meet in the LDS in order.  48 tokens of [6144, 4096], quantised: 12.3 us
// in 128 x 64 with K in five parts, 13.5 in 32 x 64 with ten stages, 9.2 in 64 x 32 with four
// groups; such workgroups have one tile each.
//
// Large tiles keep the matrix cores busy: 8192 x 14336 x 4096 418 to 440 us by card, 2.2 to
// 2.3 PFLOP/s (2.36 to 2.48 in a library product with one scale), where the scaled sums take 14%.  256 x 128 fetches
// and reads more for a product (1.15 us a block of K, of which the LDS is busy 0.6 and the
// matrix cores 0.43) and is for outputs that 256 x 256 would leave half the CUs without:
// 2047 x 4096 x 4096 40 us, 52 in 256 x 256.
template <class E, int BN, int BT, int WN, int WT, int S, int G = 1>
__global__ __launch_bounds__(G*(BN / WN) * (BT / WT) * kWave, G > 2 ? 1 : 2) void gemm_blocks_tile(
    GemmBlocksCall c, GemmBlocksPlan plan) {
  typedef typename E::type elem;
  constexpr int NW = (BN / WN) * (BT / WT), NI = WN / 16, TI = WT / 16;  // NW: of a group
  constexpr int kLoadsW = BN / 8 / NW, kLoadsX = BT / 8 / NW;  // of 8 rows, a wave
  constexpr int kLoads = kLoadsW + kLoadsX + 1;                // and one of scales
  static_assert(BN % (8 * NW) == 0 && BT % (8 * NW) == 0, "whole loads");
  static_assert(NI % 2 == 0 && 128 % WN == 0, "row tiles in pairs, of one block of the weights");
  static_assert(WT <= kWave, "a lane for each token's scale");
  constexpr int kScales = (BN + BT) * 128, kStage = kScales + NW * kWave * 4;
  static_assert(G == 1 || S * kStage >= NW * kWave * NI * TI * 16, "room to join the groups' sums");
  __shared__ __align__(16) char s_stage[G * S * kStage];
  const int lane = threadIdx.x & (kWave - 1);
  const int all_wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int group = G > 1 ? all_wave / NW : 0, wave = G > 1 ? all_wave % NW : all_wave;
  const int r16 = lane & 15, q = lane >> 4;
  const int KB = (c.K + 127) / 128;
  const int wn = wave % (BN / WN) * WN, wt = wave / (BN / WN) * WT;

  // Workgroups i, i + 8, .. run on one XCD: its share of the tiles is a
  // compact part of the output, strips of eight token tiles wide.
  const int tn = (c.N + BN - 1) / BN, tt = (c.T + BT - 1) / BT, all = tn * tt * plan.parts;
  struct Place {
    int n0, t0, part, b0, b1;  // blocks b0 .. b1 - 1 of K
  };
  auto place = [&](int i) {
    const int xcd = i & 7, each = all >> 3, more = all & 7;
    const int nth = xcd * each + min(xcd, more) + (i >> 3);
    const int part = nth / (tn * tt), at = nth - part * tn * tt;
    const int strip = at / (8 * tn), in = at - strip * 8 * tn, wide = min(8, tt - 8 * strip);
    return Place{in / wide * BN, (8 * strip + in % wide) * BT, part, part * plan.each,
                 min(KB, (part + 1) * plan.each)};
  };

  // Load i of a wave has rows 8 (NW i + wave) .. + 7 of the weights, or of x.
  const int lane_row = 8 * wave + (lane >> 3), chunk = ((lane & 7) ^ (lane >> 3)) * 16;
  const int w_row = lane_row * c.K, x_row = lane_row * (int)c.x_row;
  // What is fetched: the next block of a tile, then of the workgroup's next one.
  int tile = blockIdx.x, next, last;
  u4 rw, rx;
  const float* xs;  // of the wave's first token
  int xs_lane;
  auto open = [&] {
    const Place f = place(tile);
    next = f.b0 + group;
    last = f.b1;
    rw = dma_rsrc(static_cast<const char*>(c.W) + (size_t)f.n0 * c.K, min(BN, c.N - f.n0) * c.K);
    rx = dma_rsrc(static_cast<const char*>(c.x) + f.t0 * c.x_row,
                  (int)((min(BT, c.T - f.t0) - 1) * c.x_row) + c.K);
    const int t = min(f.t0 + wt, c.T - 1);
    xs = c.x_scale + t * c.xs_t;
    xs_lane = min(min(lane, WT - 1), c.T - 1 - t) * (int)c.xs_t * 4;
  };
  char* const my_stages = s_stage + group * S * kStage;
  const unsigned lds = lds_address(my_stages);
  auto fetch = [&](int stage) {
    if (G == 1 && next == last && tile < all) {
      tile += gridDim.x;
      if (tile < all) open();
    }
    const unsigned to = lds + stage * kStage;
    const int b = min(next, last - 1), k = next * 128 + chunk;
    const int off = next < last && k < c.K ? k : kOut;  // behind the last tile come zeros
#pragma unroll
    for (int i = 0; i < kLoadsW; ++i)
      dma16(to + (i * NW + wave) * 1024, rw, off + w_row + i * NW * 8 * c.K);
#pragma unroll
    for (int i = 0; i < kLoadsX; ++i)
      dma16(to + BN * 128 + (i * NW + wave) * 1024, rx, off + x_row + i * NW * 8 * (int)c.x_row);
    dma4(to + kScales + wave * kWave * 4, dma_rsrc(xs + b * c.xs_b, 0x7FFFFFFF), xs_lane);
    next = G > 1 ? next + G : min(next + 1, last);
  };

  f4 acc[NI][TI];
  // (the next stage is asked for behind the first reads, whose wait that fills)
  auto multiply = [&](int at, float w_scale, int ask) {
    const char* const stage = my_stages + at * kStage;
    const int s0 = (q ^ (r16 & 7)) * 16, s1 = s0 ^ 64;
    const char* const pw = stage + (wn + r16) * 128;
    const char* const px = stage + (BN + wt + r16) * 128;
    i8v x[TI];
#pragma unroll
    for (int j = 0; j < TI; ++j)
      x[j] = join(ld16(px + j * 2048 + s0), ld16(px + j * 2048 + s1));
    auto rows = [&](int i) { return join(ld16(pw + i * 2048 + s0), ld16(pw + i * 2048 + s1)); };
    i8v w[3] = {rows(0), rows(1), {}};
    fetch(ask);
    f4 p[TI];
    float scale[TI];
#pragma unroll
    for (int i = 0; i < TI; ++i)
      scale[i] = *reinterpret_cast<const float*>(stage + kScales + (wave * kWave + 16 * i + r16) * 4) *
                 w_scale;
#pragma unroll
    for (int i = 0; i < NI; ++i) {
      // the products of row tile i beside the sums of i - 1 and the reads of i + 2
      f4 now[TI];
      if (i + 2 < NI) w[(i + 2) % 3] = rows(i + 2);
#pragma unroll
      for (int j = 0; j < TI; ++j) {
        now[j] = product(w[i % 3], x[j]);
        if (i > 0) {
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i - 1][j][e] += p[j][e] * scale[j];
          // (an empty statement that holds the sums here: left free, they all sink
          // to the end and their operands do not fit the registers)
          asm volatile("" : "+v"(acc[i - 1][j]));
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // one product,
        __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);  // one read,
        __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);  // four sums
      }
#pragma unroll
      for (int j = 0; j < TI; ++j) p[j] = now[j];
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int j = 0; j < TI; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[NI - 1][j][e] += p[j][e] * scale[j];
  };
  open();
#pragma unroll
  for (int i = 0; i < S - 1; ++i) fetch(i);
  int stage = 0, free_stage = S - 1;
  for (int now = blockIdx.x; now < all; now += gridDim.x) {
    const Place here = place(now);
    const float* const ws =
        c.w_scale + (size_t)min((here.n0 + wn) / 128, (c.N - 1) / 128) * KB;
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < TI; ++j) acc[i][j] = f4{0, 0, 0, 0};
    float w_scale = scalar_load(ws + min(here.b0 + group, here.b1 - 1));
    for (int b = here.b0; b < here.b1; b += G) {
      // the oldest stage is there, for all waves, and nobody reads the one before it
      dma_barrier<(S - 2) * kLoads>();
      // (the block's scale is waited for here, before the next one is asked for)
      asm volatile("" : "+s"(w_scale));
      const float w_next = scalar_load(ws + min(b + group + G, here.b1 - 1));
      // (a group without a block is at its end, where nothing more is fetched)
      if (G == 1 || b + group < here.b1) multiply(stage, w_scale, free_stage);
      w_scale = w_next;
      stage = stage + 1 == S ? 0 : stage + 1;
      free_stage = free_stage + 1 == S ? 0 : free_stage + 1;
    }
    if constexpr (G > 1) {
      // the groups' sums, in order; the stages have no other use left (what is
      // on its way into them are zeros, waited for first)
      f4* const sums = reinterpret_cast<f4*>(s_stage) + (wave * NI * TI) * kWave + lane;
#pragma unroll
      for (int g = 1; g < G; ++g) {
        dma_barrier<0>();
        if (group == g)
#pragma unroll
          for (int i = 0; i < NI * TI; ++i) sums[i * kWave] = acc[i / TI][i % TI];
        __syncthreads();
        if (group == 0)
#pragma unroll
          for (int i = 0; i < NI * TI; ++i) acc[i / TI][i % TI] += sums[i * kWave];
      }
      if (group > 0) return;
    }
    const int n_here = here.n0 + wn, t_here = here.t0 + wt;
    if (plan.parts > 1) {
      float* const to = plan.sums + (size_t)here.part * c.T * plan.pitch;
#pragma unroll
      for (int j = 0; j < TI; ++j) {
        const int t = t_here + 16 * j + r16;
        if (t >= c.T) continue;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const int n = n_here + 16 * i + 4 * q;
          if (n < c.N) *reinterpret_cast<f4*>(to + (size_t)t * plan.pitch + n) = acc[i][j];
        }
      }
      continue;
    }
    // A lane has outputs 4 q .. + 3 of row tile i; two row tiles exchange quarters,
    // so that it has eight outputs of one of them: 8 (q / 2) .. + 7 of i + q % 2.
#pragma unroll
    for (int j = 0; j < TI; ++j) {
      const int t = t_here + 16 * j + r16;
      if (t >= c.T) continue;
#pragma unroll
      for (int i = 0; i < NI; i += 2) {
        const int n = n_here + 16 * (i + (q & 1)) + 8 * (q >> 1);
        u4 v;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          typename E::vec4 a, b;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            a[e] = (elem)acc[i][j][e];
            b[e] = (elem)acc[i + 1][j][e];
          }
          const u2 r = __builtin_amdgcn_permlane16_swap(__builtin_bit_cast(u2, a)[h],
                                                        __builtin_bit_cast(u2, b)[h], false, false);
          v[h] = r[0];
          v[2 + h] = r[1];
        }
        elem* const to = static_cast<elem*>(c.y) + (size_t)t * c.N + n;
        if (c.N % 8 == 0) {
          if (n < c.N) *reinterpret_cast<u4*>(to) = v;
        } else {
          const typename E::vec8 o = __builtin_bit_cast(typename E::vec8, v);
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (n + e < c.N) to[e] = o[e];
        }
      }
    }
  }
  dma_drain();  // what is still on its way into the LDS (zeros), before that is given back
}

// The sums of the parts of K, in order.  (A launch of its own: 3 to 5 us in all.)
template <class E>
__global__ __launch_bounds__(kThreads) void gemm_blocks_join(GemmBlocksCall c,
                                                             GemmBlocksPlan plan) {
  const int quads = plan.pitch / 4;
  const size_t at = (size_t)blockIdx.x * kThreads + threadIdx.x;
  const int t = (int)(at / quads), n = (int)(at - (size_t)t * quads) * 4;
  if (t >= c.T) return;
  const float* from = plan.sums + (size_t)t * plan.pitch + n;
  f4 sum = *reinterpret_cast<const f4*>(from);
  // five parts' loads at once, added in order
  constexpr int kLoads = 5;
  for (int p0 = 1; p0 < plan.parts; p0 += kLoads) {
    f4 v[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      v[i] = *reinterpret_cast<const f4*>(
          from + (size_t)min(p0 + i, plan.parts - 1) * c.T * plan.pitch);
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      if (p0 + i < plan.parts) sum += v[i];
  }
  store4<E>(c.y, (size_t)t * c.N + n, c.N - n, c.N % 4 == 0, sum);
}

// Shapes of the tile kernel; kFew: the kernel of few tokens.
enum Shape { kFew, k256x256, k256x128, k128x64, k128x32, k64x64, k64x32, k32x32, kShapes };
struct ShapeSize {
  int n, t, threads, slots;  // slots: workgroups a CU
  int groups;                // of waves, with a block of K each
  double step, step2;        // us of a block of K for each group, with one and with two workgroups a CU
};
constexpr ShapeSize kShape[kShapes] = {{16, 16, 512, 1, 1, 0.0, 0.0},
                                       {256, 256, 512, 1, 1, 1.95, 1.95},
                                       {256, 128, 512, 1, 1, 1.15, 1.15},
                                       {128, 64, 256, 2, 1, 0.47, 0.82},
                                       {128, 32, 256, 2, 1, 0.42, 0.62},
                                       {64, 64, 512, 1, 2, 0.58, 0.58},
                                       {64, 32, 512, 1, 4, 0.82, 0.82},
                                       {32, 32, 512, 1, 4, 0.59, 0.59}};

constexpr int kFewWaves = 8;
constexpr size_t kFewLds = 100 * 1024;  // dynamic, next to 48 KB of partial sums and tiles

size_t few_lds(int T, int K, int each) {
  const int KB = (K + 127) / 128;
  return (size_t)T * ((K + 1023) / 1024 * 1024 + KB * 4) + (size_t)(each / 128 + 2) * KB * 4;
}

// The kernel of few tokens may take more dynamic LDS than a launch has unasked.
template <class E, bool QUANT>
hipError_t launch_few(const GemmBlocksCall& c, const GemmBlocksPlan& plan, hipStream_t stream) {
  auto* const fn = gemm_blocks_few<E, QUANT, kFewWaves>;
  static std::atomic<unsigned long long> asked{0};  // devices this kernel was asked for
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return e;
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
  if (!(asked.load(std::memory_order_relaxed) & bit)) {
    e = hipFuncSetAttribute(reinterpret_cast<const void*>(fn),
                            hipFuncAttributeMaxDynamicSharedMemorySize, (int)kFewLds);
    if (e != hipSuccess) return e;
    asked.fetch_or(bit, std::memory_order_relaxed);
  }
  fn<<<plan.grid, kFewWaves * kWave, few_lds(c.T, c.K, plan.each), stream>>>(c, plan);
  return hipGetLastError();
}

template <class E>
hipError_t launch(const GemmBlocksCall& c, const GemmBlocksPlan& plan, hipStream_t stream) {
  if (plan.shape == kFew)
    return c.x_scale ? launch_few<E, false>(c, plan, stream) : launch_few<E, true>(c, plan, stream);
  auto* const fn = plan.shape == k256x256   ? gemm_blocks_tile<E, 256, 256, 128, 64, 2>
                   : plan.shape == k256x128 ? gemm_blocks_tile<E, 256, 128, 64, 64, 3>
                   : plan.shape == k128x64  ? gemm_blocks_tile<E, 128, 64, 64, 32, 3>
                   : plan.shape == k128x32  ? gemm_blocks_tile<E, 128, 32, 32, 32, 3>
                   : plan.shape == k64x64   ? gemm_blocks_tile<E, 64, 64, 32, 32, 4, 2>
                   : plan.shape == k64x32   ? gemm_blocks_tile<E, 64, 32, 32, 32, 3, 4>
                                            : gemm_blocks_tile<E, 32, 32, 32, 16, 4, 4>;
  fn<<<plan.grid, kShape[plan.shape].threads, 0, stream>>>(c, plan);
  if (plan.parts > 1) {
    const size_t quads = (size_t)c.T * plan.pitch / 4;
    gemm_blocks_join<E><<<(quads + kThreads - 1) / kThreads, kThreads, 0, stream>>>(c, plan);
  }
  return hipGetLastError();
}

}  // namespace

GemmBlocksPlan gemm_blocks_plan(int T, int K, int N, int cu_count) {
  const int KB = (K + 127) / 128;
  GemmBlocksPlan p = {};
  p.parts = 1;
  p.pitch = (N + 3) / 4 * 4;
  if (T <= 16 && !tuning().blocks_shape) {
    const int rounds = (N + 64 * cu_count - 1) / (64 * cu_count);
    p.each = ((N + rounds * cu_count - 1) / (rounds * cu_count) + 3) / 4 * 4;
    p.grid = (N + p.each - 1) / p.each;
    p.magic = KB > 1 ? 0xFFFFFFFFu / KB + 1 : 0;
    // Every workgroup quantises all of x, whatever N.  us, and with a launch for it:
    //   K = 4096, tokens   2          8          12         16
    //   N = 14336       13.0 16.4  15.6 17.0  17.8 17.6  19.5 18.1
    //   N = 4096         6.9  9.8   9.7 10.2  11.4 10.5  14.7 11.0
    //   N = 1024         6.0  8.6   8.6  8.9  10.9  9.3  13.6  9.7
    // [4096, 14336], 2 tokens 14.4 and 16.1, 4 tokens 18.2 and 16.2; [2048, 2048], 16
    // tokens 8.3 and 8.7.
    p.fused = T * KB <= 320;
    if (few_lds(T, K, p.each) <= kFewLds) return p;
    p.fused = false;
  }
  // The shape and the parts of K whose rounds of workgroups are estimated to take
  // the least time, by the steps that each shape measured.  27 sizes from 16 to 8192
  // tokens: within 4% of the best of all forced ones on 22 of them, 20% on the worst
  // (64 x 1024 x 8192, 10.6 for 8.7 us).
  double best = 0.0;
  for (int shape = k256x256; shape < kShapes; ++shape) {
    if (tuning().blocks_shape && shape != tuning().blocks_shape) continue;
    const ShapeSize& s = kShape[shape];
    const long long tiles = (long long)((N + s.n - 1) / s.n) * ((T + s.t - 1) / s.t);
    for (int parts = 1; parts <= 16 && parts <= KB; ++parts) {
      if (tuning().blocks_parts && parts != min(KB, tuning().blocks_parts)) continue;
      const int each = (KB + parts - 1) / parts, have = (KB + each - 1) / each;
      const long long work = tiles * have;
      // workgroups of 128 outputs run two to a CU, a step of two takes longer
      const long long rounds = (work + s.slots * cu_count - 1) / (s.slots * cu_count);
      const bool crowded = s.slots > 1 && work > cu_count;
      const double sums = have > 1 ? (double)have * T * p.pitch * sizeof(float) : 0.0;
      const int steps = (each + s.groups - 1) / s.groups;
      // a first tile starts cold, a workgroup's next ones cost two steps more
      const double step = crowded ? s.step2 : s.step, cold = 2.4;
      const double start = s.groups > 1 ? rounds * cold : std::max(cold, rounds * 2 * step);
      const double busy = rounds * steps * step + start;
      // The weights come at 5.5 TB/s to all CUs together; neither hides all of the other.
      const double stream = (double)K * N / 5.5e6 * std::max(1.0, (double)cu_count / work);
      const double us = std::max(busy, stream) + 0.1 * std::min(busy, stream) +
                        (have > 1 ? 4.2 + 0.1 * have + sums * 1.2 / 6e6 : 0.0);
      if (best == 0.0 || us < best) {
        best = us;
        p.shape = shape;
        p.each = each;
        p.parts = have;
        p.grid = (int)(s.groups > 1 ? work : min(work, (long long)cu_count * s.slots));
        p.bytes = have > 1 ? (size_t)have * T * p.pitch * sizeof(float) : 0;
      }
    }
  }
  return p;
}

hipError_t launch_gemm_blocks(const GemmBlocksCall& c, const GemmBlocksPlan& plan,
                              hipStream_t stream) {
  return c.bf16 ? launch<ElemBF16>(c, plan, stream) : launch<ElemF16>(c, plan, stream);
}

}  // namespace dbk
