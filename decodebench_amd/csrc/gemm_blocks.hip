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

// ------------------------------------------------------------- full tiles
// A workgroup has tiles of BN outputs by BT tokens, its waves WN by WT of them,
// and goes through K a block at a time: while a block is multiplied from one
// half of the LDS, the next one (behind the last, the first of the workgroup's
// next tile) is on its way into the other (buffer_load .. lds, no registers).
// Rows of 128 bytes lie 16 bytes at a time in the order (chunk ^ row % 8), set
// by which global chunk a lane fetches: the 16 rows that a quarter of a wave
// reads then lie in different banks.
template <class E, int BN, int BT, int WN, int WT>
__global__ __launch_bounds__((BN / WN) * (BT / WT) * kWave, 2) void gemm_blocks_tile(
    GemmBlocksCall c) {
  typedef typename E::type elem;
  constexpr int NW = (BN / WN) * (BT / WT), NI = WN / 16, TI = WT / 16;
  constexpr int kLoads = (BN + BT) / 8 / NW;  // of 8 rows, a wave
  static_assert((BN + BT) % (8 * NW) == 0 && BN % (8 * kLoads) == 0, "whole loads");
  static_assert(NI % 2 == 0 && 128 % WN == 0, "row tiles in pairs, of one block of the weights");
  constexpr int kHalf = (BN + BT) * 128;
  __shared__ __align__(16) char s_a[kHalf];
  __shared__ __align__(16) char s_b[kHalf];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int r16 = lane & 15, q = lane >> 4;
  const int KB = (c.K + 127) / 128;
  const int wn = wave % (BN / WN) * WN, wt = wave / (BN / WN) * WT;

  // Workgroups i, i + 8, .. run on one XCD: its share of the tiles is a
  // compact part of the output, strips of eight token tiles wide.
  const int tn = (c.N + BN - 1) / BN, tt = (c.T + BT - 1) / BT, all = tn * tt;
  int n0, t0;
  auto place = [&](int i) {
    const int xcd = i & 7, each = all >> 3, more = all & 7;
    const int at = xcd * each + min(xcd, more) + (i >> 3);
    const int strip = at / (8 * tn), in = at - strip * 8 * tn, wide = min(8, tt - 8 * strip);
    n0 = in / wide * BN;
    t0 = (8 * strip + in % wide) * BT;
  };

  // This wave fetches rows 8 kLoads wave .. of the BN + BT.
  const bool from_w = wave * kLoads * 8 < BN;
  const int pitch = from_w ? c.K : (int)c.x_row;
  const int row0 = ((from_w ? wave * kLoads * 8 : wave * kLoads * 8 - BN) + (lane >> 3)) * pitch;
  const int chunk = ((lane & 7) ^ (lane >> 3)) * 16;
  __amdgpu_buffer_rsrc_t rows_of;
  // scales of this lane's tokens and of the wave's outputs, loaded a block ahead
  const float *xs[TI], *ws;
  float scale[TI], ahead[TI], w_ahead;
  auto open = [&] {
    rows_of = from_w ? make_rsrc(static_cast<const char*>(c.W) + (size_t)n0 * c.K,
                                 min(BN, c.N - n0) * c.K)
                     : make_rsrc(static_cast<const char*>(c.x) + t0 * c.x_row,
                                 (int)((min(BT, c.T - t0) - 1) * c.x_row) + c.K);
#pragma unroll
    for (int i = 0; i < TI; ++i)
      xs[i] = c.x_scale + min(t0 + wt + 16 * i + r16, c.T - 1) * c.xs_t;
    ws = c.w_scale + (size_t)min((n0 + wn) / 128, (c.N - 1) / 128) * KB;
  };
  auto fetch = [&](char* half, int b) {
    const int k = b * 128 + chunk;
    const int off = (k < c.K ? k : kOut) + row0;
    char* const to = half + wave * kLoads * 1024;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      typedef __attribute__((address_space(3))) void lds;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rows_of, (lds*)(to + i * 1024), 16,
                                               off + i * 8 * pitch, 0, 0, 0);
    }
    const int in = min(b, KB - 1);
    w_ahead = ws[in];
#pragma unroll
    for (int i = 0; i < TI; ++i) ahead[i] = xs[i][in * c.xs_b];
  };

  f4 acc[NI][TI];
  auto multiply = [&](const char* half) {
    const int s0 = (q ^ (r16 & 7)) * 16, s1 = s0 ^ 64;
    const char* const pw = half + (wn + r16) * 128;
    const char* const px = half + (BN + wt + r16) * 128;
    i8v x[TI];
#pragma unroll
    for (int j = 0; j < TI; ++j)
      x[j] = join(ld16(px + j * 2048 + s0), ld16(px + j * 2048 + s1));
    auto rows = [&](int i) { return join(ld16(pw + i * 2048 + s0), ld16(pw + i * 2048 + s1)); };
    i8v w[3] = {rows(0), rows(1), {}};
    f4 p[TI];
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
  // The block of `half` is there, and nobody reads the other half any more; behind
  // the last block lie zeros, scaled by zero.
  auto ready = [&](int b) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < TI; ++i) scale[i] = b < KB ? ahead[i] * w_ahead : 0.0f;
  };

  int tile = blockIdx.x;
  place(tile);
  open();
  fetch(s_a, 0);
  while (true) {
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int j = 0; j < TI; ++j) acc[i][j] = f4{0, 0, 0, 0};
    const int n_here = n0 + wn, t_here = t0 + wt;
    for (int b = 0; b < KB; b += 2) {
      ready(b);
      fetch(s_b, b + 1);
      multiply(s_a);
      ready(b + 1);
      int next = b + 2;
      if (next >= KB) {
        tile += gridDim.x;
        if (tile < all) {
          place(tile);
          open();
          next = 0;
        }
      }
      fetch(s_a, next);
      multiply(s_b);
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
    if (tile >= all) break;
  }
}

template <class E>
void launch(const GemmBlocksCall& c, hipStream_t stream) {
  if (c.T > 64) {
    const long long large = (long long)((c.N + 255) / 256) * ((c.T + 255) / 256);
    if (large >= 256) {
      gemm_blocks_tile<E, 256, 256, 128, 64><<<min(large, 256ll), 512, 0, stream>>>(c);
    } else {
      const int n = (c.N + 127) / 128 * ((c.T + 127) / 128);
      gemm_blocks_tile<E, 128, 128, 64, 64><<<n, 256, 0, stream>>>(c);
    }
    return;
  }
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
