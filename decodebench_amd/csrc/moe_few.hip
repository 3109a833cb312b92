// moe_few.hip -- the experts of a mixture-of-experts layer for a token or a few:
// two launches, and none to sort, choose or add up.
//
//   moe_few_gate   h[p, i] = silu(Wg[e] x[t]) * (Wu[e] x[t])   for each pair p = (t, j)
//   moe_few_down   y[t, n] = sum_j w[t, j] Wd[e] h[p]
//
// Each pair reads its expert's weights itself: with few tokens hardly any expert is
// asked twice, and then its second reader finds the rows in the L2 or behind it.
// The bytes of the weights bound it.  A wave has a row (of gate and up, or of down
// for all of a token's experts): a load instruction takes 1 KB of it, the next
// kAhead items of the wave are on their way to registers, products are two 16-bit
// elements at a time (e4m3 is widened first, exactly) with fp32 sums, and a row's
// sum over the lanes comes once, at its end.  The scale of a block multiplies the
// lane's sum of its 16 elements of the block.  h stays in fp32, which the down product
// takes with fp32 multiply-adds: a layer is 1.4 times nearer to 64 bits than with h of
// 16 (bf16), and costs up to 3% more (one token, 8 of 128 experts of 768 x 2048: 23.0
// us for 22.7, e4m3 20.4 for 19.8; 2 of 8 of 14336 x 4096: the same).
//
// With the router's logits given, every workgroup of the first launch chooses its
// token's experts for itself (1 us, and no launch between): the second launch gets
// the choice from the workgroups of the first rows.
//
// One token, 8 of 128 experts of 768 x 2048, bf16 (75.5 MB): the layer 22.2 us, of which
// the gate takes 11 to 13 (4.2 TB/s), the down product 6.9 and the logits 2 to 3; 2 of 8
// of 14336 x 4096 116 us (6.1 TB/s), e4m3 66 (5.3; half the bytes on their way, and a
// load of scales with each KB).  A launch
// pays about 3 us before its stream runs at its rate: x, the choice, the first rows.
#include <atomic>

#include "db_kernels.h"
#include "moe_select.h"

namespace dbk {

namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;

__device__ __forceinline__ float dot2(h2 a, h2 b, float c) {
  return __builtin_amdgcn_fdot2(a, b, c, false);
}
__device__ __forceinline__ float dot2(b2 a, b2 b, float c) {
  return __builtin_amdgcn_fdot2_f32_bf16(a, b, c, false);
}
// (by value: a bit cast of a vector's element takes the vector's first bytes)
template <class V>
__device__ __forceinline__ V as2(unsigned v) {
  return __builtin_bit_cast(V, v);
}
template <class V>
__device__ __forceinline__ float dot8v(u4 a, u4 b, float c) {
#pragma unroll
  for (int i = 0; i < 4; ++i) c = dot2(as2<V>(a[i]), as2<V>(b[i]), c);
  return c;
}

template <class E>
struct Pair2;
template <>
struct Pair2<ElemF16> {
  typedef h2 type;
};
template <>
struct Pair2<ElemBF16> {
  typedef b2 type;
};

// A lane's 16 bytes of a row times the same columns of x in the LDS.
template <class E, bool FP8>
__device__ __forceinline__ float dot_chunk(u4 w, const char* x) {
  typedef typename Pair2<E>::type V;
  if constexpr (!FP8) {
    return dot8v<V>(w, ld16(x), 0.0f);
  } else {
    const u2 a = E::widen(w[0]), b = E::widen(w[1]), c = E::widen(w[2]), d = E::widen(w[3]);
    const float lo = dot8v<V>(u4{a[0], a[1], b[0], b[1]}, ld16(x), 0.0f);
    return dot8v<V>(u4{c[0], c[1], d[0], d[1]}, ld16(x + 16), lo);
  }
}

// The same with h in fp32: element 4 p + i of the lane's 8 (16 of e4m3) lies 1 KB * p
// behind the first one, so that lanes side by side read places side by side.
template <class E, bool FP8>
__device__ __forceinline__ float dot_chunk32(u4 w, const char* h) {
  float even = 0.0f, odd = 0.0f;
  auto add = [&](f4 v, float a, float b, float c, float d) {
    even = __builtin_fmaf(a, v[0], even);
    odd = __builtin_fmaf(b, v[1], odd);
    even = __builtin_fmaf(c, v[2], even);
    odd = __builtin_fmaf(d, v[3], odd);
  };
  constexpr int kPlane = kWave * 16;
  if constexpr (FP8) {
    typedef float v2 __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const v2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[p], false);
      const v2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[p], true);
      add(*reinterpret_cast<const f4*>(h + p * kPlane), lo[0], lo[1], hi[0], hi[1]);
    }
  } else {
    const typename E::vec8 v = __builtin_bit_cast(typename E::vec8, w);
#pragma unroll
    for (int p = 0; p < 2; ++p)
      add(*reinterpret_cast<const f4*>(h + p * kPlane), (float)v[4 * p], (float)v[4 * p + 1],
          (float)v[4 * p + 2], (float)v[4 * p + 3]);
  }
  return even + odd;
}

// The scale of the block of the lane's bytes from `off` on (zero behind the last one).
__device__ __forceinline__ float ld_scale(__amdgpu_buffer_rsrc_t r, int off) {
  return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, off / 128 * 4, 0, 0));
}

// Copies a row of K elements to the LDS, with zeros up to a whole number of chunks.
__device__ __forceinline__ void row_to_lds(char* to, const void* from, int K, int padded) {
  for (int k = threadIdx.x * 8; k < padded; k += kThreads * 8)
    *reinterpret_cast<u4*>(to + k * 2) =
        k < K ? ld16(static_cast<const unsigned short*>(from) + k) : u4{0, 0, 0, 0};
}

struct FewArgs {
  MoeFewCall f;
  int slices;    // workgroups of a pair, or of a token
  int padded;    // K in whole chunks
  unsigned magic;  // 2^32 / (padded / 4), rounded up
};

// A workgroup has every (slices)th group of kWaves rows of one pair.
template <class E, bool FP8>
__global__ __launch_bounds__(kThreads) void moe_few_gate(FewArgs a) {
  constexpr int CE = FP8 ? 1024 : 512;  // elements of a row a load instruction takes
  constexpr int CH = FP8 ? 2 : 4;       // of each matrix in an item
  constexpr int kAhead = 2;               // items on their way: 8 or 16 KB a wave
  extern __shared__ __align__(16) char s_x[];
  __shared__ MoeChoice s_choice;
  const MoeExpertsCall& c = a.f.c;
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int pair = blockIdx.x / a.slices, slice = blockIdx.x - pair * a.slices;
  const int t = pair / c.k, j = pair - t * c.k;
  const int H = c.w.H, I = c.w.I;
  const bool chooses = a.f.logits != nullptr;
  MoeLogits<kThreads> logits;
  if (chooses) logits.load(a.f.logits + (size_t)t * c.w.E, 1, 0, c.w.E);
  row_to_lds(s_x, static_cast<const typename E::type*>(c.x) + t * c.x_row, H, a.padded);
  int expert;
  if (chooses) {
    moe_rank(s_choice, logits, c.w.E, c.k);
    expert = s_choice.expert[j];
  } else {
    expert = c.experts[pair];
    __syncthreads();
  }
  expert = __builtin_amdgcn_readfirstlane(expert);
  if ((unsigned)expert >= (unsigned)c.w.E) return;

  const int KB = (H + 127) / 128, NB = (I + 127) / 128;
  constexpr int CB = FP8 ? 1 : 2;
  const size_t row_bytes = (size_t)H * CB;
  const char* const wg = static_cast<const char*>(c.w.wg) + (size_t)expert * I * row_bytes;
  const char* const wu = static_cast<const char*>(c.w.wu) + (size_t)expert * I * row_bytes;
  const int items = (a.padded / CE + CH - 1) / CH;  // of a row
  const int stride = a.slices * kWaves;
  int at_row = slice * kWaves + wave, at_item = 0;
  u4 w[kAhead][2][CH];
  float scale[kAhead][2][CH];
  auto load = [&](int u) {
    // (behind the last row nothing is read)
    const int row = min(at_row, I - 1), bytes = at_row < I ? (int)row_bytes : 0;
    const __amdgpu_buffer_rsrc_t rg = make_rsrc(wg + row * row_bytes, bytes);
    const __amdgpu_buffer_rsrc_t ru = make_rsrc(wu + row * row_bytes, bytes);
    const size_t scales = ((size_t)expert * NB + row / 128) * KB;
    const __amdgpu_buffer_rsrc_t sg = make_rsrc(c.w.sg + scales, KB * 4);
    const __amdgpu_buffer_rsrc_t su = make_rsrc(c.w.su + scales, KB * 4);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int off = ((at_item * CH + i) * kWave + lane) * 16;
      w[u][0][i] = ld_buf_stream(rg, off);
      w[u][1][i] = ld_buf_stream(ru, off);
      if constexpr (FP8) {
        scale[u][0][i] = ld_scale(sg, off);
        scale[u][1][i] = ld_scale(su, off);
      }
    }
    const bool wrap = ++at_item >= items;
    at_item = wrap ? 0 : at_item;
    at_row += wrap ? stride : 0;
  };
#pragma unroll
  for (int u = 0; u < kAhead; ++u) load(u);
  if (chooses && slice == 0) {
    moe_weigh(s_choice, c.w.E, c.k, a.f.renormalize);
    if (threadIdx.x == 0) {
      a.f.experts[pair] = expert;
      a.f.weights[pair] = s_choice.p[j] / s_choice.total;
    }
  }
  int row = slice * kWaves + wave, item = 0;
  float g = 0.0f, up = 0.0f;
  while (row < I) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (row >= I) break;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        const char* const x = s_x + ((item * CH + i) * kWave + lane) * (FP8 ? 32 : 16);
        if ((item * CH + i) * CE >= a.padded) break;
        const float pg = dot_chunk<E, FP8>(w[u][0][i], x), pu = dot_chunk<E, FP8>(w[u][1][i], x);
        g += FP8 ? pg * scale[u][0][i] : pg;
        up += FP8 ? pu * scale[u][1][i] : pu;
      }
      load(u);
      if (++item == items) {
        g = wave_sum(g);
        up = wave_sum(up);
        if (lane == 0)
          static_cast<float*>(c.h)[(size_t)pair * I + row] = g / (1.0f + expf(-g)) * up;
        g = up = 0.0f;
        item = 0;
        row += stride;
      }
    }
  }
}

// A workgroup of NW waves has every (slices)th group of NW rows of one token.
template <class E, bool FP8, int CH, int NW>
__global__ __launch_bounds__(NW* kWave) void moe_few_down(FewArgs a) {
  typedef typename E::type elem;
  constexpr int kThreads = NW * kWave;
  constexpr int CE = FP8 ? 1024 : 512;
  constexpr int kAhead = 8 / CH;  // items on their way: 8 KB a wave
  extern __shared__ __align__(16) char s_h[];
  const MoeExpertsCall& c = a.f.c;
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int t = blockIdx.x / a.slices, slice = blockIdx.x - t * a.slices;
  const int H = c.w.H, I = c.w.I, k = c.k;
  // Lane j holds the token's expert j and its weight.
  static_assert(kMostChoices <= kWave, "a lane for each");
  const int my_expert = c.experts[t * k + min(lane, k - 1)];
  const float my_weight = c.weights[t * k + min(lane, k - 1)];
  // The first pieces of h are asked for before the weights, which come in order
  // behind them.  (What h holds of a pair without an expert does not count.)
  const int row_pieces = a.padded / 4, pieces = k * row_pieces;
  const float* const h_from = static_cast<const float*>(c.h) + (size_t)t * k * I;
  auto piece = [&](int i) {
    const int j = (int)__umulhi(i, a.magic), at = (i - j * row_pieces) * 4;
    return at < I && j < k ? ld16(h_from + (size_t)j * I + at) : u4{0, 0, 0, 0};
  };
  // Piece i goes to plane i % kPlanes, place i / kPlanes, of its chunk of the row.
  constexpr int kPlanes = CE / kWave / 4;
  auto put = [&](int i, u4 v) {
    const int in = i & (CE / 4 - 1);
    *reinterpret_cast<u4*>(s_h + (size_t)(i - in + in % kPlanes * kWave + in / kPlanes) * 16) = v;
  };
  constexpr int kFirst = 8;
  u4 first[kFirst];
#pragma unroll
  for (int r = 0; r < kFirst; ++r) first[r] = piece(threadIdx.x + r * kThreads);

  const int KB = (I + 127) / 128, NB = (H + 127) / 128;
  constexpr int CB = FP8 ? 1 : 2;
  const size_t row_bytes = (size_t)I * CB;
  const int items = (a.padded / CE + CH - 1) / CH;  // of a row of one expert
  const int stride = a.slices * NW;
  int at_row = slice * NW + wave, at_j = 0, at_item = 0;
  u4 w[kAhead][CH];
  float scale[kAhead][CH];
  auto load = [&](int u) {
    const int e = __builtin_amdgcn_readlane(my_expert, at_j);
    const bool exists = at_row < H && (unsigned)e < (unsigned)c.w.E;
    const size_t row = exists ? (size_t)e * H + at_row : 0;
    const __amdgpu_buffer_rsrc_t rd = make_rsrc(
        static_cast<const char*>(c.w.wd) + row * row_bytes, exists ? (int)row_bytes : 0);
    const size_t nb = exists ? (size_t)e * NB + at_row / 128 : 0;
    const __amdgpu_buffer_rsrc_t sd = make_rsrc(c.w.sd + nb * KB, KB * 4);
#pragma unroll
    for (int i = 0; i < CH; ++i) {
      const int off = ((at_item * CH + i) * kWave + lane) * 16;
      w[u][i] = ld_buf_stream(rd, off);
      if constexpr (FP8) scale[u][i] = ld_scale(sd, off);
    }
    const bool wrap = ++at_item >= items;
    at_item = wrap ? 0 : at_item;
    at_j += wrap ? 1 : 0;
    const bool next = at_j >= k;
    at_j = next ? 0 : at_j;
    at_row += next ? stride : 0;
  };
#pragma unroll
  for (int u = 0; u < kAhead; ++u) load(u);
#pragma unroll
  for (int r = 0; r < kFirst; ++r) {
    const int i = threadIdx.x + r * kThreads;
    if (i < pieces) put(i, first[r]);
  }
  for (int i = threadIdx.x + kFirst * kThreads; i < pieces; i += kThreads) put(i, piece(i));
  __syncthreads();
  int row = slice * NW + wave, j = 0, item = 0;
  float sum = 0.0f, part = 0.0f;
  while (row < H) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      if (row >= H) break;
      const char* const h = s_h + (size_t)j * a.padded * 4;
#pragma unroll
      for (int i = 0; i < CH; ++i) {
        if ((item * CH + i) * CE >= a.padded) break;
        const float p = dot_chunk32<E, FP8>(w[u][i], h + (item * CH + i) * CE * 4 + lane * 16);
        part += FP8 ? p * scale[u][i] : p;
      }
      load(u);
      if (++item == items) {
        // (a pair without an expert adds nothing, whatever its weight was)
        if ((unsigned)__builtin_amdgcn_readlane(my_expert, j) < (unsigned)c.w.E)
          sum += part * lane_value(my_weight, j);
        part = 0.0f;
        item = 0;
        if (++j == k) {
          sum = wave_sum(sum);
          if (lane == 0) static_cast<elem*>(c.y)[(size_t)t * H + row] = (elem)sum;
          sum = 0.0f;
          j = 0;
          row += stride;
        }
      }
    }
  }
}

int chunks(int K, bool fp8) {
  const int CE = fp8 ? 1024 : 512;
  return (K + CE - 1) / CE * CE;
}

constexpr size_t kLds = 156 * 1024;  // of a CU, for h

// The down kernel may take more dynamic LDS than a launch has unasked.
template <class E, bool FP8, int CH, int NW>
hipError_t launch_down(const FewArgs& d, size_t bytes, hipStream_t stream) {
  auto* const fn = moe_few_down<E, FP8, CH, NW>;
  static std::atomic<unsigned long long> asked{0};  // devices this kernel was asked for
  int dev = 0;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return e;
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
  if (!(asked.load(std::memory_order_relaxed) & bit)) {
    e = hipFuncSetAttribute(reinterpret_cast<const void*>(fn),
                            hipFuncAttributeMaxDynamicSharedMemorySize, (int)kLds);
    if (e != hipSuccess) return e;
    asked.fetch_or(bit, std::memory_order_relaxed);
  }
  fn<<<d.f.c.T * d.slices, NW * kWave, bytes, stream>>>(d);
  return hipGetLastError();
}

template <class E, bool FP8>
hipError_t launch(const MoeFewCall& f, hipStream_t stream) {
  const MoeExpertsCall& c = f.c;
  int err = 0;
  const int cus = device_cu_count(&err);
  if (err) return (hipError_t)err;
  // waves for each CU, and no more than rows
  auto slices = [&](int groups, int rows, int waves) {
    const int want = (8 * cus / waves + groups - 1) / groups;
    return max(1, min(want, (rows + waves - 1) / waves));
  };
  const int P = c.T * c.k;
  FewArgs g = {f, slices(P, c.w.I, kWaves), chunks(c.w.H, FP8), 0};
  moe_few_gate<E, FP8><<<P * g.slices, kThreads, (size_t)g.padded * 2, stream>>>(g);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  // h in fp32 may fill most of a CU's LDS: one workgroup with the waves of two
  const size_t h_bytes = (size_t)chunks(c.w.I, FP8) * 4 * c.k;
  const int waves = h_bytes <= kLds / 2 ? kWaves : 2 * kWaves;
  FewArgs d = {f, slices(c.T, c.w.H, waves), chunks(c.w.I, FP8), 0};
  d.magic = 0xFFFFFFFFu / (d.padded / 4) + 1;
  // (rows of one load have items of one)
  const bool one = d.padded == chunks(1, FP8);
  return waves == kWaves ? (one ? launch_down<E, FP8, 1, kWaves>(d, h_bytes, stream)
                                : launch_down<E, FP8, 2, kWaves>(d, h_bytes, stream))
                         : (one ? launch_down<E, FP8, 1, 2 * kWaves>(d, h_bytes, stream)
                                : launch_down<E, FP8, 2, 2 * kWaves>(d, h_bytes, stream));
}

}  // namespace

// Few pairs, whose row of x fits the LDS that a launch has without asking and whose rows
// of h fit a CU's, and that read hardly more together than the experts they name among equally likely
// ones: the tile kernels read an expert once for all its tokens, but take 15 us more
// for sorting and adding up (80 MB at the rate of the weights, and 50 more for what the
// L2 holds of a second reading).  us here and there, at one to four tokens:
//   2 of 8 experts of 14336 x 4096, e4m3   67 103  121 142  237 184  211 204
//   the same, 16-bit                      117 165  222 263  414 344  397 374
//   8 of 128 of 768 x 2048, e4m3           21  32   29  33   39  40   43  44
//   6 of 64 of 1408 x 2048, e4m3           23  31   34  37   44  43   54  48
// The rule takes the slower one in the last two only.
bool moe_few(const db_moe& m, int T, int k) {
  const bool fp8 = m.w_dtype == DB_DTYPE_FP8_E4M3;
  const int P = T * k;
  if (T > 4 || P > 32 || (size_t)chunks(m.H, fp8) * 2 + sizeof(MoeChoice) + 1024 > 64 * 1024 ||
      (size_t)chunks(m.I, fp8) * 4 * k > 126 * 1024)
    return false;
  double missed = 1.0;  // chance that an expert is not named
  for (int t = 0; t < T; ++t) missed *= 1.0 - (double)min(k, m.E) / m.E;
  const double bytes = 3.0 * m.H * m.I * (fp8 ? 1 : 2);
  return (P - 1.06 * m.E * (1.0 - missed)) * bytes <= 130e6;
}

hipError_t launch_moe_few(const MoeFewCall& f, hipStream_t stream) {
  const bool fp8 = f.c.w.w_dtype == DB_DTYPE_FP8_E4M3;
  if (f.c.bf16)
    return fp8 ? launch<ElemBF16, true>(f, stream) : launch<ElemBF16, false>(f, stream);
  return fp8 ? launch<ElemF16, true>(f, stream) : launch<ElemF16, false>(f, stream);
}

}  // namespace dbk
