// paged_chunk.hip -- paged attention of many rows (chunks of a prompt), the
// merge of split rows, and the launches of a call.
//
// A workgroup of four waves owns one (request, KV head, row tile of 128 rows)
// and one split of the keys; wave w has rows 32 w .. 32 w + 31 and all four
// share 64-key tiles of K and V in LDS.  Bound by the MFMAs and, beside them,
// the softmax on the VALU.
//
//  * S^T = K Q^T on v_mfma_f32_32x32x16: a lane holds scores of one row (its
//    column), 32 of the tile's 64 keys, the other half in lane ^ 32, so a
//    row's maximum and sum are nearly all in-lane work.
//  * The rounded probabilities are the B operand of O^T = V^T P^T as they lie:
//    accumulator registers 8 s .. 8 s + 7 of lane half h are keys 16 s + 4 h +
//    0..3 and 16 s + 8 + 4 h + 0..3, and V^T is read from LDS in that order by
//    two transposing reads (ds_read_b64_tr_b16) per operand.
//  * The next tile's loads are in flight in registers while this one is
//    computed.  Lane i of every wave looks up the page of key i of a tile.
//  * A wave skips tiles that none of its rows sees, and masks only tiles that
//    some row sees in part (as paged_decode, an Inf or NaN among such a tile's
//    values is added key by key).
#include "paged_attn.h"

namespace dbk {

namespace {

constexpr int kWaves = kPagedThreads / kWave;
constexpr int MT = kChunkRows, KT = kChunkKeys;
constexpr int kRowsPerWave = MT / kWaves;

template <class E, bool FP8, int D>
__global__ __launch_bounds__(kPagedThreads) void paged_chunk(PagedArgs a) {
  typedef typename E::type elem;
  typedef typename E::vec8 vec8;
  constexpr int CB = FP8 ? 1 : 2;
  constexpr int LPR = D * CB / 16;                 // threads per row of a tile
  constexpr int RPI = kPagedThreads / LPR;         // rows a load instruction of the workgroup
  constexpr int NL = KT / RPI;                     // loads of K (and of V) a thread
  constexpr int KS = D + 8, VS = D + 16;           // row strides in LDS (elements)
  constexpr int QSTEPS = D / 16, NB = D / 32;

  __shared__ __align__(16) elem s_k[KT * KS];
  __shared__ __align__(16) elem s_v[KT * VS];

  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int n32 = lane & 31, half = lane >> 5;

  PagedSchedule<MT, KT> schedule(a);
  PagedWork wk;
  while (schedule.next(wk)) {
    const PagedRequest& rq = wk.req;
    int t_begin, t_end;
    paged_range<MT, KT>(a, wk, t_begin, t_end);
    t_begin = __builtin_amdgcn_readfirstlane(t_begin);
    t_end = __builtin_amdgcn_readfirstlane(t_end);
    paged_describe(a, wk, MT);
    const int limit = __builtin_amdgcn_readfirstlane(paged_limit(a, rq.len));

    // This lane's row and the keys it sees; rows past the last one see none.
    const long long left = (long long)rq.n * a.G - (long long)wk.tile * MT;
    const int rows = (int)min(left, (long long)MT);
    const int lrow = wave * kRowsPerWave + n32;
    const bool live = lrow < rows;
    const int x = wk.tile * MT + min(lrow, rows - 1);
    const int token = x / a.G, qhead = wk.head * a.G + x % a.G;
    const int pos = rq.len - rq.n + token;
    const int khi = !live ? 0 : a.causal ? min(limit, pos + 1) : limit;
    const int klo = !live ? 0x7FFFFFFF : a.window > 0 ? max(pos - a.window + 1, 0) : 0;
    // Keys that every live row sees, and keys that any of them sees.
    int all_lo = live ? klo : 0, all_hi = live ? khi : 0x7FFFFFFF, any_lo = klo, any_hi = khi;
    for (int d = 1; d < 32; d <<= 1) {
      all_lo = max(all_lo, __shfl_xor(all_lo, d));
      all_hi = min(all_hi, __shfl_xor(all_hi, d));
      any_lo = min(any_lo, __shfl_xor(any_lo, d));
      any_hi = max(any_hi, __shfl_xor(any_hi, d));
    }
    all_lo = __builtin_amdgcn_readfirstlane(all_lo);
    all_hi = __builtin_amdgcn_readfirstlane(all_hi);
    any_lo = __builtin_amdgcn_readfirstlane(any_lo);
    any_hi = __builtin_amdgcn_readfirstlane(any_hi);

    vec8 qop[QSTEPS];
    {
      const elem* qp = static_cast<const elem*>(a.q) + (rq.tok0 + token) * a.q_token +
                       qhead * a.q_head + 8 * half;
#pragma unroll
      for (int t = 0; t < QSTEPS; ++t) qop[t] = __builtin_bit_cast(vec8, ld16(qp + 16 * t));
    }
    const float scale = a.scale_log2 * (FP8 ? a.k_scale[wk.head] : 1.0f);
    const char* const kbase = static_cast<const char*>(a.k) + wk.head * a.kh * CB;
    const char* const vbase = static_cast<const char*>(a.v) + wk.head * a.vh * CB;
    const int* const trow = a.table + wk.r * a.table_row;

    // Page of key `lane` of a tile, -1 where there is none.
    auto lookup = [&](int tile) {
      const int key = tile * KT + lane;
      if (tile >= t_end || key >= limit) return -1;
      const int p = trow[page_of(a, key)];
      return (unsigned)p < (unsigned)a.pages ? p : -1;
    };
    // Absent keys read row 0 of page 0: valid memory, zero in LDS.
    auto load_tile = [&](u4 (&kt)[NL], u4 (&vt)[NL], int tile, int pg) {
#pragma unroll
      for (int j = 0; j < NL; ++j) {
        const int row = j * RPI + threadIdx.x / LPR, key = tile * KT + row;
        const int pr = __shfl(pg, row), page = max(pr, 0);
        const int off = pr < 0 ? 0 : key - page_of(a, key) * a.page;
        const int c = (threadIdx.x % LPR) * 16;
        kt[j] = ld16(kbase + (page * a.kp + off * a.kt) * CB + c);
        vt[j] = ld16(vbase + (page * a.vp + off * a.vt) * CB + c);
      }
    };
    auto store_row = [&](elem* to, u4 w) {
      if constexpr (FP8) {
        const u2 w0 = E::widen(w[0]), w1 = E::widen(w[1]);
        const u2 w2 = E::widen(w[2]), w3 = E::widen(w[3]);
        *reinterpret_cast<u4*>(to) = u4{w0[0], w0[1], w1[0], w1[1]};
        *reinterpret_cast<u4*>(to + 8) = u4{w2[0], w2[1], w3[0], w3[1]};
      } else {
        *reinterpret_cast<u4*>(to) = w;
      }
    };
    auto store_tile = [&](const u4 (&kt)[NL], const u4 (&vt)[NL], unsigned long long there) {
#pragma unroll
      for (int j = 0; j < NL; ++j) {
        const int row = j * RPI + threadIdx.x / LPR, c = (threadIdx.x % LPR) * (16 / CB);
        const bool ok = (there >> row) & 1;
        store_row(s_k + row * KS + c, ok ? kt[j] : u4{0, 0, 0, 0});
        store_row(s_v + row * VS + c, ok ? vt[j] : u4{0, 0, 0, 0});
      }
    };

    f16v o[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[b][i] = 0.0f;
    float m_run = kPagedNegInf, l_run = 0.0f;  // l: of this lane's keys

    auto compute_tile = [&](int tile, unsigned long long there) {
      const int key0 = tile * KT;
      if (key0 >= any_hi || key0 + KT <= any_lo) return;
      f16v s[2];
#pragma unroll
      for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[kb][i] = 0.0f;
#pragma unroll
        for (int t = 0; t < QSTEPS; ++t)
          s[kb] = E::mfma32(__builtin_bit_cast(
                                vec8, ld16(s_k + (32 * kb + n32) * KS + 16 * t + 8 * half)),
                            qop[t], s[kb]);
      }
      const bool partial = there != ~0ull || key0 < all_lo || key0 + KT > all_hi;
      unsigned sees[2] = {0xFFFFu, 0xFFFFu};  // bit i: register i of block kb counts
      if (partial) {
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
          sees[kb] = 0;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int kk = 32 * kb + 8 * (i >> 2) + 4 * half + (i & 3);
            const bool ok = key0 + kk >= klo && key0 + kk < khi && ((there >> kk) & 1);
            sees[kb] |= ok ? 1u << i : 0u;
            s[kb][i] = ok ? s[kb][i] : kPagedNegInf;
          }
        }
      }
      float tmax = kPagedNegInf;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) tmax = fmaxf(tmax, s[kb][i]);
      tmax = max_xor32(tmax) * scale;
      const float m_new = fmaxf(m_run, tmax);
      const float m_use = m_new == kPagedNegInf ? 0.0f : m_new;
      const float alpha = fast_exp2(m_run - m_use);
      vec8 p[4];
      float sum = 0.0f;
#pragma unroll
      for (int kb = 0; kb < 2; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const elem e = (elem)fast_exp2(fmaf(s[kb][i], scale, -m_use));
          p[2 * kb + (i >> 3)][i & 7] = e;
          sum += (float)e;
        }
      l_run = fmaf(l_run, alpha, sum);
      m_run = m_new;
      if (__any(alpha != 1.0f)) {
#pragma unroll
        for (int b = 0; b < NB; ++b) o[b] *= alpha;
      }
      if (partial) {
        bool bad = false;
        for (int i = lane; i < KT * D / 8; i += kWave) {
          const u4 w = ld16(s_v + (i / (D / 8)) * VS + (i % (D / 8)) * 8);
#pragma unroll
          for (int c = 0; c < 4; ++c) bad = bad || pair_nonfinite<E>(w[c]);
        }
        if (__any(bad)) {
          // Key by key: only keys that the row sees are added.  Two keys of
          // each half a step, the registers moving up by one pair a step.
          u4 pr[4];
#pragma unroll
          for (int t = 0; t < 4; ++t) pr[t] = __builtin_bit_cast(u4, p[t]);
          unsigned bits = sees[0] | (sees[1] << 16);
#pragma unroll 1
          for (int step = 0; step < 16; ++step) {
            const vec8 now = __builtin_bit_cast(vec8, pr[0]);
            const int i0 = 2 * step;  // accumulator register of 32
#pragma unroll
            for (int e = 0; e < 2; ++e) {
#pragma unroll
              for (int h = 0; h < 2; ++h) {
                const float pv = __shfl((float)now[e], n32 + 32 * h);
                const bool sp = (__shfl((int)bits, n32 + 32 * h) >> e) & 1;
                const int i = i0 + e;
                const elem* row = s_v + (32 * (i >> 4) + 8 * ((i & 15) >> 2) + 4 * h + (i & 3)) * VS;
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                  for (int c = 0; c < 16; ++c) {
                    const float v = (float)row[32 * b + 8 * (c >> 2) + 4 * half + (c & 3)];
                    o[b][c] += sp ? pv * v : 0.0f;
                  }
              }
            }
            bits >>= 2;
            const u4 keep[4] = {pr[0], pr[1], pr[2], pr[3]};
#pragma unroll
            for (int t = 0; t < 4; ++t)
              pr[t] = u4{keep[t][1], keep[t][2], keep[t][3], t < 3 ? keep[t < 3 ? t + 1 : 3][0] : 0u};
          }
          return;
        }
      }
#pragma unroll
      for (int t = 0; t < 4; ++t) {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const elem* at = s_v + (16 * t + 4 * half + ((lane & 15) >> 2)) * VS + 32 * b +
                           16 * ((lane >> 4) & 1) + 4 * (lane & 3);
          u2 lo = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                             (__attribute__((address_space(3))) s4*)(at)));
          u2 hi = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                             (__attribute__((address_space(3))) s4*)(at + 8 * VS)));
          o[b] = E::mfma32(__builtin_bit_cast(vec8, u4{lo[0], lo[1], hi[0], hi[1]}), p[t], o[b]);
        }
      }
    };

    u4 kt[NL], vt[NL];
    int pg = lookup(t_begin);
    if (t_begin < t_end) load_tile(kt, vt, t_begin, pg);
    for (int tile = t_begin; tile < t_end; ++tile) {
      const unsigned long long there = __ballot(pg >= 0);
      pg = lookup(tile + 1);
      __syncthreads();  // the previous tile is read
      store_tile(kt, vt, there);
      __syncthreads();
      if (tile + 1 < t_end) load_tile(kt, vt, tile + 1, pg);
      compute_tile(tile, there);
    }

    // ---- outputs -----------------------------------------------------------
    const float l = l_run + __shfl_xor(l_run, 32);
    const float vscale = FP8 ? a.v_scale[wk.head] : 1.0f;
    const int rec = wk.rec < 0 ? -1 : wk.rec + wk.split * a.Hkv;
    if (live) {
      if (rec < 0) {
        const float inv = l == 0.0f ? 0.0f : vscale / l;
        elem* op = static_cast<elem*>(a.o) + ((size_t)(rq.tok0 + token) * a.Hq + qhead) * D;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            typename E::vec4 r;
#pragma unroll
            for (int i = 0; i < 4; ++i) r[i] = (elem)(l == 0.0f ? 0.0f : o[b][4 * c + i] * inv);
            *reinterpret_cast<typename E::vec4*>(op + 32 * b + 8 * c + 4 * half) = r;
          }
      } else if (rec < a.rec.records) {
        const size_t at = (size_t)rec * MT + lrow;
        float* op = a.rec.opart + at * D;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int c = 0; c < 4; ++c)
            *reinterpret_cast<f4*>(op + 32 * b + 8 * c + 4 * half) =
                f4{o[b][4 * c], o[b][4 * c + 1], o[b][4 * c + 2], o[b][4 * c + 3]} * vscale;
        if (half == 0) a.rec.ml[at] = make_float2(m_run, l);
      }
    }
    __syncthreads();  // the tiles are read: the next piece may write them
  }
}

// Joins the records of split rows: o = sum_s e^(m_s - M) o_s / sum_s e^(m_s - M) l_s.
// A workgroup a row, its four waves a quarter of the splits each, eight records
// in flight a wave (a wave alone, one record after the other, took 45 us for
// the 64 splits of one request of 8192 tokens); the groups' count and places
// come from the first kernel.
template <class E, int D>
__global__ __launch_bounds__(kPagedThreads) void paged_merge(PagedArgs a, int mt) {
  typedef typename E::type elem;
  constexpr int PER = D / kWave;  // elements a lane
  constexpr int kAtOnce = 8;
  __shared__ float s_acc[kWaves][D], s_m[kWaves], s_l[kWaves];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int total = min(a.rec.head[0], a.rec.groups) * mt;
  for (int task = blockIdx.x; task < total; task += gridDim.x) {
    const int group = task / mt, row = task % mt;
    const int* d = a.rec.desc + (size_t)group * kDescInts;
    const int splits = d[0], rec0 = d[1], head = rec0 % a.Hkv;
    if (row >= d[4] || rec0 + (splits - 1) * a.Hkv >= a.rec.records) continue;
    float M = kPagedNegInf, L = 0.0f, acc[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) acc[i] = 0.0f;
    for (int s0 = wave; s0 < splits; s0 += kWaves * kAtOnce) {
      float2 ml[kAtOnce];
      float v[kAtOnce][PER];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        const int s = min(s0 + j * kWaves, splits - 1);
        const size_t at = (size_t)(rec0 + s * a.Hkv) * mt + row;
        ml[j] = a.rec.ml[at];
#pragma unroll
        for (int i = 0; i < PER; ++i) v[j][i] = a.rec.opart[at * D + lane * PER + i];
      }
      float Mn = M;
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        if (s0 + j * kWaves >= splits) ml[j] = make_float2(kPagedNegInf, 0.0f);
        if (ml[j].y != 0.0f) Mn = fmaxf(Mn, ml[j].x);
      }
      const float keep = L == 0.0f ? 0.0f : fast_exp2(M - Mn);
      L *= keep;
#pragma unroll
      for (int i = 0; i < PER; ++i) acc[i] *= keep;
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        if (ml[j].y == 0.0f) continue;  // saw nothing
        const float w = fast_exp2(ml[j].x - Mn);
        L = fmaf(w, ml[j].y, L);
#pragma unroll
        for (int i = 0; i < PER; ++i) acc[i] = fmaf(w, v[j][i], acc[i]);
      }
      M = Mn;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) s_acc[wave][lane * PER + i] = acc[i];
    if (lane == 0) {
      s_m[wave] = M;
      s_l[wave] = L;
    }
    __syncthreads();
    if (threadIdx.x < D) {
      float Mt = kPagedNegInf, Lt = 0.0f, o = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w)
        if (s_l[w] != 0.0f) Mt = fmaxf(Mt, s_m[w]);
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        if (s_l[w] == 0.0f) continue;
        const float e = fast_exp2(s_m[w] - Mt);
        Lt = fmaf(e, s_l[w], Lt);
        o = fmaf(e, s_acc[w][threadIdx.x], o);
      }
      const int xr = d[3] + row;
      static_cast<elem*>(a.o)[((size_t)(d[2] + xr / a.G) * a.Hq + head * a.G + xr % a.G) * D +
                              threadIdx.x] = (elem)(Lt == 0.0f ? 0.0f : o / Lt);
    }
    __syncthreads();
  }
}

template <class E, bool FP8>
PagedFn pick_size(int D) {
  return D == 64 ? paged_chunk<E, FP8, 64> : paged_chunk<E, FP8, 128>;
}

PagedFn pick_chunk(bool bf16, bool fp8, int D) {
  if (bf16) return fp8 ? pick_size<ElemBF16, true>(D) : pick_size<ElemBF16, false>(D);
  return fp8 ? pick_size<ElemF16, true>(D) : pick_size<ElemF16, false>(D);
}

void (*pick_merge(bool bf16, int D))(PagedArgs, int) {
  if (bf16) return D == 64 ? paged_merge<ElemBF16, 64> : paged_merge<ElemBF16, 128>;
  return D == 64 ? paged_merge<ElemF16, 64> : paged_merge<ElemF16, 128>;
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

// Workgroups wanted of each kernel: two a CU.
int paged_target(int cu_count) { return 2 * cu_count; }

size_t region_bytes(int target, int mt, int D) {
  const size_t records = 2 * (size_t)target, groups = (size_t)target;
  return 256 + round256(groups * kDescInts * sizeof(int)) +
         round256(records * mt * sizeof(float2)) + round256(records * mt * D * sizeof(float));
}

PagedRecords region(char* base, int target, int mt, int D) {
  PagedRecords r;
  r.records = 2 * target;
  r.groups = target;
  r.head = reinterpret_cast<int*>(base);
  base += 256;
  r.desc = reinterpret_cast<int*>(base);
  base += round256((size_t)r.groups * kDescInts * sizeof(int));
  r.ml = reinterpret_cast<float2*>(base);
  base += round256((size_t)r.records * mt * sizeof(float2));
  r.opart = reinterpret_cast<float*>(base);
  (void)D;
  return r;
}

// Whether 16 keys from a multiple of 16 on always lie in one page, at offsets
// from its first key that 32 bits hold.
bool paged_aligned(const db_paged_cache& kv) {
  constexpr long long kFar = 1 << 26;
  return kv.page_size % 16 == 0 && kv.k_token_stride < kFar && kv.v_token_stride < kFar;
}

// Which kernels a call of these bounds needs.
void kernels_of(const PagedCall& c, bool* decode, bool* chunk) {
  const int most = c.max_new > 0 && c.max_new < c.T ? c.max_new : c.T;
  *decode = true;
  *chunk = (long long)most * (c.Hq / c.cache.Hkv) > kDecodeRows;
  if (*chunk && c.R == 1) *decode = false;  // one request: many rows, or few at most
}

}  // namespace

size_t paged_workspace_bytes(const PagedCall& c, int cu_count) {
  bool decode, chunk;
  kernels_of(c, &decode, &chunk);
  const int target = paged_target(cu_count), D = c.cache.D;
  return (decode ? region_bytes(target, kDecodeRows, D) : 0) +
         (chunk ? region_bytes(target, kChunkRows, D) : 0);
}

hipError_t launch_paged_attention(const PagedCall& c, int cu_count, void* ws, hipStream_t stream) {
  const db_paged_cache& kv = c.cache;
  const bool fp8 = kv.dtype == DB_DTYPE_FP8_E4M3;
  const int target = paged_target(cu_count), D = kv.D;
  PagedArgs a;
  a.q = c.q;
  a.o = c.o;
  a.k = kv.k;
  a.v = kv.v;
  a.k_scale = kv.k_scale;
  a.v_scale = kv.v_scale;
  a.table = c.table;
  a.q_start = c.q_start;
  a.kv_len = c.kv_len;
  a.q_token = c.q_token;
  a.q_head = c.q_head;
  a.kp = kv.k_page_stride;
  a.kh = kv.k_head_stride;
  a.kt = kv.k_token_stride;
  a.vp = kv.v_page_stride;
  a.vh = kv.v_head_stride;
  a.vt = kv.v_token_stride;
  a.table_row = c.table_row;
  a.T = c.T;
  a.R = c.R;
  a.Hq = c.Hq;
  a.Hkv = kv.Hkv;
  a.G = c.Hq / kv.Hkv;
  a.pages = kv.pages;
  a.page = kv.page_size;
  a.width = c.width;
  int s = 0;
  while ((1ll << s) < kv.page_size) ++s;
  a.page_magic = s == 0 ? 0u
                        : (unsigned)(((1ull << (31 + s)) + kv.page_size - 1) / kv.page_size);
  a.page_shift = s == 0 ? 0u : (unsigned)(s - 1);
  a.causal = c.causal;
  a.window = c.window;
  a.scale_log2 = c.scale * 1.4426950408889634f;
  a.target = target;

  bool decode, chunk;
  kernels_of(c, &decode, &chunk);
  char* base = static_cast<char*>(ws);
  auto run = [&](PagedFn fn, int part, int mt, int min_tiles) {
    a.part = part;
    a.min_tiles = min_tiles;
    a.rec = region(base, target, mt, D);
    base += region_bytes(target, mt, D);
    // Row tiles of every request at most, and the splits beyond one each.
    const long long tiles = (long long)c.T * a.G / mt + c.R;
    const long long grid = tiles * a.Hkv + target;
    hipLaunchKernelGGL(fn, dim3((unsigned)(grid < 65536 ? grid : 65536)), dim3(kPagedThreads), 0,
                       stream, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(pick_merge(c.bf16, D), dim3(2048), dim3(kPagedThreads), 0, stream, a, mt);
    return hipGetLastError();
  };
  hipError_t e = hipSuccess;
  if (decode)
    e = run(paged_decode_fn(c.bf16, fp8, D, paged_aligned(kv)), chunk ? 1 : 0, kDecodeRows,
            paged_decode_min_tiles(fp8, D));
  if (e == hipSuccess && chunk)
    e = run(pick_chunk(c.bf16, fp8, D), decode ? 2 : 0, kChunkRows, 8);
  return e;
}

}  // namespace dbk
