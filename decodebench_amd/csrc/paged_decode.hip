// paged_decode.hip -- paged attention of few rows (single tokens, drafts).
//
// A workgroup of four waves owns one (request, KV head, row tile of 16 rows)
// and one split of the keys; wave w takes the 16-key tiles w, w + 4, ... of
// the split.  Bound by HBM: every key and value is read once per row tile, and
// rows beyond the few that a request has cost nothing but idle MFMA columns.
//
//  * Scores: v_mfma_f32_16x16x32, A = 16 keys straight from the cache to
//    registers (lane (g4, n16) holds 16-byte chunks g4, g4 + 4, ... of key
//    n16), B = the rows.  An e4m3 chunk is 16 elements, so its two halves are
//    two MFMA steps; the rows are loaded in the same order.
//  * Softmax with running maximum and sum, base 2, fp32, on the four keys that
//    each lane holds.  Probabilities are rounded to the element type for the
//    product and summed as rounded, so numerator and denominator agree.
//  * P.V: O^T = V^T P^T on 16x16x16 MFMAs, V^T through the wave's copy of the
//    tile in LDS and the transposing read ds_read_b64_tr_b16.
//  * A lane looks up the page of key n16 of a tile (the lookups run one tile
//    ahead of the loads); rows of V take theirs from that lane.
//  * Masked keys: scores by selection, so no Inf or NaN of a masked key counts;
//    a tile that some row sees only in part is searched for an Inf or NaN
//    among its values, and one that has any is added key by key.
#include "paged_attn.h"

namespace dbk {

namespace {

constexpr int kWaves = kPagedThreads / kWave;
constexpr int MT = kDecodeRows, KT = kDecodeKeys;

template <class E, bool FP8, int D>
__global__ __launch_bounds__(kPagedThreads) void paged_decode(PagedArgs a) {
  typedef typename E::type elem;
  typedef typename E::vec8 vec8;
  typedef typename E::vec4 vec4;
  constexpr int CB = FP8 ? 1 : 2;          // bytes of a cache element
  constexpr int NK = D * CB / 64;          // 16-byte loads of K a lane (16 keys, 4 lanes each)
  constexpr int STEPS = D / 32;            // MFMA steps of a score
  constexpr int LPR = D * CB / 16;         // lanes per row of V
  constexpr int RPI = kWave / LPR;         // rows of V a load instruction
  constexpr int NV = KT / RPI;
  constexpr int VS = D + 16;               // row stride of the V tile in LDS (elements)
  constexpr int NB = D / 16;
  constexpr size_t kRegion = sizeof(float) * MT * D;
  static_assert(kRegion >= sizeof(elem) * KT * VS, "a V tile fits the wave's outputs");

  __shared__ PagedShared s_sched;
  __shared__ __align__(16) char s_region[kWaves][kRegion];
  __shared__ float s_m[MT][kWaves], s_l[MT][kWaves];

  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int n16 = lane & 15, g4 = lane >> 4;
  elem* const vbuf = reinterpret_cast<elem*>(s_region[wave]);

  PagedSchedule<MT, KT> schedule(a, s_sched);
  PagedWork wk;
  while (schedule.next(wk)) {
    const PagedRequest& rq = wk.req;
    int t_begin, t_end;
    paged_range<MT, KT>(a, wk, t_begin, t_end);
    t_begin = __builtin_amdgcn_readfirstlane(t_begin);
    t_end = __builtin_amdgcn_readfirstlane(t_end);
    paged_describe(a, wk, MT);
    const int limit = __builtin_amdgcn_readfirstlane(paged_limit(a, rq.len));

    // This lane's row (column n16 of the products) and the keys it sees.
    const int rows = (int)min((long long)rq.n * a.G - (long long)wk.tile * MT, (long long)MT);
    const int x = wk.tile * MT + min(n16, rows - 1);
    const int token = x / a.G, qhead = wk.head * a.G + x % a.G;
    const int pos = rq.len - rq.n + token;
    const int khi = a.causal ? min(limit, pos + 1) : limit;
    const int klo = a.window > 0 ? max(pos - a.window + 1, 0) : 0;
    // Keys that every row sees.
    int all_lo = klo, all_hi = khi;
    for (int d = 1; d < 16; d <<= 1) {
      all_lo = max(all_lo, __shfl_xor(all_lo, d));
      all_hi = min(all_hi, __shfl_xor(all_hi, d));
    }
    all_lo = __builtin_amdgcn_readfirstlane(all_lo);
    all_hi = __builtin_amdgcn_readfirstlane(all_hi);

    vec8 qop[STEPS];
    {
      const elem* qp = static_cast<const elem*>(a.q) + (rq.tok0 + token) * a.q_token +
                       qhead * a.q_head;
#pragma unroll
      for (int t = 0; t < STEPS; ++t) {
        const int at = FP8 ? 16 * (g4 + 4 * (t >> 1)) + 8 * (t & 1) : 8 * (g4 + 4 * t);
        qop[t] = __builtin_bit_cast(vec8, ld16(qp + at));
      }
    }
    const float scale = a.scale_log2 * (FP8 ? a.k_scale[wk.head] : 1.0f);
    const char* const kbase = static_cast<const char*>(a.k) + wk.head * a.kh * CB;
    const char* const vbase = static_cast<const char*>(a.v) + wk.head * a.vh * CB;
    const int* const trow = a.table + wk.r * a.table_row;

    const int first = t_begin + wave;
    const int nt = first < t_end ? (t_end - first + kWaves - 1) / kWaves : 0;
    auto tile_of = [&](int k) { return first + kWaves * k; };

    // Page of key n16 of the wave's k-th tile, -1 where there is none.
    auto lookup = [&](int k) {
      const int key = tile_of(k) * KT + n16;
      if (k >= nt || key >= limit) return -1;
      const int p = trow[page_of(a, key)];
      return (unsigned)p < (unsigned)a.pages ? p : -1;
    };

    f4 o[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) o[b] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    float m_run = kPagedNegInf, l_run = 0.0f;

    // Absent keys read row 0 of page 0: valid memory, never counted.
    auto load_tile = [&](u4 (&kt)[NK], u4 (&vt)[NV], int tile, int pg) {
      {
        const int key = tile * KT + n16;
        const int off = pg < 0 ? 0 : key - page_of(a, key) * a.page;
        const char* p = kbase + (max(pg, 0) * a.kp + off * a.kt) * CB;
#pragma unroll
        for (int t = 0; t < NK; ++t) kt[t] = ld_stream(p + (g4 + 4 * t) * 16);
      }
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int row = j * RPI + lane / LPR, key = tile * KT + row;
        const int pr = __shfl(pg, row);
        const int off = pr < 0 ? 0 : key - page_of(a, key) * a.page;
        vt[j] = ld_stream(vbase + (max(pr, 0) * a.vp + off * a.vt) * CB + (lane % LPR) * 16);
      }
    };

    auto compute_tile = [&](const u4 (&kt)[NK], u4 (&vt)[NV], int tile, int pg) {
      const int key0 = tile * KT;
      const unsigned there = (unsigned)__ballot(pg >= 0) & 0xFFFFu;
      const bool partial = there != 0xFFFFu || key0 < all_lo || key0 + KT > all_hi;
      bool odd = false;  // a partly seen tile with an Inf or NaN among its values
      if (partial) {
        bool bad = false;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          if (!((there >> (j * RPI + lane / LPR)) & 1)) vt[j] = u4{0, 0, 0, 0};
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            if constexpr (FP8) {
              const unsigned w = vt[j][c] & 0x7F7F7F7Fu;  // NaN: seven bits set (no Inf in e4m3)
              bad = bad || (w & 0xFFu) == 0x7Fu || ((w >> 8) & 0xFFu) == 0x7Fu ||
                    ((w >> 16) & 0xFFu) == 0x7Fu || (w >> 24) == 0x7Fu;
            } else {
              bad = bad || pair_nonfinite<E>(vt[j][c]);
            }
          }
        }
        odd = __any(bad);
      }
      // the tile's values, rows in key order
      wave_lds_order();
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        elem* row = vbuf + (j * RPI + lane / LPR) * VS + (lane % LPR) * (16 / CB);
        if constexpr (FP8) {
          const u2 w0 = E::widen(vt[j][0]), w1 = E::widen(vt[j][1]);
          const u2 w2 = E::widen(vt[j][2]), w3 = E::widen(vt[j][3]);
          *reinterpret_cast<u4*>(row) = u4{w0[0], w0[1], w1[0], w1[1]};
          *reinterpret_cast<u4*>(row + 8) = u4{w2[0], w2[1], w3[0], w3[1]};
        } else {
          *reinterpret_cast<u4*>(row) = vt[j];
        }
      }
      wave_lds_order();

      // s[j]: score of key key0 + 4 g4 + j and row n16
      f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int t = 0; t < NK; ++t) {
        if constexpr (FP8) {
          const u2 w0 = E::widen(kt[t][0]), w1 = E::widen(kt[t][1]);
          const u2 w2 = E::widen(kt[t][2]), w3 = E::widen(kt[t][3]);
          acc = E::mfma16(__builtin_bit_cast(vec8, u4{w0[0], w0[1], w1[0], w1[1]}), qop[2 * t], acc);
          acc = E::mfma16(__builtin_bit_cast(vec8, u4{w2[0], w2[1], w3[0], w3[1]}), qop[2 * t + 1],
                          acc);
        } else {
          acc = E::mfma16(__builtin_bit_cast(vec8, kt[t]), qop[t], acc);
        }
      }
      float s[4];
      bool sees[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = key0 + 4 * g4 + j;
        sees[j] = key >= klo && key < khi && ((there >> (4 * g4 + j)) & 1);
        s[j] = sees[j] ? acc[j] * scale : kPagedNegInf;
      }
      float tmax = fmaxf(fmaxf(s[0], s[1]), fmaxf(s[2], s[3]));
      tmax = fmaxf(tmax, __shfl_xor(tmax, 16));
      tmax = fmaxf(tmax, __shfl_xor(tmax, 32));
      const float m_new = fmaxf(m_run, tmax);
      // A row that has seen nothing yet keeps -inf; its exponents use 0.
      const float m_use = m_new == kPagedNegInf ? 0.0f : m_new;
      const float alpha = fast_exp2(m_run - m_use);
      vec4 pb;
#pragma unroll
      for (int j = 0; j < 4; ++j) pb[j] = (elem)fast_exp2(s[j] - m_use);
      l_run = l_run * alpha + (((float)pb[0] + (float)pb[1]) + ((float)pb[2] + (float)pb[3]));
      m_run = m_new;
      if (__any(alpha != 1.0f)) {
#pragma unroll
        for (int b = 0; b < NB; ++b) o[b] *= alpha;
      }
      if (odd) {
        // Key by key: only keys that the row sees are added.
#pragma unroll 1
        for (int g = 0; g < 4; ++g) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float p = __shfl((float)pb[j], 16 * g + n16);
            const bool sp = __shfl((int)sees[j], 16 * g + n16) != 0;
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float v = (float)vbuf[(4 * g + j) * VS + 16 * b + 4 * g4 + i];
                o[b][i] += sp ? p * v : 0.0f;
              }
          }
        }
      } else {
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const vec4 va = __builtin_bit_cast(
              vec4, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (__attribute__((address_space(3))) s4*)(
                            vbuf + (4 * g4 + (n16 >> 2)) * VS + 16 * b + 4 * (n16 & 3))));
          o[b] = E::mfma16k16(va, pb, o[b]);
        }
      }
    };

    if (nt > 0) {
      u4 ka[NK], va[NV], kb[NK], vb[NV];
      int pa = lookup(0), pb = lookup(1);
      load_tile(ka, va, tile_of(0), pa);
      for (int k = 0; k < nt; k += 2) {
        int pn = lookup(k + 2);
        if (k + 1 < nt) load_tile(kb, vb, tile_of(k + 1), pb);
        compute_tile(ka, va, tile_of(k), pa);
        if (k + 1 >= nt) break;
        pa = pn;
        pn = lookup(k + 3);
        if (k + 2 < nt) load_tile(ka, va, tile_of(k + 2), pa);
        compute_tile(kb, vb, tile_of(k + 1), pb);
        pb = pn;
      }
    }

    // ---- the waves' rows meet in LDS ---------------------------------------
    float l_tot = l_run + __shfl_xor(l_run, 16);
    l_tot += __shfl_xor(l_tot, 32);
    wave_lds_order();
    float* const so = reinterpret_cast<float*>(s_region[wave]);
#pragma unroll
    for (int b = 0; b < NB; ++b)
      *reinterpret_cast<f4*>(so + n16 * D + 16 * b + 4 * g4) = o[b];
    if (lane < MT) {
      s_m[lane][wave] = m_run;
      s_l[lane][wave] = l_tot;
    }
    __syncthreads();
    const float vscale = FP8 ? a.v_scale[wk.head] : 1.0f;
    const int rec = wk.rec < 0 ? -1 : wk.rec + wk.split * a.Hkv;
    for (int idx = threadIdx.x; idx < rows * (D / 4); idx += kPagedThreads) {
      const int row = idx / (D / 4), d4 = idx % (D / 4);
      float M = kPagedNegInf;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) M = fmaxf(M, s_m[row][w]);
      f4 ow = {0.0f, 0.0f, 0.0f, 0.0f};
      float lw = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) {
        if (s_l[row][w] == 0.0f) continue;  // saw nothing
        const float e = fast_exp2(s_m[row][w] - M);
        ow += e * *reinterpret_cast<const f4*>(reinterpret_cast<float*>(s_region[w]) + row * D +
                                               4 * d4);
        lw += e * s_l[row][w];
      }
      ow *= vscale;
      if (rec < 0) {
        const int xr = wk.tile * MT + row;
        elem* op = static_cast<elem*>(a.o) +
                   ((size_t)(rq.tok0 + xr / a.G) * a.Hq + wk.head * a.G + xr % a.G) * D + 4 * d4;
        const float inv = lw == 0.0f ? 0.0f : 1.0f / lw;
        vec4 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = (elem)(ow[i] * inv);
        *reinterpret_cast<vec4*>(op) = r;
      } else if (rec < a.rec.records) {
        const size_t at = (size_t)rec * MT + row;
        *reinterpret_cast<f4*>(a.rec.opart + at * D + 4 * d4) = ow;
        if (d4 == 0) a.rec.ml[at] = make_float2(M, lw);
      }
    }
  }
}

template <class E, bool FP8>
PagedFn pick_size(int D) {
  return D == 64 ? paged_decode<E, FP8, 64> : paged_decode<E, FP8, 128>;
}

}  // namespace

PagedFn paged_decode_fn(bool bf16, bool fp8, int D) {
  if (bf16) return fp8 ? pick_size<ElemBF16, true>(D) : pick_size<ElemBF16, false>(D);
  return fp8 ? pick_size<ElemF16, true>(D) : pick_size<ElemF16, false>(D);
}

}  // namespace dbk
