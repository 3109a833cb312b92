// paged_chunk.hip -- paged attention of many rows: chunks of a prompt, drafts.
//
// A workgroup owns one (request, KV head, row tile) and one split of the keys; its
// waves have 32 rows each and share 64-key tiles of K and V in LDS.  Row tiles
// have 256 rows (eight waves) or, where no request has more, 64: four waves then,
// two (KP) to each 32 rows, each with half of every tile's keys, joined through
// LDS at the end (with one wave to 32 rows 16 drafts of 5 tokens took 17.9 us
// instead of 15.6).  Two such workgroups fit a CU, so the registers of a wave are
// held to 256 (300 of them and one workgroup a CU: 16.6).  A tile of 256 rows of 128 takes a CU about
// 4200 clocks, in which each SIMD has 2050 of MFMAs and 1900 of softmax, and the
// LDS 2300 (256 KB of operands for the eight waves, 32 KB written).  2048 tokens
// of 32 heads of 128, the last of 8192: 0.28 ms, 0.86 PFLOP/s, where a large
// library matrix product reaches 1.13; 12% of that is CUs whose row tiles see
// fewer keys than the longest (2048 tokens from nothing, where half is: 73 us).  Two schedules that run the MFMAs beside
// the softmax (the waves of a SIMD half a tile apart; a wave's own scores, softmax
// and values woven together) took 2% less for twice the code; 64 rows a wave,
// which halve the LDS reads, spill registers and took 1.6 times as long.
//
//  * S^T = K Q^T on v_mfma_f32_32x32x16: a lane holds scores of one row (its
//    column), 32 of the tile's 64 keys, the other half in lane ^ 32, so a
//    row's maximum and sum are nearly all in-lane work.
//  * The rounded probabilities are the B operand of O^T = V^T P^T as they lie:
//    accumulator registers 8 s .. 8 s + 7 of lane half h are keys 16 s + 4 h +
//    0..3 and 16 s + 8 + 4 h + 0..3, and V^T is read from LDS in that order by
//    two transposing reads (ds_read_b64_tr_b16) per operand.
//  * Exponents are taken against a reference that moves only when a row's
//    maximum leaves it by more than 2^12, to 2^8 below that maximum: the output
//    is rescaled a few times a row instead of at most tiles, and small
//    probabilities stay clear of fp16's subnormals.
//  * Two tiles in LDS: while tile t is computed, tile t + 1 goes from registers
//    to the other half and tile t + 2 is on its way to registers; one barrier a
//    tile.
//  * Pages of a multiple of 16 tokens (ALIGNED): lane 4 t + g holds where the
//    g-th 16 keys of the t-th of 16 tiles are, and the table entries of the
//    next 16 tiles, so an address is two scalars read from a lane.  Any other
//    page size: lane i looks up the page of key i of a tile, one tile ahead.
//  * A wave skips tiles that none of its rows sees, and masks only tiles that
//    some row sees in part (an Inf or NaN among such a tile's values as in
//    paged_decode: left out of the product, added to the rows that see it).
#include <mutex>

#include "paged_attn.h"

namespace dbk {

namespace {

constexpr int KT = kChunkKeys;
constexpr int kHold = kWave / (KT / 16);  // tiles whose places the lanes hold

// Exponent references: a row's maximum may be kAbove over its reference, which
// is set kBelow under the maximum.
constexpr float kAbove = 12.0f, kBelow = 8.0f;

template <class E, bool FP8, int D, bool ALIGNED, int NW, int KP>
__global__ __launch_bounds__(NW * kWave, 2) void paged_chunk(PagedArgs a) {
  typedef typename E::type elem;
  typedef typename E::vec8 vec8;
  constexpr int MT = 32 * NW / KP;
  constexpr int WK = KT / KP;                      // keys of a tile that a wave takes
  constexpr int CB = FP8 ? 1 : 2;
  constexpr int RW = KT / NW;                      // rows of a tile that a wave loads
  constexpr int LPR = D * CB / 16;                 // lanes per row
  constexpr int RPI = kWave / LPR;                 // rows a load instruction
  constexpr int NL = RW > RPI ? RW / RPI : 1;      // loads of K (and of V) a lane
  // Row strides in LDS (elements): 16 rows of a K read, and the four rows of 64
  // bytes that half a wave takes in a transposing read of V, lie in different banks.
  constexpr int KS = D + 8, VS = D + 32;
  constexpr int QSTEPS = D / 16, NB = D / 32;

  __shared__ __align__(16) elem s_k[2][KT * KS];
  __shared__ __align__(16) elem s_v[2][KT * VS];
  __shared__ int s_odd[2];  // tile + 1 of a tile with an Inf or NaN left out

  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int n32 = lane & 31, half = lane >> 5;
  const int block = wave % (NW / KP), kpart = wave / (NW / KP) * WK;  // rows and keys of the wave

  PagedSchedule<MT, KT> schedule(a);
  PagedWork wk;
  if (!schedule.find(wk)) return;
  if (threadIdx.x < 2) s_odd[threadIdx.x] = 0;
  __syncthreads();
  {
    const PagedRequest& rq = wk.req;
    int t_begin, t_end;
    paged_range<MT, KT>(a, wk, t_begin, t_end);
    paged_describe(a, wk, MT);
    const int limit = paged_limit(a, rq.len);

    const char* const kbase = static_cast<const char*>(a.k) + wk.head * a.kh * CB;
    const char* const vbase = static_cast<const char*>(a.v) + wk.head * a.vh * CB;
    const int* const trow = a.table + wk.r * a.table_row;

    // ---- where the keys are ------------------------------------------------
    // ALIGNED: byte offsets of this lane's 16 keys and values (of the tiles
    // held .. held + 15) and a bit for each that has a page; `ahead` is the
    // table entry for the 16 tiles after these.
    long long koff = 0, voff = 0;
    unsigned long long has = 0;
    int held = t_begin, ahead = -1;
    auto entry = [&](int tile) {  // of this lane's 16 keys, 16 tiles from `tile` on
      const int key = (tile + lane / 4) * KT + 16 * (lane % 4);
      return tile + lane / 4 < t_end && key < limit ? trow[page_of(a, key)] : -1;
    };
    auto hold = [&](int tile) {
      held = tile;
      const int p = ahead;
      ahead = entry(tile + kHold);
      const int key = (tile + lane / 4) * KT + 16 * (lane % 4);
      const bool ok = (unsigned)p < (unsigned)a.pages;
      const int off = ok ? key - page_of(a, key) * a.page : 0;
      koff = ok ? (p * a.kp + off * a.kt) * CB : 0;
      voff = ok ? (p * a.vp + off * a.vt) * CB : 0;
      has = __ballot(ok);
    };
    // Otherwise: page of key `lane` of a tile, -1 where there is none.
    auto lookup = [&](int tile) {
      const int key = tile * KT + lane;
      if (tile >= t_end || key >= limit) return -1;
      const int p = trow[page_of(a, key)];
      return (unsigned)p < (unsigned)a.pages ? p : -1;
    };
    int pg = -1;
    if constexpr (ALIGNED)
      ahead = entry(t_begin);
    else
      pg = lookup(t_begin);

    // This lane's row and the keys it sees; rows past the last one see none.
    const long long left = (long long)rq.n * a.G - (long long)wk.tile * MT;
    const int rows = (int)min(left, (long long)MT);
    const int lrow = block * 32 + n32;
    const bool live = lrow < rows;
    const int x = wk.tile * MT + min(lrow, rows - 1);
    const int token = x / a.G, qhead = wk.head * a.G + x % a.G;
    vec8 qop[QSTEPS];
    {
      const elem* qp = static_cast<const elem*>(a.q) + (rq.tok0 + token) * a.q_token +
                       qhead * a.q_head + 8 * half;
#pragma unroll
      for (int t = 0; t < QSTEPS; ++t) qop[t] = __builtin_bit_cast(vec8, ld16(qp + 16 * t));
    }
    const int past = rq.len - rq.n;
    const int khi = !live ? 0 : a.causal ? min(limit, past + token + 1) : limit;
    const int klo = !live ? 0x7FFFFFFF : first_seen(a, past + token);
    // Keys that every row of the workgroup sees (wg_), that every live row of
    // the wave sees (all_) and that any of them sees (any_), from its first and
    // last live row (none: nothing at all).
    const int wg_hi = a.causal ? min(limit, past + (wk.tile * MT) / a.G + 1) : limit;
    const int wg_lo = first_seen(a, past + (wk.tile * MT + rows - 1) / a.G);
    const bool any = block * 32 < rows;
    const int i0 = (wk.tile * MT + min(block * 32, rows - 1)) / a.G;
    const int i1 = (wk.tile * MT + min(block * 32 + 31, rows - 1)) / a.G;
    const int all_hi = a.causal ? min(limit, past + i0 + 1) : limit;
    const int any_hi = !any ? 0 : a.causal ? min(limit, past + i1 + 1) : limit;
    const int all_lo = first_seen(a, past + i1);
    const int any_lo = first_seen(a, past + i0);
    const float scale = a.scale_log2 * (FP8 ? a.k_scale[wk.head] : 1.0f);

    // ---- tiles to registers and to LDS -------------------------------------
    const int row0 = wave * RW;  // of the tile, this wave's first
    const int lrow_l = min(lane / LPR, RW - 1), lcol = (lane % LPR) * 16;
    const unsigned lane_k = (unsigned)((row0 % 16 + lrow_l) * (int)a.kt * CB + lcol);
    const unsigned lane_v = (unsigned)((row0 % 16 + lrow_l) * (int)a.vt * CB + lcol);
    // Absent keys read rows of page 0: valid memory, zero in LDS.
    auto load_tile = [&](u4 (&kt)[NL], u4 (&vt)[NL], int tile) {
      if constexpr (ALIGNED) {
        if (tile >= held + kHold) hold(tile);
#pragma unroll
        for (int j = 0; j < NL; ++j) {
          const int g = (row0 + j * RPI) / 16;  // row0 % 16 + j RPI runs on from its group
          const int in = (row0 % 16 + j * RPI) / 16 * 16;
          const long long ko = lane_i64(koff, (tile - held) * 4 + g);
          const long long vo = lane_i64(voff, (tile - held) * 4 + g);
          kt[j] = ld16(kbase + ko + (j * RPI - in) * a.kt * CB + lane_k);
          vt[j] = ld16(vbase + vo + (j * RPI - in) * a.vt * CB + lane_v);
        }
      } else {
#pragma unroll
        for (int j = 0; j < NL; ++j) {
          const int row = row0 + j * RPI + lrow_l, key = tile * KT + row;
          const int pr = __shfl(pg, row), page = max(pr, 0);
          const int off = pr < 0 ? 0 : key - page_of(a, key) * a.page;
          kt[j] = ld16(kbase + (page * a.kp + off * a.kt) * CB + lcol);
          vt[j] = ld16(vbase + (page * a.vp + off * a.vt) * CB + lcol);
        }
      }
    };
    // Keys of a tile that are in the cache and below the request's end.
    auto present = [&](int tile) -> unsigned long long {
      if constexpr (ALIGNED) {
        const unsigned b = (unsigned)(has >> ((tile - held) * 4)) & 15u;
        unsigned long long there = 0;
#pragma unroll
        for (int g = 0; g < 4; ++g) there |= (b >> g) & 1 ? 0xFFFFull << (16 * g) : 0ull;
        return there & below(limit - tile * KT);
      } else {
        return __ballot(pg >= 0);
      }
    };
    // Widens a chunk of e4m3; otherwise the chunk itself.
    auto widen = [&](u4 w, u4 (&to)[2 / CB]) {
      if constexpr (FP8) {
        const u2 w0 = E::widen(w[0]), w1 = E::widen(w[1]);
        const u2 w2 = E::widen(w[2]), w3 = E::widen(w[3]);
        to[0] = u4{w0[0], w0[1], w1[0], w1[1]};
        to[1] = u4{w2[0], w2[1], w3[0], w3[1]};
      } else {
        to[0] = w;
      }
    };
    // A tile to LDS: zeros for keys that are not there, and, in a tile that
    // some row of the workgroup sees in part, for values that are Inf or NaN:
    // a hidden key's probability is zero, but zero times those is not.
    auto store_tile = [&](u4 (&kt)[NL], u4 (&vt)[NL], int tile, unsigned long long there, int buf) {
      const bool partial = there != ~0ull || tile * KT < wg_lo || tile * KT + KT > wg_hi;
      bool odd = false;
#pragma unroll
      for (int j = 0; j < NL; ++j) {
        const int row = row0 + j * RPI + lrow_l, c = (lane % LPR) * (16 / CB);
        u4 kw[2 / CB], vw[2 / CB];
        widen(kt[j], kw);
        widen(vt[j], vw);
        if (partial) {
          const bool ok = (there >> row) & 1;
#pragma unroll
          for (int h = 0; h < 2 / CB; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const unsigned v = vw[h][i];
              const bool lo = (v & E::kExp) == E::kExp, hi = ((v >> 16) & E::kExp) == E::kExp;
              odd = odd || (ok && (lo || hi));
              vw[h][i] = ok ? v & ((lo ? 0u : 0x0000FFFFu) | (hi ? 0u : 0xFFFF0000u)) : 0u;
              kw[h][i] = ok ? kw[h][i] : 0u;
            }
        }
#pragma unroll
        for (int h = 0; h < 2 / CB; ++h) {
          *reinterpret_cast<u4*>(s_k[buf] + row * KS + c + 8 * h) = kw[h];
          *reinterpret_cast<u4*>(s_v[buf] + row * VS + c + 8 * h) = vw[h];
        }
      }
      if (odd) s_odd[buf] = tile + 1;
    };

    f16v o[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[b][i] = 0.0f;
    float m_ref = kPagedNegInf, l_run = 0.0f;  // l: of this lane's keys

    // V^T of 16 keys (step t) and 32 dims (block b): the A operand.
    auto read_v = [&](const elem* vb0, int t, int b) {
      const elem* at = vb0 + 16 * t * VS + 32 * b;
      const u2 lo = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                               (__attribute__((address_space(3))) s4*)(at)));
      const u2 hi = __builtin_bit_cast(u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                                               (__attribute__((address_space(3))) s4*)(at + 8 * VS)));
      return u4{lo[0], lo[1], hi[0], hi[1]};
    };

    // Adds the Infs and NaNs that store_tile left out to the rows that see them
    // (values read again from the cache; a rare path, kept small).
    auto add_odd = [&](int key0, unsigned long long sees) {
#pragma unroll 1
      for (int kk = 0; kk < KT; ++kk) {
        if (!__any((sees >> kk) & 1)) continue;  // also keys without a page
        const int key = key0 + kk, at = page_of(a, key);
        const char* row = vbase + (trow[at] * a.vp + (key - at * a.page) * a.vt) * CB;
        const bool ok = (sees >> kk) & 1;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const char* four = row + (32 * b + 8 * c + 4 * half) * CB;
            const u2 w = FP8 ? E::widen(*reinterpret_cast<const unsigned*>(four))
                             : *reinterpret_cast<const u2*>(four);
            const typename E::vec4 v = __builtin_bit_cast(typename E::vec4, w);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              o[b][4 * c + i] += ok && !__builtin_isfinite((float)v[i]) ? (float)v[i] : 0.0f;
            __builtin_amdgcn_sched_barrier(0);
          }
      }
    };

    auto compute_tile = [&](int tile, unsigned long long there, int buf) {
      const int key0 = tile * KT, lo = key0 + kpart, hi = lo + WK;  // lo .. hi - 1: the wave's
      if (lo >= any_hi || hi <= any_lo) return;
      const elem* const kb0 = s_k[buf] + (kpart + n32) * KS + 8 * half;
      const elem* const vb0 = s_v[buf] + (kpart + 4 * half + ((lane & 15) >> 2)) * VS +
                              16 * ((lane >> 4) & 1) + 4 * (lane & 3);
      f16v s[WK / 32];
#pragma unroll
      for (int kb = 0; kb < WK / 32; ++kb) {
#pragma unroll
        for (int i = 0; i < 16; ++i) s[kb][i] = 0.0f;
#pragma unroll
        for (int t = 0; t < QSTEPS; ++t)
          s[kb] = E::mfma32(__builtin_bit_cast(vec8, ld16(kb0 + 32 * kb * KS + 16 * t)), qop[t],
                            s[kb]);
      }
      // Keys of the tile that this lane's row sees, a bit each.  (Bits tested at
      // fixed places of words shifted by the lane's half: places that depend on
      // the lane were hoisted out of the loop, 96 registers of them.)
      const unsigned long long mine = below(WK) << kpart;
      unsigned long long sees = mine;
      if ((there & mine) != mine || lo < all_lo || hi > all_hi) {
        sees = there & mine & below(khi - key0) & ~below(klo - key0);
#pragma unroll
        for (int kb = 0; kb < WK / 32; ++kb) {
          const unsigned w = (unsigned)(sees >> (kpart + 32 * kb)) >> (4 * half);
#pragma unroll
          for (int i = 0; i < 16; ++i)
            s[kb][i] = w & (1u << (8 * (i >> 2) + (i & 3))) ? s[kb][i] : kPagedNegInf;
        }
      }
      float tmax = s[0][0];
#pragma unroll
      for (int kb = 0; kb < WK / 32; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) tmax = fmaxf(tmax, s[kb][i]);
      tmax = max_xor32(tmax) * scale;
      if (__any(tmax > m_ref + kAbove)) {
        const float m_new = fmaxf(m_ref, tmax - kBelow);
        const float alpha = m_ref == kPagedNegInf ? 0.0f : fast_exp2(m_ref - m_new);
        l_run *= alpha;
#pragma unroll
        for (int b = 0; b < NB; ++b) o[b] *= alpha;
        m_ref = m_new;
      }
      // A row that has seen nothing yet keeps -inf; its exponents use 0.
      const float m_use = m_ref == kPagedNegInf ? 0.0f : m_ref;
      // Probabilities are rounded to the element type for the product with V, half
      // a step each that the product averages over a row's keys; their sum is of
      // the fp32 values.
      vec8 p[WK / 16];
      float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int kb = 0; kb < WK / 32; ++kb)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float e = fast_exp2(fmaf(s[kb][i], scale, -m_use));
          sum[i & 3] += e;
          p[2 * kb + (i >> 3)][i & 7] = (elem)e;
        }
      l_run += (sum[0] + sum[1]) + (sum[2] + sum[3]);
#pragma unroll
      for (int t = 0; t < WK / 16; ++t)
#pragma unroll
        for (int b = 0; b < NB; ++b)
          o[b] = E::mfma32(__builtin_bit_cast(vec8, read_v(vb0, t, b)), p[t], o[b]);
      if ((there != ~0ull || key0 < wg_lo || key0 + KT > wg_hi) && s_odd[buf] == tile + 1)
        add_odd(key0, sees);
    };

    // Between barriers: tile t is read, tile t + 1 written, tile t + 2 loaded.
    if (t_begin < t_end) {
      u4 kt[NL], vt[NL];
      if constexpr (ALIGNED) hold(t_begin);
      load_tile(kt, vt, t_begin);
      unsigned long long there = present(t_begin), next = 0;
      store_tile(kt, vt, t_begin, there, 0);
      if (t_begin + 1 < t_end) {
        if constexpr (!ALIGNED) pg = lookup(t_begin + 1);
        load_tile(kt, vt, t_begin + 1);
        next = present(t_begin + 1);
        if constexpr (!ALIGNED) pg = lookup(t_begin + 2);
      }
      __syncthreads();
      for (int tile = t_begin; tile < t_end; ++tile) {
        const int buf = (tile - t_begin) & 1;
        const unsigned long long now = there;
        if (tile + 1 < t_end) {
          there = next;
          store_tile(kt, vt, tile + 1, there, buf ^ 1);
          if (tile + 2 < t_end) {
            load_tile(kt, vt, tile + 2);
            next = present(tile + 2);
            if constexpr (!ALIGNED) pg = lookup(tile + 3);
          }
        }
        compute_tile(tile, now, buf);
        __syncthreads();
      }
    }

    // ---- outputs -----------------------------------------------------------
    float l = l_run + __shfl_xor(l_run, 32);
    if constexpr (KP == 2) {  // the other keys' waves hand over what they have, through LDS
      constexpr int OS = D + 4;  // floats; rows in different banks
      static_assert(sizeof(s_k) >= sizeof(float) * MT * OS, "the keys' tiles hold the outputs");
      float* const so = reinterpret_cast<float*>(s_k) + (block * 32 + n32) * OS + 4 * half;
      float2* const sml = reinterpret_cast<float2*>(s_v) + block * 32 + n32;
      if (kpart != 0) {
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int c = 0; c < 4; ++c)
            *reinterpret_cast<f4*>(so + 32 * b + 8 * c) =
                f4{o[b][4 * c], o[b][4 * c + 1], o[b][4 * c + 2], o[b][4 * c + 3]};
        if (half == 0) *sml = make_float2(m_ref, l);
      }
      __syncthreads();
      if (kpart != 0) return;
      const float2 ml = *sml;
      if (ml.y != 0.0f) {  // else: saw nothing
        const float m_new = l != 0.0f ? fmaxf(m_ref, ml.x) : ml.x;
        const float w0 = l != 0.0f ? fast_exp2(m_ref - m_new) : 0.0f, w1 = fast_exp2(ml.x - m_new);
        l = fmaf(l, w0, ml.y * w1);
        m_ref = m_new;
#pragma unroll
        for (int b = 0; b < NB; ++b)
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            const f4 v = *reinterpret_cast<const f4*>(so + 32 * b + 8 * c);
#pragma unroll
            for (int i = 0; i < 4; ++i)
              o[b][4 * c + i] = fmaf(o[b][4 * c + i], w0, v[i] * w1);
          }
      }
    }
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
            for (int i = 0; i < 4; ++i) r[i] = (elem)(o[b][4 * c + i] * inv);
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
        if (half == 0) a.rec.ml[at] = make_float2(m_ref, l);
      }
    }
  }
}

// Joins the records of split rows: o = sum_s e^(m_s - M) o_s / sum_s e^(m_s - M) l_s.
// A workgroup of 16 waves has up to 64 rows of a row tile: a wave a row where there
// are up to 8 splits, two or four waves a row where there are more, each with
// its share of the splits and eight records in flight.  (A wave alone, one
// record after another, took 45 us for the 64 splits of one request of 8192
// tokens; four waves a row whatever the splits 47 us for 192 row tiles of 256
// rows in two splits.)  The groups' count and places come from the first kernel.
constexpr int kMergeWaves = 16;

// Rows row .. row + ROWS - 1 (below `end`) of a row tile of up to SPLITS splits, by
// one wave with all their records in flight.
template <class E, int D, int ROWS, int SPLITS>
__device__ __forceinline__ void merge_rows(const PagedArgs& a, const int* d, int mt, int row,
                                           int end, int splits, int rec0, int head) {
  constexpr int PER = D / kWave;
  const int lane = threadIdx.x & (kWave - 1);
  float2 ml[ROWS][SPLITS];
  float v[ROWS][SPLITS][PER];
#pragma unroll
  for (int r = 0; r < ROWS; ++r)
#pragma unroll
    for (int s = 0; s < SPLITS; ++s) {
      const size_t at = (size_t)(rec0 + min(s, splits - 1) * a.Hkv) * mt + min(row + r, end - 1);
      ml[r][s] = a.rec.ml[at];
#pragma unroll
      for (int i = 0; i < PER; ++i) v[r][s][i] = a.rec.opart[at * D + lane * PER + i];
    }
#pragma unroll
  for (int r = 0; r < ROWS; ++r) {
    float M = kPagedNegInf, L = 0.0f, acc[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) acc[i] = 0.0f;
#pragma unroll
    for (int s = 0; s < SPLITS; ++s)
      if (s < splits && ml[r][s].y != 0.0f) M = fmaxf(M, ml[r][s].x);  // else: saw nothing
#pragma unroll
    for (int s = 0; s < SPLITS; ++s) {
      if (s >= splits || ml[r][s].y == 0.0f) continue;
      const float w = fast_exp2(ml[r][s].x - M);
      L = fmaf(w, ml[r][s].y, L);
#pragma unroll
      for (int i = 0; i < PER; ++i) acc[i] = fmaf(w, v[r][s][i], acc[i]);
    }
    if (row + r < end) {
      const int xr = d[3] + row + r;
      typename E::type* op =
          static_cast<typename E::type*>(a.o) +
          ((size_t)(d[2] + xr / a.G) * a.Hq + head * a.G + xr % a.G) * D + lane * PER;
#pragma unroll
      for (int i = 0; i < PER; ++i)
        op[i] = (typename E::type)(L == 0.0f ? 0.0f : acc[i] / L);
    }
  }
}

template <class E, int D>
__global__ __launch_bounds__(kMergeWaves * kWave) void paged_merge(PagedArgs a, int mt) {
  typedef typename E::type elem;
  constexpr int PER = D / kWave;  // elements a lane
  constexpr int kAtOnce = 8;
  __shared__ float s_acc[kMergeWaves][D], s_m[kMergeWaves], s_l[kMergeWaves];
  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  // Rows of a workgroup's piece: 64 where that makes a piece for each workgroup, 16
  // where it does for half of them, else 4, which a workgroup joins at once however
  // many the splits (20 rows of 8 heads in 31 splits: 17 us in pieces of 16).
  const int groups = min(a.rec.head[0], a.rec.groups);
  const int grid = (int)gridDim.x;
  const int part = groups * (mt / 64) >= grid ? 64 : 2 * groups * (mt / 16) >= grid ? 16 : 4;
  const int parts = mt / part, total = groups * parts;
  for (int task = blockIdx.x; task < total; task += gridDim.x) {
    const int group = task / parts;
    const int* d = a.rec.desc + (size_t)group * kDescInts;
    const int splits = d[0], rec0 = d[1], head = rec0 % a.Hkv;
    // Nothing outside the records and o, also if another stream has changed the
    // lengths since the groups were counted and this one was not described.
    if (splits < 2 || rec0 < 0 || rec0 + (splits - 1ll) * a.Hkv >= a.rec.records || d[2] < 0 ||
        d[3] < 0 || d[4] < 1 || d[4] > mt ||
        (long long)d[2] * a.G + d[3] + d[4] > (long long)a.T * a.G)
      continue;
    const int first = task % parts * part, rows = min(d[4] - first, part);
    if (splits <= 2) {
      for (int r0 = wave * 4; r0 < rows; r0 += 4 * kMergeWaves)
        merge_rows<E, D, 4, 2>(a, d, mt, first + r0, first + rows, splits, rec0, head);
      continue;
    }
    if (splits <= 4) {
      for (int r0 = wave * 2; r0 < rows; r0 += 2 * kMergeWaves)
        merge_rows<E, D, 2, 4>(a, d, mt, first + r0, first + rows, splits, rec0, head);
      continue;
    }
    const int share = splits <= 8 ? 1 : splits <= 16 ? 2 : 4;  // waves of a row
    for (int r0 = 0; r0 < rows; r0 += kMergeWaves / share) {
      const int sub = r0 + wave / share, row = first + min(sub, rows - 1);
      float M = kPagedNegInf, L = 0.0f, acc[PER];
#pragma unroll
      for (int i = 0; i < PER; ++i) acc[i] = 0.0f;
      for (int s0 = wave % share; s0 < splits; s0 += share * kAtOnce) {
        float2 ml[kAtOnce];
        float v[kAtOnce][PER];
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
          const int s = min(s0 + j * share, splits - 1);
          const size_t at = (size_t)(rec0 + s * a.Hkv) * mt + row;
          ml[j] = a.rec.ml[at];
#pragma unroll
          for (int i = 0; i < PER; ++i) v[j][i] = a.rec.opart[at * D + lane * PER + i];
        }
        float Mn = M;
#pragma unroll
        for (int j = 0; j < kAtOnce; ++j) {
          if (s0 + j * share >= splits) ml[j] = make_float2(kPagedNegInf, 0.0f);
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
      if (share > 1) {  // the row's waves meet in the first one
#pragma unroll
        for (int i = 0; i < PER; ++i) s_acc[wave][lane * PER + i] = acc[i];
        if (lane == 0) {
          s_m[wave] = M;
          s_l[wave] = L;
        }
        __syncthreads();
        float Mt = kPagedNegInf, Lt = 0.0f;
        for (int w = wave / share * share; w < wave / share * share + share; ++w)
          if (s_l[w] != 0.0f) Mt = fmaxf(Mt, s_m[w]);
#pragma unroll
        for (int i = 0; i < PER; ++i) acc[i] = 0.0f;
        for (int w = wave / share * share; w < wave / share * share + share; ++w) {
          if (s_l[w] == 0.0f) continue;
          const float e = fast_exp2(s_m[w] - Mt);
          Lt = fmaf(e, s_l[w], Lt);
#pragma unroll
          for (int i = 0; i < PER; ++i) acc[i] = fmaf(e, s_acc[w][lane * PER + i], acc[i]);
        }
        L = Lt;
        __syncthreads();
      }
      if (sub < rows && wave % share == 0) {
        const int xr = d[3] + row;
        elem* op = static_cast<elem*>(a.o) +
                   ((size_t)(d[2] + xr / a.G) * a.Hq + head * a.G + xr % a.G) * D + lane * PER;
#pragma unroll
        for (int i = 0; i < PER; ++i) op[i] = (elem)(L == 0.0f ? 0.0f : acc[i] / L);
      }
    }
  }
}

template <class E, bool FP8, int D, int NW>
PagedFn pick_pages(bool aligned) {
  constexpr int KP = NW == 4 ? 2 : 1;
  return aligned ? paged_chunk<E, FP8, D, true, NW, KP> : paged_chunk<E, FP8, D, false, NW, KP>;
}
template <class E, bool FP8, int NW>
PagedFn pick_size(int D, bool aligned) {
  return D == 64 ? pick_pages<E, FP8, 64, NW>(aligned) : pick_pages<E, FP8, 128, NW>(aligned);
}
template <int NW>
PagedFn pick_type(bool bf16, bool fp8, int D, bool aligned) {
  if (bf16)
    return fp8 ? pick_size<ElemBF16, true, NW>(D, aligned)
               : pick_size<ElemBF16, false, NW>(D, aligned);
  return fp8 ? pick_size<ElemF16, true, NW>(D, aligned)
             : pick_size<ElemF16, false, NW>(D, aligned);
}
PagedFn pick_chunk(int rows, bool bf16, bool fp8, int D, bool aligned) {
  return rows == 64 ? pick_type<4>(bf16, fp8, D, aligned) : pick_type<8>(bf16, fp8, D, aligned);
}

void (*pick_merge(bool bf16, int D))(PagedArgs, int) {
  if (bf16) return D == 64 ? paged_merge<ElemBF16, 64> : paged_merge<ElemBF16, 128>;
  return D == 64 ? paged_merge<ElemF16, 64> : paged_merge<ElemF16, 128>;
}

size_t round256(size_t n) { return (n + 255) / 256 * 256; }

// How a call of these bounds runs: the rows of the chunk kernel's tile (0: none), and
// the workgroups wanted of each kernel.
struct PagedPlanned {
  bool decode;
  int chunk_rows, chunk_target;
  int decode_groups;  // a whole number of parts for each KV head
};
PagedPlanned planned(const PagedCall& c, int cu_count) {
  const int most = c.max_new > 0 && c.max_new < c.T ? c.max_new : c.T;
  const long long rows = (long long)most * (c.Hq / c.cache.Hkv);
  PagedPlanned p;
  p.chunk_rows = rows <= kDecodeRows ? 0 : rows <= 64 ? 64 : 256;
  // Up to 64 rows a request, or one request: the chunk kernel takes them all (16
  // drafts of 5 tokens at 4000, 4 heads a KV head: 58.7 us, on the decode kernel 81;
  // where 8 heads fill the decode kernel's row tiles, 15.8 and 14.0).
  p.decode = p.chunk_rows == 0 || (p.chunk_rows == 256 && c.R > 1);
  // Parts of a KV head's line: a workgroup a CU where requests are few (a line of
  // 32 parts and one request: 13.4 against 16.1 us with 64, at 8192 tokens, 27.9
  // against 30.4 at 32768), else two (256 requests of 500 tokens 72 against 84).
  const int per_cu = 4ll * c.R * c.cache.Hkv <= cu_count ? 1 : 2;
  p.decode_groups = max(1, per_cu * cu_count / c.cache.Hkv) * c.cache.Hkv;
  p.chunk_target = p.chunk_rows == 64 ? 2 * cu_count : cu_count;
  return p;
}

// Workspace of a call: the decode kernel's tickets (zero between calls), its
// records, then the chunk kernel's.
struct PagedSpace {
  PagedRecords decode, chunk;
  size_t bytes;
};
PagedSpace layout(const PagedPlanned& p, int D, char* base) {
  PagedSpace s = {};
  size_t at = 0;
  auto take = [&](size_t n) {
    char* const here = base + at;
    at += round256(n);
    return here;
  };
  auto records = [&](PagedRecords& r, int count, int mt) {
    r.records = count;
    r.ml = reinterpret_cast<float2*>(take((size_t)count * mt * sizeof(float2)));
    r.opart = reinterpret_cast<float*>(take((size_t)count * mt * D * sizeof(float)));
  };
  if (p.decode) {
    s.decode.tickets =
        reinterpret_cast<int*>(take((size_t)p.decode_groups * kTicketInts * sizeof(int)));
    records(s.decode, 2 * p.decode_groups, kDecodeRows);
  }
  if (p.chunk_rows) {
    s.chunk.groups = p.chunk_target;
    s.chunk.head = reinterpret_cast<int*>(take(sizeof(int)));
    s.chunk.desc =
        reinterpret_cast<int*>(take((size_t)p.chunk_target * kDescInts * sizeof(int)));
    records(s.chunk, 2 * p.chunk_target, p.chunk_rows);
  }
  s.bytes = at;
  return s;
}

// Whether 16 keys from a multiple of 16 on always lie in one page, at offsets
// from its first key that 32 bits hold.
bool paged_aligned(const db_paged_cache& kv) {
  constexpr long long kFar = 1 << 26;
  return kv.page_size % 16 == 0 && kv.k_token_stride < kFar && kv.v_token_stride < kFar;
}

}  // namespace

size_t paged_workspace_bytes(const PagedCall& c, int cu_count, size_t* zeroed) {
  const PagedPlanned p = planned(c, cu_count);
  *zeroed = p.decode ? (size_t)p.decode_groups * kTicketInts * sizeof(int) : 0;
  return layout(p, c.cache.D, nullptr).bytes;
}

hipError_t launch_paged_attention(const PagedCall& c, int cu_count, void* ws, hipStream_t stream) {
  const db_paged_cache& kv = c.cache;
  const bool fp8 = kv.dtype == DB_DTYPE_FP8_E4M3;
  const int D = kv.D;
  const PagedPlanned p = planned(c, cu_count);
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

  const bool aligned = paged_aligned(kv);
  const PagedSpace space = layout(p, D, static_cast<char*>(ws));
  // Calls of several host threads on one stream may share a workspace that one keeps
  // from call to call: a call's launches must then stand together on the stream, or
  // another's chunk kernel would overwrite records that are not joined yet.
  static std::mutex together;
  const std::lock_guard<std::mutex> hold(together);
  if (p.decode) {
    a.part = p.chunk_rows ? 1 : 0;
    a.min_tiles = 8;  // two a wave: shorter parts cost more to join than they save
    a.rec = space.decode;
    hipLaunchKernelGGL(paged_decode_fn(c.bf16, fp8, D, aligned), dim3(p.decode_groups),
                       dim3(kPagedThreads), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  if (p.chunk_rows) {
    const int mt = p.chunk_rows;
    a.part = p.decode ? 2 : 0;
    a.target = p.chunk_target;
    a.min_tiles = 4;
    a.rec = space.chunk;
    // Row tiles of every request at most, and the splits beyond one each.
    const long long grid = ((long long)c.T * a.G / mt + c.R) * a.Hkv + p.chunk_target;
    hipLaunchKernelGGL(pick_chunk(mt, c.bf16, fp8, D, aligned), dim3((unsigned)grid),
                       dim3((mt == 64 ? 4 : 8) * kWave), 0, stream, a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL(pick_merge(c.bf16, D), dim3(2 * cu_count), dim3(kMergeWaves * kWave), 0,
                       stream, a, mt);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

}  // namespace dbk
