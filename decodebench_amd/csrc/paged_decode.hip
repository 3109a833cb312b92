// paged_decode.hip -- paged attention of few rows (single tokens, drafts).
//
// A workgroup of four waves owns one (request, KV head, row tile of 16 rows)
// and one split of the keys; wave w takes the key tiles w, w + 4, ... of the
// split.  Bound by HBM: every key and value is read once per row tile, and
// rows beyond the few that a request has cost nothing but idle MFMA columns.
//
//  * A tile is 16 keys where K takes 4 KB of them, 32 (two sub-tiles of 16)
//    where it takes less (e4m3, heads of 64), so that a tile's fixed work, its
//    maximum and its rescale, is paid per 8 KB of cache.
//  * Scores: v_mfma_f32_16x16x32, A = 16 keys straight from the cache to
//    registers (lane (g4, n16) holds 16-byte chunks g4, g4 + 4, ... of key
//    n16), B = the rows.  An e4m3 chunk is 16 elements, so its two halves are
//    two MFMA steps; the rows are loaded in the same order.
//  * Softmax with running maximum and sum, base 2, fp32, on the keys that each
//    lane holds.  Probabilities are rounded to the element type for the product
//    and summed as rounded, so numerator and denominator agree.
//  * P.V: O^T = V^T P^T on 16x16x16 (two sub-tiles: 16x16x32) MFMAs, V^T
//    through the wave's copy of the tile in LDS and the transposing read
//    ds_read_b64_tr_b16.
//  * Pages of a multiple of 16 tokens (ALIGNED): a sub-tile lies in one page.
//    Lane i works out where the wave's i-th sub-tile is, 64 of them at once,
//    and a tile's addresses are two scalars read from its lane.  Any other
//    page size: a lane looks up the page of its own key, one tile ahead of the
//    loads, and rows of V take theirs from that lane.
//  * Masked keys: scores by selection, so no Inf or NaN of a masked key counts;
//    a tile that some row sees only in part is searched for an Inf or NaN
//    among its values, and one that has any is added key by key.
#include "paged_attn.h"

namespace dbk {

namespace {

constexpr int kWaves = kPagedThreads / kWave;
constexpr int MT = kDecodeRows;

constexpr float kHidden = -1.0f;  // no probability

constexpr int decode_keys(bool fp8, int D) { return D * (fp8 ? 1 : 2) >= 256 ? 16 : 32; }

// Orders a wave's LDS accesses (not its loads from memory) as written.
__device__ __forceinline__ void lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

// ------------------------------------------------------------- schedule
// All work of a call in one line: for each KV head, each request in order, each
// row tile of it, its key tiles from the first that a row sees to the last.
// The line is cut into `target` equal parts, a workgroup each, so that all of
// them end together whatever the lengths are (splitting each request by itself
// left 64 requests of 800 to 8000 tokens at 63% of the stream rate).  A part
// holds the end of one item, whole items, and the beginning of another.
struct DecodeRequest {
  int tok0, n, len;
  int t0, tiles;     // first key tile, and how many, of each row tile (none: one all the same)
  int row_tiles;
};

template <int KT>
__device__ __forceinline__ DecodeRequest decode_request(const PagedArgs& a, int r) {
  DecodeRequest q = {0, 0, 0, 0, 0, 0};
  if (r >= a.R) return q;
  q.tok0 = clamp_int(a.q_start[r], 0, a.T);
  q.n = max(clamp_int(a.q_start[r + 1], 0, a.T) - q.tok0, 0);
  q.len = max(a.kv_len[r], 0);
  const int rows = q.n * a.G;
  if (a.part != 0 && rows > kDecodeRows) q.n = 0;
  if (q.n == 0) return q;
  q.row_tiles = (rows + MT - 1) / MT;
  const int limit = paged_limit(a, q.len);
  q.t0 = a.window > 0 ? min(max(q.len - q.n - a.window + 1, 0), limit) / KT : 0;
  q.tiles = max((limit + KT - 1) / KT - q.t0, 1);
  return q;
}

__device__ __forceinline__ long long wave_scan64(long long v) {
  const int lane = threadIdx.x & (kWave - 1);
  for (int d = 1; d < kWave; d <<= 1) {
    const long long u = __shfl_up(v, d);
    if (lane >= d) v += u;
  }
  return v;
}

// A position on the line, in scalar registers but for what each lane holds of
// a request of the present 64 ones.  Every wave has its own: no LDS, no barrier.
template <int KT>
struct DecodeLine {
  const PagedArgs& a;
  DecodeRequest mine;
  long long per_head;     // key tiles of one KV head
  long long upto, all;    // of this round's requests up to this one, and in all
  long long before;       // of the rounds before
  int items_before, items_head;  // row tiles of the rounds before; of one KV head
  int round;
  long long at;           // within the KV head
  int head;

  __device__ explicit DecodeLine(const PagedArgs& args) : a(args) {
    const int lane = threadIdx.x & (kWave - 1);
    long long sum = 0;
    int items = 0;
    for (int r = (a.R - 1) / kWave * kWave; r >= 0; r -= kWave) {
      mine = decode_request<KT>(a, r + lane);
      sum += (long long)mine.row_tiles * mine.tiles;
      items += mine.row_tiles;
    }
    if (a.R > kWave)
      for (int d = 1; d < kWave; d <<= 1) sum += __shfl_xor(sum, d);
    items_head = wave_total(items);
    round = 0;
    before = 0;
    items_before = 0;
    scan();
    per_head = a.R > kWave ? lane_i64(sum, 0) : all;
  }
  __device__ void scan() {
    upto = wave_scan64((long long)mine.row_tiles * mine.tiles);
    all = lane_i64(upto, kWave - 1);
  }
  __device__ void to_round(int r) {
    round = r;
    mine = decode_request<KT>(a, r * kWave + (int)(threadIdx.x & (kWave - 1)));
    scan();
  }
  // The item at `at`: its request (lane `who` of the round), row tile and the
  // tile within it.  Positions only grow within a head.
  __device__ void locate(int& who, int& row_tile, int& tile, int& item) {
    if (at < before) {  // a new head
      before = 0;
      items_before = 0;
      to_round(0);
    }
    while (at >= before + all) {
      before += all;
      items_before += wave_total(mine.row_tiles);
      to_round(round + 1);
    }
    const long long in = at - before;
    who = __builtin_ctzll(__ballot(in < upto));
    const int tiles = __builtin_amdgcn_readlane(mine.tiles, who);
    const int rts = __builtin_amdgcn_readlane(mine.row_tiles, who);
    const long long off = in - (lane_i64(upto, who) - (long long)tiles * rts);
    row_tile = rts == 1 ? 0 : (int)(off / tiles);
    tile = (int)(off - (long long)row_tile * tiles);
    const bool earlier = (int)(threadIdx.x & (kWave - 1)) < who;
    item = head * items_head + items_before + wave_total(earlier ? mine.row_tiles : 0) + row_tile;
  }
};

template <class E, bool FP8, int D, bool ALIGNED>
__global__ __launch_bounds__(kPagedThreads, 2) void paged_decode(PagedArgs a) {
  typedef typename E::type elem;
  typedef typename E::vec8 vec8;
  typedef typename E::vec4 vec4;
  constexpr int CB = FP8 ? 1 : 2;          // bytes of a cache element
  constexpr int KT = decode_keys(FP8, D);  // keys of a tile
  constexpr int NS = KT / 16;              // sub-tiles
  constexpr int NK = D * CB / 64;          // 16-byte loads of K a lane (16 keys, 4 lanes each)
  constexpr int STEPS = D / 32;            // MFMA steps of a score
  constexpr int LPR = D * CB / 16;         // lanes per row of V
  constexpr int RPI = kWave / LPR;         // rows of V a load instruction
  constexpr int NV = 16 / RPI;
  constexpr int VS = D + 16;               // row stride of the V tile in LDS (elements)
  constexpr int NB = D / 16;
  constexpr int kTilesHeld = kWave / NS;   // tiles whose places the lanes hold
  constexpr size_t kOut = sizeof(float) * MT * D, kTile = sizeof(elem) * KT * VS;
  constexpr size_t kRegion = kOut > kTile ? kOut : kTile;

  __shared__ __align__(16) char s_region[kWaves][kRegion];
  __shared__ float s_p[kWaves][KT][16];  // probabilities of a tile added key by key
  __shared__ float s_m[MT][kWaves], s_l[MT][kWaves];

  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int n16 = lane & 15, g4 = lane >> 4;
  elem* const vbuf = reinterpret_cast<elem*>(s_region[wave]);

  DecodeLine<KT> line(a);
  // This workgroup's part [begin, end) of the line.
  const long long total = line.per_head * a.Hkv;
  if (blockIdx.x == 0 && threadIdx.x == 0) a.rec.head[0] = line.items_head * a.Hkv;
  const long long per = max((total + a.target - 1) / a.target, (long long)a.min_tiles);
  long long begin = per * blockIdx.x;
  const long long end = min(begin + per, total);
  if (begin >= end) return;
  line.head = (int)(begin / line.per_head);
  line.at = begin - line.per_head * line.head;
  for (bool once = true; begin < end; once = false) {
    if (!once) __syncthreads();  // the region is read: the next piece may write it
    DecodeRequest rq;
    int who, row_tile, tile_in, item;
    line.locate(who, row_tile, tile_in, item);
    auto of = [&](int v) { return __builtin_amdgcn_readlane(v, who); };
    rq.tok0 = of(line.mine.tok0);
    rq.n = of(line.mine.n);
    rq.len = of(line.mine.len);
    rq.t0 = of(line.mine.t0);
    rq.tiles = of(line.mine.tiles);
    const int r = line.round * kWave + who, head = line.head;
    const int take = (int)min(end - begin, (long long)(rq.tiles - tile_in));
    const int limit = paged_limit(a, rq.len);
    const int t_begin = rq.t0 + tile_in, t_end = t_begin + take;
    // Rows that other workgroups have keys of go to a record: of this
    // workgroup's two the first if it goes on with an item, else the second.
    const bool starts = tile_in == 0, whole = starts && take == rq.tiles;
    const int rec = whole ? -1 : 2 * blockIdx.x + (starts ? 1 : 0);
    const int rows = min(rq.n * a.G - row_tile * MT, MT);
    if (starts && threadIdx.x == 0 && item < a.rec.groups) {
      int* d = a.rec.desc + (size_t)item * kDescInts;
      // the workgroup of the item's last tile
      d[0] = whole ? 0 : (int)((begin + rq.tiles - 1) / per) - (int)blockIdx.x + 1;
      d[1] = blockIdx.x;
      d[2] = rq.tok0;
      d[3] = row_tile * MT;
      d[4] = rows;
      d[5] = head;
    }

    const char* const kbase = static_cast<const char*>(a.k) + head * a.kh * CB;
    const char* const vbase = static_cast<const char*>(a.v) + head * a.vh * CB;
    const int* const trow = a.table + r * a.table_row;
    const int first = t_begin + wave;
    const int nt = first < t_end ? (t_end - first + kWaves - 1) / kWaves : 0;
    auto tile_of = [&](int k) { return first + kWaves * k; };

    // ---- where the keys are ------------------------------------------------
    // ALIGNED: byte offsets of the first key and value of this lane's sub-tile
    // (of 64 from tile `held` on), and a bit per sub-tile that has a page.
    // Otherwise: page of key n16 of a sub-tile, -1 where there is none.
    long long koff = 0, voff = 0;
    unsigned long long has = 0;
    int held = 0;
    auto hold = [&](int k) {
      held = k;
      const int kk = k + lane / NS;
      const int key = kk < nt ? tile_of(kk) * KT + 16 * (lane % NS) : limit;
      int p = -1, off = 0;
      if (key < limit) {
        const int at = page_of(a, key);
        off = key - at * a.page;
        p = trow[at];
      }
      const bool ok = (unsigned)p < (unsigned)a.pages;
      koff = ok ? (p * a.kp + off * a.kt) * CB : 0;
      voff = ok ? (p * a.vp + off * a.vt) * CB : 0;
      has = __ballot(ok);
    };
    auto lookup = [&](int k, int u) {
      const int key = tile_of(k) * KT + 16 * u + n16;
      if (k >= nt || key >= limit) return -1;
      const int p = trow[page_of(a, key)];
      return (unsigned)p < (unsigned)a.pages ? p : -1;
    };

    // This lane's row (column n16 of the products) and the keys it sees.
    const int x = row_tile * MT + min(n16, rows - 1);
    const int token = x / a.G, qhead = head * a.G + x % a.G;
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
    if constexpr (ALIGNED) hold(0);
    const int past = rq.len - rq.n;
    const int khi = a.causal ? min(limit, past + token + 1) : limit;
    const int klo = a.window > 0 ? max(past + token - a.window + 1, 0) : 0;
    // Keys that every row sees: the first row's end, the last row's beginning.
    const int i0 = row_tile * MT / a.G, i1 = (row_tile * MT + rows - 1) / a.G;
    const int all_hi = a.causal ? min(limit, past + i0 + 1) : limit;
    const int all_lo = a.window > 0 ? max(past + i1 - a.window + 1, 0) : 0;
    const float scale = a.scale_log2 * (FP8 ? a.k_scale[head] : 1.0f);

    f4 o[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) o[b] = f4{0.0f, 0.0f, 0.0f, 0.0f};
    float m_run = kPagedNegInf, l_run = 0.0f;

    const unsigned lane_k = (unsigned)(n16 * (int)a.kt * CB + g4 * 16);
    const unsigned lane_v = (unsigned)((lane / LPR) * (int)a.vt * CB + (lane % LPR) * 16);
    // Absent keys read rows of page 0: valid memory, never counted.
    auto load_tile = [&](u4 (&kt)[NS][NK], u4 (&vt)[NS][NV], int k, const int (&pg)[NS]) {
      if constexpr (ALIGNED) {
        if (k >= held + kTilesHeld) hold(k);
#pragma unroll
        for (int u = 0; u < NS; ++u) {
          const int from = (k - held) * NS + u;
          const char* kp = kbase + lane_i64(koff, from);
          const char* vp = vbase + lane_i64(voff, from);
#pragma unroll
          for (int t = 0; t < NK; ++t) kt[u][t] = ld_stream(kp + (lane_k + t * 64u));
#pragma unroll
          for (int j = 0; j < NV; ++j)
            vt[u][j] = ld_stream(vp + j * RPI * a.vt * CB + lane_v);
        }
      } else {
#pragma unroll
        for (int u = 0; u < NS; ++u) {
          const int key0 = tile_of(k) * KT + 16 * u;
          {
            const int key = key0 + n16;
            const int off = pg[u] < 0 ? 0 : key - page_of(a, key) * a.page;
            const char* p = kbase + (max(pg[u], 0) * a.kp + off * a.kt) * CB;
#pragma unroll
            for (int t = 0; t < NK; ++t) kt[u][t] = ld_stream(p + (g4 + 4 * t) * 16);
          }
#pragma unroll
          for (int j = 0; j < NV; ++j) {
            const int row = j * RPI + lane / LPR, key = key0 + row;
            const int pr = __shfl(pg[u], row);
            const int off = pr < 0 ? 0 : key - page_of(a, key) * a.page;
            vt[u][j] =
                ld_stream(vbase + (max(pr, 0) * a.vp + off * a.vt) * CB + (lane % LPR) * 16);
          }
        }
      }
    };
    // Bits of the tile's keys that are in the cache.
    auto present = [&](int k, const int (&pg)[NS]) {
      unsigned there = 0;
#pragma unroll
      for (int u = 0; u < NS; ++u) {
        if constexpr (ALIGNED)
          there |= (has >> ((k - held) * NS + u)) & 1 ? 0xFFFFu << (16 * u) : 0u;
        else
          there |= ((unsigned)__ballot(pg[u] >= 0) & 0xFFFFu) << (16 * u);
      }
      return there;
    };

    auto compute_tile = [&](const u4 (&kt)[NS][NK], u4 (&vt)[NS][NV], int k, unsigned there) {
      const int key0 = tile_of(k) * KT;
      const bool partial =
          there != (unsigned)((1ull << KT) - 1) || key0 < all_lo || key0 + KT > all_hi;
      bool odd = false;  // a partly seen tile with an Inf or NaN among its values
      if (partial) {
        bool bad = false;
#pragma unroll
        for (int u = 0; u < NS; ++u)
#pragma unroll
          for (int j = 0; j < NV; ++j) {
            const int row = 16 * u + j * RPI + lane / LPR;
            if (!((there >> row) & 1) || key0 + row >= limit) vt[u][j] = u4{0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              if constexpr (FP8) {
                const unsigned w = vt[u][j][c] & 0x7F7F7F7Fu;  // NaN: seven bits set (no Inf)
                bad = bad || (w & 0xFFu) == 0x7Fu || ((w >> 8) & 0xFFu) == 0x7Fu ||
                      ((w >> 16) & 0xFFu) == 0x7Fu || (w >> 24) == 0x7Fu;
              } else {
                bad = bad || pair_nonfinite<E>(vt[u][j][c]);
              }
            }
          }
        odd = __any(bad);
      }
      // the tile's values, rows in key order
      lds_order();
#pragma unroll
      for (int u = 0; u < NS; ++u)
#pragma unroll
        for (int j = 0; j < NV; ++j) {
          elem* row = vbuf + (16 * u + j * RPI + lane / LPR) * VS + (lane % LPR) * (16 / CB);
          const u4 v = vt[u][j];
          if constexpr (FP8) {
            const u2 w0 = E::widen(v[0]), w1 = E::widen(v[1]);
            const u2 w2 = E::widen(v[2]), w3 = E::widen(v[3]);
            *reinterpret_cast<u4*>(row) = u4{w0[0], w0[1], w1[0], w1[1]};
            *reinterpret_cast<u4*>(row + 8) = u4{w2[0], w2[1], w3[0], w3[1]};
          } else {
            *reinterpret_cast<u4*>(row) = v;
          }
        }
      lds_order();

      // s[4 u + j]: score of key key0 + 16 u + 4 g4 + j and row n16
      float s[4 * NS];
#pragma unroll
      for (int u = 0; u < NS; ++u) {
        f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int t = 0; t < NK; ++t) {
          const u4 c = kt[u][t];
          if constexpr (FP8) {
            const u2 w0 = E::widen(c[0]), w1 = E::widen(c[1]);
            const u2 w2 = E::widen(c[2]), w3 = E::widen(c[3]);
            acc = E::mfma16(__builtin_bit_cast(vec8, u4{w0[0], w0[1], w1[0], w1[1]}), qop[2 * t],
                            acc);
            acc = E::mfma16(__builtin_bit_cast(vec8, u4{w2[0], w2[1], w3[0], w3[1]}),
                            qop[2 * t + 1], acc);
          } else {
            acc = E::mfma16(__builtin_bit_cast(vec8, c), qop[t], acc);
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) s[4 * u + j] = acc[j] * scale;
      }
      unsigned sees = ~0u;  // bit 4 u + j
      if (partial) {
        sees = 0;
#pragma unroll
        for (int i = 0; i < 4 * NS; ++i) {
          const int kk = 16 * (i >> 2) + 4 * g4 + (i & 3);
          const bool ok = key0 + kk >= klo && key0 + kk < khi && ((there >> kk) & 1);
          sees |= ok ? 1u << i : 0u;
          s[i] = ok ? s[i] : kPagedNegInf;
        }
      }
      float tmax = s[0];
#pragma unroll
      for (int i = 1; i < 4 * NS; ++i) tmax = fmaxf(tmax, s[i]);
      tmax = max_xor32(max_xor16(tmax));
      const float m_new = fmaxf(m_run, tmax);
      // A row that has seen nothing yet keeps -inf; its exponents use 0.
      const float m_use = m_new == kPagedNegInf ? 0.0f : m_new;
      const float alpha = fast_exp2(m_run - m_use);
      elem pb[4 * NS];
      float sum = 0.0f;
#pragma unroll
      for (int i = 0; i < 4 * NS; ++i) {
        pb[i] = (elem)fast_exp2(s[i] - m_use);
        sum += (float)pb[i];
      }
      l_run = fmaf(l_run, alpha, sum);
      m_run = m_new;
      if (__any(alpha != 1.0f)) {
#pragma unroll
        for (int b = 0; b < NB; ++b) o[b] *= alpha;
      }
      if (odd) {
        // Key by key: only keys that the row sees are added.
#pragma unroll
        for (int i = 0; i < 4 * NS; ++i)
          s_p[wave][16 * (i >> 2) + 4 * g4 + (i & 3)][n16] =
              (sees >> i) & 1 ? (float)pb[i] : kHidden;
        lds_order();
#pragma unroll 1
        for (int kk = 0; kk < KT; ++kk) {
          const float p = s_p[wave][kk][n16];
          if (p == kHidden) continue;
#pragma unroll
          for (int b = 0; b < NB; ++b)
#pragma unroll
            for (int c = 0; c < 4; ++c)
              o[b][c] += p * (float)vbuf[kk * VS + 16 * b + 4 * g4 + c];
        }
        return;
      }
      auto read_v = [&](int u, int b) {
        return __builtin_bit_cast(
            u2, __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) s4*)(
                        vbuf + (16 * u + 4 * g4 + (n16 >> 2)) * VS + 16 * b + 4 * (n16 & 3))));
      };
      if constexpr (NS == 1) {
        const vec4 p = {pb[0], pb[1], pb[2], pb[3]};
#pragma unroll
        for (int b = 0; b < NB; ++b)
          o[b] = E::mfma16k16(__builtin_bit_cast(vec4, read_v(0, b)), p, o[b]);
      } else {
        const vec8 p = {pb[0], pb[1], pb[2], pb[3], pb[4], pb[5], pb[6], pb[7]};
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const u2 v0 = read_v(0, b), v1 = read_v(1, b);
          o[b] = E::mfma16(__builtin_bit_cast(vec8, u4{v0[0], v0[1], v1[0], v1[1]}), p, o[b]);
        }
      }
    };

    // ---- this wave's tiles, two register sets of one tile each ------------
    if (nt > 0) {
      u4 ka[NS][NK], va[NS][NV], kb[NS][NK], vb[NS][NV];
      int pa[NS], pb[NS], pc[NS];
      unsigned ta, tb;
      auto find = [&](int k, int (&pg)[NS]) {
        if constexpr (!ALIGNED)
#pragma unroll
          for (int u = 0; u < NS; ++u) pg[u] = lookup(k, u);
      };
      find(0, pa);
      find(1, pb);
      load_tile(ka, va, 0, pa);
      ta = present(0, pa);
      int k = 0;
      for (; k + 3 <= nt; k += 2) {
        find(k + 2, pc);
        load_tile(kb, vb, k + 1, pb);
        tb = present(k + 1, pb);
        compute_tile(ka, va, k, ta);
        find(k + 3, pb);
        load_tile(ka, va, k + 2, pc);
        ta = present(k + 2, pc);
        compute_tile(kb, vb, k + 1, tb);
      }
      if (k + 1 < nt) {
        load_tile(kb, vb, k + 1, pb);
        tb = present(k + 1, pb);
        // all of tile k + 1 is requested before tile k is waited for
        __builtin_amdgcn_sched_barrier(0);
        compute_tile(ka, va, k, ta);
        compute_tile(kb, vb, k + 1, tb);
      } else {
        compute_tile(ka, va, k, ta);
      }
    }

    // ---- the waves' rows meet in LDS ---------------------------------------
    float l_tot = l_run + __shfl_xor(l_run, 16);
    l_tot += __shfl_xor(l_tot, 32);
    lds_order();
    float* const so = reinterpret_cast<float*>(s_region[wave]);
#pragma unroll
    for (int b = 0; b < NB; ++b)
      *reinterpret_cast<f4*>(so + n16 * D + 16 * b + 4 * g4) = o[b];
    if (lane < MT) {
      s_m[lane][wave] = m_run;
      s_l[lane][wave] = l_tot;
    }
    __syncthreads();
    const float vscale = FP8 ? a.v_scale[head] : 1.0f;
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
        const int xr = row_tile * MT + row;
        elem* op = static_cast<elem*>(a.o) +
                   ((size_t)(rq.tok0 + xr / a.G) * a.Hq + head * a.G + xr % a.G) * D + 4 * d4;
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
    begin += take;
    line.at += take;
    if (line.at >= line.per_head) {
      line.at = 0;
      ++line.head;
    }
  }
}

// Joins the records of a row that several workgroups had keys of:
// o = sum_s e^(m_s - M) o_s / sum_s e^(m_s - M) l_s.  A workgroup an item and
// row; D / 4 threads take a record, 1024 / D records at once, eight of each
// thread's in flight, so up to 64 (D = 128) splits cost one round trip.
template <class E, int D>
__global__ __launch_bounds__(kPagedThreads) void paged_decode_merge(PagedArgs a) {
  typedef typename E::type elem;
  constexpr int LPR = D / 4, GROUPS = kPagedThreads / LPR, AT_ONCE = 8;
  __shared__ __align__(16) float s_acc[GROUPS][D];
  __shared__ float s_m[GROUPS], s_l[GROUPS];
  const int group = threadIdx.x / LPR, col = threadIdx.x % LPR * 4;
  const int items = min(a.rec.head[0], a.rec.groups);
  for (int item = blockIdx.x; item < items; item += gridDim.x) {
    const int* d = a.rec.desc + (size_t)item * kDescInts;
    const int splits = d[0], wg = d[1];
    if (splits < 2 || 2 * (wg + splits - 1) >= a.rec.records) continue;
    for (int row = blockIdx.y; row < d[4]; row += gridDim.y) {
      float M = kPagedNegInf, L = 0.0f;
      f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
      for (int s0 = group; s0 < splits; s0 += GROUPS * AT_ONCE) {
        float2 ml[AT_ONCE];
        f4 v[AT_ONCE];
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
          const int s = min(s0 + j * GROUPS, splits - 1);
          const size_t at = (size_t)(2 * (wg + s) + (s == 0 ? 1 : 0)) * MT + row;
          ml[j] = a.rec.ml[at];
          v[j] = *reinterpret_cast<const f4*>(a.rec.opart + at * D + col);
        }
        float Mn = M;
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
          if (s0 + j * GROUPS >= splits) ml[j] = make_float2(kPagedNegInf, 0.0f);
          if (ml[j].y != 0.0f) Mn = fmaxf(Mn, ml[j].x);  // else: saw nothing
        }
        const float keep = L == 0.0f ? 0.0f : fast_exp2(M - Mn);
        L *= keep;
        acc *= keep;
#pragma unroll
        for (int j = 0; j < AT_ONCE; ++j) {
          if (ml[j].y == 0.0f) continue;
          const float w = fast_exp2(ml[j].x - Mn);
          L = fmaf(w, ml[j].y, L);
          acc += w * v[j];
        }
        M = Mn;
      }
      *reinterpret_cast<f4*>(&s_acc[group][col]) = acc;
      if (col == 0) {
        s_m[group] = M;
        s_l[group] = L;
      }
      __syncthreads();
      if (threadIdx.x < D) {
        float Mt = kPagedNegInf, Lt = 0.0f, o = 0.0f;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g)
          if (s_l[g] != 0.0f) Mt = fmaxf(Mt, s_m[g]);
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
          if (s_l[g] == 0.0f) continue;
          const float e = fast_exp2(s_m[g] - Mt);
          Lt = fmaf(e, s_l[g], Lt);
          o = fmaf(e, s_acc[g][threadIdx.x], o);
        }
        const int xr = d[3] + row;
        static_cast<elem*>(a.o)[((size_t)(d[2] + xr / a.G) * a.Hq + d[5] * a.G + xr % a.G) * D +
            threadIdx.x] = (elem)(Lt == 0.0f ? 0.0f : o / Lt);
      }
      __syncthreads();
    }
  }
}

template <class E, bool FP8>
PagedFn pick_size(int D, bool aligned) {
  if (D == 64)
    return aligned ? paged_decode<E, FP8, 64, true> : paged_decode<E, FP8, 64, false>;
  return aligned ? paged_decode<E, FP8, 128, true> : paged_decode<E, FP8, 128, false>;
}

}  // namespace

PagedFn paged_decode_merge_fn(bool bf16, int D) {
  if (bf16) return D == 64 ? paged_decode_merge<ElemBF16, 64> : paged_decode_merge<ElemBF16, 128>;
  return D == 64 ? paged_decode_merge<ElemF16, 64> : paged_decode_merge<ElemF16, 128>;
}

PagedFn paged_decode_fn(bool bf16, bool fp8, int D, bool aligned) {
  if (bf16)
    return fp8 ? pick_size<ElemBF16, true>(D, aligned) : pick_size<ElemBF16, false>(D, aligned);
  return fp8 ? pick_size<ElemF16, true>(D, aligned) : pick_size<ElemF16, false>(D, aligned);
}

}  // namespace dbk
