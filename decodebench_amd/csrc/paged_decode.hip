// paged_decode.hip -- paged attention of few rows (single tokens, drafts).
//
// A workgroup of four waves owns an equal part of a KV head's work (see
// DecodeLine): keys of one (request, row tile of 16 rows) after another; wave w
// takes the key tiles w, w + 4, ... of each.  Bound by HBM: every key and value
// is read once per row tile, and rows beyond the few that a request has cost
// nothing but idle MFMA columns.  64 requests of 800 to 8000 tokens (8 heads of
// 128, 1.15 GB of cache): 0.21 ms, 5.5 TB/s, where a plain read reaches 7.1; equal
// lengths in a [pages, heads, page, D] cache reach 6.1 to 6.5.
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
//    in a tile that some row sees only in part the values that are Inf or NaN
//    are left out of the product (their probability may be zero, but zero times
//    those is not) and added to the rows that do see them.
#include "paged_attn.h"

namespace dbk {

namespace {

constexpr int kWaves = kPagedThreads / kWave;
constexpr int MT = kDecodeRows;

constexpr int kSc1 = 16;         // cache policy of a buffer access: device scope
constexpr int kVmcnt0 = 0x0F70;  // s_waitcnt vmcnt(0), the other counters left alone

constexpr int decode_keys(bool fp8, int D) { return D * (fp8 ? 1 : 2) >= 256 ? 16 : 32; }

// Orders a wave's LDS accesses (not its loads from memory) as written.
__device__ __forceinline__ void lds_order() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront", "local");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront", "local");
}

// ------------------------------------------------------------- schedule
// The work of a KV head in one line: each request in order, each row tile of
// it, its key tiles from the first that a row sees to the last.  The line is cut
// into equal parts, a workgroup each, so that all of them end together whatever
// the lengths are (splitting each request by itself left 64 requests of 800 to
// 8000 tokens at 63% of the stream rate).  A part holds the end of one item,
// whole items, and the beginning of another.  The workgroups of a part's KV
// heads are neighbours, so the heads of a page, which lie side by side, are read
// at about the same time.
struct DecodeRequest {
  int tok0, n, len;
  int t0, tiles;     // first key tile, and how many, of each row tile (none: one all the same)
  int row_tiles;
  bool back;         // as PagedRequest's
};

template <int KT>
__device__ __forceinline__ DecodeRequest decode_request(const PagedArgs& a, int r, int& upto) {
  DecodeRequest q = {0, 0, 0, 0, 0, 0, false};
  const PagedRows own = paged_rows(a, r, upto);
  q.tok0 = own.tok0;
  q.back = own.n < 0;
  q.n = max(own.n, 0);
  q.len = own.len;
  const int rows = q.n * a.G;
  if (a.part != 0 && rows > kDecodeRows) q.n = 0;
  if (q.n == 0) return q;
  q.row_tiles = (rows + MT - 1) / MT;
  const int limit = paged_limit(a, q.len);
  q.t0 = min(first_seen(a, q.len - q.n), limit) / KT;
  q.tiles = max((limit + KT - 1) / KT - q.t0, 1);
  return q;
}

// The line of a KV head; what each lane holds is of a request of the present 64.
// Every wave has its own: no LDS, no barrier.  (The host has checked that all
// tiles of a line are fewer than 2^31: T rows, each of one request.)
template <int KT>
struct DecodeLine {
  const PagedArgs& a;
  DecodeRequest mine;
  int length;      // key tiles in all
  int upto, all;   // of the present 64 requests up to this one, and in all
  int before;      // of the requests before them
  int round;
  int rows_upto;   // where the present requests' rows end, or kInOrder

  __device__ explicit DecodeLine(const PagedArgs& args) : a(args), before(0), round(0) {
    const int lane = threadIdx.x & (kWave - 1);
    int sum = 0;  // of the rounds after the first
    bool back = false;
    for (int r = (a.R - 1) / kWave * kWave; r > 0; r -= kWave) {
      int far = kInOrder;
      const DecodeRequest q = decode_request<KT>(a, r + lane, far);
      sum += q.row_tiles * q.tiles;
      back = back || q.back;
    }
    rows_upto = kInOrder;
    mine = decode_request<KT>(a, lane, rows_upto);
    if (__any(back || mine.back)) {  // (apart: one loop for both took 13.6 us for 13.3)
      rows_upto = 0;
      mine = decode_request<KT>(a, lane, rows_upto);
      int far = rows_upto;
      sum = 0;
      for (int r = kWave; r < a.R; r += kWave) {
        const DecodeRequest q = decode_request<KT>(a, r + lane, far);
        sum += q.row_tiles * q.tiles;
      }
    }
    scan();
    length = all + (a.R > kWave ? wave_total(sum) : 0);
  }
  __device__ void scan() {
    upto = wave_scan(mine.row_tiles * mine.tiles);
    all = __builtin_amdgcn_readlane(upto, kWave - 1);
  }
  // The item at `at` < length: its request (lane `who` of the round), row tile and
  // the tile within it.  Positions only grow.  (False only where another stream
  // changes the lengths meanwhile: a search that must end all the same.)
  __device__ bool locate(int at, int& who, int& row_tile, int& tile) {
    while (at >= before + all) {
      if ((round + 1) * kWave >= a.R) return false;
      before += all;
      ++round;
      mine = decode_request<KT>(a, round * kWave + (int)(threadIdx.x & (kWave - 1)), rows_upto);
      scan();
    }
    const int in = at - before;
    const unsigned long long hit = __ballot(in < upto);
    if (!hit) return false;
    who = __builtin_ctzll(hit);
    const int tiles = __builtin_amdgcn_readlane(mine.tiles, who);
    const int rts = __builtin_amdgcn_readlane(mine.row_tiles, who);
    const int off = in - (__builtin_amdgcn_readlane(upto, who) - tiles * rts);
    if (off < 0 || off >= tiles * rts) return false;
    row_tile = rts == 1 ? 0 : off / tiles;
    tile = off - row_tile * tiles;
    return true;
  }
};

// Joins the `splits` records of a row tile, the first in workgroup wg0's second
// place, the others in the first places of wg0 + Hkv, + 2 Hkv, ...: a thread a
// float4 of a row and a share of the records, sixteen of them in flight, then the
// shares through LDS (`scratch`: 6 floats a thread).
template <class E, int D>
__device__ __forceinline__ void join_records(const PagedArgs& a, int tok0, int row_tile, int rows,
                                             int head, int wg0, int splits, float* scratch) {
  typedef typename E::vec4 vec4;
  constexpr int AT_ONCE = 16;
  const __amdgpu_buffer_rsrc_t r_ml = make_rsrc(a.rec.ml, a.rec.records * MT * 8);
  const __amdgpu_buffer_rsrc_t r_op = make_rsrc(a.rec.opart, a.rec.records * MT * D * 4);
  const int slots = rows * (D / 4);
  const int shares = slots >= kPagedThreads ? 1 : kPagedThreads / slots;
  for (int s_base = 0; s_base < slots; s_base += kPagedThreads / shares) {
    const int share = threadIdx.x / min(slots, kPagedThreads);
    const int slot = s_base + threadIdx.x % min(slots, kPagedThreads);
    const bool on = share < shares && slot < slots;
    const int row = slot / (D / 4), d4 = slot % (D / 4);
    float M = kPagedNegInf, L = 0.0f;
    f4 acc = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s0 = share; on && s0 < splits; s0 += shares * AT_ONCE) {
      float2 ml[AT_ONCE];
      f4 v[AT_ONCE];
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) {
        const int s = min(s0 + j * shares, splits - 1);
        const size_t at = (size_t)(2 * (wg0 + s * a.Hkv) + (s == 0 ? 1 : 0)) * MT + row;
        ml[j] = __builtin_bit_cast(
            float2, __builtin_amdgcn_raw_buffer_load_b64(r_ml, (int)at * 8, 0, kSc1));
        v[j] = __builtin_bit_cast(f4, __builtin_amdgcn_raw_buffer_load_b128(
                                          r_op, (int)(at * D + 4 * d4) * 4, 0, kSc1));
      }
      float Mn = M;
#pragma unroll
      for (int j = 0; j < AT_ONCE; ++j) {
        if (s0 + j * shares >= splits) ml[j] = make_float2(kPagedNegInf, 0.0f);
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
    float* mine = scratch + threadIdx.x * 6;
    mine[0] = M;
    mine[1] = L;
#pragma unroll
    for (int i = 0; i < 4; ++i) mine[2 + i] = acc[i];
    __syncthreads();
    if (on && share == 0) {
      float Mt = kPagedNegInf, Lt = 0.0f;
      f4 o = {0.0f, 0.0f, 0.0f, 0.0f};
      const int step = 6 * min(slots, kPagedThreads);
      for (int g = 0; g < shares; ++g)
        if (mine[g * step + 1] != 0.0f) Mt = fmaxf(Mt, mine[g * step]);
      for (int g = 0; g < shares; ++g) {
        const float* c = mine + g * step;
        if (c[1] == 0.0f) continue;
        const float e = fast_exp2(c[0] - Mt);
        Lt = fmaf(e, c[1], Lt);
        o += e * f4{c[2], c[3], c[4], c[5]};
      }
      const int xr = row_tile * MT + row;
      const float inv = Lt == 0.0f ? 0.0f : 1.0f / Lt;
      vec4 r;
#pragma unroll
      for (int i = 0; i < 4; ++i) r[i] = (typename E::type)(o[i] * inv);
      *reinterpret_cast<vec4*>(static_cast<typename E::type*>(a.o) +
                               ((size_t)(tok0 + xr / a.G) * a.Hq + head * a.G + xr % a.G) * D +
                               4 * d4) = r;
    }
    __syncthreads();
  }
}

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
  __shared__ float s_m[MT][kWaves], s_l[MT][kWaves];
  __shared__ int s_arrived;

  const int lane = threadIdx.x & (kWave - 1);
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int n16 = lane & 15, g4 = lane >> 4;
  elem* const vbuf = reinterpret_cast<elem*>(s_region[wave]);

  const __amdgpu_buffer_rsrc_t r_ml = make_rsrc(a.rec.ml, a.rec.records * MT * 8);
  const __amdgpu_buffer_rsrc_t r_op = make_rsrc(a.rec.opart, a.rec.records * MT * D * 4);
  DecodeLine<KT> line(a);
  // This workgroup's part [begin, end) of its KV head's line.
  const int part = blockIdx.x / a.Hkv, head = blockIdx.x % a.Hkv;
  const int parts = gridDim.x / a.Hkv;
  const int per = max((line.length + parts - 1) / parts, a.min_tiles);
  int begin = (int)min((long long)per * part, (long long)line.length);
  const int end = (int)min((long long)begin + per, (long long)line.length);
  for (bool once = true; begin < end; once = false) {
    if (!once) __syncthreads();  // the region is read: the next piece may write it
    DecodeRequest rq;
    int who, row_tile, tile_in;
    if (!line.locate(begin, who, row_tile, tile_in)) break;
    auto of = [&](int v) { return __builtin_amdgcn_readlane(v, who); };
    rq.tok0 = of(line.mine.tok0);
    rq.n = of(line.mine.n);
    rq.len = of(line.mine.len);
    rq.t0 = of(line.mine.t0);
    rq.tiles = of(line.mine.tiles);
    const int r = line.round * kWave + who;
    const int take = min(end - begin, rq.tiles - tile_in);
    const int limit = paged_limit(a, rq.len);
    const int t_begin = rq.t0 + tile_in, t_end = t_begin + take;
    // Rows that other workgroups have keys of go to a record: of this
    // workgroup's two the first if it goes on with an item, else the second.
    const bool starts = tile_in == 0, whole = starts && take == rq.tiles;
    const int rec = whole ? -1 : 2 * blockIdx.x + (starts ? 1 : 0);
    const int rows = min(rq.n * a.G - row_tile * MT, MT);

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
    const int klo = first_seen(a, past + token);
    // Keys that every row sees: the first row's end, the last row's beginning.
    const int i0 = row_tile * MT / a.G, i1 = (row_tile * MT + rows - 1) / a.G;
    const int all_hi = a.causal ? min(limit, past + i0 + 1) : limit;
    const int all_lo = first_seen(a, past + i1);
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

    // Adds the Infs and NaNs that a partly seen tile left out to the rows that see
    // them (values read again from the cache; a rare path, kept small).
    auto add_odd = [&](int key0, unsigned sees) {
#pragma unroll 1
      for (int kk = 0; kk < KT; ++kk) {
        const bool ok = (sees >> kk) & 1;
        if (!__any(ok)) continue;  // also keys without a page
        const int key = key0 + kk, at = page_of(a, key);
        const char* row = vbase + (trow[at] * a.vp + (key - at * a.page) * a.vt) * CB;
#pragma unroll
        for (int b = 0; b < NB; ++b) {
          const char* four = row + (16 * b + 4 * g4) * CB;
          const u2 w = FP8 ? E::widen(*reinterpret_cast<const unsigned*>(four))
                           : *reinterpret_cast<const u2*>(four);
          const vec4 v = __builtin_bit_cast(vec4, w);
#pragma unroll
          for (int c = 0; c < 4; ++c)
            o[b][c] += ok && !__builtin_isfinite((float)v[c]) ? (float)v[c] : 0.0f;
          __builtin_amdgcn_sched_barrier(0);
        }
      }
    };

    auto compute_tile = [&](const u4 (&kt)[NS][NK], u4 (&vt)[NS][NV], int k, unsigned there) {
      const int key0 = tile_of(k) * KT;
      const bool partial =
          there != (unsigned)((1ull << KT) - 1) || key0 < all_lo || key0 + KT > all_hi;
      bool odd = false;  // an Inf or NaN among the values of a partly seen tile, left out
      unsigned sees = ~0u;   // bit 16 u + 4 g4 + j: this lane's row sees that key
      if (partial) {
        const unsigned in = there & (unsigned)below(limit - key0);
        sees = in & (unsigned)(below(khi - key0) & ~below(klo - key0));
        const unsigned mine = in >> (lane / LPR);
#pragma unroll
        for (int u = 0; u < NS; ++u)
#pragma unroll
          for (int j = 0; j < NV; ++j) {
            const bool ok = mine & (1u << (16 * u + j * RPI));
#pragma unroll
            for (int c = 0; c < 4; ++c) {
              unsigned w = ok ? vt[u][j][c] : 0u;
              if constexpr (FP8) {
                // NaN: the seven low bits of a byte set (there is no Inf); 0x80
                // marks those bytes
                const unsigned n = ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u;
                odd = odd || n != 0;
                w &= ~(n | (n - (n >> 7)));
              } else {
                const bool lo = (w & E::kExp) == E::kExp, hi = ((w >> 16) & E::kExp) == E::kExp;
                odd = odd || lo || hi;
                w &= (lo ? 0u : 0x0000FFFFu) | (hi ? 0u : 0xFFFF0000u);
              }
              vt[u][j][c] = w;
            }
          }
        odd = __any(odd);
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
      if (partial) {
        const unsigned mine = sees >> (4 * g4);
#pragma unroll
        for (int i = 0; i < 4 * NS; ++i)
          s[i] = mine & (1u << (16 * (i >> 2) + (i & 3))) ? s[i] : kPagedNegInf;
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
      if (odd) add_odd(key0, sees);
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
        __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(u4, ow), r_op,
                                               (int)(at * D + 4 * d4) * 4, 0, kSc1);
        if (d4 == 0)
          __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(u2, make_float2(M, lw)), r_ml,
                                                (int)at * 8, 0, kSc1);
      }
    }
    if (rec >= 0) {
      // The last of the item's workgroups to arrive joins their records,
      //   o = sum_s e^(m_s - M) o_s / sum_s e^(m_s - M) l_s.
      // Its parts are first_part .. first_part + splits - 1; the ticket is that
      // of the part that begins it (a part begins one such item at most).
      const int item_begin = begin - tile_in;
      const int first_part = item_begin / per;
      const int splits = (item_begin + rq.tiles - 1) / per - first_part + 1;
      const int wg0 = first_part * a.Hkv + head;
      int* const ticket = a.rec.tickets + (size_t)wg0 * kTicketInts;
      // Records are written through to memory and read from there (device
      // scope, kSc1), since the item's workgroups run on any XCD; every thread's
      // stores are done before the ticket is taken.  (Plain stores released and
      // acquired by the ticket instead write back and invalidate whole L2s: one
      // request of 8192 tokens took 28 us that way.)
      __builtin_amdgcn_s_waitcnt(kVmcnt0);
      __syncthreads();
      if (threadIdx.x == 0)
        s_arrived = __hip_atomic_fetch_add(ticket, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
      __syncthreads();
      if (s_arrived == splits - 1) {
        if (threadIdx.x == 0)
          __hip_atomic_store(ticket, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        join_records<E, D>(a, rq.tok0, row_tile, rows, head, wg0, splits,
                           reinterpret_cast<float*>(&s_region[0][0]));
      }
    }
    begin += take;
  }
}

template <class E, bool FP8>
PagedFn pick_size(int D, bool aligned) {
  if (D == 64)
    return aligned ? paged_decode<E, FP8, 64, true> : paged_decode<E, FP8, 64, false>;
  return aligned ? paged_decode<E, FP8, 128, true> : paged_decode<E, FP8, 128, false>;
}

}  // namespace

PagedFn paged_decode_fn(bool bf16, bool fp8, int D, bool aligned) {
  if (bf16)
    return fp8 ? pick_size<ElemBF16, true>(D, aligned) : pick_size<ElemBF16, false>(D, aligned);
  return fp8 ? pick_size<ElemF16, true>(D, aligned) : pick_size<ElemF16, false>(D, aligned);
}

}  // namespace dbk
