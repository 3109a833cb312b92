// paged_attn.h -- what the two kernels of paged attention share: arguments,
// element types, page lookup, records; and how the chunk kernel finds its work.
//
// paged_attention computes, for the new tokens i = 0 .. n_r - 1 of every
// request r (packed one request after another, q_start[r] the first row) and
// every query head h,
//   o[i, h] = sum_j softmax_j(scale q[i, h] . K[j, h / G]) V[j, h / G]
// over the keys j of the request that token i sees: j < len_r, with `causal`
// j <= pos_i = len_r - n_r + i, with a window j > pos_i - window, and only
// keys whose page is in the cache.  A row that sees nothing is zero.
//
// Rows: the n_r G (token, query head) pairs of a (request, KV head) are the
// rows of one product, row x = token x / G, head x % G, so that K and V are
// read once for all of them; a row tile is MT of them (16 in paged_decode, 64
// or 256 in paged_chunk).
//
// Lengths live on the GPU, so the host launches a grid by its bounds and every
// workgroup finds its own work from the lengths of all requests.  This costs
// about a microsecond per workgroup, once, and no launch, no table to keep in
// step with the lengths and no read on the host.  The KV head is the fastest
// index: workgroups i and i + 8 run on one XCD, so with 8 heads all row tiles
// and splits of a head share one L2.
//
// Where a row's keys are split, each part writes its running maximum, exp-sum
// and unnormalised output as an fp32 record.  paged_decode cuts the work into
// equal parts (two records a workgroup at most) and joins the records in the
// same launch; paged_chunk splits whole row tiles and paged_merge joins them.
#pragma once

#include "db_elem.h"
#include "db_kernels.h"

namespace dbk {

constexpr float kPagedNegInf = -__builtin_huge_valf();

// ------------------------------------------------------------- arguments
// Region of the workspace of one kernel.
struct PagedRecords {
  int* tickets;   // decode: [workgroups][kTicketInts], zero between calls
  int* head;      // chunk: [0]: groups (row tiles whose rows were split) of this call
  int* desc;      // chunk: [groups][8]: splits, first record, first token, first row, rows
  float2* ml;     // [records][MT]    maximum (base 2) and exp-sum
  float* opart;   // [records][MT][D] unnormalised output
  int records, groups;  // room
};

struct PagedArgs {
  const void* q;
  void* o;
  const void* k;
  const void* v;
  const float* k_scale;
  const float* v_scale;
  const int* table;
  const int* q_start;
  const int* kv_len;
  long long q_token, q_head;      // strides in elements
  long long kp, kh, kt, vp, vh, vt;
  long long table_row;
  int T, R, Hq, Hkv, G;
  int pages, page, width;
  unsigned page_magic, page_shift;  // key / page, see page_of()
  int causal, window;
  float scale_log2;
  int part;        // 0: every request, 1: those of at most kDecodeRows rows, 2: the others
  int target;      // chunk: workgroups wanted
  int min_tiles;   // fewest key tiles of a split or part
  PagedRecords rec;
};

constexpr int kDecodeRows = 16;  // rows of the decode kernel's tile
constexpr int kChunkKeys = 64;
constexpr int kPagedThreads = 256;
constexpr int kDescInts = 8;
constexpr int kTicketInts = 64;  // a 256-byte line each: 8 tickets in one cost 1.7 us of contention

// key / page for 0 <= key < 2^31, with magic = ceil(2^(31 + s) / page), s =
// ceil(log2 page) = shift + 1: the excess magic * page - 2^(31 + s) is less
// than 2^s, so key * excess < 2^(31 + s) and the quotient is exact.
__device__ __forceinline__ int page_of(const PagedArgs& a, int key) {
  return a.page_magic ? (int)(__umulhi((unsigned)key, a.page_magic) >> a.page_shift) : key;
}

// ------------------------------------------------------------- schedule
struct PagedRequest {
  int tok0, n, len;   // first row of q, new tokens, tokens in all
  int row_tiles, tiles;  // row tiles, most key tiles of any of them
  bool back;             // q_start goes back from this request to the next
};

struct PagedWork {
  PagedRequest req;
  int r, head, tile, split, splits;
  int rec, group;  // first record and group of the row tile, -1 if it is not split
};

__device__ __forceinline__ int clamp_int(int v, int lo, int hi) { return min(max(v, lo), hi); }

// Keys a request has at most: its length and what the block table can hold.
__device__ __forceinline__ int paged_limit(const PagedArgs& a, int len) {
  const long long held = (long long)a.width * a.page;
  return (int)min((long long)min(len, 0x7FFFF000), held);
}

// The first key that a token at `pos` sees (a window may be as long as an int holds).
__device__ __forceinline__ int first_seen(const PagedArgs& a, int pos) {
  return a.window > 0 && pos >= a.window ? pos - a.window + 1 : 0;
}

// Inclusive prefix sum over the 64 lanes (DPP row shifts and broadcasts).
__device__ __forceinline__ int wave_scan(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false);  // row_shr:1
  v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false);
  v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);  // row_bcast:15
  v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);  // row_bcast:31
  return v;
}
// The same with the maximum, of values that are not negative.
__device__ __forceinline__ int wave_max_scan(int v) {
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false));
  v = max(v, __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false));
  return v;
}

// Rows of q and length of this lane's request `r`, of 64 requests in lane order.
// `upto` kInOrder: as q_start says.  Else the rows go from the furthest that a q_start up
// to its own says to the furthest up to the next one's, and `upto` is the end of
// the requests before these 64 (0 at first), which becomes theirs: no row belongs to
// two requests and at most T count, which grid, records and tickets are sized by.
// A kernel takes q_start at its word first and, if it goes back anywhere, starts again.
// (A scan in every call: drafts 16.1 us instead of 15.8, 256 requests of one token with
// no max_new 105 instead of 102.)
constexpr int kInOrder = -1;
struct PagedRows {
  int tok0, n, len;
};
__device__ __forceinline__ PagedRows paged_rows(const PagedArgs& a, int r, int& upto) {
  if (r >= a.R && upto == kInOrder) return {0, 0, 0};
  const int at = min(r, a.R - 1);
  int start = clamp_int(a.q_start[at], 0, a.T), end = clamp_int(a.q_start[at + 1], 0, a.T);
  const int len = max(a.kv_len[at], 0);
  if (upto != kInOrder) {
    const int first = max(upto, __builtin_amdgcn_readfirstlane(start));
    end = max(first, wave_max_scan(end));
    start = __builtin_amdgcn_update_dpp(first, end, 0x138, 0xf, 0xf, false);  // wave_shr:1
    upto = __builtin_amdgcn_readlane(end, kWave - 1);
  }
  return {start, end - start, len};
}

template <int MT, int KT>
__device__ __forceinline__ PagedRequest paged_request(const PagedArgs& a, int r, int& upto) {
  PagedRequest q = {0, 0, 0, 0, 0, false};
  const PagedRows own = paged_rows(a, r, upto);
  q.tok0 = own.tok0;
  q.back = own.n < 0;
  q.n = max(own.n, 0);
  q.len = own.len;
  const long long rows = (long long)q.n * a.G;
  if (a.part != 0 && (rows <= kDecodeRows) != (a.part == 1)) q.n = 0;
  if (q.n == 0) return q;
  q.row_tiles = (int)((rows + MT - 1) / MT);
  long long keys = paged_limit(a, q.len);
  // With a window a row tile of tokens i .. i + d sees at most window + d keys.
  if (a.window > 0) keys = min(keys, (long long)a.window + (MT - 1) / a.G + 1 + KT);
  q.tiles = (int)((keys + KT - 1) / KT);
  return q;
}

__device__ __forceinline__ long long lane_i64(long long v, int lane) {
  const int lo = __builtin_amdgcn_readlane((int)v, lane);
  const int hi = __builtin_amdgcn_readlane((int)(v >> 32), lane);
  return (long long)(((unsigned long long)(unsigned)hi << 32) | (unsigned)lo);
}

// The lowest n of 64 bits (none below 0, all from 64 on).
__device__ __forceinline__ unsigned long long below(int n) {
  return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1;
}

__device__ __forceinline__ int wave_total(int v) {
  return __builtin_amdgcn_readlane(wave_scan(v), kWave - 1);
}

// Max over lanes that differ in bit 5 (and in bit 4) of their number.  (The
// results are copied out before the bit casts: a bit cast of a vector's
// element reads its element 0 whatever the index.)
__device__ __forceinline__ float max_xor32(float v) {
  const unsigned a = __builtin_bit_cast(unsigned, v);
  const auto r = __builtin_amdgcn_permlane32_swap(a, a, false, false);
  const unsigned x = r[0], y = r[1];
  return fmaxf(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y));
}
__device__ __forceinline__ float max_xor16(float v) {
  const unsigned a = __builtin_bit_cast(unsigned, v);
  const auto r = __builtin_amdgcn_permlane16_swap(a, a, false, false);
  const unsigned x = r[0], y = r[1];
  return fmaxf(__builtin_bit_cast(float, x), __builtin_bit_cast(float, y));
}

// The chunk kernel's search for the piece of work of the workgroup's number:
// find() says whether there is one and leaves it in `work`, in scalar registers.
// C is the key tiles that one split may hold, all work over the workgroups that
// the chip wants; a prefix sum over the requests' split counts gives the
// (request, KV head, row tile, split).  Every wave does the search for itself, a
// lane to a request and 64 requests a round: no LDS, no barrier.  The host's grid
// holds every piece, so every group that is counted for the merge is described: the
// requests have at most T rows between them and one row tile each that is not full,
// and the splits beyond one each are at most all tiles / C.  There are fewer than 2
// `target` records: only requests of at least 1.75 C tiles split, into at most
// 8/7 tmax / C parts, and C >= (all tiles) / target.
template <int MT, int KT>
struct PagedSchedule {
  const PagedArgs& a;
  int w, round, C;
  int units0, recs0, groups0;  // of the rounds before (per KV head)
  PagedRequest mine;           // this lane's request of the round
  int upto;                    // where the round's rows end, or kInOrder
  int splits, units, before, total;

  __device__ explicit PagedSchedule(const PagedArgs& args)
      : a(args), w(blockIdx.x), round(0), units0(0), recs0(0), groups0(0) {
    const int lane = threadIdx.x & (kWave - 1);
    float work;  // its rounding may move C by one tile in 2^24
    for (int begin = kInOrder;; begin = 0) {
      bool back = false;
      int far = begin;
      work = 0.0f;
      for (int r = 0; r < a.R; r += kWave) {
        const PagedRequest q = paged_request<MT, KT>(a, r + lane, far);
        if (r == 0) {
          mine = q;
          upto = far;
        }
        work += (float)q.row_tiles * (float)q.tiles;
        back = back || q.back;
      }
      if (!__any(back)) break;  // (none goes back after a scan)
    }
    const float per = ceilf(wave_sum(work) * (float)a.Hkv / (float)a.target);
    C = max(a.min_tiles, (int)fminf(per, 1073741824.0f));
    scan();
    if (blockIdx.x == 0 && threadIdx.x < kWave) {  // the groups of the whole call, for the merge
      int groups = splits > 1 ? mine.row_tiles : 0;
      int far = upto;
      for (int r = kWave; r < a.R; r += kWave) {
        const PagedRequest q = paged_request<MT, KT>(a, r + lane, far);
        groups += splits_of(q) > 1 ? q.row_tiles : 0;
      }
      groups = wave_total(groups) * a.Hkv;
      if (lane == 0) a.rec.head[0] = groups;
    }
  }

  __device__ int splits_of(const PagedRequest& q) const {
    // Two splits only for work worth nearly two parts: halves of 192 row tiles of 80
    // key tiles on 256 CUs (C = 60) are no sooner done, and cost a merge.
    return q.row_tiles == 0 ? 0 : max(1, (int)((4ll * q.tiles + C) / (4ll * C)));
  }
  __device__ void scan() {
    splits = splits_of(mine);
    units = mine.row_tiles * splits;
    const int incl = wave_scan(units);
    before = incl - units;
    total = __builtin_amdgcn_readlane(incl, kWave - 1);
  }

  __device__ bool find(PagedWork& work) {
    const int unit = w / a.Hkv, lane = threadIdx.x & (kWave - 1);
    while (unit >= units0 + total) {
      units0 += total;
      recs0 += wave_total(splits > 1 ? units : 0);
      groups0 += wave_total(splits > 1 ? mine.row_tiles : 0);
      ++round;
      if ((long long)round * kWave >= a.R) return false;
      mine = paged_request<MT, KT>(a, round * kWave + lane, upto);
      scan();
    }
    const int at0 = unit - units0;
    const unsigned long long hit = __ballot(at0 >= before && at0 - before < units);
    if (!hit) return false;  // another stream changes the lengths meanwhile
    const int who = __builtin_ctzll(hit);
    auto of = [&](int v) { return __builtin_amdgcn_readlane(v, who); };
    work.req.tok0 = of(mine.tok0);
    work.req.n = of(mine.n);
    work.req.len = of(mine.len);
    work.req.row_tiles = of(mine.row_tiles);
    work.req.tiles = of(mine.tiles);
    work.r = round * kWave + who;
    work.head = w % a.Hkv;
    work.splits = of(splits);
    const int at = at0 - of(before);
    work.tile = work.req.row_tiles - 1 - at / work.splits;  // the longest first
    work.split = at % work.splits;
    work.rec = work.group = -1;
    if (work.splits > 1) {
      const bool mine_before = lane < who && splits > 1;
      work.rec = (recs0 + wave_total(mine_before ? units : 0) + work.tile * work.splits) * a.Hkv +
                 work.head;
      work.group =
          (groups0 + wave_total(mine_before ? mine.row_tiles : 0) + work.tile) * a.Hkv + work.head;
    }
    return true;
  }
};

// Keys that the rows of one row tile see between them, as key tiles
// [first, last), and this split's share of them.
template <int MT, int KT>
__device__ __forceinline__ void paged_range(const PagedArgs& a, const PagedWork& wk, int& first,
                                            int& last) {
  const PagedRequest& q = wk.req;
  const int limit = paged_limit(a, q.len);
  const long long row0 = (long long)wk.tile * MT;
  const int i0 = (int)(row0 / a.G);
  const int i1 = (int)min((row0 + MT - 1) / a.G, (long long)q.n - 1);
  const int past = q.len - q.n;
  const int hi = a.causal ? min(limit, past + i1 + 1) : limit;
  const int lo = first_seen(a, past + i0);
  int t0 = lo / KT, t1 = hi > lo ? (hi + KT - 1) / KT : t0;
  const int per = (t1 - t0 + wk.splits - 1) / wk.splits;
  first = min(t0 + wk.split * per, t1);
  last = min(first + per, t1);
}

__device__ __forceinline__ void paged_describe(const PagedArgs& a, const PagedWork& wk, int MT) {
  if (wk.split != 0 || wk.group < 0 || wk.group >= a.rec.groups || threadIdx.x != 0) return;
  int* d = a.rec.desc + (size_t)wk.group * kDescInts;
  const long long left = (long long)wk.req.n * a.G - (long long)wk.tile * MT;
  d[0] = wk.splits;
  d[1] = wk.rec;
  d[2] = wk.req.tok0;
  d[3] = wk.tile * MT;
  d[4] = (int)min(left, (long long)MT);
}

typedef void (*PagedFn)(PagedArgs);
PagedFn paged_decode_fn(bool bf16, bool fp8, int D, bool aligned);

}  // namespace dbk
