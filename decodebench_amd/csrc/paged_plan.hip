// paged_plan.hip -- block tables, positions and cache slots of a step's tokens,
// from the requests' lengths.
//
//   n_r = new_r (as far as the step's T rows go), q_start = exclusive sum of n,
//   kv_len_r = past_r + n_r; request r holds ceil(past_r / page) pages and takes
//   ceil(kv_len_r / page) less that many from the free list, requests in order.
//   Token i of request r: position past_r + i, slot page number * page size +
//   position % page size.
//
// A page that a request takes is begun by one of its new tokens, so the token
// at a page's start writes the table entry and no thread waits for another.
// One launch; its latency, not its few bytes, is the cost.  Workgroup b has
// the tokens 256 b .. 256 b + 255 and b + grid, ... ; each workgroup walks all
// requests in rounds of 1024 (two prefix sums: tokens, then pages) and keeps a
// round in LDS while its tokens look theirs up by bisection.  The workgroups
// repeat the prefix sums instead of waiting for one another's.
#include "db_device.h"
#include "db_kernels.h"

namespace dbk {

namespace {

constexpr int kThreads = 256;
constexpr int kPer = 4;  // requests a thread in a round
constexpr int kRound = kThreads * kPer;

struct Wave {
  unsigned long long sums[kThreads / kWave];
};

// Exclusive prefix sum of `v` over the workgroup's threads; `all` is the sum.
__device__ __forceinline__ unsigned long long block_before(unsigned long long v, Wave& sh,
                                                           unsigned long long& all) {
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  unsigned long long incl = v;
  for (int d = 1; d < kWave; d <<= 1) {
    const unsigned long long u = __shfl_up(incl, d);
    if (lane >= d) incl += u;
  }
  __syncthreads();
  if (lane == kWave - 1) sh.sums[wave] = incl;
  __syncthreads();
  unsigned long long before = incl - v;
  all = 0;
  for (int w = 0; w < kThreads / kWave; ++w) {
    if (w < wave) before += sh.sums[w];
    all += sh.sums[w];
  }
  return before;
}

__global__ __launch_bounds__(kThreads) void paged_plan_kernel(PlanCall c) {
  __shared__ Wave s_sum;
  __shared__ int s_start[kRound + 1];  // first token of the round's requests
  __shared__ int s_past[kRound], s_page[kRound];  // and where their pages begin in the free list

  const long long fs = c.free_start ? max(c.free_start[0], 0) : 0;
  unsigned long long tokens = 0, pages = 0;  // of the rounds before
  for (int r0 = 0, round = 0; r0 < c.R; r0 += kRound, ++round) {
    int past[kPer], n[kPer], want[kPer];
    unsigned long long sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int r = r0 + threadIdx.x * kPer + i;
      past[i] = r < c.R ? min(max(c.past[r], 0), 0x7FFFFFFF - c.T) : 0;
      n[i] = r < c.R ? min(max(c.fresh[r], 0), c.T) : 0;
      sum += n[i];
    }
    unsigned long long all;
    unsigned long long at = tokens + block_before(sum, s_sum, all);
    const unsigned long long round_tokens = min(tokens + all, (unsigned long long)c.T);
    unsigned long long takes = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int lo = (int)min(at, (unsigned long long)c.T);
      at += n[i];
      n[i] = (int)min(at, (unsigned long long)c.T) - lo;
      const int held = min((int)(((long long)past[i] + c.page - 1) / c.page), c.width);
      const int need = min((int)(((long long)past[i] + n[i] + c.page - 1) / c.page), c.width);
      want[i] = need - held;
      takes += want[i];
      s_start[threadIdx.x * kPer + i] = lo;
      s_past[threadIdx.x * kPer + i] = past[i];
    }
    unsigned long long more;
    unsigned long long page = pages + block_before(takes, s_sum, more);
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int r = r0 + threadIdx.x * kPer + i;
      // first free page of the request, less the pages it holds
      s_page[threadIdx.x * kPer + i] =
          (int)min(fs + (long long)page, 0x7FFFFFFFll);
      page += want[i];
      if (blockIdx.x == (unsigned)round % gridDim.x && r < c.R) {
        c.q_start[r] = s_start[threadIdx.x * kPer + i];
        c.kv_len[r] = past[i] + n[i];
        if (r == c.R - 1) c.q_start[c.R] = (int)round_tokens;
      }
    }
    if (threadIdx.x == 0) s_start[kRound] = (int)round_tokens;
    __syncthreads();
    const int t_lo = (int)min(tokens, (unsigned long long)c.T), t_hi = (int)round_tokens;
    for (int t0 = blockIdx.x * kThreads; t0 < t_hi; t0 += gridDim.x * kThreads) {
      const int t = t0 + threadIdx.x;
      if (t < t_lo || t >= t_hi) continue;
      // the last request that starts at or before token t
      int lo = 0, hi = kRound;
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_start[mid] <= t) lo = mid; else hi = mid;
      }
      const int pos = s_past[lo] + (t - s_start[lo]);
      const int p = pos / c.page;
      const int held = (int)(((long long)s_past[lo] + c.page - 1) / c.page);
      int number = -1;
      if (p < c.width) {
        int* entry = c.table + (size_t)(r0 + lo) * c.table_row + p;
        if (p < held) {
          number = *entry;
        } else {
          const long long f = (long long)s_page[lo] + (p - held);
          number = f < c.free_count ? c.free_pages[f] : -1;
          if (pos == p * c.page) *entry = number;
        }
      }
      c.position[t] = pos;
      c.slot[t] = number < 0 ? -1ll : (long long)number * c.page + (pos - p * c.page);
    }
    tokens += all;
    pages += more;
  }
  // rows behind the last token
  const int end = (int)min(tokens, (unsigned long long)c.T);
  for (int t = end + blockIdx.x * kThreads + threadIdx.x; t < c.T; t += gridDim.x * kThreads) {
    c.position[t] = 0;
    c.slot[t] = -1;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) {
    c.free_next[0] = (int)min(fs + (long long)pages, 0x7FFFFFFFll);
    if (c.R == 0) c.q_start[0] = 0;
  }
}

}  // namespace

hipError_t launch_paged_plan(const PlanCall& c, int cu_count, hipStream_t stream) {
  const int blocks = (c.T + kThreads - 1) / kThreads;
  hipLaunchKernelGGL(paged_plan_kernel, dim3(max(1, min(blocks, cu_count))), dim3(kThreads), 0,
                     stream, c);
  return hipGetLastError();
}

}  // namespace dbk
