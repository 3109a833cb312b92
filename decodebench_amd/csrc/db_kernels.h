// db_kernels.h -- host-side launchers shared by the kernel files and the C ABI.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>

#include "decodebench_hip.h"

namespace dbk {

// Launch geometry knobs; defaults are the tuned MI355X values.  They can be
// changed at run time through db_tune() for launch-shape sweeps; each host
// thread has its own set.
struct Tuning {
  int gemv_waves_per_cu = 0;   // 0: the default, 32 waves per CU
  int gemv_mfma_min_batch = 0; // smallest batch that takes the MFMA GEMV
                               // (0: the measured crossovers, 2 or 3 rows
                               // by mode and weight type, see launch_gemv)
  int f4_blocks_per_cu = 1;    // target F4 workgroups per CU
  int f4_min_tiles = 8;        // minimum 16-row tiles per F4 split
  int f4_waves = 0;            // waves per F4 workgroup (4 or 8; 0: auto)
  int f4_merge = 0;            // split merge: 0 automatic (in the same launch where
                               // the grid numbering allows), 1 the same, 2 second launch
  int f4_misplace = 0;         // test hook: F4 split s acts as if off its XCD when
                               // s % k == k - 1 (0: off)
  int f4_line = 0;             // F4 score layout: 0 auto, 1 whole-line K loads, 2 plain
  int f4_combine_groups = 0;   // split groups per F4 merge workgroup (0: auto)
  int f4_depth = 0;            // F4 tiles in flight per wave: 0 auto, 1 or 2
  int gemv_long_kc = 0;        // long-row MFMA GEMV k-steps per chunk: 0 auto, 2 or 4
  int gemv_long_gpw = 0;       // long-row MFMA GEMV row groups per workgroup: 0 auto, 1, 2, 4
  int gemv_long_stage = 0;     // long-row MFMA GEMV x: 0 auto, 1 direct, 2 LDS-staged
  int gemv_pair_min_batch = 0; // gate/up pair rows from which K = 2048 and 4096 take
                               // gemv_tile (0: 12, with the RMSNorm 17)
  int stream_waves = 0;        // db_stream_read waves per workgroup: 0 (4), 1, 2 or 4
  int gemv_pass_grid = 0;      // one-matrix MFMA GEMV above 16 rows: workgroups per
                               // 16-row pass (0: CUs / passes; else a multiple of 8)
  int gemv_xb = 0;             // 1: 32-row passes (rows 16..31 of x in LDS) on the
                               // full grid instead
  int gemv_tile = 0;           // batches of 2 rows and more (gemv_mfma_min_batch if set):
                               // 0 automatic, 1 gemv_tile, 2 never gemv_tile
  int gemv_splits = 0;         // K splits of gemv_tile where a workspace is given: 0 auto, 1..8
  int blocks_shape = 0;        // gemm_blocks: 0 automatic, 1..7 tiles of 256 x 256,
                               // 256 x 128, 128 x 64, 128 x 32, 64 x 64, 64 x 32, 32 x 32
  int blocks_parts = 0;        // parts of K of its tiles: 0 automatic, 1..16
  int f4_launch = 0;           // measurement hook for the two-launch F4: 0 both
                               // launches, 1 the split kernel only, 2 the merge only
};
Tuning& tuning();

// Compute units of the current device (cached per device ordinal).
int device_cu_count(int* err);
// XCDs (accelerator complex dies) of the current device, cached likewise.
int device_xcc_count(int* err);

enum GemvMode : int {
  kGemvPlain = 0,
  kGemvRmsNorm = 1,
  kGemvSwiGLU = 2,
  kGemvRmsNormSwiGLU = 3,
};

constexpr bool gemv_has_norm(int mode) {
  return mode == kGemvRmsNorm || mode == kGemvRmsNormSwiGLU;
}
constexpr bool gemv_is_swiglu(int mode) {
  return mode == kGemvSwiGLU || mode == kGemvRmsNormSwiGLU;
}

// Weights of one GEMV call: one matrix (two for the SwiGLU modes), fp16 or
// OCP e4m3 with one fp32 scale per output row.
struct GemvWeights {
  const void* w0;     // [N, K]  (gate in the SwiGLU modes)
  const void* w1;     // [N, K]  (up, SwiGLU modes only)
  const float* s0;    // [N]     row scales of w0 (fp8 only)
  const float* s1;    // [N]     row scales of w1 (fp8 SwiGLU only)
  bool fp8;
};

// y[B,N] = op(x[B,K]) . W^T  (fp16 activations in/out, fp32 accumulation).
//   kGemvPlain          : y = x W^T
//   kGemvRmsNorm        : y = fp16(fp16(x * rsqrt(mean(x^2) + eps)) * gamma) W^T
//   kGemvSwiGLU         : y = fp16(silu(fp16(x Wg^T)) * fp16(x Wu^T))
//   kGemvRmsNormSwiGLU  : the SwiGLU mode on the RMS-normalised x
// With fp8 weights every projection is fp32(sum) * row scale before its
// fp16 rounding.
// ws (ws_bytes of device memory, 16-byte aligned, or null) lets a call that
// gains from it split K over workgroups, see gemv_workspace_bytes.
hipError_t launch_gemv(GemvMode mode, const void* x, const void* gamma,
                       const GemvWeights& w, void* y, int B, int K, int N, float eps,
                       int cu_count, void* ws, size_t ws_bytes, hipStream_t stream);
// Bytes of workspace with which launch_gemv would split K (0: it would not).
size_t gemv_workspace_bytes(GemvMode mode, bool fp8, int B, int K, int N, int cu_count);

// MFMA variant for batches of up to 16 rows per pass (gemv_mfma.hip), fp16
// or e4m3 weights, K in {2048, 4096}.
bool gemv_mfma_supported(GemvMode mode, int B, int K, int N);
hipError_t launch_gemv_mfma(GemvMode mode, const void* x, const void* gamma,
                            const GemvWeights& w, void* y, int B, int K, int N, float eps,
                            int cu_count, hipStream_t stream);

// Batched GEMV on full 16 x 16 MFMA tiles with streamed activations
// (gemv_tile.hip): any K the contract allows, any N and batch.
// With splits > 1 the partial sums go to ws and a second launch adds them.
size_t gemv_tile_workspace_bytes(GemvMode mode, int splits, int B, int N);
hipError_t launch_gemv_tile(GemvMode mode, const void* x, const void* gamma,
                            const GemvWeights& w, void* y, int B, int K, int N, float eps,
                            int cu_count, int splits, void* ws, hipStream_t stream);

// Split-KV GQA decode attention with the log-sum-exp combine in-kernel.
size_t f4_workspace_bytes(int B, int Hq, int Hkv, int S, int D);
int f4_choose_splits(int B, int Hkv, int L, int cu_count);
// How a call of S splits runs: the splits actually used (never more than
// the 16-row tiles of L), tiles per split, whether the workgroups of a
// (batch, kv-head) pair are numbered onto one XCD, and whether the splits
// are merged in the same launch (else in a second one).
struct F4Plan {
  int splits;
  int tiles_per_split;
  bool xcd_map;
  bool fused_merge;
};
F4Plan f4_plan(int B, int Hkv, int L, int S, int nxcc, bool allow_fused_merge);
// nxcc: the device's XCD count (the in-launch merge runs only with 8).
// allow_fused_merge = false keeps the merge in the second launch whatever
// db_tune("f4_merge") says, so the workspace tickets are never read.
hipError_t launch_f4(const void* q, const void* k, const void* v, void* o,
                     void* ws, int B, int Hq, int Hkv, int L, int D, int S,
                     float scale, int nxcc, hipStream_t stream,
                     bool allow_fused_merge = true);

// Bytes of the per-device scratch array behind db_f4_splitkv_noalloc.
constexpr size_t kF4ScratchBytes = DB_F4_SCRATCH_BYTES;
// Device address of that array on the current device (looked up once per
// device with hipGetSymbolAddress).
hipError_t f4_scratch_address(void** out);

// A step over a paged KV cache: the arguments of the three entry points as the
// kernels take them (checked by the caller).
struct PlanCall {
  const int* past;       // [R] tokens of each request in the cache
  const int* fresh;      // [R] tokens of this step
  int* table;            // [R, width], rows table_row apart; taken pages are entered
  const int* free_pages; // [free_count]
  const int* free_start; // [1] or null: where the step's pages begin
  long long table_row;
  int free_count, width, page, R, T;
  int* q_start;          // [R + 1]
  int* kv_len;           // [R]
  int* position;         // [T]
  long long* slot;       // [T]
  int* free_next;        // [1]
};
hipError_t launch_paged_plan(const PlanCall& c, int cu_count, hipStream_t stream);

struct RopeCall {
  const void* qkv;         // [T, (Hq + 2 Hkv) D], rows qkv_row elements apart
  const int* position;     // [axes, T]
  const long long* slot;   // [T]
  const float* freq;       // [rot / 2]
  void* q;                 // [T, Hq, D]
  db_paged_cache cache;
  long long qkv_row;
  int T, Hq, rot, interleaved;
  bool bf16;
  unsigned axes[8];        // axis of pair i: bits 2 (i % 16) of word i / 16
};
hipError_t launch_rope_append(const RopeCall& c, int cu_count, hipStream_t stream);

struct PagedCall {
  const void* q;        // [T, Hq, D]
  void* o;              // [T, Hq, D]
  const int* table;     // [R, width]
  const int* q_start;   // [R + 1]
  const int* kv_len;    // [R]
  db_paged_cache cache;
  long long q_token, q_head, table_row;
  int T, R, Hq, width, max_new, causal, window;
  float scale;
  bool bf16;
};
// Bytes of workspace, the first *zeroed of them zero between calls.
size_t paged_workspace_bytes(const PagedCall& c, int cu_count, size_t* zeroed);
hipError_t launch_paged_attention(const PagedCall& c, int cu_count, void* ws, hipStream_t stream);

// Block-scaled e4m3 (quant_blocks.hip, gemm_blocks.hip): the arguments of the
// entry points as the kernels take them (checked by the caller).
struct QuantCall {
  const void* x;      // [T, K], rows x_row elements apart
  void* q;            // [T, K]
  float* scale;       // [T, ceil(K / 128)] at the strides below
  long long x_row, scale_t, scale_b;
  int T, K;
  bool bf16;
};
hipError_t launch_quantize_blocks(const QuantCall& c, hipStream_t stream);

struct GemmBlocksCall {
  const void* x;         // [T, K] e4m3, rows x_row apart; of y's type where plan.fused
  const float* x_scale;  // [T, ceil(K / 128)] at the strides below; null where plan.fused
  const void* W;         // [N, K] e4m3
  const float* w_scale;  // [ceil(N / 128), ceil(K / 128)]
  void* y;               // [T, N]
  long long x_row, xs_t, xs_b;
  int T, K, N;
  bool bf16;             // type of y
};
// How a product runs: the kernel's shape, K in parts of `each` blocks whose fp32
// sums a second launch adds, workgroups, bytes of workspace for the sums.
struct GemmBlocksPlan {
  int shape, parts, each, grid, pitch;  // few tokens: `each` outputs a workgroup
  unsigned magic;  // few tokens: 2^32 / blocks of K, rounded up
  bool fused;      // 16-bit activations are quantised in the same launch
  size_t bytes;
  float* sums;  // [parts, T, pitch]
};
GemmBlocksPlan gemm_blocks_plan(int T, int K, int N, int cu_count);
hipError_t launch_gemm_blocks(const GemmBlocksCall& c, const GemmBlocksPlan& plan,
                              hipStream_t stream);

// A mixture-of-experts layer (moe_route.hip, moe_experts.hip).
struct MoeRouteCall {
  const void* x;       // [T, H], rows x_row elements apart
  const void* router;  // [E, H]
  int* experts;        // [T, k]
  float* weights;      // [T, k]
  double* logits;      // [parts, T, E] workspace: sums over parts of H
  long long x_row;
  int T, H, E, k, parts;
  bool renormalize, bf16;
};
hipError_t launch_moe_route(const MoeRouteCall& c, hipStream_t stream);
int moe_logit_parts(int T, int H, int E);
hipError_t launch_moe_logits(const MoeRouteCall& c, hipStream_t stream);  // its first half

struct MoeExpertsCall {
  const void* x;         // [T, H], rows x_row elements apart
  const int* experts;    // [T, k]
  const float* weights;  // [T, k]
  void* y;               // [T, H]
  db_moe w;
  long long x_row;
  int T, k;
  bool bf16;
  // workspace
  int* order;    // [T k] pairs sorted by expert
  int* tiles;    // count, then (expert, first slot, pairs) of each tile
  void* h;       // [T k, I] by slot, of x's type; of few tokens by pair, fp32
  float* parts;  // [T k, H] by pair
};
// The experts of a few tokens (moe_few.hip), whose pairs each read their expert's
// weights: with `logits` the choice among them is theirs too, and `experts` and
// `weights` (which c has as well) are written.
struct MoeFewCall {
  MoeExpertsCall c;
  const double* logits;  // [T, E], or null: experts and weights are given
  int* experts;
  float* weights;
  bool renormalize;
};
bool moe_few(const db_moe& m, int T, int k);
hipError_t launch_moe_few(const MoeFewCall& f, hipStream_t stream);
// Lays the workspace out from ws on; returns its bytes.
size_t moe_experts_workspace(MoeExpertsCall& c, void* ws);
hipError_t launch_moe_experts(const MoeExpertsCall& c, hipStream_t stream);

// Read-only streaming probe (stream_probe.hip): `bytes` (a multiple of
// kb_per_wave KB, kb_per_wave in {4, 8, 16}) read once, kb_per_wave KB per
// wave; sink needs bytes / 16 words and is written only when the folded
// data equals `magic`.
hipError_t launch_stream_read(const void* src, size_t bytes, int kb_per_wave, unsigned magic,
                              unsigned* sink, hipStream_t stream);

}  // namespace dbk
