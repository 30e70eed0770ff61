// Kernel parameter blocks and host launchers shared by the translation units of the library.
#pragma once
#include <utility>

#include "format.cuh"

namespace okc {

struct RouteParams {
  const float* logits;
  const int32_t* ids_in;
  const float* wts_in;
  int32_t* ids_out;
  float* wts_out;
  int32_t* meta;
  int32_t* counts;
  int32_t* done;                  // per-item completion counts of the GEMM launch: the sort leaves them (and the unit counters) at zero
  int4* items;
  int32_t* sorted;
  int32_t* pos;
  float* wsorted;
  int T, E, k, kk, slots, local_start, local_count, has_shared, own_t0, own_t1, max_items, chunk_rows;
  // router: 0 = softmax top-k, 1 = sigmoid(mult * logit) + bias chooses, scores renormalised
  int router_mode;
  float router_mult;
  const float* router_bias;       // f32 [E] or null
  // logits from the token rows (null: `logits` is given)
  const float* router_w;          // f32 [E, H]
  const uint16_t* hidden;         // bf16 [T, hidden_stride]
  int64_t hidden_stride;
  int H, router_splits;
  float* router_part;             // scratch f32 [router_splits, T, E]
  // the same logits on the tensor cores: router_w as bf16 hi + lo rows [2 E, H]
  const uint16_t* router_w_split;
  CUtensorMap router_wmap, router_hmap;
  int router_kb_per_cta;
};
cudaError_t launch_router_mma(const CUtensorMap& wmap, const CUtensorMap& hmap, float* part, int32_t* meta, int T, int E, int H,
                              int kb_per_cta, cudaStream_t stream);
cudaError_t launch_router_split(const float* w, void* out, size_t n, cudaStream_t stream);
cudaError_t launch_route(const RouteParams& p, cudaStream_t stream);
cudaError_t launch_gather(const void* hidden, int64_t stride, int32_t* meta, const int32_t* sorted, int kk,
                          int H, int R, void* xg, int32_t* done, int max_items, cudaStream_t stream);

cudaError_t launch_gather_norm(const void* hidden, int64_t stride, int hidden_f32, const float* gain, float eps,
                               int32_t* meta, const int32_t* sorted, int kk, int H, int R, void* xg, int32_t* done,
                               int max_items, cudaStream_t stream);

struct RepackParams {
  const uint8_t* w;
  const uint8_t* sf;
  uint8_t* out;
  int rows, K, pairs, stages, first_slot, count, is_w13, inter;
  size_t expert_bytes;
};
cudaError_t launch_repack(const RepackParams& p, cudaStream_t stream);
struct UnpackParams {
  const uint8_t* packed;
  uint16_t* out;
  int K, pairs, stages, is_w13, inter;
};
cudaError_t launch_unpack(const UnpackParams& p, cudaStream_t stream);

// One of the two GEMM phases of a step: 0 = gate_up on w13 (token operand xg), 1 = down on w2
// (token operand inter).
struct PhaseParams {
  CUtensorMap bmap[5];        // token operand [rows, K] bf16, box = 64 elements x {4, 8, 16, 32, 64} rows
  const uint8_t* wpacked;     // stage images of every expert slot
  const float* gs;            // [slots] global scales
  int pairs;                  // units per work item
  int stages;                 // K / 256
  size_t expert_bytes;
};

// The grouped-GEMM kernel works through the units of phases [phase_lo, phase_hi]: both phases in one
// launch (gate_up units first, then down units, handed out by an atomic counter) or one phase.
struct MoeGemmParams {
  PhaseParams ph[2];
  const int32_t* meta;
  const int4* items;
  int32_t* work_counter;      // units handed out behind the first grid-size ones (zeroed by the combine kernel of the launch before)
  int32_t* done;              // [items] epilogue warps that finished a gate_up unit of the item
  int phase_lo, phase_hi;
  uint16_t* inter;            // bf16 [Rpad, I]     (phase 0 output, phase 1 token operand)
  int I;
  float* y;                   // f32 [R, H]         (phase 1 output)
  const int32_t* sorted;
  const float* wsorted;
  int H;
  int weighted;
  // Token rows of the gate_up phase taken straight from the caller's `hidden` (no gathered copy): one TMA copy
  // per row and 64-element block, the row being the token of the route at that sorted position.
  int direct_rows;
  int kk;                     // routes per token: token of sorted entry s = s / kk
  CUtensorMap hmap;           // hidden [T, H] bf16 with the caller's row stride, box = 64 elements x 1 row
};
cudaError_t launch_gemm(const MoeGemmParams& p, int grid, cudaStream_t stream);

// The exchange kernels of the expert-parallel step (ep.cu).
struct EpParams {
  uint8_t* peer[kEpMaxRanks];   // this process's mapping of every rank's exchange buffer
  int rank, world, tokens, H, E;
  size_t off_hidden, off_logits, off_partial;
  const uint16_t* hidden_own;   // push: bf16 [tokens / world, hidden_stride]
  int64_t hidden_stride;
  const float* logits_own;      // push: f32 [tokens / world, E]
  uint16_t* out;                // reduce: bf16 [tokens / world, H]
  unsigned long long wait_ns;   // limit of every wait on another rank
};
cudaError_t launch_ep_push(const EpParams& p, cudaStream_t stream);
cudaError_t launch_ep_reduce(const EpParams& p, cudaStream_t stream);
cudaError_t launch_ep_push_route_sort(const EpParams& p, const RouteParams& rp, cudaStream_t stream);
cudaError_t launch_ep_mark_arrived(const EpParams& p, int which, int from, cudaStream_t stream);

struct CombineParams {
  const float* y;
  const int32_t* pos;
  const float* wsorted;
  const uint16_t* post_w;
  void* out;
  int kk, H, out_f32;
  int32_t* meta;              // control words and per-item counts of the GEMM launch before: cleared by the first CTA
  int32_t* done;
  int max_items;
};
cudaError_t launch_combine(const CombineParams& p, int T, cudaStream_t stream);
cudaError_t launch_ep_combine_reduce(const EpParams& p, const CombineParams& c, cudaStream_t stream);

cudaError_t launch_cast(const float* in, void* out_bf16, int64_t n, cudaStream_t stream);
cudaError_t launch_wait_timeout_probe(int32_t* status, cudaStream_t stream);

// The residual stream around a block (norm.cu).
enum RowsKind { kRowsBf16 = 0, kRowsF32 = 1, kRowsInt8 = 2 };
struct BlockNormParams {
  const void* res;            // residual rows (bf16 or f32), row strides in elements
  const void* blk;            // block output rows or null: only the norm before a block runs
  const void* gate;           // or null
  void* res_out;
  void* out;
  float* out_scale;           // int8 rows only
  const float* post_gain;     // f32 [H] or null: no norm after the block
  const float* pre_gain;      // f32 [H] or null: no norm before the next block
  int64_t res_stride, blk_stride, gate_stride, res_out_stride, out_stride;
  int gate_col_stride;        // 0: one value a row, 1: one a channel
  int H, res_f32, blk_f32, gate_f32, gate_sigmoid, out_kind;
  float res_scale, blk_scale, eps;
};
cudaError_t launch_block_norm(const BlockNormParams& p, int64_t rows, bool vec, cudaStream_t stream);

struct QuantizeParams {
  const void* x;
  int8_t* q;
  float* scale;
  int64_t x_stride, q_stride;
  int cols, x_f32;
  int product_follows;        // the next launch is the product of these rows: it may start early
};
cudaError_t launch_quantize_rows(const QuantizeParams& p, int64_t rows, bool x_vec, bool q_vec, cudaStream_t stream);
cudaError_t norm_read_status(cudaStream_t stream, int32_t* code);
cudaError_t launch_norm_probe_timeout(cudaStream_t stream);

// The int8 products (int8.cu).
struct Int8Params {
  const void* x;              // token rows: int8 with x_scale, or (one token only) bf16 / f32 rows quantised in the kernel
  const float* x_scale;
  const int8_t* w;            // weight rows, K int8 values each
  const float* w_scale;       // f32, one per weight row
  const float* bias;          // f32 [N] or null
  void* out;
  int64_t x_stride, w_stride, out_stride;
  int x_kind;                 // RowsKind
  int x_vec;                  // 16-byte loads of the token rows are possible
  int out_f32, out_vec;       // out_vec: 16-byte stores of an output row are possible from any column that is a multiple of 8
  int T, K, N;                // N = outputs: weight rows, or half of them for the gated product
};
constexpr int kInt8OneMaxK = 16384;         // up to here the product of one token quantises it itself
constexpr int kInt8MaxK = 131071;          // 128 * 128 * K stays below 2^31
cudaError_t launch_int8_one(const Int8Params& p, bool gated, cudaStream_t stream);
// quantised_here: launched right behind the kernel that quantised its tokens
cudaError_t launch_int8_mid(const Int8Params& p, bool gated, bool quantised_here, cudaStream_t stream);
cudaError_t launch_int8_many(const Int8Params& p, bool gated, bool quantised_here, cudaStream_t stream);
bool int8_use_many(int T, int K, int N, bool gated);
cudaError_t int8_read_status(cudaStream_t stream, int32_t* code);
cudaError_t launch_int8_probe_timeout(cudaStream_t stream);
// Tensor map of int8 rows (abi.cu): box = 128 bytes x box_rows, 128-byte swizzle, zero fill outside.
bool encode_bytes_map(CUtensorMap* map, const void* base, uint64_t rows, uint64_t K, uint64_t row_stride, uint32_t box_rows);
bool encode_blocks_map(CUtensorMap* map, const void* base, uint64_t rows, uint32_t halves, uint64_t K, uint64_t row_stride,
                       uint32_t box_rows, uint32_t blocks);
// Tensor map of bf16 result rows (row stride in elements): box = 32 columns x 32 rows, 64-byte swizzle.
bool encode_bf16_out_map(CUtensorMap* map, void* base, uint64_t rows, uint64_t cols, uint64_t row_stride);

// The largest dynamic shared memory a kernel may be launched with is state of the kernel on its device, not of a call: a
// launch sets it to one constant of the kernel, the most that any call asks for.  Set to each call's own size, a call of
// another thread lowers it between this call's setting and its launch, which then fails.
constexpr int kMostDynamicSmem = 226 * 1024;      // for kernels that declare less than a kilobyte themselves

// Launch with (pdl = true) or without the programmatic-serialization attribute.
template <typename... KArgs, typename... Args>
inline cudaError_t launch_kernel(void (*kernel)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream,
                                 bool pdl, Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = pdl ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

}  // namespace okc
