// The residual stream at a block's two ends, and the quantiser of the int8 products.
//
// okc_block_norm, per token row (r: residual, y: the block's output, both bf16 or f32, all arithmetic in f32):
//   z  = y * rsqrt(mean(y^2) + eps) * post_gain      (norm after the block; optional)
//   r' = residual_scale * r + block_scale * g * z    (gate g per channel, token or element, optionally a sigmoid's)
//   x  = r' * rsqrt(mean(r'^2) + eps) * pre_gain     (norm before the next block; optional) -> bf16, f32 or int8 rows
// r' is normalised as it is in registers, before it is rounded to its own type.
//
// What bounds it: HBM for many rows (each tensor is read or written once; the row stays in registers between the two
// norms), the latency of one row's three dependent reductions for few.  A CTA per row: the thread count is chosen so
// that a thread holds 8 values for few rows (short chains) and up to 32 for many (fewer barriers a byte).
#include "rows.cuh"

namespace okc {

// most threads of a CTA: with 32 values of each tensor in registers a thread needs up to 128 registers
constexpr int row_threads(int chunks) { return chunks == 4 ? 512 : 1024; }

template <int kChunks, bool kVec>
__global__ void __launch_bounds__(row_threads(kChunks)) okc_block_norm(const BlockNormParams p) {
  __shared__ float red_post[32], red_pre[32];
  __shared__ uint32_t red_max[32];
  const int tid = threadIdx.x, nt = blockDim.x, H = p.H;
  const int64_t row = blockIdx.x;
  float r[kChunks][8];
  {
    const void* src = p.res_f32 ? static_cast<const void*>(static_cast<const float*>(p.res) + row * p.res_stride)
                                : static_cast<const void*>(static_cast<const uint16_t*>(p.res) + row * p.res_stride);
#pragma unroll
    for (int j = 0; j < kChunks; ++j) load_chunk<kVec>(src, p.res_f32, j, tid, nt, H, r[j]);
  }
  if (p.blk) {
    float y[kChunks][8];
    const void* src = p.blk_f32 ? static_cast<const void*>(static_cast<const float*>(p.blk) + row * p.blk_stride)
                                : static_cast<const void*>(static_cast<const uint16_t*>(p.blk) + row * p.blk_stride);
#pragma unroll
    for (int j = 0; j < kChunks; ++j) load_chunk<kVec>(src, p.blk_f32, j, tid, nt, H, y[j]);
    float mul = p.blk_scale;
    if (p.gate && p.gate_col_stride == 0) {       // one gate value for the row
      const int64_t o = row * p.gate_stride;
      float g = p.gate_f32 ? static_cast<const float*>(p.gate)[o]
                           : __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(p.gate)[o]) << 16);
      if (p.gate_sigmoid) g = 1.f / (1.f + __expf(-g));
      mul *= g;
    }
    if (p.post_gain) {
      float ss = 0.f;
#pragma unroll
      for (int j = 0; j < kChunks; ++j)
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(y[j][e], y[j][e], ss);
      const float rstd = rsqrtf(cta_sum(ss, red_post) / static_cast<float>(H) + p.eps);
#pragma unroll
      for (int j = 0; j < kChunks; ++j) {
        float g[8];
        load_chunk<kVec>(p.post_gain, true, j, tid, nt, H, g);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[j][e] = y[j][e] * rstd * g[e];
      }
    }
    if (p.gate && p.gate_col_stride != 0) {
      const int64_t o = row * p.gate_stride;
      const void* gsrc = p.gate_f32 ? static_cast<const void*>(static_cast<const float*>(p.gate) + o)
                                    : static_cast<const void*>(static_cast<const uint16_t*>(p.gate) + o);
#pragma unroll
      for (int j = 0; j < kChunks; ++j) {
        float g[8];
        load_chunk<kVec>(gsrc, p.gate_f32, j, tid, nt, H, g);
#pragma unroll
        for (int e = 0; e < 8; ++e) y[j][e] *= p.gate_sigmoid ? 1.f / (1.f + __expf(-g[e])) : g[e];
      }
    }
    void* dst = p.res_f32 ? static_cast<void*>(static_cast<float*>(p.res_out) + row * p.res_out_stride)
                          : static_cast<void*>(static_cast<uint16_t*>(p.res_out) + row * p.res_out_stride);
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
#pragma unroll
      for (int e = 0; e < 8; ++e) r[j][e] = p.res_scale * r[j][e] + mul * y[j][e];
      store_chunk<kVec>(dst, p.res_f32, j, tid, nt, H, r[j]);
    }
  }
  if (!p.pre_gain) return;
  float ss = 0.f;
#pragma unroll
  for (int j = 0; j < kChunks; ++j)
#pragma unroll
    for (int e = 0; e < 8; ++e)
      // columns past the row's end hold zeros that a non-finite `mul` would have turned into NaN
      if (row_col<kVec>(j, e, tid, nt) < H) ss = fmaf(r[j][e], r[j][e], ss);
  const float rstd = rsqrtf(cta_sum(ss, red_pre) / static_cast<float>(H) + p.eps);
  uint32_t amax = 0;
#pragma unroll
  for (int j = 0; j < kChunks; ++j) {
    float g[8];
    load_chunk<kVec>(p.pre_gain, true, j, tid, nt, H, g);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      r[j][e] = r[j][e] * rstd * g[e];
      if (row_col<kVec>(j, e, tid, nt) < H) amax = max(amax, abs_bits(r[j][e]));
    }
  }
  if (p.out_kind == kRowsInt8) {
    const RowScale s = row_scale(cta_max(amax, red_max));
    int8_t* dst = static_cast<int8_t*>(p.out) + row * p.out_stride;
#pragma unroll
    for (int j = 0; j < kChunks; ++j) store_chunk_q<kVec>(dst, j, tid, nt, H, r[j], s.inv);
    if (tid == 0) p.out_scale[row] = s.scale;
  } else {
    const bool f32 = p.out_kind == kRowsF32;
    void* dst = f32 ? static_cast<void*>(static_cast<float*>(p.out) + row * p.out_stride)
                    : static_cast<void*>(static_cast<uint16_t*>(p.out) + row * p.out_stride);
#pragma unroll
    for (int j = 0; j < kChunks; ++j) store_chunk<kVec>(dst, f32, j, tid, nt, H, r[j]);
  }
}

// Rows -> int8 values and a scale per row.  A CTA per row; a row that fits the CTA's registers is read once, a longer
// one (more than 16384 columns) a second time, from L2.
template <int kChunks, bool kVec>
__global__ void __launch_bounds__(row_threads(kChunks)) okc_quantize_rows(const QuantizeParams p) {
  __shared__ uint32_t red[32];
  griddep_launch_dependents();     // a product kernel behind this one may set itself up; it waits before it reads the rows
  const int tid = threadIdx.x, nt = blockDim.x;
  const int64_t row = blockIdx.x;
  const void* src = p.x_f32 ? static_cast<const void*>(static_cast<const float*>(p.x) + row * p.x_stride)
                            : static_cast<const void*>(static_cast<const uint16_t*>(p.x) + row * p.x_stride);
  int8_t* dst = p.q + row * p.q_stride;
  float v[kChunks][8];
  uint32_t amax = 0;
  const int passes = (p.cols + nt * 8 * kChunks - 1) / (nt * 8 * kChunks);
  for (int s = 0; s < passes; ++s) {
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      load_chunk<kVec>(src, p.x_f32, s * kChunks + j, tid, nt, p.cols, v[j]);
#pragma unroll
      for (int e = 0; e < 8; ++e) amax = max(amax, abs_bits(v[j][e]));
    }
  }
  const RowScale rs = row_scale(cta_max(amax, red));
  if (tid == 0) p.scale[row] = rs.scale;
  for (int s = 0; s < passes; ++s) {
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      if (passes > 1) load_chunk<kVec>(src, p.x_f32, s * kChunks + j, tid, nt, p.cols, v[j]);
      store_chunk_q<kVec>(dst, s * kChunks + j, tid, nt, p.cols, v[j], rs.inv);
    }
  }
}

// Threads of a row's CTA and chunks of eight columns a thread holds.
static void row_shape(int64_t rows, int cols, int& threads, int& chunks) {
  const int units = (cols + 7) / 8;
  chunks = 1;
  if (rows >= 2 * 148) chunks = units > 1024 ? 4 : units > 256 ? 2 : 1;
  while (chunks < 4 && (units + chunks - 1) / chunks > row_threads(chunks)) chunks *= 2;
  threads = ((units + chunks - 1) / chunks + 31) / 32 * 32;
  if (threads > row_threads(chunks)) threads = row_threads(chunks);
}

cudaError_t launch_block_norm(const BlockNormParams& p, int64_t rows, bool vec, cudaStream_t stream) {
  int threads, chunks;
  row_shape(rows, p.H, threads, chunks);
  const dim3 grid(static_cast<unsigned>(rows)), block(threads);
  if (chunks == 1) return vec ? launch_kernel(okc_block_norm<1, true>, grid, block, 0, stream, false, p) : launch_kernel(okc_block_norm<1, false>, grid, block, 0, stream, false, p);
  if (chunks == 2) return vec ? launch_kernel(okc_block_norm<2, true>, grid, block, 0, stream, false, p) : launch_kernel(okc_block_norm<2, false>, grid, block, 0, stream, false, p);
  return vec ? launch_kernel(okc_block_norm<4, true>, grid, block, 0, stream, false, p) : launch_kernel(okc_block_norm<4, false>, grid, block, 0, stream, false, p);
}

cudaError_t launch_quantize_rows(const QuantizeParams& p, int64_t rows, bool vec, cudaStream_t stream) {
  int threads, chunks;
  row_shape(rows, p.cols, threads, chunks);
  const dim3 grid(static_cast<unsigned>(rows)), block(threads);
  if (chunks == 1) return vec ? launch_kernel(okc_quantize_rows<1, true>, grid, block, 0, stream, false, p) : launch_kernel(okc_quantize_rows<1, false>, grid, block, 0, stream, false, p);
  if (chunks == 2) return vec ? launch_kernel(okc_quantize_rows<2, true>, grid, block, 0, stream, false, p) : launch_kernel(okc_quantize_rows<2, false>, grid, block, 0, stream, false, p);
  return vec ? launch_kernel(okc_quantize_rows<4, true>, grid, block, 0, stream, false, p) : launch_kernel(okc_quantize_rows<4, false>, grid, block, 0, stream, false, p);
}

}  // namespace okc
