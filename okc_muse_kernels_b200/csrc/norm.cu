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
//
// These kernels are launched plainly: each starts when the one before it has completed.  Only the tiled int8 products
// start early, behind the quantiser of their own tokens.  With every launch programmatic, CTAs of the next call that wait
// hold registers that clusters of the product before them still need, and long queues of calls came to a stop.
#include "rows.cuh"

namespace okc {

__device__ int32_t g_norm_status;      // code of the first wait that ran out since the last read

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
    for (int j = 0; j < kChunks; ++j) store_chunk_q<kVec>(dst, j, tid, nt, H, r[j], s);
    if (tid == 0) p.out_scale[row] = s.scale;
  } else {
    const bool f32 = p.out_kind == kRowsF32;
    void* dst = f32 ? static_cast<void*>(static_cast<float*>(p.out) + row * p.out_stride)
                    : static_cast<void*>(static_cast<uint16_t*>(p.out) + row * p.out_stride);
#pragma unroll
    for (int j = 0; j < kChunks; ++j) store_chunk<kVec>(dst, f32, j, tid, nt, H, r[j]);
  }
}

// The same for many rows that 16-byte accesses can reach: persistent CTAs, each with a ring of rows in shared memory that
// bulk copies fill ahead of it, so that HBM does not wait for the two dependent sums of a row.  What is left is issue
// slots: pairs of f32 an instruction, and as many CTAs an SM as registers allow (the gains stay in L1, not in shared
// memory, for that).  4096 x 5120, everything bf16, a gate per element, inputs larger than L2: 43.0 us in a graph (210 MB: 4.9
// TB/s), 45.3 call after call (4.6); with one vector for both gains 38.6, a CTA per row then 65.1.  Without the gate 32.8 us
// (168 MB: 5.1 TB/s).  f32 residual, 4096 x 4096 int8 rows out: 39.7 us with a bf16 block (184 MB: 4.6 TB/s), 46 with an f32
// one (218 MB: 4.7).
constexpr int kStreamStages = 2;                 // rows of a ring; more do not help (4096 x 4096: 2 / 3 / 8 rows 37.8 / 38.7 / 39.4 us)
constexpr int kStreamSmem = 200 * 1024;          // an SM's shared memory for rings; L1 keeps the rest, for the gains
template <int kChunks, bool kInt8>
__global__ void __launch_bounds__(512, kChunks == 4 ? 1 : 2) okc_block_norm_stream(const BlockNormParams p, int rows, int row_bytes) {
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ uint64_t bar_full[kStreamStages];
  __shared__ int abort_code;
  __shared__ float red_post[2][32], red_pre[2][32];
  __shared__ uint32_t red_max[2][32];
  const int tid = threadIdx.x, nt = blockDim.x, H = p.H;
  const uint32_t res_bytes = static_cast<uint32_t>(H) * (p.res_f32 ? 4 : 2), blk_bytes = static_cast<uint32_t>(H) * (p.blk_f32 ? 4 : 2);
  const bool gate_rows = p.gate && p.gate_col_stride != 0 && p.gate_stride != 0, gate_cols = p.gate && p.gate_col_stride != 0 && p.gate_stride == 0;
  const uint32_t gate_bytes = gate_rows ? static_cast<uint32_t>(H) * (p.gate_f32 ? 4 : 2) : 0;
  auto fetch = [&](int row, int st) {
    const uint32_t bar = smem_u32(&bar_full[st]);
    const uint32_t dst = smem_u32(ring) + st * row_bytes;
    mbar_expect_tx(bar, res_bytes + blk_bytes + gate_bytes);
    bulk_g2s(dst, static_cast<const uint8_t*>(p.res) + row * p.res_stride * (p.res_f32 ? 4 : 2), res_bytes, bar);
    bulk_g2s(dst + res_bytes, static_cast<const uint8_t*>(p.blk) + row * p.blk_stride * (p.blk_f32 ? 4 : 2), blk_bytes, bar);
    if (gate_rows) bulk_g2s(dst + res_bytes + blk_bytes, static_cast<const uint8_t*>(p.gate) + row * p.gate_stride * (p.gate_f32 ? 4 : 2), gate_bytes, bar);
  };
  if (tid == 0) {
    for (int i = 0; i < kStreamStages; ++i) mbar_init(smem_u32(&bar_full[i]), 1);
    abort_code = 0;
    mbar_fence_init();
    for (int i = 0; i < kStreamStages && blockIdx.x + i * gridDim.x < static_cast<unsigned>(rows); ++i) fetch(blockIdx.x + i * gridDim.x, i);
  }
  __syncthreads();
  const float over_h = 1.f / static_cast<float>(H);
  const F2 res_scale = f2_pack(p.res_scale, p.res_scale);
  int st = 0, n = 0;
  uint32_t ph = 0;
  for (int row = blockIdx.x; row < rows; row += gridDim.x, ++n) {
    float mul = p.blk_scale;
    if (p.gate && p.gate_col_stride == 0) {
      const int64_t o = row * p.gate_stride;
      float g = p.gate_f32 ? static_cast<const float*>(p.gate)[o]
                           : __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(p.gate)[o]) << 16);
      if (p.gate_sigmoid) g = 1.f / (1.f + __expf(-g));
      mul *= g;
    }
    // a wait that runs out does not leave the loop (the other threads count on this one's barriers): the row's result is
    // then undefined and the status word says so
    const bool landed = mbar_wait(smem_u32(&bar_full[st]), ph, &abort_code, 0x81);
    const uint8_t* const src = ring + st * row_bytes;
    F2 r[kChunks][4];
    {
      F2 y[kChunks][4];
#pragma unroll
      for (int j = 0; j < kChunks; ++j) {
        const int c = (j * nt + tid) * 8;
        y[j][0] = y[j][1] = y[j][2] = y[j][3] = 0ull;
        if (c < H) load8_f2(src + res_bytes, p.blk_f32, c, y[j]);
      }
      if (p.post_gain) {
        F2 sum = 0ull;
#pragma unroll
        for (int j = 0; j < kChunks; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e) sum = f2_fma(y[j][e], y[j][e], sum);
        float lo, hi;
        f2_unpack(sum, lo, hi);
        const float rstd = rsqrtf(cta_sum(lo + hi, red_post[n & 1]) * over_h + p.eps);
        const F2 rstd2 = f2_pack(rstd, rstd);
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
          const int c = (j * nt + tid) * 8;
          if (c < H) {
            F2 g[4];
            load8_f2(p.post_gain, true, c, g);
#pragma unroll
            for (int e = 0; e < 4; ++e) y[j][e] = f2_mul(f2_mul(y[j][e], rstd2), g[e]);
          }
        }
      }
      if (gate_rows || gate_cols) {
        const void* gsrc = gate_rows ? static_cast<const void*>(src + res_bytes + blk_bytes) : p.gate;
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
          const int c = (j * nt + tid) * 8;
          if (c < H) {
            F2 g[4];
            load8_f2(gsrc, p.gate_f32, c, g);
            if (p.gate_sigmoid) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                float lo, hi;
                f2_unpack(g[e], lo, hi);
                g[e] = f2_pack(1.f / (1.f + __expf(-lo)), 1.f / (1.f + __expf(-hi)));
              }
            }
#pragma unroll
            for (int e = 0; e < 4; ++e) y[j][e] = f2_mul(y[j][e], g[e]);
          }
        }
      }
      const F2 mul2 = f2_pack(mul, mul);
#pragma unroll
      for (int j = 0; j < kChunks; ++j) {
        const int c = (j * nt + tid) * 8;
        r[j][0] = r[j][1] = r[j][2] = r[j][3] = 0ull;
        if (c < H) {
          load8_f2(src, p.res_f32, c, r[j]);
#pragma unroll
          for (int e = 0; e < 4; ++e) r[j][e] = f2_fma(r[j][e], res_scale, f2_mul(y[j][e], mul2));
        }
      }
    }
    void* rdst = p.res_f32 ? static_cast<void*>(static_cast<float*>(p.res_out) + row * p.res_out_stride)
                           : static_cast<void*>(static_cast<uint16_t*>(p.res_out) + row * p.res_out_stride);
    F2 sum = 0ull;
#pragma unroll
    for (int j = 0; j < kChunks; ++j) {
      const int c = (j * nt + tid) * 8;
      if (c < H) store8_f2(rdst, p.res_f32, c, r[j]);
#pragma unroll
      for (int e = 0; e < 4; ++e) sum = f2_fma(r[j][e], r[j][e], sum);
    }
    float rstd = 0.f;
    if (p.pre_gain) {
      float lo, hi;
      f2_unpack(sum, lo, hi);
      rstd = rsqrtf(cta_sum(lo + hi, red_pre[n & 1]) * over_h + p.eps);
    }
    // every thread has read its part of the slot once it is past that sum's barrier
    if (!p.pre_gain || nt == 32) __syncthreads();
    // (not into a slot whose copy is late: its barrier still counts that one)
    if (tid == 0 && row + static_cast<int64_t>(kStreamStages) * gridDim.x < rows && landed) fetch(row + kStreamStages * gridDim.x, st);
    if (p.pre_gain) {
      const F2 rstd2 = f2_pack(rstd, rstd);
      uint32_t amax = 0;
#pragma unroll
      for (int j = 0; j < kChunks; ++j) {
        const int c = (j * nt + tid) * 8;
        if (c < H) {
          F2 g[4];
          load8_f2(p.pre_gain, true, c, g);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            r[j][e] = f2_mul(f2_mul(r[j][e], rstd2), g[e]);
            if (kInt8) {
              float lo, hi;
              f2_unpack(r[j][e], lo, hi);
              amax = max(amax, max(abs_bits(lo), abs_bits(hi)));
            }
          }
          if (!kInt8) {
            const bool f32 = p.out_kind == kRowsF32;
            store8_f2(f32 ? static_cast<void*>(static_cast<float*>(p.out) + row * p.out_stride)
                          : static_cast<void*>(static_cast<uint16_t*>(p.out) + row * p.out_stride), f32, c, r[j]);
          }
        }
      }
      if (kInt8) {
        const RowScale s = row_scale(cta_max(amax, red_max[n & 1]));
        int8_t* dst = static_cast<int8_t*>(p.out) + row * p.out_stride;
#pragma unroll
        for (int j = 0; j < kChunks; ++j) {
          const int c = (j * nt + tid) * 8;
          float f[8];
#pragma unroll
          for (int e = 0; e < 4; ++e) f2_unpack(r[j][e], f[2 * e], f[2 * e + 1]);
          if (c < H) *reinterpret_cast<uint2*>(dst + c) = make_uint2(quant8x4(f[0], f[1], f[2], f[3], s), quant8x4(f[4], f[5], f[6], f[7], s));
        }
        if (tid == 0) p.out_scale[row] = s.scale;
      }
    }
    if (++st == kStreamStages) { st = 0; ph ^= 1; }
  }
  __syncthreads();
  if (tid == 0 && abort_code != 0) {
    publish_timeout(&g_norm_status, abort_code);
    const long long c0 = clock64();      // copies that are late get some time before the CTA's memory is another's
    while (clock64() - c0 < kWaitLimitCycles / 100) {}
  }
}

// The same ring for rows of any width and alignment: a copy takes the 16-byte pieces that a row lies in (never past the
// row's last piece, so never out of its allocation), and the threads find the row behind the bytes in front of it.
// Neighbouring threads take neighbouring columns.  Bounded by its instructions: one element an access, to shared memory and to
// global memory, where the aligned rows move eight (and 40 bytes of spills a thread at 32 values).  4096 x 5121, bf16, a gate per
// element: 86.7 us (210 MB: 2.4 TB/s), a CTA per row with plain loads 138.5.
template <int kChunks>
__global__ void __launch_bounds__(512, kChunks == 4 ? 1 : 2) okc_block_norm_stream_any(const BlockNormParams p, int rows, int row_bytes) {
  extern __shared__ __align__(16) uint8_t ring[];
  constexpr int kVals = kChunks * 8;
  __shared__ uint64_t bar_full[kStreamStages];
  __shared__ int abort_code;
  __shared__ float red_post[2][32], red_pre[2][32];
  __shared__ uint32_t red_max[2][32];
  const int tid = threadIdx.x, nt = blockDim.x, H = p.H;
  const bool gate_rows = p.gate && p.gate_col_stride != 0 && p.gate_stride != 0, gate_cols = p.gate && p.gate_col_stride != 0 && p.gate_stride == 0;
  const int res_size = p.res_f32 ? 4 : 2, blk_size = p.blk_f32 ? 4 : 2, gate_size = p.gate_f32 ? 4 : 2;
  const int res_room = (H * res_size + 30) & ~15, blk_room = (H * blk_size + 30) & ~15;      // any row's pieces fit
  auto pieces = [&](const uint8_t* row, int bytes) {     // length of the pieces that a row lies in
    return (static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row) & 15) + bytes + 15) & ~15u;
  };
  auto aligned_down = [](const uint8_t* row) { return reinterpret_cast<const uint8_t*>(reinterpret_cast<uintptr_t>(row) & ~static_cast<uintptr_t>(15)); };
  auto head = [](const uint8_t* row) { return static_cast<int>(reinterpret_cast<uintptr_t>(row) & 15); };
  auto res_row = [&](int row) { return static_cast<const uint8_t*>(p.res) + row * p.res_stride * res_size; };
  auto blk_row = [&](int row) { return static_cast<const uint8_t*>(p.blk) + row * p.blk_stride * blk_size; };
  auto gate_row = [&](int row) { return static_cast<const uint8_t*>(p.gate) + row * p.gate_stride * gate_size; };
  auto fetch = [&](int row, int st) {
    const uint32_t bar = smem_u32(&bar_full[st]);
    const uint32_t dst = smem_u32(ring) + st * row_bytes;
    const uint32_t a = pieces(res_row(row), H * res_size), b = pieces(blk_row(row), H * blk_size), c = gate_rows ? pieces(gate_row(row), H * gate_size) : 0;
    mbar_expect_tx(bar, a + b + c);
    bulk_g2s(dst, aligned_down(res_row(row)), a, bar);
    bulk_g2s(dst + res_room, aligned_down(blk_row(row)), b, bar);
    if (gate_rows) bulk_g2s(dst + res_room + blk_room, aligned_down(gate_row(row)), c, bar);
  };
  // this thread's values of a row; the type is asked once
  auto take = [&](const void* row, bool f32, float (&v)[kVals]) {
    if (f32) {
#pragma unroll
      for (int e = 0; e < kVals; ++e) { const int c = e * nt + tid; v[e] = c < H ? static_cast<const float*>(row)[c] : 0.f; }
    } else {
      uint32_t u[kVals];
#pragma unroll
      for (int e = 0; e < kVals; ++e) { const int c = e * nt + tid; u[e] = c < H ? static_cast<const uint16_t*>(row)[c] : 0u; }
#pragma unroll
      for (int e = 0; e < kVals; ++e) v[e] = __uint_as_float(u[e] << 16);
    }
  };
  auto put = [&](void* row, bool f32, const float (&v)[kVals]) {
    if (f32) {
#pragma unroll
      for (int e = 0; e < kVals; ++e) { const int c = e * nt + tid; if (c < H) static_cast<float*>(row)[c] = v[e]; }
    } else {
#pragma unroll
      for (int e = 0; e < kVals; ++e) { const int c = e * nt + tid; if (c < H) static_cast<__nv_bfloat16*>(row)[c] = __float2bfloat16_rn(v[e]); }
    }
  };
  if (tid == 0) {
    for (int i = 0; i < kStreamStages; ++i) mbar_init(smem_u32(&bar_full[i]), 1);
    abort_code = 0;
    mbar_fence_init();
    for (int i = 0; i < kStreamStages && blockIdx.x + i * gridDim.x < static_cast<unsigned>(rows); ++i) fetch(blockIdx.x + i * gridDim.x, i);
  }
  __syncthreads();
  const float over_h = 1.f / static_cast<float>(H);
  int st = 0, n = 0;
  uint32_t ph = 0;
  for (int row = blockIdx.x; row < rows; row += gridDim.x, ++n) {
    float mul = p.blk_scale;
    if (p.gate && p.gate_col_stride == 0) {
      float g;
      if (p.gate_f32) g = *reinterpret_cast<const float*>(gate_row(row));
      else g = __uint_as_float(static_cast<uint32_t>(*reinterpret_cast<const uint16_t*>(gate_row(row))) << 16);
      if (p.gate_sigmoid) g = 1.f / (1.f + __expf(-g));
      mul *= g;
    }
    mbar_wait(smem_u32(&bar_full[st]), ph, &abort_code, 0x82);     // (as in the kernel above: no thread leaves the loop)
    const uint8_t* const src = ring + st * row_bytes;
    float r[kVals], y[kVals];
    take(src + res_room + head(blk_row(row)), p.blk_f32, y);
    if (p.post_gain) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < kVals; ++e) ss = fmaf(y[e], y[e], ss);
      const float rstd = rsqrtf(cta_sum(ss, red_post[n & 1]) * over_h + p.eps);
      take(p.post_gain, true, r);
#pragma unroll
      for (int e = 0; e < kVals; ++e) y[e] = y[e] * rstd * r[e];
    }
    if (gate_rows || gate_cols) {
      take(gate_rows ? src + res_room + blk_room + head(gate_row(row)) : static_cast<const uint8_t*>(p.gate), p.gate_f32, r);
      if (p.gate_sigmoid) {
#pragma unroll
        for (int e = 0; e < kVals; ++e) r[e] = 1.f / (1.f + __expf(-r[e]));
      }
#pragma unroll
      for (int e = 0; e < kVals; ++e) y[e] *= r[e];
    }
    take(src + head(res_row(row)), p.res_f32, r);
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < kVals; ++e) {
      r[e] = p.res_scale * r[e] + mul * y[e];
      if (e * nt + tid < H) ss = fmaf(r[e], r[e], ss);
    }
    put(p.res_f32 ? static_cast<void*>(static_cast<float*>(p.res_out) + row * p.res_out_stride)
                  : static_cast<void*>(static_cast<uint16_t*>(p.res_out) + row * p.res_out_stride), p.res_f32, r);
    float rstd = 0.f;
    if (p.pre_gain) rstd = rsqrtf(cta_sum(ss, red_pre[n & 1]) * over_h + p.eps);
    if (!p.pre_gain || nt == 32) __syncthreads();
    if (tid == 0 && row + static_cast<int64_t>(kStreamStages) * gridDim.x < rows && abort_code == 0) fetch(row + kStreamStages * gridDim.x, st);
    if (p.pre_gain) {
      take(p.pre_gain, true, y);
#pragma unroll
      for (int e = 0; e < kVals; ++e) r[e] = r[e] * rstd * y[e];
      if (p.out_kind == kRowsInt8) {
        uint32_t amax = 0;
#pragma unroll
        for (int e = 0; e < kVals; ++e)
          if (e * nt + tid < H) amax = max(amax, abs_bits(r[e]));
        const RowScale s = row_scale(cta_max(amax, red_max[n & 1]));
        int8_t* dst = static_cast<int8_t*>(p.out) + row * p.out_stride;
#pragma unroll
        for (int e = 0; e < kVals; ++e) { const int c = e * nt + tid; if (c < H) dst[c] = static_cast<int8_t>(quant8(r[e], s)); }
        if (tid == 0) p.out_scale[row] = s.scale;
      } else {
        const bool f32 = p.out_kind == kRowsF32;
        put(f32 ? static_cast<void*>(static_cast<float*>(p.out) + row * p.out_stride)
                : static_cast<void*>(static_cast<uint16_t*>(p.out) + row * p.out_stride), f32, r);
      }
    }
    if (++st == kStreamStages) { st = 0; ph ^= 1; }
  }
  __syncthreads();
  if (tid == 0 && abort_code != 0) {
    publish_timeout(&g_norm_status, abort_code);
    const long long c0 = clock64();
    while (clock64() - c0 < kWaitLimitCycles / 100) {}
  }
}

// Rows -> int8 values and a scale per row.  A CTA per row; a row that fits the CTA's registers is read once, a longer
// one (more than 16384 columns) a second time, from L2.
template <int kChunks, bool kVec>
__global__ void __launch_bounds__(row_threads(kChunks)) okc_quantize_rows(const QuantizeParams p) {
  __shared__ uint32_t red[32];
  if (p.product_follows) griddep_launch_dependents();     // it may set itself up; it waits before it reads the rows
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
      store_chunk_q<kVec>(dst, s * kChunks + j, tid, nt, p.cols, v[j], rs);
    }
  }
}

// The same for many rows of bf16: a warp per row, which it holds in registers as it is (up to 8192 columns in 128 of them).
// Nothing waits on other warps, and a dozen warps an SM have their whole rows on the way at once.  A row may start
// anywhere: the loads are those of the 16-byte pieces that it lies in (with up to 7 values before and behind it, which
// count as zeros), and the int8 values move down by as many lanes' bytes before they are stored eight at a time.
// 4096 x 7168: a CTA per row 27.7 us, this kernel 15.1 (88 MB: 5.8 TB/s); 4096 x 7167 24.9.
template <int kVecs>
__global__ void __launch_bounds__(128) okc_quantize_rows_warp(const QuantizeParams p, int64_t rows) {
  if (p.product_follows) griddep_launch_dependents();
  const int lane = threadIdx.x & 31;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  if (row >= rows) return;
  const uintptr_t start = reinterpret_cast<uintptr_t>(static_cast<const uint16_t*>(p.x) + row * p.x_stride);
  const int head = static_cast<int>(start & 15) >> 1;         // values in front of the row in its first piece
  const uint4* src = reinterpret_cast<const uint4*>(start & ~static_cast<uintptr_t>(15));
  const int end = head + p.cols, units = (end + 7) / 8;
  uint4 v[kVecs];
#pragma unroll
  for (int j = 0; j < kVecs; ++j) {
    v[j] = make_uint4(0, 0, 0, 0);
    if (j * 32 + lane < units) v[j] = __ldg(src + j * 32 + lane);
  }
  const bool ragged = (head | (end & 7)) != 0;
  if (ragged) {
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      const int u = j * 32 + lane;
      if (u == 0 || u == units - 1) {
        uint32_t w[4] = {v[j].x, v[j].y, v[j].z, v[j].w};
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (u * 8 + i < head || u * 8 + i >= end) w[i >> 1] &= (i & 1) ? 0x0000FFFFu : 0xFFFF0000u;
        v[j] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    }
  }
  uint32_t m = 0;      // two running maxima of the magnitudes' bits, 16 bits each
#pragma unroll
  for (int j = 0; j < kVecs; ++j)
    m = __vmaxu2(__vmaxu2(__vmaxu2(m, v[j].x & 0x7FFF7FFFu), v[j].y & 0x7FFF7FFFu), __vmaxu2(v[j].z & 0x7FFF7FFFu, v[j].w & 0x7FFF7FFFu));
  const RowScale s = row_scale(__reduce_max_sync(0xffffffffu, max(m & 0xFFFF0000u, m << 16)));
  if (lane == 0) p.scale[row] = s.scale;
  uint2* dst = reinterpret_cast<uint2*>(p.q + row * p.q_stride);
  auto quantised = [&](int j) {
    float f[8];
    unpack_bf16x8(v[j], f);
    return make_uint2(quant8x4(f[0], f[1], f[2], f[3], s), quant8x4(f[4], f[5], f[6], f[7], s));
  };
  const int out_units = (p.cols + 7) / 8;
  if (head == 0) {
#pragma unroll
    for (int j = 0; j < kVecs; ++j)
      if (j * 32 + lane < out_units) dst[j * 32 + lane] = quantised(j);
  } else {
    uint2 cur = quantised(0);
#pragma unroll
    for (int j = 0; j < kVecs; ++j) {
      const uint2 next = j + 1 < kVecs ? quantised(j + 1) : make_uint2(0, 0);
      // the eight values behind this lane's: the next lane's, or the first lane's of the next step
      const uint2 give = lane == 0 ? next : cur;
      const uint2 from = make_uint2(__shfl_sync(0xffffffffu, give.x, (lane + 1) & 31), __shfl_sync(0xffffffffu, give.y, (lane + 1) & 31));
      const uint64_t lo = cur.x | (static_cast<uint64_t>(cur.y) << 32), hi = from.x | (static_cast<uint64_t>(from.y) << 32);
      const uint64_t out = (lo >> (8 * head)) | (hi << (64 - 8 * head));
      if (j * 32 + lane < out_units) dst[j * 32 + lane] = make_uint2(static_cast<uint32_t>(out), static_cast<uint32_t>(out >> 32));
      cur = next;
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

// The streaming kernels, if there is a block (without one a CTA per row takes them: 4096 x 5120 bf16 26 to 27 us for 84 MB, not
// looked at further) and the rows are many (4 an SM and more: bf16, a gate per channel, 500 / 600 rows of 4096 take 6.3 us
// a CTA each and 7.2 streamed; at 4096 rows the streamed ones take 29.6 of 44) and a ring fits; false: not launched.
static bool try_stream(const BlockNormParams& p, int64_t rows, bool vec, cudaStream_t stream, cudaError_t& e) {
  if (!p.blk || rows < 4 * 148 || rows > INT32_MAX / 2) return false;
  const int units = (p.H + 7) / 8;
  const int chunks = units > 1024 ? 4 : units > 256 ? 2 : 1;
  const int threads = ((units + chunks - 1) / chunks + 31) / 32 * 32;
  const bool rows_gate = p.gate && p.gate_col_stride != 0 && p.gate_stride != 0;
  auto room = [&](int f32) { return vec ? p.H * (f32 ? 4 : 2) : (p.H * (f32 ? 4 : 2) + 30) & ~15; };
  const int row_bytes = room(p.res_f32) + room(p.blk_f32) + (rows_gate ? room(p.gate_f32) : 0);
  // CTAs an SM by registers, then by shared memory
  const int regs = vec ? (chunks == 4 ? 96 : chunks == 2 ? 56 : 40) : (chunks == 4 ? 128 : 64);
  int per_sm = 65536 / (threads * regs);
  if (per_sm > 16) per_sm = 16;
  if (per_sm < 1) per_sm = 1;
  while (per_sm > 1 && kStreamStages * row_bytes * per_sm > kStreamSmem) --per_sm;
  const size_t smem = static_cast<size_t>(kStreamStages) * row_bytes;
  if (smem > kStreamSmem) return false;
  const int64_t most = 148LL * per_sm;
  const dim3 grid(static_cast<unsigned>(rows < most ? rows : most)), block(threads);
  const bool q = p.pre_gain && p.out_kind == kRowsInt8;
  auto kernel = !vec ? (chunks == 1 ? okc_block_norm_stream_any<1> : chunks == 2 ? okc_block_norm_stream_any<2> : okc_block_norm_stream_any<4>)
              : q ? (chunks == 1 ? okc_block_norm_stream<1, true> : chunks == 2 ? okc_block_norm_stream<2, true> : okc_block_norm_stream<4, true>)
                  : (chunks == 1 ? okc_block_norm_stream<1, false> : chunks == 2 ? okc_block_norm_stream<2, false> : okc_block_norm_stream<4, false>);
  e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kStreamSmem);     // (never less: see params.cuh)
  if (e == cudaSuccess) e = launch_kernel(kernel, grid, block, smem, stream, false, p, static_cast<int>(rows), row_bytes);
  return true;
}

cudaError_t launch_block_norm(const BlockNormParams& p, int64_t rows, bool vec, cudaStream_t stream) {
  cudaError_t e;
  if (try_stream(p, rows, vec, stream, e)) return e;
  int threads, chunks;
  row_shape(rows, p.H, threads, chunks);
  const dim3 grid(static_cast<unsigned>(rows)), block(threads);
  if (chunks == 1) return vec ? launch_kernel(okc_block_norm<1, true>, grid, block, 0, stream, false, p) : launch_kernel(okc_block_norm<1, false>, grid, block, 0, stream, false, p);
  if (chunks == 2) return vec ? launch_kernel(okc_block_norm<2, true>, grid, block, 0, stream, false, p) : launch_kernel(okc_block_norm<2, false>, grid, block, 0, stream, false, p);
  return vec ? launch_kernel(okc_block_norm<4, true>, grid, block, 0, stream, false, p) : launch_kernel(okc_block_norm<4, false>, grid, block, 0, stream, false, p);
}

// f32 rows, and bf16 rows of more than 8192 columns, do not fit a warp's registers and take a CTA each: 4096 x 7168 f32 30.9 us
// (147 MB: 4.8 TB/s), 4096 x 14336 bf16 38.9 (176 MB: 4.5 TB/s).
cudaError_t launch_quantize_rows(const QuantizeParams& p, int64_t rows, bool x_vec, bool q_vec, cudaStream_t stream) {
  const bool vec = x_vec && q_vec && (p.cols % 8) == 0;
  const int span = vec ? p.cols : p.cols + 7;
  if (q_vec && !p.x_f32 && span <= 8192 && rows >= 4 * 148) {
    const dim3 grid(static_cast<unsigned>((rows + 3) / 4)), block(128);
    if (span <= 1024) return launch_kernel(okc_quantize_rows_warp<4>, grid, block, 0, stream, false, p, rows);
    if (span <= 2048) return launch_kernel(okc_quantize_rows_warp<8>, grid, block, 0, stream, false, p, rows);
    if (span <= 4096) return launch_kernel(okc_quantize_rows_warp<16>, grid, block, 0, stream, false, p, rows);
    return launch_kernel(okc_quantize_rows_warp<32>, grid, block, 0, stream, false, p, rows);
  }
  int threads, chunks;
  row_shape(rows, p.cols, threads, chunks);
  const dim3 grid(static_cast<unsigned>(rows)), block(threads);
  if (chunks == 1) return vec ? launch_kernel(okc_quantize_rows<1, true>, grid, block, 0, stream, false, p) : launch_kernel(okc_quantize_rows<1, false>, grid, block, 0, stream, false, p);
  if (chunks == 2) return vec ? launch_kernel(okc_quantize_rows<2, true>, grid, block, 0, stream, false, p) : launch_kernel(okc_quantize_rows<2, false>, grid, block, 0, stream, false, p);
  return vec ? launch_kernel(okc_quantize_rows<4, true>, grid, block, 0, stream, false, p) : launch_kernel(okc_quantize_rows<4, false>, grid, block, 0, stream, false, p);
}

__global__ void okc_norm_probe_timeout() { probe_timeout(&g_norm_status, 0x7d); }
cudaError_t launch_norm_probe_timeout(cudaStream_t stream) {
  okc_norm_probe_timeout<<<1, 32, 0, stream>>>();
  return cudaGetLastError();
}

// Reads the word and, where it holds a code, clears that code: one that another stream's kernel records after the read stays.
__global__ void okc_norm_clear_status(int32_t code) { atomicCAS(&g_norm_status, code, 0); }
cudaError_t norm_read_status(cudaStream_t stream, int32_t* code) {
  cudaError_t e = cudaMemcpyFromSymbolAsync(code, g_norm_status, sizeof(int32_t), 0, cudaMemcpyDeviceToHost, stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
  if (e != cudaSuccess || *code == 0) return e;
  okc_norm_clear_status<<<1, 1, 0, stream>>>(*code);
  e = cudaGetLastError();
  return e != cudaSuccess ? e : cudaStreamSynchronize(stream);
}

}  // namespace okc
