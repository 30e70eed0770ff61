// Products of int8 rows with a scale per token and per weight row (W8A8):
//   y[t][n] = (sum_k qx[t][k] * qw[n][k]) * (sx[t] * sw[n]) (+ bias[n])         okc_moe_int8_linear
//   h[t][i] = g / (1 + exp(-g)) * u,  g = y[t][i], u = y[t][I + i]              okc_moe_int8_gated
// The integer sum is exact in 32 bits (K <= 131071), so its value does not depend on how K is split, and every kernel
// below turns it into the result with the same f32 operations: a token's bits do not depend on the batch it is in.
//
// Three kernels, by what bounds the product:
//   okc_int8_one   one token        the weights stream through shared memory and are multiplied on the integer dot-product
//                                   units; the token is quantised in the kernel (one launch)
//   okc_int8_mid   to some hundred  the weights fill M of a tcgen05.mma (kind::i8), the tokens are N; K is split over a
//                                   cluster of CTAs that add their integer sums through distributed shared memory
//   okc_int8_many  beyond           CTA pairs (cta_group::2) on tiles of 256 tokens x up to 256 weight rows, persistent
// The tiled kernels start early (programmatic launch) behind the quantiser of their own tokens and only there: it is
// launched plainly, so everything before it, the weights too, is complete, and all its CTAs are on their SMs by then.
// Every wait on a barrier is bounded; one that runs out is reported through a status word (okc_moe_dense_status).
#include <cooperative_groups.h>

#include <type_traits>

#include "rows.cuh"

namespace okc {

namespace cg = cooperative_groups;

__device__ int32_t g_int8_status;      // code of the first wait that ran out since the last read

// ------------------------------------------------------------------ what every kernel does with an integer sum
__device__ __forceinline__ float int8_value(int acc, float sx, float sw) { return __fmul_rn(__int2float_rn(acc), __fmul_rn(sx, sw)); }
__device__ __forceinline__ float silu_mul(float g, float u) { return __fmul_rn(__fdividef(g, 1.f + __expf(-g)), u); }

__device__ __forceinline__ void store_out(const Int8Params& p, int64_t o, float v) {
  if (p.out_f32) static_cast<float*>(p.out)[o] = v;
  else static_cast<__nv_bfloat16*>(p.out)[o] = __float2bfloat16_rn(v);
}

// ------------------------------------------------------------------ one token
constexpr int kOneWarps = 16;          // that multiply; one more brings the weights
constexpr int kOneThreads = 32 * kOneWarps + 32;
constexpr int kOneOutMax = 1024;       // most outputs of a CTA
constexpr int kOneSlots = 32;
constexpr int kOneSmem = 208 * 1024;

// Eight values of the token at column i (zeros past K), as f32.
__device__ __forceinline__ void one_load_x(const Int8Params& p, int i, float (&v)[8]) {
  if (p.x_vec && i + 8 <= p.K) {
    if (p.x_kind == kRowsF32) {
      const float4* s = reinterpret_cast<const float4*>(static_cast<const float*>(p.x) + i);
      const float4 a = s[0], b = s[1];
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      unpack_bf16x8(*reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(p.x) + i), v);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      v[j] = 0.f;
      if (i + j < p.K)
        v[j] = p.x_kind == kRowsF32 ? static_cast<const float*>(p.x)[i + j]
                                    : __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(p.x)[i + j]) << 16);
    }
  }
}

struct OneShape {
  int outs;          // neighbouring outputs of a CTA
  int group;         // pairs of weight rows of a ring slot
  int slots;
};

// A CTA owns `outs` neighbouring outputs and all of K.  One warp starts bulk copies of the weight rows into a ring that
// takes as much of them as shared memory holds (28 rows of 7168 bytes are all of a CTA's of 4096 outputs): what is on its
// way is not bounded by registers, and it starts before the token has been looked at.  Meanwhile the other warps quantise
// the token into shared memory (every CTA the whole row: a few KB from L2, where another launch would take longer).  Then
// a warp takes a slot: pairs of rows (two neighbours, or a gate row and its up row) against the token, 16 bytes a lane of
// each, integer dot products, one warp sum a row, and the outputs leave from there.
// The 16 bytes at a row's end may reach past K, never past the row's next 16-byte boundary; the token is zero there.
// bf16 token, in a graph: K = 4096, N = 4096 3.9 us with the weights of three layers in turn (50 MB, in L2) and 5.6 with all of
// them from HBM (16.8 MB: 3.0 TB/s), gated, K = 7168, 2 x 2048 rows 6.0 and 8.5 (29.4 MB: 3.5 TB/s).  Measured side by side, in
// L2: the quantiser and okc_int8_mid 6.5 us, rows held in registers, 16 a warp on their way, 5.7, this kernel 4.4 (gated 8.3,
// 8.2, 5.5); a token and one weight tile alone 3.3.  More tokens go through the tiles: the dot-product instruction gives an SM
// some 14 lanes a clock, and 2 / 4 / 8 tokens took 5.3 / 7.3 / 11.6 us here (gated 9.7 / 13.2 / 22.8) against 6.5 (8.3).
template <bool kGated>
__global__ void __launch_bounds__(kOneThreads) okc_int8_one(const Int8Params p, const OneShape q) {
  extern __shared__ __align__(16) uint8_t one_smem[];
  __shared__ uint64_t bar_full[kOneSlots], bar_empty[kOneSlots];
  __shared__ uint32_t amax_s[kOneWarps];
  __shared__ int abort_code;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int kpad = (p.K + 15) & ~15;
  const int n0 = blockIdx.x * q.outs, nr = min(q.outs, p.N - n0);
  const int per_unit = kGated ? q.group : 2 * q.group;         // outputs of a slot
  const int units = (nr + per_unit - 1) / per_unit;
  const uint32_t slot_bytes = 2u * q.group * kpad;
  uint8_t* const xq_s = one_smem;                              // [kpad] int8
  uint8_t* const ring = xq_s + kpad;
  float* const sw_s = reinterpret_cast<float*>(ring + static_cast<size_t>(q.slots) * slot_bytes);      // [outs] (gated: and [outs] of the up rows)
  float* const sb_s = sw_s + q.outs;                           // bias or up rows' scales
  const uint32_t full0 = smem_u32(&bar_full[0]), empty0 = smem_u32(&bar_empty[0]);

  if (warp == kOneWarps) {
    // unit u of weight rows into its slot, started by the calling thread
    auto fetch = [&](int u, int slot) {
      const int first = u * per_unit, v = min(per_unit, nr - first);
      const uint32_t bar = full0 + 8 * slot, dst = smem_u32(ring) + slot * slot_bytes;
      mbar_expect_tx(bar, static_cast<uint32_t>(kGated ? 2 * v : v) * kpad);
#pragma unroll
      for (int half = 0; half < (kGated ? 2 : 1); ++half) {
        const int8_t* src = p.w + (static_cast<int64_t>(half) * p.N + n0 + first) * p.w_stride;
        const uint32_t to = dst + half * q.group * kpad;
        if (p.w_stride == kpad) bulk_g2s(to, src, static_cast<uint32_t>(v) * kpad, bar);
        else
          for (int r = 0; r < v; ++r) bulk_g2s(to + r * kpad, src + r * p.w_stride, kpad, bar);
      }
    };
    if (lane == 0) {
      for (int i = 0; i < q.slots; ++i) { mbar_init(full0 + 8 * i, 1); mbar_init(empty0 + 8 * i, 1); }
      abort_code = 0;
      mbar_fence_init();
    }
    __syncwarp();
    if (lane < min(q.slots, units)) fetch(lane, lane);         // (at most 32 slots)
    __syncwarp();
    __syncthreads();
    __syncthreads();
    int slot = 0;
    uint32_t ph = 0;
    for (int u = q.slots; u < units; ++u) {
      if (!mbar_wait(empty0 + 8 * slot, ph, &abort_code, 0x51)) break;
      if (elect_one()) fetch(u, slot);
      if (++slot == q.slots) { slot = 0; ph ^= 1; }
    }
    __syncwarp();
  } else {
    for (int j = tid; j < nr; j += 32 * kOneWarps) {
      sw_s[j] = p.w_scale[n0 + j];
      if (kGated) sb_s[j] = p.w_scale[p.N + n0 + j];
      else if (p.bias) sb_s[j] = p.bias[n0 + j];
    }
    RowScale rs;
    if (p.x_kind != kRowsInt8) {
      uint32_t m = 0;
      for (int i = tid * 8; i < p.K; i += 256 * kOneWarps) {
        float v[8];
        one_load_x(p, i, v);
#pragma unroll
        for (int j = 0; j < 8; ++j) m = max(m, abs_bits(v[j]));
      }
      m = __reduce_max_sync(0xffffffffu, m);
      if (lane == 0) amax_s[warp] = m;
      __syncthreads();
      rs = row_scale(__reduce_max_sync(0xffffffffu, amax_s[lane % kOneWarps]));
      for (int i = tid * 8; i < kpad; i += 256 * kOneWarps) {
        float v[8];
        one_load_x(p, i, v);
        *reinterpret_cast<uint2*>(xq_s + i) = make_uint2(quant8x4(v[0], v[1], v[2], v[3], rs), quant8x4(v[4], v[5], v[6], v[7], rs));
      }
    } else {
      rs.scale = p.x_scale[0];
      for (int i = tid * 4; i < kpad; i += 128 * kOneWarps) {
        uint32_t w = *reinterpret_cast<const uint32_t*>(static_cast<const int8_t*>(p.x) + i);
        if (i + 4 > p.K) w = i < p.K ? w & ((1u << (8 * (p.K - i))) - 1u) : 0u;
        *reinterpret_cast<uint32_t*>(xq_s + i) = w;
      }
      __syncthreads();
    }
    __syncthreads();
    // A parity wait tells phases one apart only, so a slot that is used again has to be the same warp's each time: with
    // fewer slots than warps, as many warps work as there are slots.
    const int step = min(q.slots, kOneWarps);
    for (int u = warp < step ? warp : units; u < units; u += step) {
      const int slot = u % q.slots;
      if (!mbar_wait(full0 + 8 * slot, (u / q.slots) & 1, &abort_code, 0x52)) break;
      const uint8_t* const base = ring + static_cast<size_t>(slot) * slot_bytes;
      for (int g = 0; g < q.group; ++g) {
        const int j = u * per_unit + (kGated ? g : 2 * g);     // the pair's (first) output
        if (j >= nr) break;
        const uint8_t* const a = base + (kGated ? g : 2 * g) * kpad;
        const uint8_t* const b = kGated ? base + (q.group + g) * kpad : a + kpad;
        int da = 0, db = 0;
#pragma unroll 4
        for (int k = lane * 16; k < kpad; k += 512) {
          const uint4 x = *reinterpret_cast<const uint4*>(xq_s + k);
          const uint4 wa = *reinterpret_cast<const uint4*>(a + k), wb = *reinterpret_cast<const uint4*>(b + k);
          da = __dp4a(static_cast<int>(wa.x), static_cast<int>(x.x), da); db = __dp4a(static_cast<int>(wb.x), static_cast<int>(x.x), db);
          da = __dp4a(static_cast<int>(wa.y), static_cast<int>(x.y), da); db = __dp4a(static_cast<int>(wb.y), static_cast<int>(x.y), db);
          da = __dp4a(static_cast<int>(wa.z), static_cast<int>(x.z), da); db = __dp4a(static_cast<int>(wb.z), static_cast<int>(x.z), db);
          da = __dp4a(static_cast<int>(wa.w), static_cast<int>(x.w), da); db = __dp4a(static_cast<int>(wb.w), static_cast<int>(x.w), db);
        }
        da = __reduce_add_sync(0xffffffffu, da);
        db = __reduce_add_sync(0xffffffffu, db);               // (of a last row without a neighbour: not used)
        if (kGated) {
          if (lane == 0) store_out(p, n0 + j, silu_mul(int8_value(da, rs.scale, sw_s[j]), int8_value(db, rs.scale, sb_s[j])));
        } else if (lane < 2 && j + lane < nr) {
          float v = int8_value(lane ? db : da, rs.scale, sw_s[j + lane]);
          if (p.bias) v = __fadd_rn(v, sb_s[j + lane]);
          store_out(p, n0 + j + lane, v);
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(empty0 + 8 * slot);
    }
  }
  __syncthreads();
  if (tid == 0 && abort_code != 0) {
    publish_timeout(&g_int8_status, abort_code);
    const long long c0 = clock64();      // copies that are late get some time before the CTA's memory is another's
    while (clock64() - c0 < kWaitLimitCycles / 100) {}
  }
}

cudaError_t launch_int8_one(const Int8Params& p, bool gated, cudaStream_t stream) {
  const int kpad = (p.K + 15) & ~15;
  OneShape q;
  q.outs = (p.N + 147) / 148;
  if (q.outs > kOneOutMax) q.outs = kOneOutMax;
  q.group = 4096 / kpad;               // short rows go several pairs to a slot
  if (q.group < 1) q.group = 1;
  if (q.group > 8) q.group = 8;
  const int per_unit = gated ? q.group : 2 * q.group, units = (q.outs + per_unit - 1) / per_unit;
  const int slot_bytes = 2 * q.group * kpad, scales = 8 * q.outs;
  q.slots = (kOneSmem - kpad - scales) / slot_bytes;           // at K = 16384, the most, five
  if (q.slots > kOneSlots) q.slots = kOneSlots;
  if (q.slots > units) q.slots = units;
  else if (q.slots > kOneWarps) q.slots = q.slots / kOneWarps * kOneWarps;     // a slot that is used again is always the same warp's
  const size_t smem = static_cast<size_t>(kpad) + static_cast<size_t>(q.slots) * slot_bytes + scales;
  const dim3 grid((p.N + q.outs - 1) / q.outs), block(kOneThreads);
  auto kernel = gated ? okc_int8_one<true> : okc_int8_one<false>;
  const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kOneSmem);     // (never less: see params.cuh)
  if (e != cudaSuccess) return e;
  return launch_kernel(kernel, grid, block, smem, stream, false, p, q);
}

// ------------------------------------------------------------------ tcgen05 pieces shared by the two tiled kernels
// Instruction descriptor: int8 x int8 -> int32, both operands K-major, M = m, N = n.
__device__ __forceinline__ uint32_t idesc_i8(uint32_t m, uint32_t n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
// The shared-memory descriptors come as halves: only the low ones, which hold the addresses, change.
__device__ __forceinline__ void mma_i8(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t desc_hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 ad, bd;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 ad, {%1, %3};\n\t"
      "mov.b64 bd, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], ad, bd, %4, p;\n\t}"
      ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(desc_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_i8_pair(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t desc_hi, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 ad, bd;\n\t"
      "setp.ne.b32 p, %5, 0;\n\t"
      "mov.b64 ad, {%1, %3};\n\t"
      "mov.b64 bd, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::2.kind::i8 [%0], ad, bd, %4, p;\n\t}"
      ::"r"(d_tmem), "r"(a_lo), "r"(b_lo), "r"(desc_hi), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Low half of smem_desc_sw128 (ptx.cuh), and its high half, which is the same for every address.
__device__ __forceinline__ uint32_t desc_lo(uint32_t saddr) { return ((saddr & 0x3FFFF) >> 4) | (1u << 16); }
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
// 32 consecutive 32-bit columns of this thread's lane.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
// ------------------------------------------------------------------ some hundred tokens
constexpr int kMidThreads = 256;       // warps 0..3 read the accumulator, 4 and 6 bring weights and tokens, 5 issues the MMAs; all finish the rows
constexpr int kMidMaxStages = 16;
constexpr int kMidRing = 216 * 1024;
constexpr int kMidMaxSmem = 225 * 1024;      // an SM's 227 KB less what the kernel declares itself (1.3 KB)
constexpr int kMidMinSmem = 200 * 1024;      // one CTA an SM, and little beside it: clusters cannot wait in a circle for tensor memory
constexpr int kMidMaxBlocks = 8;       // most K blocks of a stage
constexpr int kKb = 128;               // K elements of a stage: one 128-byte swizzled row
constexpr int kTileW = 128;            // weight rows of a tile

struct Int8MidParams {
  CUtensorMap wmap;      // int8 weight rows: [block] (gated: [gate, up]) [outs rows] [128]; of single blocks 2D, box 128 x outs rows
  CUtensorMap xmap;      // int8 token rows: [block] [tn rows] [128]
  Int8Params p;
  int outs;              // outputs of a tile: a multiple of 8, at most 128, gated 64 (the MMA's other rows are not looked at)
  int blocks;            // K blocks of 128 a stage
  int tn, stages, n_kb, tmem_cols;
};

// The producers and the issuer run as whole warps with one elected lane acting: in code that only one thread runs, every
// MMA costs it about 100 cycles (its operands go through vector registers), which with four MMAs and a commit a stage was
// more than the stage's copy takes (K = 4096, N = 4096, 16 tokens, no split: 20.0 us; as whole warps 10.4).
// A copy costs an SM some 150 cycles besides its bytes, however many warps issue them, so a stage takes several K blocks with
// one copy of weights and one of tokens (8 tokens, K = 7168, N = 2048, blocks 1 / 2 / 7: 7.9 / 7.4 / 6.5 us; gated, 32 tokens,
// K = 4096, 2 x 2560 rows, 1 / 2 / 4: 8.6 / 8.0 / 7.0), and the first weights are on their way before the CTA has set itself up.
// Bounded by the copies into the SMs for most sizes while the weights are in L2, by those and the way from HBM when they are not:
// int8 tokens, 32, K = 4096, N = 7168 7.1 / 10.3 us (29.4 MB of weights, in L2 / from HBM), gated, 128 tokens, K = 7168, 2 x
// 2048 rows 9.8 / 12.0 us (29.4 MB), of which about 4 us are the launch and the sums' way through the cluster.
template <bool kGated, int kSplits, bool kSingle>      // kSingle: one K block a stage
__global__ void __launch_bounds__(kMidThreads) okc_int8_mid(const __grid_constant__ Int8MidParams q) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = smem_u32(smem_raw);
  const uint32_t smem0 = (smem_base + 1023u) & ~1023u;
  __shared__ uint64_t bar_full[kMidMaxStages], bar_empty[kMidMaxStages], bar_done;
  __shared__ float xs[256];
  __shared__ uint32_t tmem_base_s;
  __shared__ int abort_code;
  const Int8Params& p = q.p;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rank = blockIdx.x % kSplits, tile = blockIdx.x / kSplits;
  const int w0 = tile * q.outs;      // first output of the tile
  const int t0 = blockIdx.y * q.tn;
  const int kb0 = static_cast<int>(static_cast<long long>(q.n_kb) * rank / kSplits);
  const int nkb = static_cast<int>(static_cast<long long>(q.n_kb) * (rank + 1) / kSplits) - kb0;
  const int blocks = kSingle ? 1 : q.blocks;
  const int nst = (nkb + blocks - 1) / blocks, first = min(nst, q.stages);
  const int a_rows = kGated ? 2 * q.outs : q.outs;
  const uint32_t a_bytes = static_cast<uint32_t>(a_rows) * kKb, x_bytes = static_cast<uint32_t>(q.tn) * kKb;
  const uint32_t a_stage = a_bytes * blocks, x_stage = x_bytes * blocks, stage_bytes = a_stage + x_stage;
  const uint32_t full0 = smem_u32(&bar_full[0]), empty0 = smem_u32(&bar_empty[0]);

  auto load_w = [&](int i, uint32_t st) {
    const uint32_t bar = full0 + 8 * st, dst = smem0 + st * stage_bytes;
    const int kb = kb0 + i * blocks;
    if (elect_one()) {
      mbar_expect_tx(bar, a_stage);
      if (!kSingle) {
        if (kGated) tma_4d_g2s(dst, &q.wmap, 0, w0, 0, kb, bar);
        else tma_3d_g2s(dst, &q.wmap, 0, w0, kb, bar);
      } else {
        tma_2d_g2s(dst, &q.wmap, kb * kKb, w0, bar);
        if (kGated) tma_2d_g2s(dst + q.outs * kKb, &q.wmap, kb * kKb, p.N + w0, bar);
      }
    }
  };
  auto load_x = [&](int i, uint32_t st) {
    const uint32_t bar = full0 + 8 * st, dst = smem0 + st * stage_bytes + a_stage;
    const int kb = kb0 + i * blocks;
    if (elect_one()) {
      mbar_expect_tx(bar, x_stage);
      if (!kSingle) tma_3d_g2s(dst, &q.xmap, 0, t0, kb, bar);
      else tma_2d_g2s(dst, &q.xmap, kb * kKb, t0, bar);
    }
  };
  if (warp == 4) {
    if (lane == 0) {
      for (int i = 0; i < q.stages; ++i) { mbar_init(full0 + 8 * i, 2); mbar_init(empty0 + 8 * i, 1); }
      mbar_init(smem_u32(&bar_done), 1);
      abort_code = 0;
      mbar_fence_init();
    }
    __syncwarp();
    // the weights do not depend on the kernel before this one, the token rows may
    for (int i = 0; i < first; ++i) load_w(i, i);
    __syncwarp();
  } else if (warp == 5) {
    tmem_alloc(smem_u32(&tmem_base_s), static_cast<uint32_t>(q.tmem_cols));
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_base_s;
  cg::cluster_group cluster = cg::this_cluster();
  int* const part = reinterpret_cast<int*>(smem_raw + (smem0 - smem_base));
  // a thread finishes four neighbouring outputs of every few tokens
  constexpr int kQuads = kGated ? kTileW / 8 : kTileW / 4;
  const int o4 = (tid % kQuads) * 4, n = w0 + o4;
  float sw[4], su[4] = {}, sb[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const bool in = n + j < p.N;
    sw[j] = in ? __ldg(p.w_scale + n + j) : 0.f;
    if (kGated) su[j] = in ? __ldg(p.w_scale + p.N + n + j) : 0.f;
    sb[j] = !kGated && p.bias && in ? __ldg(p.bias + n + j) : -0.f;      // v + -0 is v, whatever v
  }

  int posted = 0;        // stages whose copies this warp has started
  if (warp == 4 || warp == 6) {
    const bool tokens = warp == 6;
    int i = first;
    if (tokens) {
      griddep_wait();
      for (i = 0; i < first; ++i) load_x(i, i);
    }
    uint32_t st = 0, ph = 0;
    for (; i < nst; ++i) {
      if (!mbar_wait(empty0 + 8 * st, ph, &abort_code, 0x61)) break;
      if (tokens) load_x(i, st); else load_w(i, st);
      if (++st == static_cast<uint32_t>(q.stages)) { st = 0; ph ^= 1; }
    }
    posted = i;
    __syncwarp();
  } else if (warp == 5) {
    const uint32_t idesc = idesc_i8(128, static_cast<uint32_t>(q.tn));
    const uint32_t lo0 = desc_lo(smem0);
    uint32_t st = 0, ph = 0, more = 0;
    for (int left = nkb; left > 0; left -= blocks) {
      if (!mbar_wait(full0 + 8 * st, ph, &abort_code, 0x62)) break;
      tc_fence_after();
      uint32_t a = lo0 + st * (stage_bytes >> 4), b = a + (a_stage >> 4);
      for (int j = min(left, blocks); j > 0; --j) {
        if (elect_one()) {
          mma_i8(tmem, a, b, kDescHi, idesc, more);          // K = 32 each: 32 bytes further along the swizzled rows
          mma_i8(tmem, a + 2, b + 2, kDescHi, idesc, 1);
          mma_i8(tmem, a + 4, b + 4, kDescHi, idesc, 1);
          mma_i8(tmem, a + 6, b + 6, kDescHi, idesc, 1);
        }
        more = 1;
        a += a_bytes >> 4;
        b += x_bytes >> 4;
      }
      if (elect_one()) mma_commit(empty0 + 8 * st);
      if (++st == static_cast<uint32_t>(q.stages)) { st = 0; ph ^= 1; }
    }
    if (elect_one()) mma_commit(smem_u32(&bar_done));
    __syncwarp();
  } else if (warp < 4) {
    griddep_wait();        // the token scales come from the kernel before this one
    for (int i = tid; i < q.tn; i += 128) xs[i] = t0 + i < p.T ? p.x_scale[t0 + i] : 0.f;
    const bool ok = mbar_wait<20>(smem_u32(&bar_done), 0, &abort_code, 0x63);
    tc_fence_after();
    if (ok && warp * 32 < a_rows) {
      // this CTA's sums, [token][weight row], over the ring slots (every copy has landed and every MMA has read them)
      const uint32_t taddr = tmem + (static_cast<uint32_t>(warp * 32) << 16);
      int* mine = part + warp * 32 + lane;
      int c0 = 0;
      for (; c0 + 32 <= q.tn; c0 += 32) {
        uint32_t r[32];
        tmem_ld32(taddr + c0, r);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 32; ++j) mine[(c0 + j) * kTileW] = static_cast<int>(r[j]);
      }
      if (c0 < q.tn) {
        uint32_t r[16];
        tmem_ld16(taddr + c0, r);
        tmem_wait_ld();
#pragma unroll
        for (int j = 0; j < 16; ++j) mine[(c0 + j) * kTileW] = static_cast<int>(r[j]);
      }
    }
    tc_fence_before();
  }
  if (kSplits > 1) cluster.sync(); else __syncthreads();
  const int gave_up = abort_code;

  // Each CTA of the cluster finishes tn / kSplits tokens: it adds the integer sums of all CTAs (the loads from all of them
  // under way at once) and stores the rows.  A few tokens of a thread go together, all loads and arithmetic first, and what
  // differs between calls is decided once for them: with eight warps an SM, one token at a time was a chain of latencies
  // (256 tokens, K = 256, N = 2048, no split: 8.8 us; so 6.3).  What is left, and rows off the 8-byte grid, go one by one.
  {
    const int* src[kSplits];
#pragma unroll
    for (int s = 0; s < kSplits; ++s) src[s] = (kSplits > 1 ? cluster.map_shared_rank(part, s) : part) + o4;
    const int per = q.tn / kSplits, last = o4 < q.outs ? min((rank + 1) * per, p.T - t0) : 0;
    const bool vec = p.out_vec && n + 4 <= p.N;
    constexpr int kStep = kMidThreads / kQuads, kBatch = kSplits >= 4 ? 2 : 4;
    auto finish = [&](auto tokens, int col0) {
      constexpr int kTokens = decltype(tokens)::value;
      float v[kTokens][4];
#pragma unroll
      for (int u = 0; u < kTokens; ++u) {
        const int col = col0 + u * kStep;
        int4 a[kSplits], b[kSplits];
#pragma unroll
        for (int s = 0; s < kSplits; ++s) {
          a[s] = *reinterpret_cast<const int4*>(src[s] + col * kTileW);
          if (kGated) b[s] = *reinterpret_cast<const int4*>(src[s] + col * kTileW + q.outs);
        }
#pragma unroll
        for (int s = 1; s < kSplits; ++s) {
          a[0].x += a[s].x; a[0].y += a[s].y; a[0].z += a[s].z; a[0].w += a[s].w;
          if (kGated) { b[0].x += b[s].x; b[0].y += b[s].y; b[0].z += b[s].z; b[0].w += b[s].w; }
        }
        const float sx = xs[col];
        const int av[4] = {a[0].x, a[0].y, a[0].z, a[0].w}, bv[4] = {b[0].x, b[0].y, b[0].z, b[0].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[u][j] = int8_value(av[j], sx, sw[j]);
          if (kGated) v[u][j] = silu_mul(v[u][j], int8_value(bv[j], sx, su[j]));
          else v[u][j] = __fadd_rn(v[u][j], sb[j]);
        }
      }
      const int64_t o = static_cast<int64_t>(t0 + col0) * p.out_stride + n, step = static_cast<int64_t>(kStep) * p.out_stride;
      if (vec && p.out_f32) {
#pragma unroll
        for (int u = 0; u < kTokens; ++u)
          *reinterpret_cast<float4*>(static_cast<float*>(p.out) + o + u * step) = make_float4(v[u][0], v[u][1], v[u][2], v[u][3]);
      } else if (vec) {
#pragma unroll
        for (int u = 0; u < kTokens; ++u)
          *reinterpret_cast<uint2*>(static_cast<uint16_t*>(p.out) + o + u * step) = make_uint2(pack_bf16x2(v[u][0], v[u][1]), pack_bf16x2(v[u][2], v[u][3]));
      } else if (kTokens == 1) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (n + j < p.N) store_out(p, o + j, v[0][j]);
      }
    };
    int col = rank * per + tid / kQuads;
    if (vec)
      for (; col + (kBatch - 1) * kStep < last; col += kBatch * kStep) finish(std::integral_constant<int, kBatch>{}, col);
    for (; col < last; col += kStep) finish(std::integral_constant<int, 1>{}, col);
  }
  // A wait ran out, whoever's it was (the producers of a short K have started all their copies by then and are done): the
  // copies on their way get a bounded chance to land before the CTA's memory is another's.
  if (gave_up != 0) {
    const long long c0 = clock64();
    for (int j = max(0, posted - q.stages); j < posted; ++j)
      while (!mbar_try(full0 + 8 * (j % q.stages), (j / q.stages) & 1) && clock64() - c0 < kWaitLimitCycles) {}
  }
  if (kSplits > 1) cluster.sync(); else __syncthreads();   // no CTA leaves while another reads its sums
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, static_cast<uint32_t>(q.tmem_cols));
  }
  if (tid == 0 && gave_up != 0) publish_timeout(&g_int8_status, gave_up);
}

static int tmem_cols_for(int n) { return n <= 32 ? 32 : n <= 64 ? 64 : n <= 128 ? 128 : n <= 256 ? 256 : 512; }

// How the two tiled kernels would cut a product, and what each is expected to take.  The estimates are a start-up time, a
// time for the end of a tile, and a time for the K blocks: what a CTA needs for one alone, or, with all SMs busy, what its
// bytes take at the 83 to 90 KB/us that an SM takes in then (from L2: the fit is to weights that are there).  Of 323 measured
// shapes (3 to 512 tokens, K 256 to 7168, N 300 to 7168, plain and gated) the choice of the kernel and of the split over a
// cluster costs 0.5 % of the best of the five on average and 20 % at worst with the weights in L2, 0.6 % and 16 % with all
// of them from HBM.
struct TileShape {
  int tokens, outs, blocks;      // mid: tokens and outputs of a tile, K blocks of a stage
  int t_tiles, tiles, splits;
  int bn;            // many: weight rows of a tile
  double us;
};
static TileShape mid_shape(int T, int K, int N, bool gated) {
  TileShape s = {};
  const int most = gated ? kTileW / 2 : kTileW, n_kb = (K + kKb - 1) / kKb;
  s.outs = most;
  s.tiles = (N + most - 1) / most;
  s.t_tiles = (T + 255) / 256;
  s.tokens = ((T + s.t_tiles - 1) / s.t_tiles + 15) & ~15;
  // As many CTAs a cluster as one round of them fits the SMs (a cluster lives in one group of 16 to 20 SMs: 33 clusters of
  // 4 and 15 of 8 fit at once).  K = 4096, N = 4096, 16 tokens (32 tiles), 1 / 2 / 4 / 8 CTAs a cluster: 10.5 / 7.8 / 6.6 /
  // 13.9 us; gated, K = 7168, 2 x 2048 rows, 128 tokens: 18.4 / 12.9 / 10.6 / 26.0 us.
  const int64_t clusters = static_cast<int64_t>(s.tiles) * s.t_tiles;
  const int fit = clusters <= 14 ? 14 : clusters <= 32 ? 32 : clusters <= 74 ? 74 : 148;
  s.splits = fit == 14 ? 8 : fit == 32 ? 4 : fit == 74 ? 2 : 1;
  // A cluster costs 1.2 us and adding up more with more tokens, so there have to be K blocks for it, for eight or four CTAs one
  // or two each, for two, which gain least, more (32 tokens, K = 1024, N = 1024, 1 / 2 / 4 / 8: 4.9 / 5.2 / 4.7 / 5.0 us; 256
  // tokens, K = 512, N = 2048, 1 / 2 / 4: 6.9 / 8.1 / 8.5).  A gated tile has half the outputs, and where outputs are stored
  // one by one, sharing them out is worth it by itself (333 tokens, K = 1000, N = 1537: 11.8 / 10.7 / 8.8).
  const bool odd = N % 4 != 0;
  auto too_few = [&](int splits) { return n_kb < (splits == 2 ? 9 : splits == 4 ? 4 : 10) + (gated || odd ? 0.0 : splits * s.tokens / 128.0); };
  while (s.splits > 1 && too_few(s.splits)) s.splits /= 2;
  // Tiles of fewer weight rows, down to half, where many SMs had none.  K = 7168, N = 512, 128 tokens: 8 tiles of 64 in place
  // of 4 of 128, 7.6 us in place of 8.7; gated, K = 4096, 2 x 2560 rows, 32 tokens: 64 of 40 in place of 40, 7.1 in place of 7.5.
  // Not for fewer SMs (K = 4096, N = 7168, 128 tokens, 69 in place of 56: 11.7 against 11.6) or more tokens, which each tile
  // copies (K = 4096, N = 5120, 200 tokens: 13.2 against 12.5).
  const int room = s.splits == 8 ? 14 : s.splits == 4 ? 32 : s.splits == 2 ? 74 : 148;
  if (clusters * 4 <= room * 3 && s.tokens <= 128) {
    const int tiles = room / s.t_tiles;
    int outs = ((N + tiles - 1) / tiles + 7) & ~7;
    if (outs < most / 2) outs = most / 2;
    if (outs < s.outs) { s.outs = outs; s.tiles = (N + outs - 1) / outs; }
  }
  // K blocks of a stage: what a third of the ring takes, two (which gain less) a quarter (128 tokens, K = 4096, N = 7168, of
  // 32 KB a block: 11.7 us with two, 11.3 with one), in stages of equal size, two at least.  Only whole blocks can go several
  // to a copy.
  const int per = (n_kb + s.splits - 1) / s.splits, block = ((gated ? 2 : 1) * s.outs + s.tokens) * kKb;
  s.blocks = K % kKb ? 1 : kMidRing / 3 / block;
  if (s.blocks < 3 && s.blocks > kMidRing / 4 / block) s.blocks = kMidRing / 4 / block;
  if (s.blocks > (per + 1) / 2) s.blocks = (per + 1) / 2;
  if (s.blocks > kMidMaxBlocks) s.blocks = kMidMaxBlocks;
  if (s.blocks < 1) s.blocks = 1;
  s.blocks = (per + (per + s.blocks - 1) / s.blocks - 1) / ((per + s.blocks - 1) / s.blocks);
  const double ctas = static_cast<double>(s.tiles) * s.t_tiles * s.splits;
  const double rounds = static_cast<double>((static_cast<int64_t>(s.tiles) * s.t_tiles * s.splits + 147) / 148);
  const double kbytes = (gated ? 2 : 1) * s.outs / 8.0 + s.tokens / 8.0;
  const double alone = kbytes / 126.0, busy = kbytes / 83.0 * (ctas < 148 ? ctas / 148.0 : 1.0);
  const double token = 0.010 + ((gated ? 0.006 : 0.0) + (odd ? 0.026 : 0.0)) / s.splits;
  s.us = (s.splits > 1 ? 4.95 : 3.75) + rounds * (token * s.tokens + per * (alone > busy ? alone : busy));
  return s;
}
static TileShape many_shape(int T, int K, int N, bool gated) {
  TileShape s = {};
  const int n_kb = (K + kKb - 1) / kKb;
  const int64_t cols = static_cast<int64_t>(gated ? 2 : 1) * N;
  s.t_tiles = (T + 255) / 256;
  // The tile width with the least work in whole rounds of the 74 pairs.  A round of tiles bn wide takes a time in proportion
  // to bn + 120 (K = 7168, bn 64 / 96 / 128 / 160 / 192 / 224 / 256: 11.1 / 11.4 / 12.4 / 14.1 / 15.0 / 18.1 / 18.9 us): the
  // token rows of a tile are copied whatever its width.  Narrow tiles win where wide ones leave pairs without work.
  long long best = -1, rounds = 0;
  for (int bn = 256; bn >= 64; bn -= gated ? 64 : 32) {
    const long long n = (cols + bn - 1) / bn, r = (n * s.t_tiles + 73) / 74;
    if (best < 0 || r * (bn + 120) < best) { best = r * (bn + 120); rounds = r; s.bn = bn; s.tiles = static_cast<int>(n); }
  }
  const double ctas = 2.0 * s.tiles * s.t_tiles;
  const double alone = s.bn <= 96 ? 0.19 : 0.00088 * (s.bn + 120);
  const double busy = (16 + s.bn / 16.0) / 90.0 * (ctas < 148 ? ctas / 148.0 : 1.0);
  s.us = 4.3 + rounds * (0.018 * s.bn + n_kb * (alone > busy ? alone : busy));
  return s;
}

using MidKernel = void (*)(const Int8MidParams);
template <bool kGated, bool kSingle>
static MidKernel mid_kernel(int splits) {
  return splits == 1 ? okc_int8_mid<kGated, 1, kSingle> : splits == 2 ? okc_int8_mid<kGated, 2, kSingle>
       : splits == 4 ? okc_int8_mid<kGated, 4, kSingle> : okc_int8_mid<kGated, 8, kSingle>;
}

cudaError_t launch_int8_mid(const Int8Params& p, bool gated, bool quantised_here, cudaStream_t stream) {
  Int8MidParams q;
  q.p = p;
  const TileShape shape = mid_shape(p.T, p.K, p.N, gated);
  const int tiles = shape.tiles, ttiles = shape.t_tiles, splits = shape.splits;
  q.outs = shape.outs;
  q.tn = shape.tokens;
  q.n_kb = (p.K + kKb - 1) / kKb;
  q.blocks = shape.blocks;
  const int a_bytes = (gated ? 2 : 1) * q.outs * kKb, x_bytes = q.tn * kKb, stage = (a_bytes + x_bytes) * q.blocks;
  q.stages = kMidRing / stage;
  if (q.stages > kMidMaxStages) q.stages = kMidMaxStages;
  const int most = (q.n_kb + splits * q.blocks - 1) / (splits * q.blocks) + 1;      // stages of a CTA (or one more)
  if (q.stages > most) q.stages = most;
  q.tmem_cols = tmem_cols_for(q.tn);
  if (!encode_blocks_map(&q.wmap, p.w, p.N, gated ? 2 : 1, p.K, p.w_stride, q.outs, q.blocks) ||
      !encode_blocks_map(&q.xmap, p.x, p.T, 1, p.K, p.x_stride, q.tn, q.blocks))
    return cudaErrorInvalidValue;
  // the MMA reads 128 rows, of the last block past the stage's end where a tile has fewer
  const int past = kTileW * kKb - a_bytes - x_bytes * q.blocks;
  size_t smem = 1024 + static_cast<size_t>(q.stages) * stage + (past > 0 ? past : 0);
  if (smem < kMidMinSmem) smem = kMidMinSmem;
  const size_t sums = 1024 + static_cast<size_t>(q.tn) * kTileW * 4;
  if (smem < sums) smem = sums;
  const bool one = q.blocks == 1;
  auto kernel = gated ? (one ? mid_kernel<true, true>(splits) : mid_kernel<true, false>(splits))
                      : (one ? mid_kernel<false, true>(splits) : mid_kernel<false, false>(splits));
  if (smem > kMidMaxSmem) return cudaErrorInvalidValue;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMidMaxSmem);     // (never less: see params.cuh)
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(tiles * splits, ttiles);
  cfg.blockDim = dim3(kMidThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = splits; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = quantised_here ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, q);
}

// ------------------------------------------------------------------ many tokens
// A pair of CTAs works on tiles of 256 tokens x bn weight rows: each CTA brings its 128 token rows and half of the weight
// rows into shared memory, the leader issues the MMAs of both (cta_group::2), each keeps its rows of the sums in its own
// tensor memory, two tiles side by side, so that the end of one tile runs under the next one's MMAs.  Half the operand
// bytes a CTA against two single tiles is what the rate needs: 64 bytes a clock and SM at 256 x 256.
// Bounded by the tensor cores, in long runs by the power they draw: 4096 x 7168 x 7168 123 us at 1965 MHz (3.4e15 operations/s;
// twice the bf16 burst of the measured peaks is 3.25e15) and 147 us at the 1340 MHz that seconds of it leave (2.9e15; 2.8e15);
// gated 4096 x 5120 x 2 x 2048 59 us (2.9e15: 3.5 rounds of tiles) and 66 us at 1560 MHz.
constexpr int kManyThreads = 384;      // warps 0 TMA producer, 1 MMA issuer (leader CTA), 2 TMEM, 3 weight scales, 4..11 epilogue
constexpr int kManyEpilogueWarps = 8;  // one warp a scheduler kept up with one instruction in five cycles only
constexpr int kManyStages = 6;
constexpr int kManyStageBytes = 2 * 128 * kKb;
constexpr int kManyStore = 2048;       // staging of an epilogue warp: 32 rows x 64 bytes
constexpr int kManySmem = 1024 + kManyStages * kManyStageBytes + kManyEpilogueWarps * kManyStore;

struct Int8ManyParams {
  CUtensorMap xmap;      // int8 token rows, box 128 x 128 rows
  CUtensorMap wmap;      // int8 weight rows, box 128 x bn / 2 rows
  CUtensorMap omap;      // bf16 result rows, box 32 columns x 32 rows (only with tma_out)
  Int8Params p;
  int bn;                // weight rows of a pair's tile (columns of its accumulator): a multiple of 32 (gated: 64), at most 256
  int n_kb, tiles_t, tiles_n, tma_out;
};

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
// The same shared-memory address in CTA `rank` of the cluster.
__device__ __forceinline__ uint32_t map_rank(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try_cluster(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred P;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 P, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, P;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
// Bounded wait on a barrier that the other CTA of the pair takes part in (see mbar_wait).
__device__ __forceinline__ bool pair_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int code) {
  if (mbar_try_cluster(bar, parity)) return true;
  const uint32_t c0 = static_cast<uint32_t>(clock());
#pragma unroll 1
  for (;;) {
    if (mbar_try_cluster(bar, parity)) return true;
    if (*abort_flag != 0) return false;
    if (static_cast<uint32_t>(clock()) - c0 > kWaitLimit) break;
  }
  atomicCAS(const_cast<int*>(abort_flag), 0, code);
  return false;
}
// TMA load into this CTA's shared memory whose bytes count on a barrier of either CTA of the pair.
__device__ __forceinline__ void tma_2d_pair(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
      ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(bar)
      : "memory");
}
// Arrives on the barrier at this offset in both CTAs once every MMA of the pair issued so far has completed.
__device__ __forceinline__ void mma_commit_pair(uint32_t bar) {
  asm volatile(
      "{\n\t.reg .b16 m;\n\t"
      "mov.b16 m, 3;\n\t"
      "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], m;\n\t}"
      ::"r"(bar)
      : "memory");
}

__device__ __forceinline__ void st_shared_v4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// 2-D tiled tensor store shared -> global; elements outside the tensor are not written.
__device__ __forceinline__ void tma_2d_s2g(const CUtensorMap* map, uint32_t src, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(c0), "r"(c1), "r"(src)
               : "memory");
}
// 32 bf16 results of a thread's row into its warp's staging: rows of 64 bytes, 16-byte pieces in the 64-byte swizzle.
__device__ __forceinline__ void stage_bf16_row(uint32_t at, int lane, const uint32_t (&r)[32]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack_bf16x2(__uint_as_float(r[8 * j + 2 * i]), __uint_as_float(r[8 * j + 2 * i + 1]));
    st_shared_v4(at + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4), w[0], w[1], w[2], w[3]);
  }
}

template <bool kGated>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kManyThreads) okc_int8_many(const __grid_constant__ Int8ManyParams q) {
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
  __shared__ uint64_t bar_full[kManyStages], bar_empty[kManyStages], bar_acc_full[2], bar_acc_empty[2], bar_sc_full[2], bar_sc_empty[2];
  __shared__ __align__(16) float scale_s[2][256], bias_s[2][256];
  __shared__ uint32_t tmem_base_s;
  __shared__ int abort_code;
  const Int8Params& p = q.p;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t rank = cluster_rank();
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int tiles = q.tiles_t * q.tiles_n;

  if (tid == 0) {
    for (int i = 0; i < kManyStages; ++i) { mbar_init(smem_u32(&bar_full[i]), 1); mbar_init(smem_u32(&bar_empty[i]), 1); }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&bar_acc_full[i]), 1); mbar_init(smem_u32(&bar_acc_empty[i]), 2 * kManyEpilogueWarps);
      mbar_init(smem_u32(&bar_sc_full[i]), 1); mbar_init(smem_u32(&bar_sc_empty[i]), kManyEpilogueWarps);
    }
    abort_code = 0;
    mbar_fence_init();
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&tmem_base_s)), "r"(512u) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  cg::this_cluster().sync();
  tc_fence_after();
  const uint32_t tmem = tmem_base_s;

  if (warp == 0) {
    griddep_wait();
    const uint32_t half_bytes = 128u * kKb + static_cast<uint32_t>(q.bn / 2) * kKb;
    const uint32_t full0 = map_rank(smem_u32(&bar_full[0]), 0);      // the bytes of both CTAs count on the leader's barriers
    const uint32_t empty0 = smem_u32(&bar_empty[0]);
    uint32_t st = 0, ph = 1;
    bool ok = true;
    for (int tile = pair; tile < tiles && ok; tile += pairs) {
      const int tt = tile % q.tiles_t, tw = tile / q.tiles_t;
      const int xrow = tt * 256 + static_cast<int>(rank) * 128;
      const int wrow = kGated ? static_cast<int>(rank) * p.N + tw * (q.bn / 2) : tw * q.bn + static_cast<int>(rank) * (q.bn / 2);
      for (int kb = 0; kb < q.n_kb; ++kb) {
        ok = pair_wait(empty0 + 8 * st, ph, &abort_code, 0x71);      // (the first round finds the slots empty)
        if (!ok) break;
        const uint32_t bar = full0 + 8 * st, dst = smem0 + st * kManyStageBytes;
        if (elect_one()) {
          if (rank == 0) mbar_expect_tx(smem_u32(&bar_full[st]), 2 * half_bytes);
          tma_2d_pair(dst, &q.xmap, kb * kKb, xrow, bar);
          tma_2d_pair(dst + 128 * kKb, &q.wmap, kb * kKb, wrow, bar);
        }
        if (++st == kManyStages) { st = 0; ph ^= 1; }
      }
    }
    // The issuer's last arrivals at this CTA's empty barriers come from the other CTA of the pair and nobody has waited for
    // them yet: they have to land before this CTA's memory becomes another's.  (Empty barriers that were never used, or
    // whose last arrival has been seen, pass at once.)
    for (int i = 0; ok && i < kManyStages; ++i) {
      ok = pair_wait(empty0 + 8 * st, ph, &abort_code, 0x77);
      if (++st == kManyStages) { st = 0; ph ^= 1; }
    }
    // Every copy has landed once the epilogue has seen the last tile; a producer that gave up leaves them some time.
    if (!ok) {
      const long long c0 = clock64();
      while (clock64() - c0 < kWaitLimitCycles / 100) {}
    }
    __syncwarp();
  } else if (warp == 1) {
    if (rank == 0) {
      const uint32_t idesc = idesc_i8(256, static_cast<uint32_t>(q.bn));
      const uint32_t full0 = smem_u32(&bar_full[0]), empty0 = smem_u32(&bar_empty[0]), lo0 = desc_lo(smem0);
      uint32_t st = 0, ph = 0, buf = 0, bph = 1;
      bool ok = true;
      for (int tile = pair; tile < tiles && ok; tile += pairs) {
        ok = pair_wait(smem_u32(&bar_acc_empty[buf]), bph, &abort_code, 0x72);     // (the first two tiles find it empty)
        tc_fence_after();
        const uint32_t d = tmem + buf * 256;
        for (int kb = 0; ok && kb < q.n_kb; ++kb) {
          ok = pair_wait(full0 + 8 * st, ph, &abort_code, 0x73);
          if (!ok) break;
          tc_fence_after();
          const uint32_t a = lo0 + st * (kManyStageBytes >> 4), b = a + (128 * kKb >> 4);
          if (elect_one()) {
            mma_i8_pair(d, a, b, kDescHi, idesc, kb != 0);
            mma_i8_pair(d, a + 2, b + 2, kDescHi, idesc, 1);
            mma_i8_pair(d, a + 4, b + 4, kDescHi, idesc, 1);
            mma_i8_pair(d, a + 6, b + 6, kDescHi, idesc, 1);
            mma_commit_pair(empty0 + 8 * st);
          }
          if (++st == kManyStages) { st = 0; ph ^= 1; }
        }
        if (ok && elect_one()) mma_commit_pair(smem_u32(&bar_acc_full[buf]));
        buf ^= 1;
        if (buf == 0) bph ^= 1;
      }
    }
    __syncwarp();
  } else if (warp == 3) {
    // the weight scales (and bias) of the tiles ahead of the epilogue, into shared memory
    const int half = q.bn / 2, width = kGated ? half : q.bn;
    uint32_t buf = 0, ph = 1;
    for (int tile = pair; tile < tiles; tile += pairs) {
      if (!pair_wait(smem_u32(&bar_sc_empty[buf]), ph, &abort_code, 0x75)) break;
      const int tw = tile / q.tiles_t;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = i * 32 + lane;
        const bool up = kGated && c >= half;
        const int o = tw * width + (up ? c - half : c);
        if (c < q.bn) {
          scale_s[buf][c] = o < p.N ? __ldg(p.w_scale + (up ? p.N + o : o)) : 0.f;
          if (!kGated) bias_s[buf][c] = p.bias && o < p.N ? __ldg(p.bias + o) : -0.f;      // v + -0 is v, whatever v
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_u32(&bar_sc_full[buf]));
      buf ^= 1;
      if (buf == 0) ph ^= 1;
    }
  } else if (warp >= 4) {
    griddep_wait();        // the token scales come from the kernel before this one
    const int ew = warp - 4, half = q.bn / 2;
    const int width = kGated ? half : q.bn;        // outputs of a tile
    const int first = (ew >> 2) * 32;              // two warps share a quarter of the rows: every second 32 columns each
    const int row_in = static_cast<int>(rank) * 128 + (ew & 3) * 32;
    const uint32_t taddr = tmem + (static_cast<uint32_t>((ew & 3) * 32) << 16);
    const uint32_t at = smem0 + kManyStages * kManyStageBytes + ew * kManyStore;
    uint32_t buf = 0, ph = 0;
    int t = (pair % q.tiles_t) * 256 + row_in + lane;
    float sx_next = pair < tiles && t < p.T ? p.x_scale[t] : 0.f;
    for (int tile = pair; tile < tiles; tile += pairs) {
      const int tw = tile / q.tiles_t, row0 = (tile % q.tiles_t) * 256 + row_in;
      const float sx = sx_next;
      t = ((tile + pairs) % q.tiles_t) * 256 + row_in + lane;
      if (tile + pairs < tiles && t < p.T) sx_next = p.x_scale[t];
      t = row0 + lane;
      if (!pair_wait(smem_u32(&bar_sc_full[buf]), ph, &abort_code, 0x76)) break;
      if (!pair_wait(smem_u32(&bar_acc_full[buf]), ph, &abort_code, 0x74)) break;
      tc_fence_after();
      const uint32_t acc_empty = map_rank(smem_u32(&bar_acc_empty[buf]), 0);
      if (first >= width) {
        if (lane == 0) mbar_arrive_cluster(acc_empty);
      }
      for (int c0 = first; c0 < width; c0 += 64) {
        uint32_t r[32], u[32];
        tmem_ld32(taddr + buf * 256 + c0, r);
        if (kGated) tmem_ld32(taddr + buf * 256 + half + c0, u);
        tmem_wait_ld();
        if (c0 + 64 >= width) {       // read for the last time: the pair's next tile but one may overwrite it
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_cluster(acc_empty);
        }
        // four scales (and biases) a load, and no branch: what is left of the last tile after its MMAs is this (512 tokens,
        // K = 4096, N = 4096: 13.0 us, one by one 13.2; 256 tokens, one K block, tiles 256 wide: 8.4, 8.9)
        const float4* ws = reinterpret_cast<const float4*>(scale_s[buf] + c0);
        const float4* bs = reinterpret_cast<const float4*>(kGated ? scale_s[buf] + half + c0 : bias_s[buf] + c0);
#pragma unroll
        for (int j4 = 0; j4 < 8; ++j4) {
          const float4 w4 = ws[j4], b4 = bs[j4];
          const float wv[4] = {w4.x, w4.y, w4.z, w4.w}, bv[4] = {b4.x, b4.y, b4.z, b4.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int j = 4 * j4 + i;
            float v = int8_value(static_cast<int>(r[j]), sx, wv[i]);
            if (kGated) v = silu_mul(v, int8_value(static_cast<int>(u[j]), sx, bv[i]));
            else v = __fadd_rn(v, bv[i]);
            r[j] = __float_as_uint(v);
          }
        }
        // A thread has 32 neighbouring results of its own row.  As bf16 they leave through shared memory and a TMA store a
        // warp, whole sectors at a time (stored by the threads themselves, 16 bytes each, 4096x1024x4096 takes 28.6 us for
        // 25.3); as f32 the thread has whole sectors.
        // A store that ends a row off a 16-byte boundary fills up to that with zeros, over what a caller has behind the row:
        // such last columns go the third way.
        const int col = tw * width + c0;
        if (q.tma_out) {
          if (lane == 0) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");
          __syncwarp();
        }
        if (q.tma_out && (col + 32 <= p.N || p.N % 8 == 0)) {
          stage_bf16_row(at, lane, r);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) {
            if (row0 < p.T && col < p.N) tma_2d_s2g(&q.omap, at, col, row0);
            asm volatile("cp.async.bulk.commit_group;" ::: "memory");
          }
        } else if (p.out_f32 && p.out_vec && col + 32 <= p.N) {
          if (t < p.T) {
            uint4* dst = reinterpret_cast<uint4*>(static_cast<float*>(p.out) + static_cast<int64_t>(t) * p.out_stride + col);
#pragma unroll
            for (int j = 0; j < 8; ++j) dst[j] = make_uint4(r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
          }
        } else {
          // rows off the 16-byte grid, or the last columns: through shared memory, so that a warp stores neighbours of a row
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (h == 1 && !p.out_f32) break;
            if (p.out_f32) {
#pragma unroll
              for (int j = 0; j < 4; ++j) st_shared_v4(at + lane * 64 + ((j ^ ((lane >> 1) & 3)) << 4), r[16 * h + 4 * j], r[16 * h + 4 * j + 1], r[16 * h + 4 * j + 2], r[16 * h + 4 * j + 3]);
            } else {
              stage_bf16_row(at, lane, r);
            }
            __syncwarp();
            if (p.out_f32) {       // 16 columns of two rows a step
              const int cc = col + 16 * h + (lane & 15);
#pragma unroll 4
              for (int i = lane >> 4; i < 32; i += 2) {
                uint32_t v;
                asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(at + i * 64 + ((((lane & 15) >> 2) ^ ((i >> 1) & 3)) << 4) + (lane & 3) * 4));
                if (cc < p.N && row0 + i < p.T) static_cast<float*>(p.out)[static_cast<int64_t>(row0 + i) * p.out_stride + cc] = __uint_as_float(v);
              }
            } else {
              const int cc = col + lane;
#pragma unroll 8
              for (int i = 0; i < 32; ++i) {
                uint16_t v;
                asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at + i * 64 + (((lane >> 3) ^ ((i >> 1) & 3)) << 4) + (lane & 7) * 2));
                if (cc < p.N && row0 + i < p.T) static_cast<uint16_t*>(p.out)[static_cast<int64_t>(row0 + i) * p.out_stride + cc] = v;
              }
            }
            __syncwarp();
          }
        }
        __syncwarp();      // the next load from tensor memory is one of the whole warp
      }
      if (lane == 0) mbar_arrive(smem_u32(&bar_sc_empty[buf]));
      buf ^= 1;
      if (buf == 0) ph ^= 1;
    }
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
    __syncwarp();
  }
  tc_fence_before();
  cg::this_cluster().sync();     // no CTA frees its tensor memory or leaves while the pair's MMAs and arrivals may touch it
  if (warp == 2) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
  }
  if (tid == 0 && abort_code != 0) publish_timeout(&g_int8_status, abort_code);
}

bool int8_use_many(int T, int K, int N, bool gated) { return T > 512 || many_shape(T, K, N, gated).us < mid_shape(T, K, N, gated).us; }

cudaError_t launch_int8_many(const Int8Params& p, bool gated, bool quantised_here, cudaStream_t stream) {
  Int8ManyParams q;
  q.p = p;
  q.n_kb = (p.K + kKb - 1) / kKb;
  const TileShape shape = many_shape(p.T, p.K, p.N, gated);
  const int64_t cols = static_cast<int64_t>(gated ? 2 : 1) * p.N;
  q.tiles_t = shape.t_tiles;
  q.bn = shape.bn;
  q.tiles_n = shape.tiles;      // (of a gated product: n tiles of bn / 2 outputs cover as many as n tiles of bn rows)
  if (!encode_bytes_map(&q.xmap, p.x, p.T, p.K, p.x_stride, 128) ||
      !encode_bytes_map(&q.wmap, p.w, static_cast<uint64_t>(cols), p.K, p.w_stride, q.bn / 2))
    return cudaErrorInvalidValue;
  q.tma_out = p.out_vec && !p.out_f32;
  if (q.tma_out && !encode_bf16_out_map(&q.omap, p.out, p.T, p.N, p.out_stride)) return cudaErrorInvalidValue;
  const long long tiles = static_cast<long long>(q.tiles_t) * q.tiles_n;
  const int grid = static_cast<int>(tiles < 74 ? 2 * tiles : 148);
  auto kernel = gated ? okc_int8_many<true> : okc_int8_many<false>;
  cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kManySmem);
  if (e != cudaSuccess) return e;
  return launch_kernel(kernel, dim3(grid), dim3(kManyThreads), kManySmem, stream, quantised_here, q);
}

__global__ void okc_int8_probe_timeout() { probe_timeout(&g_int8_status, 0x7c); }
cudaError_t launch_int8_probe_timeout(cudaStream_t stream) {
  okc_int8_probe_timeout<<<1, 32, 0, stream>>>();
  return cudaGetLastError();
}

// Reads the word and, where it holds a code, clears that code: one that another stream's kernel records after the read stays.
__global__ void okc_int8_clear_status(int32_t code) { atomicCAS(&g_int8_status, code, 0); }
cudaError_t int8_read_status(cudaStream_t stream, int32_t* code) {
  cudaError_t e = cudaMemcpyFromSymbolAsync(code, g_int8_status, sizeof(int32_t), 0, cudaMemcpyDeviceToHost, stream);
  if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
  if (e != cudaSuccess || *code == 0) return e;
  okc_int8_clear_status<<<1, 1, 0, stream>>>(*code);
  e = cudaGetLastError();
  return e != cudaSuccess ? e : cudaStreamSynchronize(stream);
}

}  // namespace okc
