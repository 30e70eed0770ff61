// Row helpers shared by the norm, quantising and int8 product kernels: loads of eight consecutive values as f32, the
// rounding to bf16 and to int8, and sums / maxima over the threads of a CTA that share a row.
#pragma once
#include <cuda_bf16.h>

#include <cstdint>

#include "params.cuh"

namespace okc {

// Rows of int8 values.  With a = max |x| of the row: scale = a / 127, value = rint(x * (127 / a)), both quotients
// rounded to f32 once per row and the product rounded to f32 once, so every kernel that quantises (and a caller that
// does it elsewhere) gets the same integers.  A row with a < 2^-120 (127 / a would leave the range of f32) counts as
// zeros: scale 0.  A row that holds an infinity or a NaN gets scale NaN and zeros, so that every product of the row
// is NaN instead of a number made from part of it.
struct RowScale {
  float scale, inv;
  uint32_t keep;      // all ones, or zero for a row that is not finite
};
__device__ __forceinline__ RowScale row_scale(uint32_t amax_bits) {
  RowScale s;
  const float a = __uint_as_float(amax_bits);
  const bool zero = a < 7.52316385e-37f;                        // 2^-120
  s.keep = amax_bits < 0x7F800000u ? 0xFFFFFFFFu : 0u;
  s.scale = zero ? 0.f : s.keep ? __fdiv_rn(a, 127.f) : __uint_as_float(0x7FC00000u);
  s.inv = zero || !s.keep ? 0.f : __fdiv_rn(127.f, a);
  return s;
}
// rint(x * inv) as a byte.  Below 2^22 in magnitude, v + 1.5 * 2^23 rounds v to an integer, halves to even, which then is
// the low end of the sum's bits: one addition instead of a conversion, which runs at a quarter of its rate or less.
// |x * inv| is at most 127 * (1 + 2^-23), so the value needs no clamp; a row that is not finite has its bytes cleared.
__device__ __forceinline__ uint32_t quant_bits(float x, float inv) { return __float_as_uint(__fadd_rn(__fmul_rn(x, inv), 12582912.f)); }
__device__ __forceinline__ uint32_t quant8(float x, const RowScale& s) { return quant_bits(x, s.inv) & s.keep & 0xFFu; }
__device__ __forceinline__ uint32_t quant8x4(float a, float b, float c, float d, const RowScale& s) {
  const uint32_t lo = __byte_perm(quant_bits(a, s.inv), quant_bits(b, s.inv), 0x0040);
  const uint32_t hi = __byte_perm(quant_bits(c, s.inv), quant_bits(d, s.inv), 0x0040);
  return __byte_perm(lo, hi, 0x5410) & s.keep;
}
// Bits of |x|: compared as integers a NaN is above every number, so a maximum of these never loses one.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }

__device__ __forceinline__ void unpack_bf16x8(uint4 u, float (&v)[8]) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    v[2 * j] = __uint_as_float(w[j] << 16);
    v[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ uint32_t pack_bf16x2(float lo, float hi) {
  const __nv_bfloat162 b = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&b);
}

// Two f32 in one 64-bit register: sm_100 multiplies and adds such pairs in one instruction, each half rounded as usual.
using F2 = unsigned long long;
__device__ __forceinline__ F2 f2_pack(float lo, float hi) {
  F2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ void f2_unpack(F2 v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ F2 f2_mul(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ F2 f2_fma(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
// Eight neighbouring values at column c of an aligned row, as four pairs.
__device__ __forceinline__ void load8_f2(const void* row, bool f32, int c, F2 (&v)[4]) {
  if (f32) {
    const float4 a = reinterpret_cast<const float4*>(static_cast<const float*>(row) + c)[0];
    const float4 b = reinterpret_cast<const float4*>(static_cast<const float*>(row) + c)[1];
    v[0] = f2_pack(a.x, a.y); v[1] = f2_pack(a.z, a.w); v[2] = f2_pack(b.x, b.y); v[3] = f2_pack(b.z, b.w);
  } else {
    const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(row) + c);
    const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = f2_pack(__uint_as_float(w[j] << 16), __uint_as_float(w[j] & 0xFFFF0000u));
  }
}
__device__ __forceinline__ void store8_f2(void* row, bool f32, int c, const F2 (&v)[4]) {
  float f[8];
#pragma unroll
  for (int j = 0; j < 4; ++j) f2_unpack(v[j], f[2 * j], f[2 * j + 1]);
  if (f32) {
    float4* d = reinterpret_cast<float4*>(static_cast<float*>(row) + c);
    d[0] = make_float4(f[0], f[1], f[2], f[3]);
    d[1] = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    *reinterpret_cast<uint4*>(static_cast<uint16_t*>(row) + c) =
        make_uint4(pack_bf16x2(f[0], f[1]), pack_bf16x2(f[2], f[3]), pack_bf16x2(f[4], f[5]), pack_bf16x2(f[6], f[7]));
  }
}

// The columns of a row belong to threads in chunks of eight.  With kVec a chunk is eight neighbours (16- and 32-byte
// accesses; the host checks that the width and every stride and address allow them); without, neighbouring threads
// take neighbouring columns, so that single-element accesses still coalesce.
template <bool kVec>
__device__ __forceinline__ int row_col(int chunk, int e, int tid, int nt) {
  return kVec ? (chunk * nt + tid) * 8 + e : (chunk * 8 + e) * nt + tid;
}
template <bool kVec>
__device__ __forceinline__ void load_chunk(const void* row, bool f32, int chunk, int tid, int nt, int cols, float (&v)[8]) {
  if (kVec) {
    const int c = row_col<true>(chunk, 0, tid, nt);
    if (c < cols) {
      if (f32) {
        const float4 a = reinterpret_cast<const float4*>(static_cast<const float*>(row) + c)[0];
        const float4 b = reinterpret_cast<const float4*>(static_cast<const float*>(row) + c)[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
      } else {
        unpack_bf16x8(*reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(row) + c), v);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 0.f;
    }
  } else {
    // (the type is asked once, not for every value: the eight loads have to be under way together)
    if (f32) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int c = row_col<false>(chunk, e, tid, nt);
        v[e] = c < cols ? static_cast<const float*>(row)[c] : 0.f;
      }
    } else {
      uint32_t u[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int c = row_col<false>(chunk, e, tid, nt);
        u[e] = c < cols ? static_cast<const uint16_t*>(row)[c] : 0u;
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = __uint_as_float(u[e] << 16);
    }
  }
}
template <bool kVec>
__device__ __forceinline__ void store_chunk(void* row, bool f32, int chunk, int tid, int nt, int cols, const float (&v)[8]) {
  if (kVec) {
    const int c = row_col<true>(chunk, 0, tid, nt);
    if (c >= cols) return;
    if (f32) {
      float4* d = reinterpret_cast<float4*>(static_cast<float*>(row) + c);
      d[0] = make_float4(v[0], v[1], v[2], v[3]);
      d[1] = make_float4(v[4], v[5], v[6], v[7]);
    } else {
      *reinterpret_cast<uint4*>(static_cast<uint16_t*>(row) + c) =
          make_uint4(pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3]), pack_bf16x2(v[4], v[5]), pack_bf16x2(v[6], v[7]));
    }
  } else {
    if (f32) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int c = row_col<false>(chunk, e, tid, nt);
        if (c < cols) static_cast<float*>(row)[c] = v[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int c = row_col<false>(chunk, e, tid, nt);
        if (c < cols) static_cast<__nv_bfloat16*>(row)[c] = __float2bfloat16_rn(v[e]);
      }
    }
  }
}
template <bool kVec>
__device__ __forceinline__ void store_chunk_q(int8_t* row, int chunk, int tid, int nt, int cols, const float (&v)[8], const RowScale& s) {
  if (kVec) {
    const int c = row_col<true>(chunk, 0, tid, nt);
    if (c < cols) *reinterpret_cast<uint2*>(row + c) = make_uint2(quant8x4(v[0], v[1], v[2], v[3], s), quant8x4(v[4], v[5], v[6], v[7], s));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int c = row_col<false>(chunk, e, tid, nt);
      if (c < cols) row[c] = static_cast<int8_t>(quant8(v[e], s));
    }
  }
}

// Sum / maximum over all threads of the CTA (a multiple of 32, at most 1024).  `red` is 32 words of shared memory that
// no other call of the kernel uses, so one barrier is enough.  The order of the additions depends on the thread count
// alone.
__device__ __forceinline__ float cta_sum(float x, float* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  if (blockDim.x == 32) return x;
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = x;
  __syncthreads();
  x = (threadIdx.x & 31) < (blockDim.x >> 5) ? red[threadIdx.x & 31] : 0.f;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}
__device__ __forceinline__ uint32_t cta_max(uint32_t x, uint32_t* red) {
  x = __reduce_max_sync(0xffffffffu, x);
  if (blockDim.x == 32) return x;
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = x;
  __syncthreads();
  x = (threadIdx.x & 31) < (blockDim.x >> 5) ? red[threadIdx.x & 31] : 0u;
  return __reduce_max_sync(0xffffffffu, x);
}

// The code of a wait that ran out, into the module's status word: the first since the word was read stays.
__device__ __forceinline__ void publish_timeout(int32_t* word, int code) { atomicCAS(word, 0, code); }
// A wait, with a short limit, on a barrier that nothing completes (one warp): what the kernels do when theirs run out.
__device__ __forceinline__ void probe_timeout(int32_t* word, int code) {
  __shared__ uint64_t bar;
  __shared__ int abort_code;
  if (threadIdx.x == 0) {
    mbar_init(smem_u32(&bar), 1);
    abort_code = 0;
    mbar_fence_init();
  }
  __syncthreads();
  mbar_wait(smem_u32(&bar), 0, &abort_code, code, 1u << 14);
  __syncthreads();
  if (threadIdx.x == 0 && abort_code != 0) publish_timeout(word, abort_code);
}

}  // namespace okc
