// Read-back of int32 accumulators with one scale per row and one per column.
#pragma once

#include "ptx.cuh"

namespace smb {

// z = (float(acc) * row scale) * column scale: the same three roundings in every kernel of the int8
// product, so that all of them give the same bits.
__device__ __forceinline__ float scale_i32(uint32_t acc, float row_scale, float col_scale) {
  return __fmul_rn(__fmul_rn(__int2float_rn(static_cast<int>(acc)), row_scale), col_scale);
}

// silu(gate) * up = gate / (1 + exp(-gate)) * up.  ex2.approx and rcp.approx are within 2^-22 relative, the
// rounded exponent argument adds |gate| 2^-24: far below the 2^-8 of the bf16 that follows.  For gate below
// -88 the exponential overflows to infinity and the result is -0.
__device__ __forceinline__ float silu_mul(float gate, float up) {
  float e, r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(gate * -1.4426950408889634f));
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + e));
  return gate * r * up;
}

// The scales of columns [col0, col0 + kCols) to the front of the warp's staging buffer; columns from
// `n` on (never stored) get 0.  kTma: the TMA stores that read the buffer have to finish first.
template <int kCols, bool kTma>
__device__ __forceinline__ void stage_column_scales(uint32_t sbuf, const float* sb, int col0, int n, int lane) {
  float v[kCols / 32];
#pragma unroll
  for (int i = 0; i < kCols / 32; ++i) {
    const int c = col0 + i * 32 + lane;
    v[i] = c < n ? sb[c] : 0.0f;
  }
  if (kTma) {
    if (lane == 0) bulk_wait_group_read<0>();
  }
  __syncwarp();
#pragma unroll
  for (int i = 0; i < kCols / 32; ++i)
    asm volatile("st.shared.f32 [%0], %1;" ::"r"(sbuf + (i * 32 + lane) * 4), "f"(v[i]) : "memory");
  __syncwarp();
}

// kCols int32 columns of this warp's 32 lanes (lane = row), scaled and packed to bf16 pairs;
// kSwiglu: columns 2n, 2n + 1 are up, gate of output n.  kAhead: the next 32 columns travel from tensor
// memory while the current ones are scaled (32 more registers).
template <int kCols, bool kSwiglu, bool kAhead>
__device__ __forceinline__ void drain_columns_i8(uint32_t taddr, uint32_t sbuf, float sa,
                                                 uint32_t (&packed)[(kSwiglu ? kCols / 2 : kCols) / 2]) {
  uint32_t v[kAhead ? 2 : 1][32];
  tmem_ld_32x32b_x32(taddr, v[0]);
#pragma unroll
  for (int g = 0; g < kCols / 32; ++g) {
    uint32_t(&w)[32] = v[kAhead ? g & 1 : 0];
    if (!kAhead && g > 0) tmem_ld_32x32b_x32(taddr + g * 32, w);
    tmem_ld_wait();
    if (kAhead && g + 1 < kCols / 32) tmem_ld_32x32b_x32(taddr + (g + 1) * 32, v[(g + 1) & 1]);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      uint32_t s0, s1, s2, s3;
      ld_shared_v4(sbuf + (g * 32 + 4 * i) * 4, s0, s1, s2, s3);
      const float z0 = scale_i32(w[4 * i], sa, __uint_as_float(s0));
      const float z1 = scale_i32(w[4 * i + 1], sa, __uint_as_float(s1));
      const float z2 = scale_i32(w[4 * i + 2], sa, __uint_as_float(s2));
      const float z3 = scale_i32(w[4 * i + 3], sa, __uint_as_float(s3));
      if (kSwiglu) {
        packed[g * 8 + i] = pack_bf16x2(__float_as_uint(silu_mul(z1, z0)), __float_as_uint(silu_mul(z3, z2)));
      } else {
        packed[g * 16 + 2 * i] = pack_bf16x2(__float_as_uint(z0), __float_as_uint(z1));
        packed[g * 16 + 2 * i + 1] = pack_bf16x2(__float_as_uint(z2), __float_as_uint(z3));
      }
    }
  }
  __syncwarp();   // every lane has read its scales before the buffer takes the packed box
}

}  // namespace smb
