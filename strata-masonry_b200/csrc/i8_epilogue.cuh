// Read-back of int32 accumulators with one scale per row and one per column.
#pragma once

#include "ptx.cuh"

namespace smb {

// z = (float(acc) * row scale) * column scale: the same three roundings in every kernel of the int8
// product, so that all of them give the same bits.
__device__ __forceinline__ float scale_i32(uint32_t acc, float row_scale, float col_scale) {
  return __fmul_rn(__fmul_rn(__int2float_rn(static_cast<int>(acc)), row_scale), col_scale);
}

// Two floats to a bf16 pair, round to nearest even.  Not volatile: the compiler may move it between the
// shuffles and loads of neighbouring outputs.
__device__ __forceinline__ uint32_t bf16_pair(float lo, float hi) {
  uint32_t out;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(out) : "f"(hi), "f"(lo));
  return out;
}

// silu(gate) * up = gate / (1 + exp(-gate)) * up.  ex2.approx and rcp.approx are within 2^-22 relative, the
// rounded exponent argument adds |gate| 2^-24: far below the 2^-8 of the bf16 that follows.  For gate below
// -87 the reciprocal would be subnormal, and the result is -0.
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
        packed[g * 8 + i] = bf16_pair(silu_mul(z1, z0), silu_mul(z3, z2));
      } else {
        packed[g * 16 + 2 * i] = bf16_pair(z0, z1);
        packed[g * 16 + 2 * i + 1] = bf16_pair(z2, z3);
      }
    }
  }
  __syncwarp();   // every lane has read its scales before the buffer takes the packed box
}

// For kernels whose accumulator lanes are channels (columns of D) and whose columns are tokens (rows of D):
// kCount tokens of this lane's channel n, from row pointer `d` on, `valid` of them inside D (<= 0: none).
// `scale`: lane i holds the scale of token i.  Neighbouring lanes trade halves, so that even lanes write two
// channels of the even tokens and odd lanes two of the odd ones; with the gated epilogue the two are up and
// gate of one output.  kPairs: D takes 4-byte stores.  Nothing branches before the stores, so that the
// shuffles and exponentials of all tokens overlap.
template <int kCount, bool kSwiglu, bool kPairs>
__device__ __forceinline__ void store_tokens(const uint32_t (&acc)[kCount], float scale, float sb, uint16_t* d, int ldd,
                                             int n_total, int valid, int n) {
  float z[kCount];
#pragma unroll
  for (int i = 0; i < kCount; ++i) z[i] = scale_i32(acc[i], __shfl_sync(0xffffffffu, scale, i), sb);
  if (!kSwiglu && !kPairs) {
#pragma unroll
    for (int i = 0; i < kCount; ++i) {
      if (i < valid && n < n_total)
        d[static_cast<long long>(i) * ldd + n] = static_cast<uint16_t>(bf16_pair(z[i], 0.0f) & 0xFFFFu);
    }
    return;
  }
  const bool odd = n & 1;
  const int n0 = n & ~1;
  uint32_t out[kCount / 2];
#pragma unroll
  for (int i = 0; i < kCount; i += 2) {
    const float other = __shfl_xor_sync(0xffffffffu, odd ? z[i] : z[i + 1], 1);
    const float lo = odd ? other : z[i], hi = odd ? z[i + 1] : other;
    out[i / 2] = kSwiglu ? bf16_pair(silu_mul(hi, lo), 0.0f) : bf16_pair(lo, hi);
  }
  if (n0 >= n_total) return;
  const int left = valid - (odd ? 1 : 0);
  uint16_t* row = d + (odd ? ldd : 0) + (kSwiglu ? n0 >> 1 : n0);
  const bool whole = kSwiglu || n0 + 1 < n_total;
#pragma unroll
  for (int i = 0; i < kCount; i += 2) {
    if (i < left) {
      if (kSwiglu || !whole) row[0] = static_cast<uint16_t>(out[i / 2] & 0xFFFFu);
      else *reinterpret_cast<uint32_t*>(row) = out[i / 2];
    }
    row += 2 * static_cast<long long>(ldd);
  }
}

}  // namespace smb
