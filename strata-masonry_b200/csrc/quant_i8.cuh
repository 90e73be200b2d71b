// Per-row int8 quantiser, shared by the plain quantiser and the one that copies rows to experts.
//
//   amax  = max(max_k |x[k]|, 2^-100)           (the floor keeps 127 / amax finite)
//   scale = fl32(amax / 127),  inv = fl32(127 / amax)
//   code  = round_half_even(fl32(x[k] * inv)),  in [-127, 127]
//
// The definition is in these fp32 operations, so that host, device and any other program agree on
// every code.  A row with an infinity or a NaN gets codes 0 and scale NaN: its products are NaN.
#pragma once

#include <cstdint>

#include "ptx.cuh"

namespace smb {
namespace qi8 {

constexpr float kMinAmax = 7.8886090522101181e-31f;   // 2^-100

// Eight consecutive elements as they are loaded.
template <bool kBf16>
struct Vec {
  uint32_t w[kBf16 ? 4 : 8];
};

template <bool kBf16>
__device__ __forceinline__ Vec<kBf16> load_vec(const void* row, int64_t k) {
  Vec<kBf16> v;
  const uint4* p = reinterpret_cast<const uint4*>(static_cast<const char*>(row) + k * (kBf16 ? 2 : 4));
#pragma unroll
  for (int i = 0; i < (kBf16 ? 1 : 2); ++i) {
    const uint4 q = p[i];
    v.w[4 * i] = q.x;
    v.w[4 * i + 1] = q.y;
    v.w[4 * i + 2] = q.z;
    v.w[4 * i + 3] = q.w;
  }
  return v;
}

// Largest magnitude as an fp32 bit pattern: magnitudes order like their bits, and infinities and
// NaNs come out above every finite value.
template <bool kBf16>
__device__ __forceinline__ uint32_t abs_max_bits(const Vec<kBf16>& v, uint32_t m) {
  if (kBf16) {
    uint32_t pair = v.w[0] & 0x7FFF7FFFu;
#pragma unroll
    for (int i = 1; i < 4; ++i) pair = __vmaxu2(pair, v.w[i] & 0x7FFF7FFFu);
    return max(m, max(pair << 16, pair & 0xFFFF0000u));
  }
#pragma unroll
  for (int i = 0; i < (kBf16 ? 4 : 8); ++i) m = max(m, v.w[i] & 0x7FFFFFFFu);
  return m;
}

// Bits of the rounded code in the low byte: adding 1.5 * 2^23 to |q| <= 127 leaves no room for a
// fraction, so the addition itself rounds half to even.
__device__ __forceinline__ uint32_t code_bits(float x, float inv) {
  return __float_as_uint(__fadd_rn(__fmul_rn(x, inv), 12582912.0f));
}

__device__ __forceinline__ uint32_t pack4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}

template <bool kBf16>
__device__ __forceinline__ uint2 encode(const Vec<kBf16>& v, float inv) {
  uint32_t c[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    float x;
    if (kBf16) x = __uint_as_float((i & 1) ? (v.w[i >> 1] & 0xFFFF0000u) : (v.w[i >> 1] << 16));
    else x = __uint_as_float(v.w[kBf16 ? 0 : i]);
    c[i] = code_bits(x, inv);
  }
  return make_uint2(pack4(c[0], c[1], c[2], c[3]), pack4(c[4], c[5], c[6], c[7]));
}

template <bool kBf16>
__device__ __forceinline__ float load_one(const void* row, int64_t k) {
  if (kBf16) return __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(row)[k]) << 16);
  return static_cast<const float*>(row)[k];
}

struct RowScale {
  float scale, inv;
  bool bad;
};

__host__ __device__ inline RowScale row_scale(float amax, bool finite) {
  RowScale r;
  r.bad = !finite;
  const float a = amax > kMinAmax ? amax : kMinAmax;
#ifdef __CUDA_ARCH__
  r.scale = __fdiv_rn(a, 127.0f);
  r.inv = __fdiv_rn(127.0f, a);
#else
  r.scale = a / 127.0f;
  r.inv = 127.0f / a;
#endif
  return r;
}

constexpr int kHeldVecs = 4;      // vectors of a row that a thread keeps between the two passes
constexpr int kHeldWords = 16;    // the same where rows take no vectors, for a warp with single elements twice as many
constexpr int kMaxRowWarps = 16;

// Threads that share a row of K elements as a CTA of their own.  Many rows: as few as hold the row in registers,
// since few threads with four vectors each keep more rows in flight than many with one (4095 x 4160 bf16 10.0
// against 12.2 us).  Few rows: as many as there are vectors, for the shortest way through one row (rows
// of 4096 for 16 tokens to 8 experts each, in the chain that sorts and sums them: 6.3 against 7.1 us).
inline int row_threads(int64_t K, int64_t rows, int per) {
  const int elems = rows <= 4 * 148 ? 8 : (per == 8 ? 8 * kHeldVecs : (per == 2 ? 32 : 16));
  int64_t t = (K + elems - 1) / elems;
  t = (t + 31) / 32 * 32;
  return static_cast<int>(t < 64 ? 64 : (t > kMaxRowWarps * 32 ? kMaxRowWarps * 32 : t));
}

// Elements a load: 8 (rows on 16-byte boundaries), 2 (bf16 on 4-byte ones, an even number of them) or 1.
inline int row_per(const void* src, int64_t ld_src, const void* codes, int64_t ld_bytes, int64_t K, bool bf16) {
  const uintptr_t s = reinterpret_cast<uintptr_t>(src), c = reinterpret_cast<uintptr_t>(codes);
  const int64_t pitch = ld_src * (bf16 ? 2 : 4);
  if (s % 16 == 0 && pitch % 16 == 0 && c % 8 == 0 && ld_bytes % 8 == 0) return 8;
  return bf16 && s % 4 == 0 && pitch % 4 == 0 && c % 2 == 0 && ld_bytes % 2 == 0 && K % 2 == 0 ? 2 : 1;
}

// The largest magnitude over the threads of a row: a warp (kWarp, no CTA barrier), or the whole CTA, `red`
// then holding a word per warp.
template <bool kWarp>
__device__ __forceinline__ RowScale join_max(uint32_t m, int tid, int threads, uint32_t* red) {
  m = __reduce_max_sync(0xffffffffu, m);
  __syncwarp();   // what the caller put into shared memory is there for store8 / store1
  if (!kWarp) {
    if ((tid & 31) == 0) red[tid >> 5] = m;
    __syncthreads();
    m = (tid & 31) < (threads >> 5) ? red[tid & 31] : 0u;
    m = __reduce_max_sync(0xffffffffu, m);
  }
  return row_scale(__uint_as_float(m), m < 0x7F800000u);
}

// One row by `threads` threads.  `store8(k, codes)`, `store2(k, codes)` and `store1(k, code)` receive the codes,
// after a barrier of the row's threads; returns the row's scale.  Rows too long for the registers are read
// again (from L2).  kPer = 2 and 1: rows on no 16-byte boundaries, a pair or an element a load and consecutive
// lanes on consecutive ones, with as many loads in flight as the registers hold.  Bound by instructions: 4095
// rows of 4161 bf16 23 us, of 4162 15.6, of 4160 9.9.
// kMany: the stores are long, so what no thread needs of them is jumped over (a branch between short stores
// would cost a third of the time).
template <bool kBf16, bool kWarp, int kPer, bool kMany, class Store8, class Store2, class Store1>
__device__ __forceinline__ float quantize_row(const void* row, int K, int tid, int threads, uint32_t* red, Store8 store8,
                                              Store2 store2, Store1 store1) {
  RowScale rs;
  if constexpr (kPer == 8) {
    const int nvec = K / 8;
    Vec<kBf16> held[kHeldVecs];
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kHeldVecs; ++i) {
      const int v = tid + i * threads;
      if (v < nvec) held[i] = load_vec<kBf16>(row, static_cast<int64_t>(v) * 8);
    }
#pragma unroll
    for (int i = 0; i < kHeldVecs; ++i)
      if (tid + i * threads < nvec) m = abs_max_bits<kBf16>(held[i], m);
    for (int v = tid + kHeldVecs * threads; v < nvec; v += threads)
      m = abs_max_bits<kBf16>(load_vec<kBf16>(row, static_cast<int64_t>(v) * 8), m);
    for (int k = nvec * 8 + tid; k < K; k += threads)
      m = max(m, __float_as_uint(load_one<kBf16>(row, k)) & 0x7FFFFFFFu);
    rs = join_max<kWarp>(m, tid, threads, red);
#pragma unroll
    for (int i = 0; i < kHeldVecs; ++i) {
      const int v = tid + i * threads;
      if (v < nvec) store8(v * 8, rs.bad ? make_uint2(0, 0) : encode<kBf16>(held[i], rs.inv));
    }
    for (int v = tid + kHeldVecs * threads; v < nvec; v += threads)
      store8(v * 8, rs.bad ? make_uint2(0, 0) : encode<kBf16>(load_vec<kBf16>(row, static_cast<int64_t>(v) * 8), rs.inv));
    for (int k = nvec * 8 + tid; k < K; k += threads)
      store1(k, rs.bad ? 0 : static_cast<int8_t>(code_bits(load_one<kBf16>(row, k), rs.inv) & 0xFFu));
  } else {
    static_assert(kPer == 1 || kBf16, "pairs of bf16");
    constexpr int kHeld = kWarp && !kMany && kPer == 1 ? 2 * kHeldWords : kHeldWords;
    const int words = K / kPer;
    uint32_t held[kHeld];   // a pair, or the bits of a float
    auto load = [&](int w0) {
#pragma unroll
      for (int i = 0; i < kHeld; ++i) {
        const int w = w0 + i * threads;
        if (kPer == 2) held[i] = w < words ? static_cast<const uint32_t*>(row)[w] : 0u;
        else held[i] = w < words ? __float_as_uint(load_one<kBf16>(row, w)) : 0u;
      }
    };
    const int batch = kHeld * threads;
    uint32_t m = 0;
    for (int w0 = tid; w0 < words; w0 += batch) {
      load(w0);
#pragma unroll
      for (int i = 0; i < kHeld; ++i)
        m = kPer == 2 ? __vmaxu2(m, held[i] & 0x7FFF7FFFu) : max(m, held[i] & 0x7FFFFFFFu);
    }
    if (kPer == 2) m = max(m << 16, m & 0xFFFF0000u);
    rs = join_max<kWarp>(m, tid, threads, red);
    for (int w0 = tid; w0 < words; w0 += batch) {
      if (words > batch) load(w0);
#pragma unroll
      for (int i0 = 0; i0 < kHeld; i0 += 4) {
        if (kMany && w0 - tid + i0 * threads >= words) break;
#pragma unroll
        for (int i = i0; i < i0 + 4; ++i) {
          const int w = w0 + i * threads;
          if (w >= words) continue;
          if (kPer == 2) {
            const uint32_t lo = code_bits(__uint_as_float(held[i] << 16), rs.inv) & 0xFFu;
            const uint32_t hi = code_bits(__uint_as_float(held[i] & 0xFFFF0000u), rs.inv) & 0xFFu;
            store2(2 * w, rs.bad ? uint16_t(0) : static_cast<uint16_t>(lo | hi << 8));
          } else {
            store1(w, rs.bad ? 0 : static_cast<int8_t>(code_bits(__uint_as_float(held[i]), rs.inv) & 0xFFu));
          }
        }
      }
    }
  }
  return rs.bad ? __uint_as_float(0x7FC00000u) : rs.scale;
}

}  // namespace qi8
}  // namespace smb
