// Rows to experts and back: the layout the grouped GEMMs read, and the weighted sum of what they write.
//
//   dispatch   ids [tokens, top_k] -> a stable counting sort of the slots by expert: row offsets of the
//              experts, slot -> row and row -> slot maps
//   gather     row_of_slot[t, j] = r: row r of the sorted buffer becomes row t of x (bf16, or int8 codes
//              with the row's scale)
//   combine    y[t] = sum_j weights[t, j] * rows[row_of_slot[t, j]], and its gradients
//
// A slot that goes nowhere (id outside [0, experts)) has row -1 and is skipped everywhere; rows that no
// slot names are never written.  The order of every sum and of the rows is fixed (the only atomics are
// integer counts in shared memory).
//
// The copies and sums are bound by HBM: 8192 tokens x 8 rows of 2048 bf16, gather 48 us (6.2 TB/s written and
// read), quantised 28.6 us (5.9), combine 49 us (6.0), its gradients 92 us (6.1); a call for 16 tokens costs a
// launch, about 2 us.
#include "i8_common.cuh"
#include "ptx.cuh"
#include "quant_i8.cuh"

namespace smb {
namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kMaxDispatchGroups = 1024;
constexpr int kMaxTopKRows = 32;

cudaLaunchConfig_t pdl_config(dim3 grid, dim3 block, size_t smem, cudaStream_t st, cudaLaunchAttribute* attr) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  attr->id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr->val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cfg;
}

// --------------------------------------------------------------------------- dispatch
struct DispatchParams {
  const int* ids;
  int n;               // slots
  int groups, align;
  int cap;             // rows of the sorted buffer
  int per_warp;        // slots per warp, a multiple of 32
  int sorters;         // warps of a CTA that own slots; the rest only help with groups and rows
  int* offsets;
  int* row_of_slot;
  int* slot_of_row;
  int* mtile_group;
};

// One cluster sorts everything: warp w of the cluster owns the slots [w * per_warp, + per_warp), so
// "earlier slots" means earlier lanes, earlier chunks, earlier warps, earlier CTAs, and the counts of the
// CTAs meet through distributed shared memory instead of a second launch.
//   shared: hist[sorters][groups] | total[groups] | start[groups] | count[groups] | warp_sums[32], all of it asked
//   for by the launch, since what a kernel declares itself counts towards the 48 KB that need no asking too
// Bound by latency: the ids of a warp are fetched together (8 x 32 at a time) and stay in registers
// between the count and the placement where they fit.  128 slots of 256 groups 2.3 us, 4096 of 64 4.3 us; 65536
// slots 9.8 us on the eight SMs of a cluster, where the copies that follow take 190.
constexpr int kHeldIds = 8;

__device__ __forceinline__ int clean_id(int e, int groups) { return e >= 0 && e < groups ? e : -1; }

// Lanes with this lane's id, from a ballot per bit of it (`bits` cover every id and the -1 of dropped slots).
// match.any takes longer, and longer still the more ids differ: 65536 slots of 64 groups 24 us with it.
__device__ __forceinline__ unsigned same_id(int e, int bits) {
  unsigned same = kFull;
  for (int b = 0; b < bits; ++b) {
    const bool bit = (e >> b) & 1;
    const unsigned set = __ballot_sync(kFull, bit);
    same &= bit ? set : ~set;
  }
  return same;
}

template <bool kCluster>
__global__ void __launch_bounds__(1024) dispatch_kernel(const DispatchParams p) {
  extern __shared__ int sm[];
  griddep_launch_dependents();
  const int all_warps = blockDim.x >> 5, warps = p.sorters;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int ctas = kCluster ? static_cast<int>(cluster_nctarank()) : 1;
  const int rank = kCluster ? static_cast<int>(cluster_ctarank()) : 0;
  const int G = p.groups;
  int* hist = sm;
  int* total = hist + warps * G;
  int* start = total + G;
  int* count = start + G;
  int* warp_sums = count + G;

  const long long first = warp < warps ? static_cast<long long>(rank * warps + warp) * p.per_warp : p.n;
  const int lo = static_cast<int>(first < p.n ? first : p.n);
  const int hi = static_cast<int>(first + p.per_warp < p.n ? first + p.per_warp : p.n);
  int* mine = hist + warp * G;   // of sorters
  if (warp < warps)
    for (int e = lane; e < G; e += 32) mine[e] = 0;
  griddep_wait();
  int held[kHeldIds];
#pragma unroll
  for (int i = 0; i < kHeldIds; ++i) {
    const int s = lo + i * 32 + lane;
    held[i] = s < hi ? p.ids[s] : -1;
  }
  __syncwarp();
  const bool fits = hi - lo <= kHeldIds * 32;
  for (int s0 = lo; s0 < hi; s0 += kHeldIds * 32) {
    if (s0 != lo) {
#pragma unroll
      for (int i = 0; i < kHeldIds; ++i) {
        const int s = s0 + i * 32 + lane;
        held[i] = s < hi ? p.ids[s] : -1;
      }
    }
#pragma unroll
    for (int i = 0; i < kHeldIds; ++i) {
      if (s0 + i * 32 >= hi) break;
      const int e = clean_id(held[i], G);
      if (e >= 0) atomicAdd(mine + e, 1);   // the warp's own words; a count does not depend on the order
    }
  }
  __syncthreads();
  // Exclusive prefix of every group over the warps of this CTA.
  for (int e = threadIdx.x; e < G; e += blockDim.x) {
    int before = 0;
    for (int w0 = 0; w0 < warps; w0 += 8) {
      int c[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = w0 + i < warps ? hist[(w0 + i) * G + e] : 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (w0 + i < warps) hist[(w0 + i) * G + e] = before;
        before += c[i];
      }
    }
    total[e] = before;
  }
  if (kCluster) cluster_sync_all();   // also a CTA barrier
  else __syncthreads();
  // Threads take runs of groups; counts over all CTAs, then an exclusive scan of the padded sizes.
  const int per = (G + blockDim.x - 1) / blockDim.x;   // 1 unless there are more groups than threads
  const int e_lo = min(static_cast<int>(threadIdx.x) * per, G), e_hi = min(e_lo + per, G);
  auto padded = [&](int c) { return p.align == 1 ? c : (c + p.align - 1) / p.align * p.align; };
  int sum = 0;
  for (int e = e_lo; e < e_hi; ++e) {
    int before = 0, all = 0;
    if (kCluster) {
      const uint32_t addr = smem_u32(total + e);
      int v[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) v[c] = c < ctas ? static_cast<int>(ld_shared_cluster_u32(mapa_u32(addr, c))) : 0;
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        if (c < rank) before += v[c];
        all += v[c];
      }
    } else {
      all = total[e];
    }
    start[e] = before;
    count[e] = all;
    sum += padded(all);
  }
  int inclusive = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int up = __shfl_up_sync(kFull, inclusive, d);
    if (lane >= d) inclusive += up;
  }
  if (lane == 31) warp_sums[warp] = inclusive;
  if (kCluster) cluster_sync_all();   // nobody's totals are read by another CTA after this
  else __syncthreads();
  const int others = lane < all_warps ? warp_sums[lane] : 0;
  int base = __reduce_add_sync(kFull, lane < warp ? others : 0) + inclusive - sum;
  const int used = __reduce_add_sync(kFull, others);
  const int id_bits = 32 - __clz(G);   // G < 2^bits, so the low bits of -1 are no id either
  for (int e = e_lo; e < e_hi; ++e) {
    total[e] = base;                  // first row of the group, from here on
    start[e] += base;
    if (rank == 0) p.offsets[e] = base;
    base += padded(count[e]);
  }
  if (rank == 0 && threadIdx.x == 0) p.offsets[G] = used;
  __syncthreads();
  for (int s0 = lo; s0 < hi; s0 += kHeldIds * 32) {
    if (!fits) {
#pragma unroll
      for (int i = 0; i < kHeldIds; ++i) {
        const int s = s0 + i * 32 + lane;
        held[i] = s < hi ? p.ids[s] : -1;
      }
    }
#pragma unroll
    for (int i = 0; i < kHeldIds; ++i) {
      const int s = s0 + i * 32 + lane;
      if (s0 + i * 32 >= hi) break;
      const int e = clean_id(held[i], G);
      const unsigned same = same_id(e, id_bits);
      const int row = e >= 0 ? start[e] + mine[e] + __popc(same & ((1u << lane) - 1u)) : -1;
      __syncwarp();
      if (e >= 0 && lane == __ffs(same) - 1) mine[e] += __popc(same);
      __syncwarp();
      if (s < hi) p.row_of_slot[s] = row;
      if (row >= 0) p.slot_of_row[row] = s;
    }
  }
  // Rows that no slot names: the padding of every group, and everything behind the last one.  Unsigned, since
  // a step past the last row may leave 31 bits.
  const unsigned threads = ctas * blockDim.x;
  const unsigned me = rank * blockDim.x + threadIdx.x;
  if (p.align > 1) {
    for (int e = me >> 5; e < G; e += threads >> 5) {
      const unsigned end = e + 1 < G ? total[e + 1] : used;
      for (unsigned r = total[e] + count[e] + lane; r < end; r += 32) p.slot_of_row[r] = -1;
    }
  }
  for (unsigned r = used + me; r < static_cast<unsigned>(p.cap); r += threads) p.slot_of_row[r] = -1;
  if (p.mtile_group != nullptr) {
    for (int e = me >> 5; e < G; e += threads >> 5) {
      const int end = e + 1 < G ? total[e + 1] : used;
      for (int t = total[e] / 256 + lane; t < end / 256; t += 32) p.mtile_group[t] = e;
    }
    for (int t = used / 256 + static_cast<int>(me); t < p.cap / 256; t += threads) p.mtile_group[t] = G - 1;
  }
}

// --------------------------------------------------------------------------- gather
constexpr int kCta = 256;

// Rows are read and written in words of 16, 4 or 2 bytes, the widest that bases, pitches and width allow,
// consecutive lanes on consecutive words; a thread has kWords of them in flight.
template <class W>
struct Words {
  static constexpr int kElems = sizeof(W) / 2;
  static constexpr int kWords = sizeof(W) == 16 ? 1 : 4;
};

template <class W>
__global__ void __launch_bounds__(kCta) gather_bf16_kernel(const uint16_t* x, int64_t ld_x, const int* row_of_slot, int top_k,
                                                           int width, int max_rows, uint16_t* out, int64_t ld_out) {
  constexpr int kE = Words<W>::kElems, kN = Words<W>::kWords;
  griddep_launch_dependents();
  griddep_wait();
  const int64_t t = blockIdx.x;
  const int* rows = row_of_slot + t * top_k;
  const W* src = reinterpret_cast<const W*>(x + t * ld_x);
  const int words = width / kE;
  const int c0 = blockIdx.y * kN * blockDim.x + threadIdx.x;
  W v[kN];
#pragma unroll
  for (int i = 0; i < kN; ++i)
    if (c0 + i * blockDim.x < words) v[i] = src[c0 + i * blockDim.x];
  for (int j = 0; j < top_k; ++j) {
    const int r = rows[j];
    if (r < 0 || r >= max_rows) continue;
    W* dst = reinterpret_cast<W*>(out + static_cast<int64_t>(r) * ld_out);
#pragma unroll
    for (int i = 0; i < kN; ++i)
      if (c0 + i * blockDim.x < words) dst[c0 + i * blockDim.x] = v[i];
  }
}

template <bool kWarp, int kPer>
__global__ void __launch_bounds__(kWarp ? kCta : 32 * qi8::kMaxRowWarps)
gather_i8_kernel(const uint16_t* x, int64_t ld_x, const int* row_of_slot, int64_t tokens, int top_k, int width, int max_rows,
                 int8_t* codes, int64_t ld_bytes, float* scales) {
  __shared__ uint32_t red[qi8::kMaxRowWarps];
  __shared__ int rows_all[kWarp ? kCta / 32 : 1][kMaxTopKRows];
  griddep_launch_dependents();
  griddep_wait();
  const int threads = kWarp ? 32 : blockDim.x;
  const int tid = kWarp ? threadIdx.x & 31 : threadIdx.x;
  const int64_t t = kWarp ? static_cast<int64_t>(blockIdx.x) * (kCta / 32) + (threadIdx.x >> 5) : blockIdx.x;
  if (t >= tokens) return;   // whole warps
  // The destinations are fetched along with the row; quantize_row has a barrier between its loads and
  // its stores.
  int* rows = rows_all[kWarp ? threadIdx.x >> 5 : 0];
  if (tid < top_k) rows[tid] = row_of_slot[t * top_k + tid];
  const float scale = qi8::quantize_row<true, kWarp, kPer, true>(
      x + t * ld_x, width, tid, threads, red,
      [&](int k, uint2 c) {
        for (int j = 0; j < top_k; ++j) {
          const int r = rows[j];
          if (r >= 0 && r < max_rows) *reinterpret_cast<uint2*>(codes + static_cast<int64_t>(r) * ld_bytes + k) = c;
        }
      },
      [&](int k, uint16_t c) {
        for (int j = 0; j < top_k; ++j) {
          const int r = rows[j];
          if (r >= 0 && r < max_rows) *reinterpret_cast<uint16_t*>(codes + static_cast<int64_t>(r) * ld_bytes + k) = c;
        }
      },
      [&](int k, int8_t c) {
        for (int j = 0; j < top_k; ++j) {
          const int r = rows[j];
          if (r >= 0 && r < max_rows) codes[static_cast<int64_t>(r) * ld_bytes + k] = c;
        }
      });
  if (tid < top_k) {
    const int r = rows[tid];
    if (r >= 0 && r < max_rows) scales[r] = scale;
  }
}

// --------------------------------------------------------------------------- combine
__device__ __forceinline__ float bf16_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf16_hi(uint32_t w) { return __uint_as_float(w & 0xFFFF0000u); }

// A word of bf16 as 32-bit pairs (a single element as the low half of one).
__device__ __forceinline__ uint32_t pair_of(const uint4& q, int i) { return i == 0 ? q.x : (i == 1 ? q.y : (i == 2 ? q.z : q.w)); }
__device__ __forceinline__ uint32_t pair_of(uint32_t q, int) { return q; }
__device__ __forceinline__ uint32_t pair_of(uint16_t q, int) { return q; }
__device__ __forceinline__ void set_word(uint4& q, const uint32_t* p) { q = make_uint4(p[0], p[1], p[2], p[3]); }
__device__ __forceinline__ void set_word(uint32_t& q, const uint32_t* p) { q = p[0]; }
__device__ __forceinline__ void set_word(uint16_t& q, const uint32_t* p) { q = static_cast<uint16_t>(p[0] & 0xFFFFu); }

// fp32 sum in slot order, one rounding to bf16.
template <class W>
__global__ void __launch_bounds__(kCta) combine_kernel(const uint16_t* rows_in, int64_t ld_rows, const int* row_of_slot,
                                                       const float* weights, int top_k, int width, int max_rows, uint16_t* y,
                                                       int64_t ld_y) {
  constexpr int kE = Words<W>::kElems, kN = Words<W>::kWords, kPairs = (kE + 1) / 2;
  griddep_launch_dependents();
  griddep_wait();
  const int64_t t = blockIdx.x;
  const int* rows = row_of_slot + t * top_k;
  const int words = width / kE;
  const int c0 = blockIdx.y * kN * blockDim.x + threadIdx.x;
  if (c0 >= words) return;
  float acc[kN][2 * kPairs] = {};
  const float* w_row = weights != nullptr ? weights + t * top_k : nullptr;
  // Eight slots at a time: their rows, then all their loads, are in flight together.
  for (int j0 = 0; j0 < top_k; j0 += 8) {
    int r[8];
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      r[i] = j0 + i < top_k ? rows[j0 + i] : -1;
      w[i] = w_row != nullptr && j0 + i < top_k ? w_row[j0 + i] : 1.0f;
      if (r[i] >= max_rows) r[i] = -1;
    }
    W q[8][kN];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const W* src = reinterpret_cast<const W*>(rows_in + static_cast<int64_t>(r[i]) * ld_rows);
#pragma unroll
      for (int n = 0; n < kN; ++n)
        if (r[i] >= 0 && c0 + n * blockDim.x < words) q[i][n] = src[c0 + n * blockDim.x];
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if (r[i] < 0) continue;
#pragma unroll
      for (int n = 0; n < kN; ++n)
#pragma unroll
        for (int k = 0; k < kPairs; ++k) {
          acc[n][2 * k] = fmaf(w[i], bf16_lo(pair_of(q[i][n], k)), acc[n][2 * k]);
          if (kE > 1) acc[n][2 * k + 1] = fmaf(w[i], bf16_hi(pair_of(q[i][n], k)), acc[n][2 * k + 1]);
        }
    }
  }
  W* dst = reinterpret_cast<W*>(y + t * ld_y);
#pragma unroll
  for (int n = 0; n < kN; ++n) {
    uint32_t o[kPairs];
#pragma unroll
    for (int k = 0; k < kPairs; ++k) o[k] = pack_bf16x2(__float_as_uint(acc[n][2 * k]), __float_as_uint(acc[n][2 * k + 1]));
    if (c0 + n * blockDim.x < words) set_word(dst[c0 + n * blockDim.x], o);
  }
}

// A warp per slot: its row's gradient w * dy and its weight's gradient <dy, row>.  The warps of a token
// are neighbours, so dy comes from L1 after the first of them.
template <class W>
__global__ void __launch_bounds__(kCta) combine_grad_kernel(const uint16_t* grad_y, int64_t ld_gy, const uint16_t* rows_in,
                                                            int64_t ld_rows, const int* row_of_slot, const float* weights,
                                                            int64_t slots, int top_k, int width, int max_rows,
                                                            uint16_t* grad_rows, int64_t ld_gr, float* grad_weights) {
  constexpr int kE = Words<W>::kElems, kN = kE == 1 ? 8 : Words<W>::kWords, kPairs = (kE + 1) / 2;
  griddep_launch_dependents();
  griddep_wait();
  const int lane = threadIdx.x & 31;
  const int64_t s = static_cast<int64_t>(blockIdx.x) * (kCta / 32) + (threadIdx.x >> 5);
  if (s >= slots) return;
  const int r = row_of_slot[s];
  if (r < 0 || r >= max_rows) {
    if (lane == 0 && grad_weights != nullptr) grad_weights[s] = 0.0f;
    return;
  }
  const float w = weights != nullptr ? weights[s] : 1.0f;
  const W* gy = reinterpret_cast<const W*>(grad_y + s / top_k * ld_gy);
  const W* in = grad_weights != nullptr ? reinterpret_cast<const W*>(rows_in + static_cast<int64_t>(r) * ld_rows) : nullptr;
  W* out = reinterpret_cast<W*>(grad_rows + static_cast<int64_t>(r) * ld_gr);
  float dot = 0.0f;
  const int words = width / kE;
  for (int c = lane; c < words; c += 32 * kN) {
    W g[kN], v[kN];
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      if (c + 32 * n >= words) continue;
      g[n] = gy[c + 32 * n];
      if (in != nullptr) v[n] = in[c + 32 * n];
    }
#pragma unroll
    for (int n = 0; n < kN; ++n) {
      if (c + 32 * n >= words) continue;
      uint32_t o[kPairs];
#pragma unroll
      for (int k = 0; k < kPairs; ++k) {
        const float lo = bf16_lo(pair_of(g[n], k)), hi = bf16_hi(pair_of(g[n], k));   // hi of a single element: 0
        if (in != nullptr) {
          dot = fmaf(lo, bf16_lo(pair_of(v[n], k)), dot);
          if (kE > 1) dot = fmaf(hi, bf16_hi(pair_of(v[n], k)), dot);
        }
        o[k] = pack_bf16x2(__float_as_uint(w * lo), __float_as_uint(w * hi));
      }
      set_word(out[c + 32 * n], o);
    }
  }
  if (grad_weights != nullptr) {
#pragma unroll
    for (int d = 16; d > 0; d >>= 1) dot += __shfl_xor_sync(kFull, dot, d);
    if (lane == 0) grad_weights[s] = dot;
  }
}

// Whether rows of 2-byte elements consist of words of n bytes.
bool rows_take(int n, const void* p, int64_t ld, int width) {
  return reinterpret_cast<uintptr_t>(p) % n == 0 && ld * 2 % n == 0 && static_cast<int64_t>(width) * 2 % n == 0;
}
bool aligned_to(const void* p, int n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

int finish(cudaError_t e, const char* what) {
  if (e == cudaSuccess) e = cudaGetLastError();
  return e == cudaSuccess ? SMB_OK : set_cuda_error(e, what);
}

// What the row copies and sums share.
int check_rows(const char* what, const void* row_of_slot, int64_t tokens, int top_k, int width, int64_t max_rows) {
  if (tokens != 0 && row_of_slot == nullptr) return set_error(SMB_ERR_INVALID, "%s: null row map", what);
  if (!aligned_to(row_of_slot, 4)) return set_error(SMB_ERR_INVALID, "%s: row map is not 4-byte aligned", what);
  if (tokens < 0 || tokens > 0x7FFFFFFFLL) return set_error(SMB_ERR_INVALID, "%s: bad token count", what);
  if (top_k < 1 || top_k > kMaxTopKRows)
    return set_error(SMB_ERR_INVALID, "%s: top_k=%d outside 1..%d", what, top_k, kMaxTopKRows);
  if (width < 1 || width > 65535 * 8 * 32) return set_error(SMB_ERR_INVALID, "%s: width %d out of range", what, width);
  if (max_rows < (tokens != 0 ? 1 : 0) || max_rows > 0x7FFFFFFFLL)
    return set_error(SMB_ERR_INVALID, "%s: bad row capacity", what);
  return SMB_OK;
}

// Threads for a row in words: whole warps, at most 128; the rest goes to the grid's y.
template <class W>
void row_grid(int64_t tokens, int width, dim3* grid, dim3* block) {
  const int words = width / Words<W>::kElems;
  int threads = (words + Words<W>::kWords * 32 - 1) / (Words<W>::kWords * 32) * 32;
  if (threads > 128) threads = 128;
  const int per_cta = threads * Words<W>::kWords;
  *block = dim3(static_cast<unsigned>(threads), 1, 1);
  *grid = dim3(static_cast<unsigned>(tokens), static_cast<unsigned>((words + per_cta - 1) / per_cta), 1);
}

template <class W>
int launch_gather(const uint16_t* x, int64_t ld_x, const int32_t* row_of_slot, int64_t tokens, int top_k, int width, int max_rows,
                  uint16_t* out, int64_t ld_out, void* stream) {
  dim3 grid, block;
  row_grid<W>(tokens, width, &grid, &block);
  cudaLaunchAttribute attr;
  cudaLaunchConfig_t cfg = pdl_config(grid, block, 0, static_cast<cudaStream_t>(stream), &attr);
  return finish(cudaLaunchKernelEx(&cfg, gather_bf16_kernel<W>, x, ld_x, row_of_slot, top_k, width, max_rows, out, ld_out),
                "gather launch");
}

template <class W>
int launch_combine(const uint16_t* rows, int64_t ld_rows, const int32_t* row_of_slot, const float* weights, int64_t tokens,
                   int top_k, int width, int max_rows, uint16_t* y, int64_t ld_y, void* stream) {
  dim3 grid, block;
  row_grid<W>(tokens, width, &grid, &block);
  cudaLaunchAttribute attr;
  cudaLaunchConfig_t cfg = pdl_config(grid, block, 0, static_cast<cudaStream_t>(stream), &attr);
  return finish(cudaLaunchKernelEx(&cfg, combine_kernel<W>, rows, ld_rows, row_of_slot, weights, top_k, width, max_rows, y, ld_y),
                "combine launch");
}

template <class W>
int launch_combine_grad(const uint16_t* grad_y, int64_t ld_gy, const uint16_t* rows, int64_t ld_rows, const int32_t* row_of_slot,
                        const float* weights, int64_t slots, int top_k, int width, int max_rows, uint16_t* grad_rows,
                        int64_t ld_gr, float* grad_weights, void* stream) {
  cudaLaunchAttribute attr;
  cudaLaunchConfig_t cfg = pdl_config(dim3(static_cast<unsigned>((slots + kCta / 32 - 1) / (kCta / 32)), 1, 1), dim3(kCta, 1, 1),
                                      0, static_cast<cudaStream_t>(stream), &attr);
  return finish(cudaLaunchKernelEx(&cfg, combine_grad_kernel<W>, grad_y, ld_gy, rows, ld_rows, row_of_slot, weights, slots, top_k,
                                   width, max_rows, grad_rows, ld_gr, grad_weights),
                "combine backward launch");
}

}  // namespace
}  // namespace smb

using namespace smb;

extern "C" int64_t smb_moe_max_rows(int64_t tokens, int top_k, int groups, int align) {
  if (tokens < 0 || top_k < 1 || groups < 1 || align < 1) return 0;
  const int64_t n = tokens * top_k;
  const int64_t hit = groups < n ? groups : n;
  return (n + hit * (align - 1)) / align * align;
}

extern "C" int smb_moe_dispatch_device(const int32_t* ids, int64_t tokens, int top_k, int groups, int align, int64_t max_rows,
                                       int32_t* offsets, int32_t* row_of_slot, int32_t* slot_of_row, int32_t* mtile_group,
                                       void* stream) {
  // An empty batch has no ids and no row map, and with align 1 no rows either.
  if (offsets == nullptr || (tokens != 0 && (ids == nullptr || row_of_slot == nullptr)) ||
      (max_rows != 0 && slot_of_row == nullptr))
    return set_error(SMB_ERR_INVALID, "dispatch: null pointer");
  if (!aligned_to(ids, 4) || !aligned_to(offsets, 4) || !aligned_to(row_of_slot, 4) || !aligned_to(slot_of_row, 4) ||
      !aligned_to(mtile_group, 4))
    return set_error(SMB_ERR_INVALID, "dispatch: pointers must be 4-byte aligned");
  if (groups < 1 || groups > kMaxDispatchGroups)
    return set_error(SMB_ERR_UNSUPPORTED, "dispatch: %d groups outside 1..%d", groups, kMaxDispatchGroups);
  if (tokens < 0 || top_k < 1 || top_k > kMaxTopKRows)
    return set_error(SMB_ERR_INVALID, "dispatch: bad extents (tokens=%lld top_k=%d)", static_cast<long long>(tokens), top_k);
  if (align < 1 || align > 65536) return set_error(SMB_ERR_INVALID, "dispatch: alignment %d outside 1..65536", align);
  if (mtile_group != nullptr && align % 256 != 0)
    return set_error(SMB_ERR_INVALID, "dispatch: the tile map needs groups aligned to 256 rows, not %d", align);
  if (tokens > (1LL << 30) / top_k) return set_error(SMB_ERR_UNSUPPORTED, "dispatch: more than 2^30 slots");
  const int64_t need = smb_moe_max_rows(tokens, top_k, groups, align);
  if (max_rows < need || max_rows > 0x7FFFFFFFLL)
    return set_error(SMB_ERR_INVALID, "dispatch: room for %lld rows, up to %lld may be needed",
                     static_cast<long long>(max_rows), static_cast<long long>(need));
  DispatchParams p = {};
  p.ids = ids;
  p.n = static_cast<int>(tokens * top_k);
  p.groups = groups;
  p.align = align;
  p.cap = static_cast<int>(max_rows);
  p.offsets = offsets;
  p.row_of_slot = row_of_slot;
  p.slot_of_row = slot_of_row;
  p.mtile_group = mtile_group;
  // Warps: as many as have 32 slots each, up to 32 in a CTA and 8 CTAs; the histograms bound them too.
  int warps = (p.n + 31) / 32;
  if (warps < 4) warps = 4;
  int ctas = 1;
  while (ctas < 8 && warps > 32 * ctas) ctas *= 2;
  warps = (warps + ctas - 1) / ctas;
  if (warps > 32) warps = 32;
  p.sorters = warps;
  p.per_warp = static_cast<int>((p.n + static_cast<int64_t>(ctas) * warps * 32 - 1) / (static_cast<int64_t>(ctas) * warps * 32)) * 32;
  auto shared = [](int sorters, int groups) { return (static_cast<size_t>(sorters + 3) * groups + 32) * sizeof(int); };
  const size_t smem = shared(warps, groups);
  // More warps where there are many groups or rows to walk at the end: 60 slots of 388 groups of 256 rows
  // 22 us with the four that sort, 7 with 32.
  const int64_t walk = align > 1 ? groups / 8 : 0;
  const int64_t help = walk > max_rows / 512 ? walk : max_rows / 512;
  const int all_warps = help <= warps ? warps : (help < 32 ? static_cast<int>(help) : 32);
  auto kernel = ctas > 1 ? dispatch_kernel<true> : dispatch_kernel<false>;
  if (smem > 48 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         static_cast<int>(shared(32, kMaxDispatchGroups)));
    if (e != cudaSuccess) return set_cuda_error(e, "dispatch shared memory");
  }
  cudaLaunchAttribute attr[2];
  cudaLaunchConfig_t cfg = pdl_config(dim3(ctas, 1, 1), dim3(all_warps * 32, 1, 1), smem, static_cast<cudaStream_t>(stream), attr);
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(ctas);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.numAttrs = ctas > 1 ? 2 : 1;
  return finish(cudaLaunchKernelEx(&cfg, kernel, p), "dispatch launch");
}

extern "C" int smb_moe_gather_bf16_device(const uint16_t* x, int64_t ld_x, const int32_t* row_of_slot, int64_t tokens,
                                          int top_k, int width, int64_t max_rows, uint16_t* out, int64_t ld_out,
                                          void* stream) {
  if (tokens != 0 && (x == nullptr || out == nullptr)) return set_error(SMB_ERR_INVALID, "gather: null pointer");
  if (int rc = check_rows("gather", row_of_slot, tokens, top_k, width, max_rows)) return rc;
  if (ld_x < width || ld_out < width) return set_error(SMB_ERR_INVALID, "gather: pitch smaller than the row");
  if (!aligned_to(x, 2) || !aligned_to(out, 2)) return set_error(SMB_ERR_INVALID, "gather: rows are not 2-byte aligned");
  if (tokens == 0) return SMB_OK;
  auto take = [&](int n) { return rows_take(n, x, ld_x, width) && rows_take(n, out, ld_out, width); };
  auto launch = take(16) ? launch_gather<uint4> : (take(4) ? launch_gather<uint32_t> : launch_gather<uint16_t>);
  return launch(x, ld_x, row_of_slot, tokens, top_k, width, static_cast<int>(max_rows), out, ld_out, stream);
}

extern "C" int smb_moe_gather_i8_device(const uint16_t* x, int64_t ld_x, const int32_t* row_of_slot, int64_t tokens, int top_k,
                                        int width, int64_t max_rows, int8_t* codes, int64_t ld_bytes, float* scales,
                                        void* stream) {
  if (tokens != 0 && (x == nullptr || codes == nullptr || scales == nullptr))
    return set_error(SMB_ERR_INVALID, "i8 gather: null pointer");
  if (int rc = check_rows("i8 gather", row_of_slot, tokens, top_k, width, max_rows)) return rc;
  if (ld_x < width || ld_bytes < width) return set_error(SMB_ERR_INVALID, "i8 gather: pitch smaller than the row");
  if (!aligned_to(x, 2) || !aligned_to(scales, 4))
    return set_error(SMB_ERR_INVALID, "i8 gather: rows must be 2-byte, scales 4-byte aligned");
  if (tokens == 0) return SMB_OK;
  const int per = qi8::row_per(x, ld_x, codes, ld_bytes, width, true);
  const bool warp = width <= 1024;   // a warp holds such a row in registers
  const int64_t per_cta = warp ? kCta / 32 : 1;
  cudaLaunchAttribute attr;
  cudaLaunchConfig_t cfg = pdl_config(dim3(static_cast<unsigned>((tokens + per_cta - 1) / per_cta), 1, 1),
                                      dim3(static_cast<unsigned>(warp ? kCta : qi8::row_threads(width, tokens, per)), 1, 1), 0,
                                      static_cast<cudaStream_t>(stream), &attr);
  auto kernel = warp ? (per == 8 ? gather_i8_kernel<true, 8> : (per == 2 ? gather_i8_kernel<true, 2> : gather_i8_kernel<true, 1>))
                     : (per == 8 ? gather_i8_kernel<false, 8> : (per == 2 ? gather_i8_kernel<false, 2> : gather_i8_kernel<false, 1>));
  return finish(cudaLaunchKernelEx(&cfg, kernel, x, ld_x, row_of_slot, tokens, top_k, width, static_cast<int>(max_rows), codes,
                                   ld_bytes, scales),
                "i8 gather launch");
}

extern "C" int smb_moe_combine_device(const uint16_t* rows, int64_t ld_rows, const int32_t* row_of_slot, const float* weights,
                                      int64_t tokens, int top_k, int width, int64_t max_rows, uint16_t* y, int64_t ld_y,
                                      void* stream) {
  if (tokens != 0 && (rows == nullptr || y == nullptr)) return set_error(SMB_ERR_INVALID, "combine: null pointer");
  if (int rc = check_rows("combine", row_of_slot, tokens, top_k, width, max_rows)) return rc;
  if (ld_rows < width || ld_y < width) return set_error(SMB_ERR_INVALID, "combine: pitch smaller than the row");
  if (!aligned_to(rows, 2) || !aligned_to(y, 2) || !aligned_to(weights, 4))
    return set_error(SMB_ERR_INVALID, "combine: rows must be 2-byte, weights 4-byte aligned");
  if (tokens == 0) return SMB_OK;
  auto take = [&](int n) { return rows_take(n, rows, ld_rows, width) && rows_take(n, y, ld_y, width); };
  auto launch = take(16) ? launch_combine<uint4> : (take(4) ? launch_combine<uint32_t> : launch_combine<uint16_t>);
  return launch(rows, ld_rows, row_of_slot, weights, tokens, top_k, width, static_cast<int>(max_rows), y, ld_y, stream);
}

extern "C" int smb_moe_combine_backward_device(const uint16_t* grad_y, int64_t ld_grad_y, const uint16_t* rows,
                                               int64_t ld_rows, const int32_t* row_of_slot, const float* weights,
                                               int64_t tokens, int top_k, int width, int64_t max_rows, uint16_t* grad_rows,
                                               int64_t ld_grad_rows, float* grad_weights, void* stream) {
  if (tokens != 0 && (grad_y == nullptr || grad_rows == nullptr))
    return set_error(SMB_ERR_INVALID, "combine backward: null pointer");
  if (tokens != 0 && grad_weights != nullptr && rows == nullptr)
    return set_error(SMB_ERR_INVALID, "combine backward: the weights' gradient needs the rows");
  if (int rc = check_rows("combine backward", row_of_slot, tokens, top_k, width, max_rows)) return rc;
  if (ld_grad_y < width || ld_grad_rows < width || (rows != nullptr && ld_rows < width))
    return set_error(SMB_ERR_INVALID, "combine backward: pitch smaller than the row");
  if (!aligned_to(grad_y, 2) || !aligned_to(rows, 2) || !aligned_to(grad_rows, 2) || !aligned_to(weights, 4) ||
      !aligned_to(grad_weights, 4))
    return set_error(SMB_ERR_INVALID, "combine backward: rows must be 2-byte, weights 4-byte aligned");
  if (tokens == 0) return SMB_OK;
  const int64_t slots = tokens * top_k;
  if ((slots + kCta / 32 - 1) / (kCta / 32) > 0x7FFFFFFFLL) return set_error(SMB_ERR_UNSUPPORTED, "combine backward: too many slots");
  auto take = [&](int n) {
    return rows_take(n, grad_y, ld_grad_y, width) && rows_take(n, grad_rows, ld_grad_rows, width) &&
           (grad_weights == nullptr || rows_take(n, rows, ld_rows, width));
  };
  auto launch = take(16) ? launch_combine_grad<uint4> : (take(4) ? launch_combine_grad<uint32_t> : launch_combine_grad<uint16_t>);
  return launch(grad_y, ld_grad_y, rows, ld_rows, row_of_slot, weights, slots, top_k, width, static_cast<int>(max_rows),
                grad_rows, ld_grad_rows, grad_weights, stream);
}
