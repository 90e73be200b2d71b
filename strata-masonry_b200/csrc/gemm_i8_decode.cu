// int8 GEMM for few rows per weight matrix (decode batches, experts with a handful of tokens): bound by
// reading B once.  Same result, bit for bit, as gemm_i8.cu.  Measured in a CUDA graph: 16 x 28672 x 8192 with its
// quantiser 38 us (6.1 TB/s), 128 experts x 256 rows (1536 x 2048 each, gated) 63 us (6.4 TB/s), DRAM reads the
// operands once (ncu: 235.2 and 404.0 MB).
//
// The operands swap roles: 128 rows of B (output channels) fill the rows of a 1-CTA tcgen05.mma and up
// to 128 rows of A (tokens) its columns, so the instruction does no more work than the tokens need and a
// stage is mostly weights.  Accumulator lane = channel, column = token.
//
// Two CTAs per SM walk the (row chunk, channel tile) pairs; warp 0 loads (TMA), warp 1 issues the MMAs,
// warps 2-9 drain.  Where there are fewer pairs than SMs, a cluster of up to 8 CTAs for every pair cuts the K loop of
// the pair and adds its int32 partial sums through distributed shared memory: the sums are exact, so their
// order does not matter, and there is neither workspace nor atomic.
//
// Up to 4 bf16 tokens are quantised in the kernel itself: every CTA finds the scales of all rows (4 x K
// bf16 come from L2) and writes the codes of its own K range where the MMA reads them.
// That saves a launch and a trip of the codes through L2 in front of the first MMA.
#include "gemm_common.cuh"
#include "i8_common.cuh"
#include "i8_epilogue.cuh"
#include "ptx.cuh"
#include "quant_i8.cuh"

namespace smb {

namespace i8d {

constexpr int kTileRows = 128;        // channels per tile
constexpr int kBlockK = 128;
constexpr int kThreads = 320;
constexpr int kMaxSplit = 8;
constexpr int kPushTokens = 32;       // most tokens per tile whose partial sums have room beside the ring
constexpr int kWBytes = kTileRows * kBlockK;
constexpr int kMaxStages = 12;
constexpr int kPrefetchBlocks = 4;    // K blocks of weights sent to L2 before the offsets are known
constexpr int kBarBytes = 384;
constexpr int kFusedTokens = 4;       // most tokens quantised in the kernel
constexpr int kFusedRows = 8;         // rows of their codes in shared memory: the smallest N of the MMA
// K blocks of codes (1 KB each) beside the ring, which keeps five stages.  us with the quantiser inside / as
// a launch of its own, 1 and 4 tokens: 4096 x 4096 (8 blocks per CTA) 6.6 / 7.6, 7.3 / 7.8 (8 tokens, before the last
// steps: 8.5 / 8.4); 28672 x 8192 (64 blocks, two stages left) 44.6 / 39.9.
constexpr int kFusedMaxBlocks = 24;
constexpr int kTableBytes = (kI8MaxGroups + 8) * 4;
// Half of an SM's shared memory, and at most half of its tensor memory: two CTAs share an SM, so the next
// launch on the stream starts its prologue (and the loads of weights nobody writes) while this one drains.
// Never less, so that there are never three, and an allocation of tensor memory always succeeds at once: a
// CTA that holds some may be waiting for the very kernel that asks for more.  (Of the other kernels that
// allocate it, the narrow BF16 and FP4 tiles take half an SM of both; the rest leave no room beside them.)
constexpr int kTotal = 111 * 1024;
static_assert(kTotal >= kHolderShared, "least of a holder of tensor memory");
constexpr int kRingBudget = kTotal - 1024 - kBarBytes - kTableBytes;

struct Params {
  int M, N, K;
  int tiles_n;
  int chunk;          // tokens per tile, a multiple of 16 up to 128
  int box_rows;       // tokens per TMA box: the chunk, or 16 where groups are ragged
  int stages, stage_bytes;
  int tmem_cols, bank_cols;
  int kb_per;         // K blocks per CTA of a cluster
  int recv_offset;    // bytes from the ring's start to the partial sums received from other CTAs
  int ldd;
  uint16_t* d_ptr;
  const float* sa;
  const float* sb;
  const int* offsets;
  int groups;
  int* status;
  int weights_static;
  int prefetch;
  const uint16_t* x;  // fused quantiser: bf16 tokens [M, K], 16-byte rows, and their pitch
  long long ldx;
};

struct Tile {
  int row0, rows;     // tokens [row0, row0 + rows)
  int group, col0;    // channels [col0, col0 + 128) of the group
};

__device__ __forceinline__ void group_rows(const Params& p, int g, int& lo, int& hi) {
  if (p.offsets == nullptr) {
    lo = 0;
    hi = p.M;
    return;
  }
  lo = min(max(ld_global_s32(p.offsets + g), 0), p.M);
  hi = min(max(ld_global_s32(p.offsets + g + 1), lo), p.M);
}

// Number of row chunks before every group, groups + 1 words at `table`.  First warp of the CTA.
__device__ __forceinline__ void build_chunks(const Params& p, int* table, int lane) {
  constexpr int kPer = kI8MaxGroups / 32;
  int count[kPer];
  int sum = 0;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int g = lane * kPer + i;
    int lo = 0, hi = 0;
    if (g < p.groups) group_rows(p, g, lo, hi);
    count[i] = (hi - lo + p.chunk - 1) / p.chunk;
    sum += count[i];
  }
  int before = sum;
#pragma unroll
  for (int d = 1; d < 32; d <<= 1) {
    const int up = __shfl_up_sync(0xffffffffu, before, d);
    if (lane >= d) before += up;
  }
  before -= sum;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    const int g = lane * kPer + i;
    if (g <= p.groups) table[g] = before;
    before += count[i];
  }
  if (lane == 31 && p.groups == kI8MaxGroups) table[kI8MaxGroups] = before;
}

// Tiles of a group run chunk-fastest: the chunks that read the same weights are neighbours in time.
__device__ __forceinline__ Tile find_tile(const Params& p, const int* table, int t, int lane) {
  constexpr int kPer = kI8MaxGroups / 32;
  const int c = t / p.tiles_n;
  int g = 0;
  if (p.groups > 1) {
    const int first = lane * kPer;
    const unsigned seg_mask = __ballot_sync(0xffffffffu, first < p.groups && table[min(first, p.groups)] <= c);
    const int seg = 31 - __clz(seg_mask | 1u);
    const int g0 = seg * kPer + (lane & (kPer - 1));
    const unsigned in_mask = __ballot_sync(0xffffffffu, lane < kPer && g0 < p.groups && table[min(g0, p.groups)] <= c);
    g = seg * kPer + 31 - __clz(in_mask | 1u);
  }
  const int chunks = table[g + 1] - table[g];
  const int local = t - table[g] * p.tiles_n;
  const int nt = local / chunks;
  int lo, hi;
  group_rows(p, g, lo, hi);
  Tile r;
  r.group = g;
  r.col0 = nt * kTileRows;
  r.row0 = lo + (local - nt * chunks) * p.chunk;
  r.rows = min(p.chunk, hi - r.row0);
  return r;
}

__device__ __forceinline__ float token_scale(const float* sa, const Tile& tile, int c) {
  return c < tile.rows ? sa[tile.row0 + c] : 0.0f;
}

// The eight epilogue warps quantise the tokens, 8 / (M rounded up to a power of two) warps a row: the
// scale of every row to `sa`, the codes of K blocks [kb0, kb1) to x_base ([block][8 rows][128 bytes],
// 128-byte swizzle).  The loads for the codes go out together with the first loads for the maximum and
// wait in registers (up to kHeld per thread; the rest is read again).  `red`: eight words.
__device__ __forceinline__ void quantize_tokens(const Params& p, int kb0, int kb1, uint32_t x_base, uint32_t sa, uint32_t red,
                                                int warp, int lane) {
  const int share = p.M <= 1 ? 8 : (p.M <= 2 ? 4 : 2);   // warps per row
  const int r = warp / share;
  const int threads = share * 32, tid = (warp % share) * 32 + lane;
  const bool live = r < p.M;
  const uint16_t* row = p.x + r * p.ldx;
  constexpr int kBlockVecs = kBlockK / 8;
  const int nvec = live ? p.K / 8 : 0;
  const int first = kb0 * kBlockVecs + tid, end = min(nvec, kb1 * kBlockVecs);
  constexpr int kHeld = 4, kBatch = 8;
  qi8::Vec<true> held[kHeld];
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (first + threads * i < end) held[i] = qi8::load_vec<true>(row, static_cast<int64_t>(first + threads * i) * 8);
  uint32_t m = 0;
  for (int v0 = tid; v0 < nvec; v0 += threads * kBatch) {
    qi8::Vec<true> q[kBatch];
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (v0 + threads * i < nvec) q[i] = qi8::load_vec<true>(row, static_cast<int64_t>(v0 + threads * i) * 8);
#pragma unroll
    for (int i = 0; i < kBatch; ++i)
      if (v0 + threads * i < nvec) m = qi8::abs_max_bits<true>(q[i], m);
  }
  m = __reduce_max_sync(0xffffffffu, m);
  if (lane == 0) asm volatile("st.shared.u32 [%0], %1;" ::"r"(red + 4u * warp), "r"(m) : "memory");
  asm volatile("bar.sync 1, 256;" ::: "memory");   // the eight epilogue warps
  uint32_t other;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(other) : "r"(red + 4u * (r * share + lane % share)) : "memory");
  m = __reduce_max_sync(0xffffffffu, other);
  if (!live) return;
  const qi8::RowScale rs = qi8::row_scale(__uint_as_float(m), m < 0x7F800000u);
  auto store = [&](int v, const qi8::Vec<true>& q) {
    const uint2 c = rs.bad ? make_uint2(0, 0) : qi8::encode<true>(q, rs.inv);
    const int in_block = v % kBlockVecs;
    const uint32_t dst = x_base + (v / kBlockVecs - kb0) * (kFusedRows * kBlockK) + r * kBlockK +
                         (((in_block >> 1) ^ (r & 7)) << 4) + (in_block & 1) * 8;
    asm volatile("st.shared.v2.b32 [%0], {%1, %2};" ::"r"(dst), "r"(c.x), "r"(c.y) : "memory");
  };
#pragma unroll
  for (int i = 0; i < kHeld; ++i)
    if (first + threads * i < end) store(first + threads * i, held[i]);
  for (int v0 = first + threads * kHeld; v0 < end; v0 += threads * kHeld) {
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (v0 + threads * i < end) held[i] = qi8::load_vec<true>(row, static_cast<int64_t>(v0 + threads * i) * 8);
#pragma unroll
    for (int i = 0; i < kHeld; ++i)
      if (v0 + threads * i < end) store(v0 + threads * i, held[i]);
  }
  if (tid == 0)
    asm volatile("st.shared.f32 [%0], %1;" ::"r"(sa + 4u * r), "f"(rs.bad ? __uint_as_float(0x7FC00000u) : rs.scale) : "memory");
}

// kSplit: the CTAs of a cluster share the K loop of ONE tile (the grid has a cluster for every tile), and each
// finishes a share of its tokens.  kPush (up to 32 tokens): partial sums are written straight into the
// owner's shared memory, beside its ring, and one cluster barrier later the owner adds what it received;
// kPull (more, for which there is no room): everyone writes its own into the idle ring, the owners fetch
// them after the barrier, and a second barrier keeps them in place.  1 x 4096 x 4096: accumulator complete to
// kernel end 1.3 us pushed, 2.1 pulled.
enum { kWhole = 0, kPull = 1, kPush = 2 };

// kFused: bf16 tokens (at most 4, a plain product), codes and scales made here.
template <bool kSwiglu, bool kPairs, int kSplitForm, bool kFused>
__global__ void __launch_bounds__(kThreads, 2)
gemm_i8_decode_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                      const __grid_constant__ Params p) {
  constexpr bool kSplit = kSplitForm != kWhole;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t ring_base = smem_base;
  const uint32_t bar_base = ring_base + kRingBudget / 1024 * 1024;
  int* table = reinterpret_cast<int*>(smem_raw + (bar_base + kBarBytes - smem_u32(smem_raw)));
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (kMaxStages + s); };
  auto acc_full_bar = [&](int b) { return bar_base + 8u * (2 * kMaxStages + b); };
  auto acc_empty_bar = [&](int b) { return bar_base + 8u * (2 * kMaxStages + 2 + b); };
  const uint32_t tmem_slot = bar_base + 8u * (2 * kMaxStages + 4);
  const uint32_t x_bar = bar_base + 8u * (2 * kMaxStages + 5);
  const float* sa_smem = reinterpret_cast<const float*>(smem_raw + (bar_base + 320u - smem_u32(smem_raw)));
  const uint32_t x_base = ring_base + p.stages * p.stage_bytes;   // kFused: codes of this CTA's K range
  const float* scales = kFused ? sa_smem : p.sa;
  constexpr int kWOnly = kFused ? 1 : 0;   // stages hold weights alone

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const int split = kSplit ? static_cast<int>(cluster_nctarank()) : 1;
  const int rank = kSplit ? static_cast<int>(cluster_ctarank()) : 0;
  const int unit = blockIdx.x / split;
  const int units = gridDim.x / split;
  const int per = ((p.chunk + split - 1) / split + 1) & ~1;   // tokens of a CTA's share
  const uint32_t recv_base = ring_base + p.recv_offset;        // kPush: [CTA][share][channel] words
  const int num_kb = (p.K + kBlockK - 1) / kBlockK;
  const int kb0 = rank * p.kb_per;
  const int kb1 = min(num_kb, kb0 + p.kb_per);

  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) {
      mbar_init(full_bar(s), 1);
      mbar_init(empty_bar(s), 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full_bar(b), 1);
      mbar_init(acc_empty_bar(b), 8);
    }
    if (kFused) mbar_init(x_bar, 8);
    fence_mbar_init_cluster();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmap_w);
    if (!kFused) tma_prefetch_desc(&tmap_x);
  }
  if (warp == 1) {
    tmem_alloc<1>(tmem_slot, p.tmem_cols);
    tmem_relinquish<1>();
  }
  const bool grouped = p.offsets != nullptr;
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  griddep_launch_dependents();   // not before this CTA holds its tensor memory
  if (kSplitForm == kPush) cluster_arrive();   // the others may write into this CTA from here on
  const uint64_t pol_w = l2_policy_evict_first();
  const uint64_t pol_x = l2_policy_evict_last();
  // Weights that nobody on the stream writes are on their way while the kernel that makes the
  // activations still runs: the first ring's worth of the first tile (a plain product knows its tiles).
  int early = 0;
  if (!grouped && p.weights_static) {
    early = min(p.stages, kb1 - kb0);
    if (warp == 0) {
      const int nt = unit / ((p.M + p.chunk - 1) / p.chunk);
      const int rows = min(p.chunk, p.M);   // every chunk is loaded as whole boxes
      const uint32_t bytes = kWBytes + (kWOnly ? 0 : ((rows + p.box_rows - 1) / p.box_rows) * p.box_rows * kBlockK);
      for (int s = 0; s < early; ++s) {
        if (elect_one()) {
          mbar_arrive_expect_tx(full_bar(s), bytes);
          tma_load_2d_cta_hint(ring_base + s * p.stage_bytes, &tmap_w, full_bar(s), (kb0 + s) * kBlockK, nt * kTileRows, pol_w);
        }
        __syncwarp();
      }
      if (kSplit && elect_one()) {   // what the ring has no room for waits in L2
        for (int kb = kb0 + early; kb < min(kb1, kb0 + early + kPrefetchBlocks); ++kb)
          tma_prefetch_l2_2d(&tmap_w, kb * kBlockK, nt * kTileRows);
      }
      __syncwarp();
    }
  }
  if (p.prefetch != 0 && warp == 0) {
    // The offsets are not there yet, but with rows for every group the walk starts with the weights of the
    // first groups in order: the first blocks of what this CTA would take if every group were one chunk go to
    // L2, where whichever CTA needs them finds them (an int8 expert layer of 512 tokens: 107.2 -> 104.3 us).
    const int g = unit / p.tiles_n, nt = unit % p.tiles_n;
    if (g < p.groups && elect_one()) {
      for (int kb = 0; kb < min(kPrefetchBlocks, num_kb); ++kb)
        tma_prefetch_l2_2d(&tmap_w, kb * kBlockK, g * p.N + nt * kTileRows);
    }
    __syncwarp();
  }
  griddep_wait();
  if (grouped) {
    if (warp == 0) build_chunks(p, table, lane);
  } else if (threadIdx.x == 0) {
    table[0] = 0;
    table[1] = (p.M + p.chunk - 1) / p.chunk;
  }
  __syncthreads();
  if (kSplitForm == kPush) cluster_wait();
  uint32_t tmem_base;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem_base) : "r"(tmem_slot) : "memory");
  int num_tiles = table[p.groups] * p.tiles_n;
  if (kSplit) num_tiles = min(num_tiles, units);   // offsets that overlap could ask for more

  if (warp == 0) {
    // ------------------------------------------------------------- TMA producer
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    for (int t = unit; t < num_tiles && ok; t += units) {
      const Tile tile = find_tile(p, table, t, lane);
      const int boxes = kWOnly ? 0 : (tile.rows + p.box_rows - 1) / p.box_rows;
      const uint32_t bytes = kWBytes + boxes * p.box_rows * kBlockK;
      const int row_w = tile.group * p.N + tile.col0;
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(empty_bar(s), ph ^ 1u)) {
          report_status(p.status, kDevTimeoutProducer);
          ok = false;
          break;
        }
        const uint32_t dst = ring_base + s * p.stage_bytes;
        if (elect_one()) {
          if (early == 0) {
            mbar_arrive_expect_tx(full_bar(s), bytes);
            tma_load_2d_cta_hint(dst, &tmap_w, full_bar(s), kb * kBlockK, row_w, pol_w);
          }
          for (int b = 0; b < boxes; ++b)
            tma_load_2d_cta_hint(dst + kWBytes + b * p.box_rows * kBlockK, &tmap_x, full_bar(s), kb * kBlockK,
                                 tile.row0 + b * p.box_rows, pol_x);
        }
        if (early > 0) --early;
        __syncwarp();
        if (++s == p.stages) { s = 0; ph ^= 1u; }
      }
    }
    if (!ok) {
      for (int i = 0; i < 64; ++i) __nanosleep(1000);   // copies in flight land before shared memory goes away
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------- MMA issue
    int s = 0;
    uint32_t ph = 0;
    int local = 0;
    bool ok = true;
    if (kFused && !mbar_wait(x_bar, 0)) {
      report_status(p.status, kDevTimeoutActivations);
      ok = false;
    }
    for (int t = unit; t < num_tiles && ok; t += units, ++local) {
      const Tile tile = find_tile(p, table, t, lane);
      const int boxes = (tile.rows + p.box_rows - 1) / p.box_rows;
      const uint32_t idesc = make_idesc_i8(128, boxes * p.box_rows);
      const int bank = local & 1;
      if (!mbar_wait(acc_empty_bar(bank), (static_cast<uint32_t>(local >> 1) & 1u) ^ 1u)) {
        report_status(p.status, kDevTimeoutMmaAcc);
        break;
      }
      tc_fence_after_sync();
      const uint32_t tmem_d = tmem_base + static_cast<uint32_t>(bank * p.bank_cols);
      for (int kb = kb0; kb < kb1; ++kb) {
        if (!mbar_wait(full_bar(s), ph)) {
          report_status(p.status, kDevTimeoutMmaFull);
          ok = false;
          break;
        }
        tc_fence_after_sync();
        const uint32_t w_addr = ring_base + s * p.stage_bytes;
        const uint64_t desc_w = make_smem_desc(w_addr, 1024, 16, kSwizzle128B);
        const uint64_t desc_x = make_smem_desc(kFused ? x_base + (kb - kb0) * (kFusedRows * kBlockK) : w_addr + kWBytes, 1024, 16,
                                               kSwizzle128B);
        if (elect_one()) {
#pragma unroll
          for (int k = 0; k < kBlockK / 32; ++k)
            mma_i8_ss<1>(tmem_d, desc_w + 2u * k, desc_x + 2u * k, idesc, (kb > kb0 || k > 0) ? 1u : 0u);
          mma_commit_1cta(empty_bar(s));
        }
        __syncwarp();
        if (++s == p.stages) { s = 0; ph ^= 1u; }
      }
      if (ok && elect_one()) mma_commit_1cta(acc_full_bar(bank));
      __syncwarp();
    }
  } else {
    // ------------------------------------------------------------- epilogue (8 warps)
    // Warp quarter = the 32 lanes it may read; the two warps of a quarter take every other 16 tokens.
    const int quarter = warp & 3;
    const int half = (warp - 2) >> 2;
    int local = 0;
    if (kFused) {
      quantize_tokens(p, kb0, kb1, x_base, bar_base + 320u, bar_base + 352u, warp - 2, lane);
      fence_proxy_async_smem();   // the MMA reads the codes through the async proxy
      __syncwarp();
      if (lane == 0) mbar_arrive(x_bar);
      if (!mbar_wait(x_bar, 0) && lane == 0) report_status(p.status, kDevTimeoutActivations);   // all scales are there
    }
    for (int t = unit; t < num_tiles; t += units, ++local) {
      const Tile tile = find_tile(p, table, t, lane);
      const int bank = local & 1;
      const int n = tile.col0 + quarter * 32 + lane;
      const float sb = !kSplit && n < p.N ? p.sb[static_cast<long long>(tile.group) * p.N + n] : 0.0f;
      // Lane i holds the scale of token i of the warp's current 16.
      float sa = !kSplit ? token_scale(scales, tile, half * 16 + (lane & 15)) : 0.0f;
      if (!mbar_wait(acc_full_bar(bank), static_cast<uint32_t>(local >> 1) & 1u)) {
        if (lane == 0) report_status(p.status, kDevTimeoutEpilogue);
        break;
      }
      tc_fence_after_sync();
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + static_cast<uint32_t>(bank * p.bank_cols);
      for (int c0 = half * 16; c0 < tile.rows; c0 += 32) {
        uint32_t v[16];
        tmem_ld_32x32b_x16(taddr + c0, v);
        tmem_ld_wait();
        if (kSplitForm == kPush) {
          // Token c belongs to CTA c / per: to its slot for this rank, [rank][token of the share][channel].
          int owner = c0 / per, slot = c0 - owner * per;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            if (c0 + i < tile.rows) {
              const uint32_t local = recv_base + ((rank * per + slot) * kTileRows + quarter * 32 + lane) * 4;
              st_shared_cluster_u32(mapa_u32(local, owner), v[i]);
            }
            if (++slot == per) {
              slot = 0;
              ++owner;
            }
          }
        } else if (kSplit) {
          // The ring is idle: its only tile's MMAs are complete.  [token][channel] words.
#pragma unroll
          for (int i = 0; i < 16; ++i)
            asm volatile("st.shared.b32 [%0], %1;" ::"r"(ring_base + ((c0 + i) * kTileRows + quarter * 32 + lane) * 4), "r"(v[i])
                         : "memory");
        } else {
          const float scale = sa;
          sa = token_scale(scales, tile, c0 + 32 + (lane & 15));
          store_tokens<16, kSwiglu, kPairs>(v, scale, sb, p.d_ptr + static_cast<long long>(tile.row0 + c0) * p.ldd, p.ldd, p.N,
                                            tile.rows - c0, n);
        }
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(acc_empty_bar(bank));
    }
  }
  __syncwarp();
  if (kSplit) {
    // CTA r of the cluster owns tokens [r * per, (r + 1) * per) of the tile; its warps take them four at a
    // time, all partial sums of the four in flight together.
    Tile tile = {0, 0, 0, 0};
    if (unit < num_tiles) tile = find_tile(p, table, unit, lane);
    const int quarter = warp & 3;
    const int n = tile.col0 + quarter * 32 + lane;
    const int end = min(tile.rows, (rank + 1) * per);
    float sb = 0.0f;
    if (warp >= 2 && n < p.N && tile.rows > 0) sb = p.sb[static_cast<long long>(tile.group) * p.N + n];
    const int c_first = rank * per + ((warp - 2) >> 2) * 4;
    float sa = warp >= 2 ? token_scale(scales, tile, c_first + (lane & 3)) : 0.0f;
    cluster_sync_all();
    if (warp >= 2) {
      for (int c = c_first; c < end; c += 8) {
        uint32_t part[kMaxSplit][4];
#pragma unroll
        for (int q = 0; q < kMaxSplit; ++q) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            part[q][i] = 0u;
            if (kSplitForm == kPush) {
              if (q < split && c + i < end)
                part[q][i] = ld_shared_u32(recv_base + ((q * per + c + i - rank * per) * kTileRows + quarter * 32 + lane) * 4);
            } else if (q < split) {
              part[q][i] = ld_shared_cluster_u32(mapa_u32(ring_base + ((c + i) * kTileRows + quarter * 32 + lane) * 4, q));
            }
          }
        }
        uint32_t sum[4] = {};
#pragma unroll
        for (int q = 0; q < kMaxSplit; ++q)
#pragma unroll
          for (int i = 0; i < 4; ++i) sum[i] += part[q][i];
        store_tokens<4, kSwiglu, kPairs>(sum, sa, sb, p.d_ptr + static_cast<long long>(tile.row0 + c) * p.ldd, p.ldd, p.N, end - c, n);
        sa = token_scale(scales, tile, c + 8 + (lane & 3));
      }
    }
    if (kSplitForm == kPull) cluster_sync_all();   // partial sums stay until every CTA has read them
  }
  tc_fence_before_sync();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc<1>(tmem_base, p.tmem_cols);
  }
}

}  // namespace i8d

namespace {

template <bool kSwiglu, bool kPairs, int kSplit, bool kFused>
int launch_i8_decode(const I8Launch& L, const i8d::Params& p, int ctas, int split, cudaStream_t stream) {
  auto kernel = i8d::gemm_i8_decode_kernel<kSwiglu, kPairs, kSplit, kFused>;
  static thread_local int configured_device = -1;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return set_error(SMB_ERR_CUDA, "cudaGetDevice failed");
  if (configured_device != dev) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, i8d::kTotal);
    if (e != cudaSuccess) return set_cuda_error(e, "cudaFuncSetAttribute(i8 decode smem)");
    configured_device = dev;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas, 1, 1);
  cfg.blockDim = dim3(i8d::kThreads, 1, 1);
  cfg.dynamicSmemBytes = i8d::kTotal;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = static_cast<unsigned>(split);
  attr[1].val.clusterDim.y = 1;
  attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = kSplit != i8d::kWhole ? 2 : 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, L.tmap_b, L.tmap_a, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error(e, "i8 decode GEMM launch");
  return SMB_OK;
}

int usable_sms() {
  const int slots = device_cluster_slots();
  return slots > 0 ? 2 * slots : 148;
}

// CTAs that share the K loop of a tile: with SMs to spare, the number of the lowest estimate in cycles, the K
// blocks at the 48 bytes per cycle that reach a CTA from HBM and the exchange of the sums, which is short
// where they are pushed.  us with 1 / 2 / 4 CTAs: 48 x 1024 x 512 3.9 / 6.1 / -, 64 x 1024 x 1024 - / 7.5 / 6.1.
// (As many as fill both places of every SM: 1 x 4096 x 4096 from bf16 7.3 instead of 6.6 us, 128 x 4096 x 4096
// 12.7 instead of 11.3.)
int k_split(long long tiles, int K, int chunk, int sms, int* kb_per) {
  const int num_kb = (K + i8d::kBlockK - 1) / i8d::kBlockK;
  const bool push = chunk <= i8d::kPushTokens;
  const int block = (i8d::kWBytes + chunk * i8d::kBlockK) / 48;
  int best = 1, best_cost = num_kb * block;
  for (int split = 2; split <= i8d::kMaxSplit && tiles * split <= sms && num_kb >= 2 * split; split *= 2) {
    const int cost = (num_kb + split - 1) / split * block + (push ? 800 + chunk / split * 60 : 1500 + chunk / split * 130);
    if (cost < best_cost) {
      best = split;
      best_cost = cost;
    }
  }
  *kb_per = (num_kb + best - 1) / best;
  return (num_kb + *kb_per - 1) / *kb_per;
}

}  // namespace

bool i8_pick_decode(int M, int N, int K, int groups, bool tma_store, bool force, int* chunk, int* box_rows) {
  if (groups == 1) {
    // us here / best tiled kernel: 128 x 28672 x 8192 43 / 56, 128 x 4096 x 4096 11.3 / 14.1, 128 x 1024 x 8192
    // 9.6 / 16.5, but 64 x 8192 x 2048 9.3 / 8.2: a short K loop over enough 128-wide tiles for most clusters
    // leaves little to gain over 64 rows.
    if (M > 128 && !force) {
      // A few tiles with a long K, which only this kernel cuts: cycles of 256 x 128 tiles on as many clusters
      // against a share of the K loop and the exchange of 128 x 128 sums.  us tiled / here: 209 x 43 x 5141
      // 12.6 / 7.8, 1024 x 256 x 8192 16.1 / 11.3, 256 x 1024 x 4096 9.9 / 10.1, 2048 x 512 x 8192 17 / 24.
      const long long tiles = static_cast<long long>((M + 127) / 128) * ((N + 127) / 128);
      int kb_per = 0;
      const int split = k_split(tiles, K, 128, usable_sms(), &kb_per);
      if (split == 1) return false;
      const int num_kb = (K + i8d::kBlockK - 1) / i8d::kBlockK;
      if (num_kb * 400 + (tma_store ? 1800 : 3700) <= kb_per * 680 + 7500 + 128 / split * 130) return false;
    }
    if (M >= 64 && N >= 8192 && K <= 2048 && !force) return false;
    *chunk = M >= 128 ? 128 : (M + 15) / 16 * 16;
    *box_rows = *chunk;
    return true;
  }
  // Small chunks keep the stages small and the ring deep; large ones keep experts in one chunk.  us with
  // chunks of 16 / 32 / 64 / 128: 128 experts of 1536 x 2048 with 4 rows on average 61.9 / 65.1 / 66.2 / 69.0, 12
  // rows 67.7 / 66.7 / 67.7 / 69.9, 48 rows - / 73.9 / 69.4 / 73.1, 95 rows - / - / 85.5 / 75.8.  Above 96 rows the
  // 256-row tiles win: 64 experts of 2048 x 2048, 95 rows 52.4 here and 58.6 tiled, 127 rows 60.5 and 59.2.
  const int average = (M + groups - 1) / groups;
  if (average > 96 && !force) return false;
  *chunk = average <= 8 ? 16 : (average <= 16 ? 32 : (average <= 64 ? 64 : 128));
  *box_rows = 16;
  return true;
}

namespace {

template <int kSplit, bool kFused>
int launch_store(const I8Launch& L, const i8d::Params& p, int ctas, int split, cudaStream_t stream) {
  const bool pairs = L.ldd % 2 == 0 && reinterpret_cast<uintptr_t>(L.d) % 4 == 0 && L.tma_store;
  if (L.swiglu) return launch_i8_decode<true, true, kSplit, kFused>(L, p, ctas, split, stream);
  return pairs ? launch_i8_decode<false, true, kSplit, kFused>(L, p, ctas, split, stream)
               : launch_i8_decode<false, false, kSplit, kFused>(L, p, ctas, split, stream);
}

}  // namespace

int i8_decode_launch(const I8Launch& L, cudaStream_t stream) {
  int dev = 0, sms = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess)
    return set_error(SMB_ERR_CUDA, "i8 decode: no current device");
  const int all_sms = sms;
  if (L.max_clusters > 0 && sms > 2 * L.max_clusters) sms = 2 * L.max_clusters;
  i8d::Params p = {};
  p.M = L.M;
  p.N = L.N;
  p.K = L.K;
  p.tiles_n = (L.N + i8d::kTileRows - 1) / i8d::kTileRows;
  p.chunk = L.chunk;
  p.box_rows = L.box_rows;
  p.stage_bytes = i8d::kWBytes + L.chunk * i8d::kBlockK;
  p.bank_cols = L.chunk <= 16 ? 16 : (L.chunk <= 32 ? 32 : (L.chunk <= 64 ? 64 : 128));
  p.tmem_cols = 2 * p.bank_cols;
  p.ldd = L.ldd;
  p.d_ptr = static_cast<uint16_t*>(L.d);
  p.sa = L.sa;
  p.sb = L.sb;
  p.offsets = L.offsets;
  p.groups = L.groups;
  p.status = L.status;
  p.weights_static = L.weights_static ? 1 : 0;
  p.prefetch = L.weights_static && L.offsets != nullptr && L.M >= 8 * L.groups ? 1 : 0;   // hardly a group is empty
  // Upper bound of the (chunk, channel tile) pairs; exact for a plain product.
  const long long full = (static_cast<long long>(L.M) + L.chunk - 1) / L.chunk;
  long long chunks = full;
  if (L.offsets != nullptr) chunks = L.M / L.chunk + (L.groups < L.M ? L.groups : L.M);
  const long long tiles = chunks * p.tiles_n;
  if (tiles > 0x7FFFFFFFLL) return set_error(SMB_ERR_UNSUPPORTED, "i8 decode: too many tiles");
  const int split = k_split(tiles, L.K, L.x != nullptr ? i8d::kFusedRows : L.chunk, L.x != nullptr ? all_sms : sms, &p.kb_per);   // as the plan decided
  long long ctas;
  if (split > 1) {
    ctas = tiles * split;
  } else {
    // Two CTAs per SM, equal shares: the CTAs that t = ceil(tiles / slots) tiles each leave busy.  16 x 28672 x
    // 8192 from bf16: 38.6 us with two CTAs per SM, 43.7 with one of the same size, 40.5 with one of twice
    // the ring; 128 experts x 256 rows gated 63.5 / 65.9 / 65.9.
    const int slots = 2 * sms;
    const long long per = (tiles + slots - 1) / slots;
    ctas = (tiles + per - 1) / per;
    if (L.offsets != nullptr && ctas < slots && tiles >= slots) ctas = slots;   // the bound says little about the count
  }
  int room = i8d::kRingBudget / 1024 * 1024;
  if (L.x != nullptr) {
    // The stages hold weights alone; behind the ring lie the codes of the CTA's K range.
    p.x = L.x;
    p.ldx = L.ldx;
    p.chunk = p.box_rows = i8d::kFusedRows;
    p.stage_bytes = i8d::kWBytes;
    room -= p.kb_per * i8d::kFusedRows * i8d::kBlockK;
  }
  const bool push = split > 1 && p.chunk <= i8d::kPushTokens;
  if (push) room -= ((split * (((p.chunk + split - 1) / split + 1) & ~1) * i8d::kTileRows * 4) + 1023) / 1024 * 1024;
  p.stages = room / p.stage_bytes;
  if (p.stages > i8d::kMaxStages) p.stages = i8d::kMaxStages;
  p.recv_offset = p.stages * p.stage_bytes + (L.x != nullptr ? p.kb_per * i8d::kFusedRows * i8d::kBlockK : 0);
  const int c = static_cast<int>(ctas);
  if (L.x != nullptr)
    return split > 1 ? launch_store<i8d::kPush, true>(L, p, c, split, stream) : launch_store<i8d::kWhole, true>(L, p, c, split, stream);
  if (split == 1) return launch_store<i8d::kWhole, false>(L, p, c, split, stream);
  return push ? launch_store<i8d::kPush, false>(L, p, c, split, stream) : launch_store<i8d::kPull, false>(L, p, c, split, stream);
}

bool i8_decode_fuses(const I8Launch& L, const void* x, long long ldx) {
  if (!L.decode || L.offsets != nullptr || L.M > i8d::kFusedTokens || L.K % 8 != 0 || ldx % 8 != 0 ||
      reinterpret_cast<uintptr_t>(x) % 16 != 0)
    return false;
  int kb_per = 0;
  k_split((L.N + i8d::kTileRows - 1) / i8d::kTileRows, L.K, i8d::kFusedRows, usable_sms(), &kb_per);
  return kb_per <= i8d::kFusedMaxBlocks;
}

}  // namespace smb
