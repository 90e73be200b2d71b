// Dense and grouped int8 GEMM for sm_100a:
//   D[m,n] = bf16( (float(sum_k A[m,k] B[n,k]) * sa[m]) * sb[n] ),  A, B int8, the sum exact in int32.
// Gated form: z as above with its rounding left out, D[m,n] = bf16( silu(z[m,2n+1]) * z[m,2n] ).
//
// Same skeleton as the BF16 kernel (one 2-CTA cluster per 256 x (NB * TN) tile, TMA ring of 128-byte
// rows, tcgen05.mma.cta_group::2 with accumulators in tensor memory), because a 128-byte row of int8
// holds twice the K of a bf16 one at twice the MMA rate: bytes and cycles per stage are the same.
// What differs: kind::i8 with int32 accumulators, the scales applied on the way out of tensor memory,
// and groups whose row offsets live in device memory (written by an earlier kernel on the stream).
//
// Bound by the tensor cores, from a second of load on by the 1 kW power cap: 8192^3 in 311 us (3.53 PFLOP/s, the
// tensor pipe busy 91 % of the cycles) in bursts and 366 us (3.0 PFLOP/s) sustained, 2.1 times the bf16
// rate either way; DRAM reads 340 MB of 134 MB of operands.  A grouped launch of 64 experts x 32768 rows (gated,
// 4096 x 2048 each) takes 230 to 240 us / 287 us sustained: 161 row tiles where 128 full ones would do.  With a
// K below about 768 the epilogue bounds it, 5.6K cycles for a 256 x 256 tile.
//
// Rounding: the int32 sum becomes fp32 (half a step, 2^-24 relative), two fp32 products follow
// (2^-24 each), one rounding to bf16 (2^-8) ends it.
#include "epilogue.cuh"
#include "i8_common.cuh"
#include "i8_epilogue.cuh"
#include "ptx.cuh"

namespace smb {

namespace i8k {

constexpr int kBlockM = 128;          // rows of A per CTA
constexpr int kBlockK = 128;          // int8 per stage row
constexpr int kThreads = 320;
constexpr int kEpiWarps = 8;
constexpr int kABytes = kBlockM * kBlockK;            // 16 KiB
enum { kStorePlain = 0, kStoreTma = 1, kStoreSwiglu = 2 };

template <int TN, int NB>
struct Cfg {
  static_assert(TN == 128 || TN == 256, "tile width");
  static_assert(NB == 1 || (NB == 2 && TN == 256), "two sub-blocks only at full width");
  static constexpr int kTmemCols = 512;                            // two accumulator slots of up to 256
  static constexpr int kBBytes = (TN / 2) * kBlockK;               // one sub-block, one CTA
  static constexpr int kStageBytes = kABytes + NB * kBBytes;
  static constexpr int kStages = 192 * 1024 / kStageBytes;         // 8, 6 or 4
  static constexpr int kRingBytes = kStages * kStageBytes;
  static constexpr int kTileN = TN * NB;
  static constexpr int kGroupsPerSlot = (NB == 2) ? 1 : 2;
  static constexpr int kStoreBytes = kEpiWarps * kStoreBufBytes;
  static constexpr int kBarrierBytes = 256;
  static constexpr int kTableBytes = (kI8MaxGroups + 8) * 2;       // row-tile table of grouped launches
  static constexpr int kTotal = 1024 + kRingBytes + kStoreBytes + kBarrierBytes + kTableBytes;
  static constexpr int kColsPerWarp = TN / kGroupsPerSlot;
  static constexpr int kSlotReaders = 2 * 4 * kGroupsPerSlot;      // arrivals per drained slot
  static_assert(kTotal <= 232448, "shared memory budget");
  static_assert(fills_sm(kTotal), "the next kernel starts before the allocation");
};

struct Params {
  int M, N, K;
  int tiles_m, tiles_n;      // tiles_m: plain launches; grouped ones count their own
  int group_m;
  int ldd;
  uint16_t* d_ptr;
  const float* sa;
  const float* sb;
  const int* offsets;
  int groups;
  int* status;
  PeerCopies peers;          // always empty; the store path asks
};

// First row and end of the rows of row tile `tm`, and its group.
struct RowTile {
  int row0, row_end, group;
};

// Rows of group g, kept inside [0, M] whatever the offsets hold.
__device__ __forceinline__ void group_rows(const Params& p, int g, int& lo, int& hi) {
  lo = min(max(ld_global_s32(p.offsets + g), 0), p.M);
  hi = min(max(ld_global_s32(p.offsets + g + 1), lo), p.M);
}

// Cumulative count of 256-row tiles before every group, as 16-bit words at `table` (groups + 1 of
// them).  All threads of the CTA call this.
__device__ __forceinline__ void build_row_tiles(const Params& p, uint16_t* table) {
  // One warp, 16 groups a lane: the loads of a lane are independent, the scan is five shuffles.
  if (threadIdx.x < 32) {
    const int lane = threadIdx.x;
    constexpr int kPer = kI8MaxGroups / 32;
    int count[kPer];
    int sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int g = lane * kPer + i;
      int lo = 0, hi = 0;
      if (g < p.groups) group_rows(p, g, lo, hi);
      count[i] = (hi - lo + 255) >> 8;
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
      if (g <= p.groups) table[g] = static_cast<uint16_t>(min(before, 65535));
      before += count[i];
    }
    if (lane == 31 && p.groups == kI8MaxGroups) table[kI8MaxGroups] = static_cast<uint16_t>(min(before, 65535));
  }
}

// The group whose tiles hold tile `tm` is the last one with table[g] <= tm.  Whole warp.
__device__ __forceinline__ RowTile find_row_tile(const Params& p, const uint16_t* table, int tm, int lane) {
  constexpr int kPer = kI8MaxGroups / 32;
  const int first = lane * kPer;
  const unsigned seg_mask = __ballot_sync(0xffffffffu, first < p.groups && table[min(first, p.groups)] <= tm);
  const int seg = 31 - __clz(seg_mask | 1u);
  const int g0 = seg * kPer + (lane & (kPer - 1));
  const unsigned in_mask = __ballot_sync(0xffffffffu, lane < kPer && g0 < p.groups && table[min(g0, p.groups)] <= tm);
  RowTile r;
  r.group = seg * kPer + 31 - __clz(in_mask | 1u);
  int lo, hi;
  group_rows(p, r.group, lo, hi);
  r.row0 = lo + (tm - table[r.group]) * 256;
  r.row_end = hi;
  return r;
}

template <int TN, int NB, int kStore>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
gemm_i8_kernel(const __grid_constant__ CUtensorMap tmap_a, const __grid_constant__ CUtensorMap tmap_a32,
               const __grid_constant__ CUtensorMap tmap_b, const __grid_constant__ CUtensorMap tmap_d,
               const __grid_constant__ Params p) {
  using C = Cfg<TN, NB>;
  constexpr bool kTmaStore = (kStore != kStorePlain);
  constexpr bool kSwiglu = (kStore == kStoreSwiglu);
  static_assert(!kSwiglu || C::kColsPerWarp % 128 == 0, "gated epilogue: 64 output columns per box");
  constexpr int kStages = C::kStages;
  extern __shared__ uint8_t smem_raw[];
  const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t ring_base = smem_base;
  const uint32_t store_base = ring_base + C::kRingBytes;
  const uint32_t bar_base = store_base + C::kStoreBytes;
  uint16_t* table = reinterpret_cast<uint16_t*>(smem_raw + (bar_base + C::kBarrierBytes - smem_u32(smem_raw)));
  auto full_bar = [&](int s) { return bar_base + 8u * s; };
  auto empty_bar = [&](int s) { return bar_base + 8u * (kStages + s); };
  auto acc_full_bar = [&](int b) { return bar_base + 8u * (2 * kStages + b); };
  auto acc_empty_bar = [&](int b) { return bar_base + 8u * (2 * kStages + 2 + b); };
  const uint32_t tmem_slot = bar_base + 8u * (2 * kStages + 4);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const int cluster = static_cast<int>(cluster_id_x());
  const int n_clusters = static_cast<int>(num_clusters_x());
  const int num_kb = (p.K + kBlockK - 1) / kBlockK;

  griddep_launch_dependents();
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(full_bar(s), 1);    // the leader's arrive.expect_tx covers both CTAs' bytes
      mbar_init(empty_bar(s), 1);   // one tcgen05.commit
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(acc_full_bar(b), 1);                 // one tcgen05.commit
      mbar_init(acc_empty_bar(b), C::kSlotReaders);  // every epilogue warp that reads the slot
    }
    fence_mbar_init_cluster();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tmap_a);
    tma_prefetch_desc(&tmap_b);
    if (kTmaStore) tma_prefetch_desc(&tmap_d);
  }
  if (warp == 1) {
    tmem_alloc<2>(tmem_slot, C::kTmemCols);
    tmem_relinquish<2>();
  }
  const bool grouped = p.offsets != nullptr;
  // Operands, scales and offsets may be the previous kernel's output: nothing of theirs is read
  // before it has completed.
  griddep_wait();
  if (grouped) build_row_tiles(p, table);
  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after_sync();
  uint32_t tmem_base;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(tmem_base) : "r"(tmem_slot) : "memory");
  const int tiles_m = grouped ? table[p.groups] : p.tiles_m;
  const int num_tiles = tiles_m * p.tiles_n;
  const int group_m = min(p.group_m, max(tiles_m, 1));

  if (warp == 0) {
    // ------------------------------------------------------------- TMA producer
    const uint32_t leader_full0 = mapa_u32(full_bar(0), 0);
    int s = 0;
    uint32_t ph = 0;
    bool ok = true;
    const uint64_t pol = l2_policy_evict_last();
    for (int t = cluster; t < num_tiles && ok; t += n_clusters) {
      int tm, tn;
      tile_coords(t, tiles_m, p.tiles_n, group_m, tm, tn);
      RowTile rt = {tm * 256, p.M, 0};
      if (grouped) rt = find_row_tile(p, table, tm, lane);
      // B is read on past N (columns that are never stored).
      const int row_a = rt.row0 + static_cast<int>(rank) * kBlockM;
      const bool ragged = grouped && row_a + kBlockM > rt.row_end;   // the group ends in this CTA's half
      const int row_b = rt.group * p.N + tn * C::kTileN + static_cast<int>(rank) * (TN / 2);
      for (int kb = 0; kb < num_kb; ++kb) {
        if (!mbar_wait(empty_bar(s), ph ^ 1u)) {
          report_status(p.status, kDevTimeoutProducer);
          ok = false;
          break;
        }
        const uint32_t bar = leader_full0 + 8u * s;
        const uint32_t dst_a = ring_base + s * C::kStageBytes;
        if (elect_one()) {
          if (rank == 0) mbar_arrive_expect_tx(full_bar(s), 2 * C::kStageBytes);
          if (ragged) {
            // Rows of other groups would be multiplied in vain; in steps of 32 they are fetched from beyond
            // the end of A instead, as zeros, which cost the tensor cores less power and L2 nothing.
#pragma unroll
            for (int q = 0; q < kBlockM; q += 32)
              tma_load_2d_pair_hint(dst_a + q * kBlockK, &tmap_a32, bar, kb * kBlockK, row_a + q < rt.row_end ? row_a + q : p.M,
                                    pol);
          } else {
            tma_load_2d_pair_hint(dst_a, &tmap_a, bar, kb * kBlockK, row_a, pol);
          }
#pragma unroll
          for (int h = 0; h < NB; ++h)
            tma_load_2d_pair_hint(dst_a + kABytes + h * C::kBBytes, &tmap_b, bar, kb * kBlockK, row_b + h * TN, pol);
        }
        __syncwarp();
        if (++s == kStages) { s = 0; ph ^= 1u; }
      }
    }
    if (!ok) {
      // Give copies already in flight time to land before this CTA's shared memory goes away.
      for (int i = 0; i < 64; ++i) __nanosleep(1000);
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------- MMA issue (leader CTA only)
    if (rank == 0) {
      constexpr uint32_t idesc = make_idesc_i8(256, TN);
      int s = 0;
      uint32_t ph = 0;
      int local = 0;
      bool ok = true;
      for (int t = cluster; t < num_tiles && ok; t += n_clusters, ++local) {
        const int bank = (NB == 1) ? (local & 1) : 0;
        const uint32_t use_parity = static_cast<uint32_t>((NB == 1) ? (local >> 1) : local) & 1u;
        for (int kb = 0; kb < num_kb && ok; ++kb) {
          if (!mbar_wait(full_bar(s), ph)) {
            report_status(p.status, kDevTimeoutMmaFull);
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t a_addr = ring_base + s * C::kStageBytes;
          const uint64_t desc_a = make_smem_desc(a_addr, 1024, 16, kSwizzle128B);
#pragma unroll
          for (int h = 0; h < NB; ++h) {
            const int slot = (NB == 1) ? bank : h;
            if (kb == 0) {
              if (!mbar_wait(acc_empty_bar(slot), use_parity ^ 1u)) {
                report_status(p.status, kDevTimeoutMmaAcc);
                ok = false;
                break;
              }
              tc_fence_after_sync();
            }
            const uint32_t tmem_d = tmem_base + static_cast<uint32_t>(slot * TN);
            const uint64_t desc_b = make_smem_desc(a_addr + kABytes + h * C::kBBytes, 1024, 16, kSwizzle128B);
            if (elect_one()) {
#pragma unroll
              for (int k = 0; k < kBlockK / 32; ++k)   // 32 int8 = 32 bytes further inside the swizzled row
                mma_i8_ss<2>(tmem_d, desc_a + 2u * k, desc_b + 2u * k, idesc, (kb > 0 || k > 0) ? 1u : 0u);
            }
            __syncwarp();
          }
          if (!ok) break;
          if (elect_one()) mma_commit_pair(empty_bar(s), 0x3);
          __syncwarp();
          if (++s == kStages) { s = 0; ph ^= 1u; }
        }
        if (ok && elect_one()) mma_commit_pair(acc_full_bar(bank), 0x3);
        __syncwarp();
      }
    }
  } else {
    // ------------------------------------------------------------- epilogue (8 warps)
    const int quarter = warp & 3;           // TMEM lane quarter this warp may read
    const int group = (warp - 2) >> 2;      // 0: warps 2-5, 1: warps 6-9
    const uint32_t leader_acc_empty0 = mapa_u32(acc_empty_bar(0), 0);
    const uint32_t sbuf = store_base + (warp - 2) * kStoreBufBytes;
    StoreTarget out;
    out.tmap_d = &tmap_d;
    out.d_ptr = p.d_ptr;
    out.ldd = p.ldd;
    out.M = p.M;
    out.N = kSwiglu ? p.N / 2 : p.N;
    out.peers = &p.peers;
    out.alpha = 1.0f;
    out.keep_padding = true;
    int local = 0;
    for (int t = cluster; t < num_tiles; t += n_clusters, ++local) {
      int tm, tn;
      tile_coords(t, tiles_m, p.tiles_n, group_m, tm, tn);
      RowTile rt = {tm * 256, p.M, 0};
      if (grouped) rt = find_row_tile(p, table, tm, lane);
      const int row0 = rt.row0 + static_cast<int>(rank) * kBlockM + quarter * 32;
      out.row_end = rt.row_end;
      const int bank = (NB == 1) ? (local & 1) : 0;
      const int slot = (NB == 1) ? bank : group;
      const uint32_t use_parity = static_cast<uint32_t>((NB == 1) ? (local >> 1) : local) & 1u;
      const int tile_col = (NB == 1) ? group * C::kColsPerWarp : group * TN;
      const int col0 = tn * C::kTileN + tile_col;
      // The scales of this warp's rows and columns are fetched while the tile is being multiplied.
      const int row = row0 + lane;
      const float sa = row < rt.row_end ? p.sa[row] : 0.0f;
      stage_column_scales<C::kColsPerWarp, kTmaStore>(sbuf, p.sb + static_cast<long long>(rt.group) * p.N, col0, p.N,
                                                      lane);
      if (!mbar_wait(acc_full_bar(bank), use_parity)) {
        if (lane == 0) report_status(p.status, kDevTimeoutEpilogue);
        break;
      }
      tc_fence_after_sync();
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) +
                             static_cast<uint32_t>((NB == 1) ? bank * TN + tile_col : tile_col);
      constexpr int kOutCols = kSwiglu ? C::kColsPerWarp / 2 : C::kColsPerWarp;
      uint32_t packed[kOutCols / 2];
      drain_columns_i8<C::kColsPerWarp, kSwiglu, NB == 1>(taddr, sbuf, sa, packed);
      release_columns(leader_acc_empty0 + 8u * slot, lane);
      store_columns<kOutCols, kTmaStore>(packed, sbuf, out, row0, kSwiglu ? col0 / 2 : col0, lane);
    }
    drain_store_groups<kTmaStore>(lane);
  }
  __syncwarp();

  tc_fence_before_sync();
  __syncthreads();
  cluster_sync_all();
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc<2>(tmem_base, C::kTmemCols);
  }
}

}  // namespace i8k

// -----------------------------------------------------------------------------------
// Host side
// -----------------------------------------------------------------------------------
namespace {

template <int TN, int NB, int kStore>
int launch_i8(const I8Launch& L, cudaStream_t stream) {
  using C = i8k::Cfg<TN, NB>;
  auto kernel = i8k::gemm_i8_kernel<TN, NB, kStore>;
  static thread_local int configured_device = -1;
  static thread_local int max_clusters = 0;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return set_error(SMB_ERR_CUDA, "cudaGetDevice failed");
  if (configured_device != dev) {
    cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kTotal);
    if (e != cudaSuccess) return set_cuda_error(e, "cudaFuncSetAttribute(i8 smem)");
    cudaLaunchConfig_t probe = {};
    probe.gridDim = dim3(2, 1, 1);
    probe.blockDim = dim3(i8k::kThreads, 1, 1);
    probe.dynamicSmemBytes = C::kTotal;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2;
    attr.val.clusterDim.y = 1;
    attr.val.clusterDim.z = 1;
    probe.attrs = &attr;
    probe.numAttrs = 1;
    int n = 0;
    e = cudaOccupancyMaxActiveClusters(&n, kernel, &probe);
    if (e != cudaSuccess) return set_cuda_error(e, "cudaOccupancyMaxActiveClusters(i8)");
    if (n <= 0) return set_error(SMB_ERR_CUDA, "no 2-CTA cluster of the i8 kernel fits on this device");
    max_clusters = n;
    configured_device = dev;
  }
  i8k::Params p = {};
  p.M = L.M;
  p.N = L.N;
  p.K = L.K;
  p.tiles_m = (L.M + 255) / 256;
  p.tiles_n = (L.N + C::kTileN - 1) / C::kTileN;
  p.group_m = L.group_m > 0 ? L.group_m : raster_group_rows(p.tiles_m, L.K, static_cast<long long>(L.N) * L.K);
  p.ldd = L.ldd;
  p.d_ptr = static_cast<uint16_t*>(L.d);
  p.sa = L.sa;
  p.sb = L.sb;
  p.offsets = L.offsets;
  p.groups = L.groups;
  p.status = L.status;
  // Grouped: at most one partly filled row tile per group on top of the full ones.
  const long long rows = L.offsets != nullptr ? static_cast<long long>(p.tiles_m) + L.groups : p.tiles_m;
  const long long tiles = rows * p.tiles_n;
  if (tiles > 0x7FFFFFFFLL) return set_error(SMB_ERR_UNSUPPORTED, "i8: too many tiles");
  int clusters = static_cast<int>(tiles < max_clusters ? tiles : max_clusters);
  if (L.max_clusters > 0 && clusters > L.max_clusters) clusters = L.max_clusters;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(2 * clusters, 1, 1);
  cfg.blockDim = dim3(i8k::kThreads, 1, 1);
  cfg.dynamicSmemBytes = C::kTotal;
  cfg.stream = stream;
  cudaLaunchAttribute pdl;
  pdl.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &pdl;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, L.tmap_a, L.tmap_a32, L.tmap_b, L.tmap_d, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error(e, "i8 GEMM launch");
  return SMB_OK;
}

template <int TN, int NB>
int launch_i8_store(const I8Launch& L, cudaStream_t stream) {
  if (L.swiglu) {
    if constexpr (TN == 256) {
      return launch_i8<TN, NB, i8k::kStoreSwiglu>(L, stream);
    } else {
      return set_error(SMB_ERR_UNSUPPORTED, "i8: the gated epilogue needs 256-wide tiles");
    }
  }
  return L.tma_store ? launch_i8<TN, NB, i8k::kStoreTma>(L, stream) : launch_i8<TN, NB, i8k::kStorePlain>(L, stream);
}

}  // namespace

// Estimated cycles of the three tiles.  A K block (24, 32 or 48 KB) takes 630, 756 or 1432 cycles in a chain of
// launches (from the 64 bytes per cycle that an SM takes in through TMA, at the clock that their power leaves);
// draining and storing a tile takes 14 cycles a column, 29 without TMA stores, half hidden (three quarters
// with TMA) behind the next tile's K loop.  The 512-wide tile has no second accumulator: only loads hide its
// drain, from the second wave on.
// Measured, us, 128 / 256 / 512 wide: 256 x 4096 x 4096 11.2 / 14.9 / 25.5, 256 x 28672 x 8192 70 / 58 / 59,
// 1151 x 4040 x 90 6.9 / 8.1 / 9.0, 1000 deep 12.6 / 12.0 / 13.5; without TMA stores 4095 x 12289 x 4160 200 / 146 /
// 173, 1151 x 4039 x 90 8.6 / 10.5 / 10.6.
void i8_pick_tile(int M, int N, int K, int clusters, bool tma_store, int* tile_n, int* sub_blocks) {
  if (clusters < 1) clusters = 74;
  const long long tiles_m = (M + 255) / 256;
  const long long kb = (K + 127) / 128;
  const double column = tma_store ? 14.0 : 29.0;
  auto waves = [&](int width) { return static_cast<double>((tiles_m * ((N + width - 1) / width) + clusters - 1) / clusters); };
  auto cost = [&](int width, double block) {
    const double loop = kb * block, drain = width * column;
    const double more = loop < drain ? loop : drain, open = tma_store ? 0.25 : 0.5;
    return waves(width) * (loop + drain - more + open * more) + (1.0 - open) * more;
  };
  const double cost128 = cost(128, 630.0), cost256 = cost(256, 756.0);
  const double loop512 = kb * 1432.0, drain512 = 512 * column;
  const double shown = (drain512 > loop512 ? drain512 - loop512 : 0.0) + (tma_store ? 2500.0 : 8000.0);
  const double cost512 = waves(512) * (loop512 + shown) - shown + 0.85 * drain512;
  *tile_n = cost128 <= cost256 && cost128 <= cost512 ? 128 : 256;
  *sub_blocks = *tile_n == 256 && cost512 < cost256 ? 2 : 1;
}

int i8_launch(const I8Launch& L, cudaStream_t stream) {
  if (L.sub_blocks == 2 && L.tile_n == 256) return launch_i8_store<256, 2>(L, stream);
  if (L.sub_blocks != 1) return set_error(SMB_ERR_INVALID, "i8: two sub-blocks need 256-wide tiles");
  switch (L.tile_n) {
    case 256: return launch_i8_store<256, 1>(L, stream);
    case 128: return launch_i8_store<128, 1>(L, stream);
    default: return set_error(SMB_ERR_INVALID, "i8 tile width must be 128 or 256");
  }
}

}  // namespace smb
