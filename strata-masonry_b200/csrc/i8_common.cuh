// Shared between the int8 product's kernels (gemm_i8.cu, gemm_i8_decode.cu), its quantiser
// (quant_i8.cu) and its C-ABI layer (api_i8.cu).
#pragma once

#include "gemm_common.cuh"

namespace smb {

constexpr int kI8MaxGroups = 512;        // grouped plans: entries of the kernels' row-tile table
constexpr int kI8MaxRows = 8 << 20;      // ... whose 16-bit counts hold 65535 tiles of 256 rows
constexpr int kI8MaxExtent = 1 << 30;    // M and N: tiles that end behind them stay within 31 bits
constexpr int kI8MaxK = 131071;          // 128 * 128 * K stays below 2^31: int32 sums never wrap

struct I8Launch {
  CUtensorMap tmap_a, tmap_b, tmap_d;
  CUtensorMap tmap_a32;   // grouped tiled kernel: A in boxes of 32 rows
  int M, N, K;           // M: rows of A (grouped: upper bound of the rows in use)
  int tile_n;            // tiled kernel: width of one N sub-block, 128 or 256
  int sub_blocks;        // 1, or 2 (256 x 512 tiles)
  bool tma_store;        // false: D rows are not 16-byte aligned
  bool swiglu;           // gated epilogue, D is [M, N/2] (tma_store only)
  int group_m;           // raster group height (0 = default)
  int max_clusters;      // 0 = as many as fit
  void* d;
  int ldd;
  const float* sa;       // scale per row of A
  const float* sb;       // scale per row of B (grouped: groups * N)
  int groups;            // 1: plain product
  const int* offsets;    // grouped: groups + 1 row offsets (device), else null
  bool decode;           // the kernel for few rows per weight matrix (tmap boxes differ)
  int chunk;             // decode: rows of A per tile, a multiple of 16 up to 128
  int box_rows;          // decode: rows of A per TMA box
  bool weights_static;   // B and sb are not written by work that may still run on the stream
  const uint16_t* x;     // decode: bf16 rows that the kernel quantises itself (i8_decode_fuses), else null
  long long ldx;
  int* status;
};

void i8_pick_tile(int M, int N, int K, int clusters, bool tma_store, int* tile_n, int* sub_blocks);
int i8_launch(const I8Launch& L, cudaStream_t stream);
// Whether the decode kernel is taken for M rows in `groups` groups, with its chunk and box heights.
bool i8_pick_decode(int M, int N, int K, int groups, bool tma_store, bool force, int* chunk, int* box_rows);
int i8_decode_launch(const I8Launch& L, cudaStream_t stream);
bool i8_decode_fuses(const I8Launch& L, const void* x, long long ldx);   // for plain plans fed with bf16 rows

// Rows of `src` (bf16 or fp32) to int8 codes and one scale per row.  The next kernel on the stream may
// start its prologue early.
int quantize_i8_launch(const void* src, bool bf16, int64_t ld_src, int8_t* codes, int64_t ld_bytes, float* scales,
                       int64_t rows, int64_t K, cudaStream_t st);

}  // namespace smb
