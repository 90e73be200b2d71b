// int8 quantiser, one scale per row: the activations of a token, or the weights of an output channel
// of the int8 product.  Bound by HBM: bf16 rows move 3 bytes per element, 8192 x 8192 in 30.2 us (6.7 TB/s); a row
// stays in registers between the search for its maximum and the coding, so it is read once.  A few rows
// cost a launch: 1 x 8192 1.6 us, 128 x 8192 3.0 us behind another kernel.
#include <cmath>
#include <cstring>

#include "i8_common.cuh"
#include "quant_i8.cuh"

namespace smb {
namespace {

constexpr int kWarpRows = 8;        // rows of a CTA where a warp takes a row
constexpr int kWarpMaxK = 1024;     // ... which it holds in registers

template <bool kBf16, bool kWarp, int kPer>
__global__ void __launch_bounds__(kWarp ? 32 * kWarpRows : 32 * qi8::kMaxRowWarps)
quantize_i8_kernel(const void* src, int64_t ld_src, int8_t* codes, int64_t ld_bytes, float* scales, int64_t rows, int K) {
  __shared__ uint32_t red[qi8::kMaxRowWarps];
  griddep_launch_dependents();
  griddep_wait();
  const int threads = kWarp ? 32 : blockDim.x;
  const int tid = kWarp ? threadIdx.x & 31 : threadIdx.x;
  const int64_t r = kWarp ? static_cast<int64_t>(blockIdx.x) * kWarpRows + (threadIdx.x >> 5) : blockIdx.x;
  if (r >= rows) return;   // whole warps
  const void* row = static_cast<const char*>(src) + r * ld_src * (kBf16 ? 2 : 4);
  int8_t* out = codes + r * ld_bytes;
  const float scale = qi8::quantize_row<kBf16, kWarp, kPer, false>(
      row, K, tid, threads, red, [&](int k, uint2 c) { *reinterpret_cast<uint2*>(out + k) = c; },
      [&](int k, uint16_t c) { *reinterpret_cast<uint16_t*>(out + k) = c; },
      [&](int k, int8_t c) { out[k] = c; });
  if (tid == 0) scales[r] = scale;
}

template <bool kBf16, int kPer>
cudaError_t launch_quantize(const cudaLaunchConfig_t& base, const void* src, int64_t ld_src, int8_t* codes,
                            int64_t ld_bytes, float* scales, int64_t rows, int K) {
  cudaLaunchConfig_t cfg = base;
  if (K <= kWarpMaxK) {
    cfg.gridDim = dim3(static_cast<unsigned>((rows + kWarpRows - 1) / kWarpRows), 1, 1);
    cfg.blockDim = dim3(32 * kWarpRows, 1, 1);
    return cudaLaunchKernelEx(&cfg, quantize_i8_kernel<kBf16, true, kPer>, src, ld_src, codes, ld_bytes, scales, rows, K);
  }
  cfg.gridDim = dim3(static_cast<unsigned>(rows), 1, 1);
  cfg.blockDim = dim3(static_cast<unsigned>(qi8::row_threads(K, rows, kPer)), 1, 1);
  return cudaLaunchKernelEx(&cfg, quantize_i8_kernel<kBf16, false, kPer>, src, ld_src, codes, ld_bytes, scales, rows, K);
}

int check_quantize(const void* src, int64_t ld_src, const void* codes, int64_t ld_bytes, const void* scales, int64_t rows,
                   int64_t K) {
  if (rows != 0 && (src == nullptr || codes == nullptr || scales == nullptr))
    return set_error(SMB_ERR_INVALID, "i8 quantize: null pointer");
  if (rows < 0 || rows > 0x7FFFFFFFLL || K <= 0 || K > (1LL << 30))   // 32-bit steps through a row
    return set_error(SMB_ERR_INVALID, "i8 quantize: bad extents (rows=%lld K=%lld)", static_cast<long long>(rows),
                     static_cast<long long>(K));
  if (ld_src < K || ld_bytes < K) return set_error(SMB_ERR_INVALID, "i8 quantize: pitch smaller than K");
  return SMB_OK;
}

}  // namespace

int quantize_i8_launch(const void* src, bool bf16, int64_t ld_src, int8_t* codes, int64_t ld_bytes, float* scales,
                       int64_t rows, int64_t K, cudaStream_t st) {
  if (rows == 0) return SMB_OK;
  int per = qi8::row_per(src, ld_src, codes, ld_bytes, K, bf16);
  // A warp a row: pairs win by throughput alone.  us by elements / by pairs: 1026 x 162 2.1 / 2.9, 1026 x 1002 2.7 /
  // 3.6, 4000 x 602 3.9 / 3.9, 16000 x 162 10.5 / 7.8, 16000 x 1002 28 / 11.4.
  if (per == 2 && K <= kWarpMaxK && rows <= 4000) per = 1;
  cudaLaunchConfig_t cfg = {};
  cfg.stream = st;
  cudaLaunchAttribute pdl;
  pdl.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &pdl;
  cfg.numAttrs = 1;
  const int k = static_cast<int>(K);
  cudaError_t e;
  if (bf16)
    e = per == 8 ? launch_quantize<true, 8>(cfg, src, ld_src, codes, ld_bytes, scales, rows, k)
        : per == 2 ? launch_quantize<true, 2>(cfg, src, ld_src, codes, ld_bytes, scales, rows, k)
                   : launch_quantize<true, 1>(cfg, src, ld_src, codes, ld_bytes, scales, rows, k);
  else
    e = per == 8 ? launch_quantize<false, 8>(cfg, src, ld_src, codes, ld_bytes, scales, rows, k)
                 : launch_quantize<false, 1>(cfg, src, ld_src, codes, ld_bytes, scales, rows, k);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error(e, "i8 quantize launch");
  return SMB_OK;
}

}  // namespace smb

using namespace smb;

extern "C" int smb_quantize_i8_device(const float* src, int64_t ld_src, int8_t* codes, int64_t ld_bytes, float* scales,
                                      int64_t rows, int64_t K, void* stream) {
  if (int rc = check_quantize(src, ld_src, codes, ld_bytes, scales, rows, K)) return rc;
  if (reinterpret_cast<uintptr_t>(src) % 4 != 0 || reinterpret_cast<uintptr_t>(scales) % 4 != 0)
    return set_error(SMB_ERR_INVALID, "i8 quantize: source and scales must be 4-byte aligned");
  return quantize_i8_launch(src, false, ld_src, codes, ld_bytes, scales, rows, K, static_cast<cudaStream_t>(stream));
}

extern "C" int smb_quantize_i8_bf16_device(const uint16_t* src, int64_t ld_src, int8_t* codes, int64_t ld_bytes,
                                           float* scales, int64_t rows, int64_t K, void* stream) {
  if (int rc = check_quantize(src, ld_src, codes, ld_bytes, scales, rows, K)) return rc;
  if (reinterpret_cast<uintptr_t>(src) % 2 != 0 || reinterpret_cast<uintptr_t>(scales) % 4 != 0)
    return set_error(SMB_ERR_INVALID, "i8 quantize: source must be 2-byte, scales 4-byte aligned");
  return quantize_i8_launch(src, true, ld_src, codes, ld_bytes, scales, rows, K, static_cast<cudaStream_t>(stream));
}

extern "C" int smb_quantize_i8_host(const float* src, int64_t ld_src, int8_t* codes, int64_t ld_bytes, float* scales,
                                    int64_t rows, int64_t K) {
  if (int rc = check_quantize(src, ld_src, codes, ld_bytes, scales, rows, K)) return rc;
  for (int64_t r = 0; r < rows; ++r) {
    const float* row = src + r * ld_src;
    uint32_t m = 0;
    for (int64_t k = 0; k < K; ++k) {
      uint32_t bits;
      memcpy(&bits, row + k, 4);
      bits &= 0x7FFFFFFFu;
      m = bits > m ? bits : m;
    }
    float amax;
    memcpy(&amax, &m, 4);
    const qi8::RowScale rs = qi8::row_scale(amax, m < 0x7F800000u);
    for (int64_t k = 0; k < K; ++k)
      codes[r * ld_bytes + k] = rs.bad ? 0 : static_cast<int8_t>(std::nearbyintf(row[k] * rs.inv));
    scales[r] = rs.bad ? NAN : rs.scale;
  }
  return SMB_OK;
}
