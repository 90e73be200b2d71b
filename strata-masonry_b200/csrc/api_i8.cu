// C-ABI of the int8 GEMM: plans (tensor maps + tile choice), launch, status check, host-buffer form.
#include <cstdio>
#include <new>

#include "i8_common.cuh"

using namespace smb;

struct smb_i8_plan {
  I8Launch launch;
  int* status_dev;
  int device;              // current at creation: pointers, codes and status word live there
  const void* act_src;     // plans fed with bf16 activations: the rows quantised by every run
  int64_t act_ld;
  int8_t* act_codes;       // owned by the plan
  int64_t act_pitch;
  float* act_scales;       // owned by the plan
};

namespace {

constexpr unsigned kKnownFlags = SMB_FLAG_FORCE_PLAIN_STORE | SMB_FLAG_TILE_N_128 | SMB_FLAG_TILE_N_256 |
                                 SMB_FLAG_TILE_N_512 | SMB_FLAG_NO_DECODE | SMB_FLAG_EPILOGUE_SWIGLU |
                                 SMB_FLAG_WEIGHTS_STATIC | SMB_FLAG_DECODE_SINGLE;

struct I8Args {
  const void* a;
  const float* sa;
  const void* b;
  const float* sb;
  void* d;
  int M, N, K;
  int64_t lda, ldb, ldd;
  int groups;
  const int* offsets;
  unsigned flags;
};

bool aligned4(const void* p) { return reinterpret_cast<uintptr_t>(p) % 4 == 0; }

// What does not depend on where A comes from.
int check_args(const I8Args& g) {
  if (g.b == nullptr || g.sb == nullptr || g.d == nullptr) return set_error(SMB_ERR_INVALID, "i8 plan: null operand pointer");
  if (g.M <= 0 || g.N <= 0 || g.K <= 0)
    return set_error(SMB_ERR_INVALID, "i8 plan: dimensions must be positive (M=%d N=%d K=%d)", g.M, g.N, g.K);
  if (g.M > kI8MaxExtent || g.N > kI8MaxExtent)
    return set_error(SMB_ERR_UNSUPPORTED, "i8 plan: M=%d N=%d above %d", g.M, g.N, kI8MaxExtent);
  if (g.K > kI8MaxK)
    return set_error(SMB_ERR_UNSUPPORTED, "i8 plan: K=%d above %d, where an int32 sum could wrap", g.K, kI8MaxK);
  if (g.flags & ~kKnownFlags) return set_error(SMB_ERR_UNSUPPORTED, "i8 plan: flags 0x%x have no int8 form", g.flags & ~kKnownFlags);
  const bool swiglu = (g.flags & SMB_FLAG_EPILOGUE_SWIGLU) != 0;
  if (swiglu && g.N % 2 != 0)
    return set_error(SMB_ERR_INVALID, "i8 plan: the gated epilogue needs an even N (up/gate row pairs of B)");
  if (g.ldb < g.K || g.ldb % 16 != 0)
    return set_error(SMB_ERR_INVALID, "i8 plan: ldb=%lld must be >= K and a multiple of 16", static_cast<long long>(g.ldb));
  if (g.ldd < (swiglu ? g.N / 2 : g.N)) return set_error(SMB_ERR_INVALID, "i8 plan: ldd smaller than the row length");
  if (g.ldd > 0x7FFFFFFFLL || g.ldb > 0x7FFFFFFFLL)
    return set_error(SMB_ERR_UNSUPPORTED, "i8 plan: leading dimensions above 2^31 - 1 elements");
  if (reinterpret_cast<uintptr_t>(g.d) % 2 != 0) return set_error(SMB_ERR_INVALID, "i8 plan: D is not 2-byte aligned");
  if (!aligned4(g.sb)) return set_error(SMB_ERR_INVALID, "i8 plan: scales of B are not 4-byte aligned");
  if (g.groups < 1 || g.groups > kI8MaxGroups)
    return set_error(SMB_ERR_UNSUPPORTED, "i8 grouped plan: %d groups outside 1..%d", g.groups, kI8MaxGroups);
  if (static_cast<long long>(g.groups) * g.N > 0x7FFFFFFFLL)
    return set_error(SMB_ERR_UNSUPPORTED, "i8 grouped plan: groups * N too large");
  return SMB_OK;
}

int plan_create(smb_i8_plan** out, const I8Args& g, const void* act_src, int64_t act_ld) {
  if (out == nullptr) return set_error(SMB_ERR_INVALID, "i8 plan: null output handle");
  *out = nullptr;
  if (int rc = check_args(g)) return rc;
  if (act_src == nullptr) {
    if (g.a == nullptr || g.sa == nullptr) return set_error(SMB_ERR_INVALID, "i8 plan: null operand pointer");
    if (g.lda < g.K || g.lda % 16 != 0 || g.lda > 0x7FFFFFFFLL)
      return set_error(SMB_ERR_INVALID, "i8 plan: lda=%lld must be >= K and a multiple of 16", static_cast<long long>(g.lda));
    if (!aligned4(g.sa)) return set_error(SMB_ERR_INVALID, "i8 plan: scales of A are not 4-byte aligned");
  } else {
    if (act_ld < g.K) return set_error(SMB_ERR_INVALID, "i8 plan: activation pitch smaller than K");
    if (reinterpret_cast<uintptr_t>(act_src) % 2 != 0)
      return set_error(SMB_ERR_INVALID, "i8 plan: activations are not 2-byte aligned");
  }
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return set_error(SMB_ERR_CUDA, "i8 plan: no current CUDA device");

  smb_i8_plan* p = new (std::nothrow) smb_i8_plan();
  if (p == nullptr) return set_error(SMB_ERR_NOMEM, "i8 plan: out of host memory");
  p->device = device;
  p->act_src = act_src;
  p->act_ld = act_ld;
  I8Launch& L = p->launch;
  L.M = g.M;
  L.N = g.N;
  L.K = g.K;
  L.d = g.d;
  L.ldd = static_cast<int>(g.ldd);
  L.swiglu = (g.flags & SMB_FLAG_EPILOGUE_SWIGLU) != 0;
  L.sb = g.sb;
  L.groups = g.groups;
  L.offsets = g.offsets;
  L.weights_static = (g.flags & SMB_FLAG_WEIGHTS_STATIC) != 0;
  L.tma_store = g.ldd % 8 == 0 && reinterpret_cast<uintptr_t>(g.d) % 16 == 0 && !(g.flags & SMB_FLAG_FORCE_PLAIN_STORE);
  // Groups end inside a row tile: half a tile each on average.
  i8_pick_tile(g.offsets != nullptr ? g.M + g.groups * 128 : g.M, g.N, g.K, device_cluster_slots(), L.tma_store, &L.tile_n,
               &L.sub_blocks);
  if (g.flags & SMB_FLAG_TILE_N_512) { L.tile_n = 256; L.sub_blocks = 2; }
  if (g.flags & SMB_FLAG_TILE_N_256) { L.tile_n = 256; L.sub_blocks = 1; }
  if (g.flags & SMB_FLAG_TILE_N_128) { L.tile_n = 128; L.sub_blocks = 1; }
  int rc = SMB_OK;
  if (L.swiglu) {
    if (!L.tma_store)
      rc = set_error(SMB_ERR_UNSUPPORTED, "i8 plan: the gated epilogue needs a 16-byte-aligned D with ldd %% 8 == 0");
    L.tile_n = 256;
  }
  const bool tiled_only = (g.flags & (SMB_FLAG_NO_DECODE | SMB_FLAG_TILE_N_128 | SMB_FLAG_TILE_N_256 | SMB_FLAG_TILE_N_512)) != 0;
  L.decode = !tiled_only && i8_pick_decode(g.M, g.N, g.K, g.offsets != nullptr ? (g.groups < 2 ? 2 : g.groups) : 1,
                                           L.tma_store, (g.flags & SMB_FLAG_DECODE_SINGLE) != 0, &L.chunk, &L.box_rows);
  if (act_src != nullptr && i8_decode_fuses(L, act_src, act_ld)) {
    L.x = static_cast<const uint16_t*>(act_src);
    L.ldx = act_ld;
  }
  const bool own_codes = act_src != nullptr && L.x == nullptr;
  const void* a = g.a;
  int64_t lda = g.lda;
  L.sa = g.sa;
  if (rc == SMB_OK) {
    cudaError_t e = cudaMalloc(&p->status_dev, sizeof(int));
    if (e == cudaSuccess) e = cudaMemset(p->status_dev, 0, sizeof(int));
    if (own_codes) {
      p->act_pitch = (static_cast<int64_t>(g.K) + 15) / 16 * 16;
      if (e == cudaSuccess) e = cudaMalloc(&p->act_codes, static_cast<size_t>(g.M) * p->act_pitch);
      if (e == cudaSuccess) e = cudaMalloc(&p->act_scales, static_cast<size_t>(g.M) * sizeof(float));
      a = p->act_codes;
      lda = p->act_pitch;
      L.sa = p->act_scales;
    }
    if (e != cudaSuccess) rc = set_cuda_error(e, "i8 plan: allocation");
  }
  if (rc == SMB_OK && L.x == nullptr)
    rc = encode_tmap_2d(&L.tmap_a, a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, g.M, g.K, lda, L.decode ? L.box_rows : 128, 128,
                        true);
  if (rc == SMB_OK && L.offsets != nullptr && !L.decode)
    rc = encode_tmap_2d(&L.tmap_a32, a, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, g.M, g.K, lda, 32, 128, true);
  if (rc == SMB_OK)
    rc = encode_tmap_2d(&L.tmap_b, g.b, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1, static_cast<uint64_t>(g.groups) * g.N, g.K, g.ldb,
                        L.decode ? 128 : L.tile_n / 2, 128, true);
  if (rc == SMB_OK) {
    if (L.tma_store)
      rc = encode_tmap_2d(&L.tmap_d, g.d, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, g.M, L.swiglu ? g.N / 2 : g.N, g.ldd * 2, 32,
                          64, true);
    else
      L.tmap_d = L.tmap_a;   // never dereferenced by the plain-store kernel
  }
  if (rc != SMB_OK) {
    smb_i8_plan_destroy(p);
    return rc;
  }
  L.status = p->status_dev;
  *out = p;
  return SMB_OK;
}

}  // namespace

extern "C" int smb_i8_plan_create(smb_i8_plan** out, const void* a, const float* sa, const void* b, const float* sb, void* d,
                                  int M, int N, int K, int64_t lda, int64_t ldb, int64_t ldd, unsigned flags) {
  const I8Args g = {a, sa, b, sb, d, M, N, K, lda, ldb, ldd, 1, nullptr, flags};
  return plan_create(out, g, nullptr, 0);
}

extern "C" int smb_i8_plan_create_bf16_activations(smb_i8_plan** out, const void* x_bf16, int64_t ldx, const void* b,
                                                   const float* sb, void* d, int M, int N, int K, int64_t ldb, int64_t ldd,
                                                   unsigned flags) {
  if (out != nullptr) *out = nullptr;
  if (x_bf16 == nullptr) return set_error(SMB_ERR_INVALID, "i8 plan: null activations");
  const I8Args g = {nullptr, nullptr, b, sb, d, M, N, K, 0, ldb, ldd, 1, nullptr, flags};
  return plan_create(out, g, x_bf16, ldx);
}

extern "C" int smb_i8_grouped_plan_create(smb_i8_plan** out, const void* a, const float* sa, const void* b_stacked,
                                          const float* sb_stacked, void* d, int max_rows, int N, int K, int64_t lda,
                                          int64_t ldb, int64_t ldd, int groups, const int* group_offsets_dev,
                                          unsigned flags) {
  if (out != nullptr) *out = nullptr;
  if (group_offsets_dev == nullptr) return set_error(SMB_ERR_INVALID, "i8 grouped plan: null offsets");
  if (!aligned4(group_offsets_dev)) return set_error(SMB_ERR_INVALID, "i8 grouped plan: offsets are not 4-byte aligned");
  if (max_rows > kI8MaxRows)
    return set_error(SMB_ERR_UNSUPPORTED, "i8 grouped plan: max_rows=%d above %d", max_rows, kI8MaxRows);
  const I8Args g = {a, sa, b_stacked, sb_stacked, d, max_rows, N, K, lda, ldb, ldd, groups, group_offsets_dev, flags};
  return plan_create(out, g, nullptr, 0);
}

extern "C" int smb_i8_plan_tune(smb_i8_plan* plan, int group_m, int max_clusters) {
  if (plan == nullptr) return set_error(SMB_ERR_INVALID, "i8 plan: null handle");
  if (group_m < 0 || max_clusters < 0) return set_error(SMB_ERR_INVALID, "i8 plan: negative tuning value");
  plan->launch.group_m = group_m;
  plan->launch.max_clusters = max_clusters;
  return SMB_OK;
}

extern "C" int smb_i8_plan_run(smb_i8_plan* plan, void* stream) {
  if (plan == nullptr) return set_error(SMB_ERR_INVALID, "i8 plan: null handle");
  int device = -1;
  if (cudaGetDevice(&device) != cudaSuccess || device != plan->device)
    return set_error(SMB_ERR_INVALID, "i8 plan: created on device %d, run with device %d current", plan->device, device);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (plan->act_src != nullptr && plan->launch.x == nullptr) {
    const I8Launch& L = plan->launch;
    int rc = quantize_i8_launch(plan->act_src, true, plan->act_ld, plan->act_codes, plan->act_pitch, plan->act_scales, L.M,
                                L.K, st);
    if (rc != SMB_OK) return rc;
  }
  return plan->launch.decode ? i8_decode_launch(plan->launch, st) : i8_launch(plan->launch, st);
}

extern "C" int smb_i8_plan_check(smb_i8_plan* plan, void* stream) {
  if (plan == nullptr) return set_error(SMB_ERR_INVALID, "i8 plan: null handle");
  cudaError_t e = cudaStreamSynchronize(static_cast<cudaStream_t>(stream));
  if (e != cudaSuccess) return set_cuda_error(e, "i8 plan check: stream synchronize");
  int status = 0;
  e = cudaMemcpy(&status, plan->status_dev, sizeof(int), cudaMemcpyDeviceToHost);
  if (e != cudaSuccess) return set_cuda_error(e, "i8 plan check: status read");
  if (status != 0) {
    cudaMemset(plan->status_dev, 0, sizeof(int));
    return set_error(SMB_ERR_DEVICE, "i8 GEMM kernel reported status %d: %s", status, device_status_name(status));
  }
  return SMB_OK;
}

extern "C" int smb_i8_plan_describe(smb_i8_plan* plan, char* out, size_t capacity) {
  if (plan == nullptr || out == nullptr || capacity == 0) return set_error(SMB_ERR_INVALID, "i8 plan describe: null argument");
  const I8Launch& L = plan->launch;
  if (L.decode) {
    snprintf(out, capacity, "i8 decode chunk=%d%s%s%s", L.chunk, L.swiglu ? " swiglu" : "",
             L.offsets != nullptr ? " grouped" : "",
             plan->act_src == nullptr ? "" : (L.x != nullptr ? " bf16-activations fused" : " bf16-activations"));
    return SMB_OK;
  }
  snprintf(out, capacity, "i8 tile 256x%d store=%s%s%s", L.tile_n * L.sub_blocks,
           L.swiglu ? "swiglu" : (L.tma_store ? "tma" : "plain"), L.offsets != nullptr ? " grouped" : "",
           plan->act_src != nullptr ? " bf16-activations" : "");
  return SMB_OK;
}

extern "C" int smb_i8_plan_wait_probe(smb_i8_plan* plan, long long budget_cycles, void* stream) {
  if (plan == nullptr) return set_error(SMB_ERR_INVALID, "i8 plan: null handle");
  return wait_probe_launch(plan->status_dev, budget_cycles, nullptr, static_cast<cudaStream_t>(stream));
}

extern "C" int smb_i8_plan_destroy(smb_i8_plan* plan) {
  if (plan == nullptr) return SMB_OK;
  if (plan->status_dev) cudaFree(plan->status_dev);
  if (plan->act_codes) cudaFree(plan->act_codes);
  if (plan->act_scales) cudaFree(plan->act_scales);
  delete plan;
  return SMB_OK;
}

extern "C" int smb_dense_gemm_i8(const void* a, const float* sa, const void* b, const float* sb, void* d, int M, int N, int K,
                                 void* stream) {
  smb_i8_plan* plan = nullptr;
  int rc = smb_i8_plan_create(&plan, a, sa, b, sb, d, M, N, K, K, K, N, SMB_FLAG_NONE);
  if (rc != SMB_OK) return rc;
  rc = smb_i8_plan_run(plan, stream);
  if (rc == SMB_OK) rc = smb_i8_plan_check(plan, stream);
  smb_i8_plan_destroy(plan);
  return rc;
}

extern "C" int smb_dense_gemm_i8_host(const int8_t* a, const float* sa, const int8_t* b, const float* sb, uint16_t* d, int M,
                                      int N, int K) {
  if (a == nullptr || sa == nullptr || b == nullptr || sb == nullptr || d == nullptr)
    return set_error(SMB_ERR_INVALID, "i8 host GEMM: null operand pointer");
  if (M <= 0 || N <= 0 || K <= 0) return set_error(SMB_ERR_INVALID, "i8 host GEMM: bad dimensions");
  const size_t pitch = (static_cast<size_t>(K) + 15) / 16 * 16;
  const size_t ldd = (static_cast<size_t>(N) + 7) / 8 * 8;
  void *da = nullptr, *db = nullptr, *dd = nullptr;
  float *dsa = nullptr, *dsb = nullptr;
  cudaError_t e = cudaMalloc(&da, M * pitch);
  if (e == cudaSuccess) e = cudaMalloc(&db, N * pitch);
  if (e == cudaSuccess) e = cudaMalloc(&dd, M * ldd * 2);
  if (e == cudaSuccess) e = cudaMalloc(&dsa, M * sizeof(float));
  if (e == cudaSuccess) e = cudaMalloc(&dsb, N * sizeof(float));
  if (e == cudaSuccess) e = cudaMemcpy2D(da, pitch, a, K, K, M, cudaMemcpyHostToDevice);
  if (e == cudaSuccess) e = cudaMemcpy2D(db, pitch, b, K, K, N, cudaMemcpyHostToDevice);
  if (e == cudaSuccess) e = cudaMemcpy(dsa, sa, M * sizeof(float), cudaMemcpyHostToDevice);
  if (e == cudaSuccess) e = cudaMemcpy(dsb, sb, N * sizeof(float), cudaMemcpyHostToDevice);
  int rc = e == cudaSuccess ? SMB_OK : set_cuda_error(e, "i8 host GEMM: upload");
  smb_i8_plan* plan = nullptr;
  if (rc == SMB_OK) rc = smb_i8_plan_create(&plan, da, dsa, db, dsb, dd, M, N, K, pitch, pitch, ldd, SMB_FLAG_NONE);
  if (rc == SMB_OK) rc = smb_i8_plan_run(plan, nullptr);
  if (rc == SMB_OK) rc = smb_i8_plan_check(plan, nullptr);
  if (rc == SMB_OK) {
    e = cudaMemcpy2D(d, static_cast<size_t>(N) * 2, dd, ldd * 2, static_cast<size_t>(N) * 2, M, cudaMemcpyDeviceToHost);
    if (e != cudaSuccess) rc = set_cuda_error(e, "i8 host GEMM: download");
  }
  smb_i8_plan_destroy(plan);
  cudaFree(da);
  cudaFree(db);
  cudaFree(dd);
  cudaFree(dsa);
  cudaFree(dsb);
  return rc;
}
