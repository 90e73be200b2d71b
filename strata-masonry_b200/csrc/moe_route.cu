// Routing of tokens to experts, forward and backward.
//
// Forward, one warp per token.  With the token's logits l[e]:
//   p[e]   = softmax(l)[e] or 1 / (1 + exp(-l[e]))
//   s[e]   = p[e] + bias[e]; without a bias the logits are what is compared
//   groups = n_groups equal runs of experts, valued by their best s (or the sum of their two best);
//            the top_groups best stay open
//   chosen = the top_k best open experts, best first, ties to the lowest index
//   weight = scale * p (or scale * p / sum of the chosen p); the bias has no part in it
// An expert whose logit (or bias) is -inf or NaN is closed to the token; slots for which no expert is left get
// id -1 and weight 0, so a padding row of -inf logits goes nowhere.
//
// Scores are fp32.  Where two neighbours in the order (or the last chosen and the first left out) lie
// closer together than the fp32 error of p, the warp repeats the choice on fp64 scores, so the ids are
// those of the exact scores whatever exp rounds to.  Choices on logits need no such care.
//
// Renormalised weights are formed from exponentials relative to the largest chosen one, so tiny
// probabilities do not underflow before they are divided.
#include <cfloat>

#include "gemm_common.cuh"
#include "ptx.cuh"

namespace smb {
namespace {

constexpr int kMaxExperts = 512;
constexpr int kMaxTopK = 32;
constexpr int kMaxRouteGroups = 32;
constexpr int kWarps = 4;
constexpr unsigned kFull = 0xffffffffu;

struct RouteParams {
  const void* logits;
  int64_t ld;
  const float* bias;
  int tokens, experts, top_k, n_groups, top_groups;
  unsigned flags;
  float scale;
  int* ids;
  float* weights;
};

// Bit patterns that order like the values; 0 is below every value and stands for "closed".
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t b = __float_as_uint(v);
  return b ^ ((b >> 31) ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ unsigned long long order_key(double v) {
  const unsigned long long b = static_cast<unsigned long long>(__double_as_longlong(v));
  return b ^ ((b >> 63) ? ~0ull : 0x8000000000000000ull);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ uint32_t warp_max(uint32_t k) { return __reduce_max_sync(kFull, k); }
__device__ __forceinline__ unsigned long long warp_max(unsigned long long k) {
  const uint32_t hi = static_cast<uint32_t>(k >> 32);
  const uint32_t top = __reduce_max_sync(kFull, hi);
  const uint32_t low = __reduce_max_sync(kFull, hi == top ? static_cast<uint32_t>(k) : 0u);
  return (static_cast<unsigned long long>(top) << 32) | low;
}

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(kFull, v, d);
  return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(kFull, v, d);
  return v;
}
__device__ __forceinline__ float warp_max_float(float v) {
  return key_value(__reduce_max_sync(kFull, order_key(v)));
}

// Logits as this file uses them: closed experts are -inf, +inf is the largest finite value.
__device__ __forceinline__ float clean_logit(float l) {
  if (!(l > -INFINITY)) return -INFINITY;
  return fminf(l, FLT_MAX);
}

template <bool kBf16>
__device__ __forceinline__ float load_logit(const void* row, int e) {
  if (kBf16) return __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(row)[e]) << 16);
  return static_cast<const float*>(row)[e];
}

__device__ __forceinline__ float exp_of(float x) { return expf(x); }
__device__ __forceinline__ double exp_of(double x) { return exp(x); }

// Scores p + bias of this lane's V experts (closed ones -inf); also p's largest value over the token.
template <int V, class S>
__device__ __forceinline__ void scores(const float (&l)[V], const float (&bias)[V], bool sigmoid, float top, S (&s)[V],
                                       float& p_max) {
  S sum = 0;
  float mine = 0.0f;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const bool open = l[i] > -INFINITY;
    if (sigmoid) s[i] = open ? S(1) / (S(1) + exp_of(-S(l[i]))) : S(0);
    else s[i] = open ? exp_of(S(l[i]) - S(top)) : S(0);
    sum += s[i];
  }
  if (!sigmoid) {
    sum = warp_sum(sum);
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = sum > S(0) ? s[i] / sum : S(0);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    mine = fmaxf(mine, static_cast<float>(s[i]));
    s[i] = l[i] > -INFINITY ? s[i] + S(bias[i]) : S(-INFINITY);
  }
  p_max = warp_max_float(mine);
}

// Bit g set: group g stays open.  `close` is raised when the choice hangs on less than `tol` (fp32).
template <int V, class S>
__device__ __forceinline__ uint32_t choose_groups(const RouteParams& p, const S (&s)[V], S* buf, int lane, float p_max,
                                                  bool& close) {
#pragma unroll
  for (int i = 0; i < V; ++i)
    if (lane * V + i < p.experts) buf[lane * V + i] = s[i];
  __syncwarp();
  const int size = p.experts / p.n_groups;
  S best = S(-INFINITY), second = S(-INFINITY);
  if (lane < p.n_groups) {
    for (int i = 0; i < size; ++i) {
      const S v = buf[lane * size + i];
      if (v > best) {
        second = best;
        best = v;
      } else if (v > second) {
        second = v;
      }
    }
  }
  __syncwarp();
  if ((p.flags & SMB_ROUTE_GROUP_TOP2) && second > S(-INFINITY)) best += second;
  auto key = best > S(-INFINITY) ? order_key(best) : decltype(order_key(best))(0);
  uint32_t kept = 0;
  float prev = 0.0f;
  for (int j = 0; j <= p.top_groups; ++j) {
    const auto m = warp_max(key);
    if (m == 0) break;
    const int win = __ffs(__ballot_sync(kFull, key == m)) - 1;
    const float value = static_cast<float>(__shfl_sync(kFull, best, win));
    // Inside the kept set the order does not matter; only the border between kept and left out does.
    if (j == p.top_groups) {
      close = prev - value <= 0x1p-19f * p_max + 0x1p-21f * (fabsf(value) + fabsf(prev));
      break;
    }
    kept |= 1u << win;
    if (lane == win) key = 0;
    prev = value;
  }
  return kept;
}

// The top_k best keys, best first: lane j ends up with the id of choice j (or -1).
template <int V, class K>
__device__ __forceinline__ int choose_experts(int top_k, K (&key)[V], int lane, bool check, float p_max, bool& close) {
  int my_id = -1;
  float prev = 0.0f;
  for (int j = 0; j < top_k + (check ? 1 : 0); ++j) {
    K best = key[0];
    int at = 0;
#pragma unroll
    for (int i = 1; i < V; ++i)
      if (key[i] > best) {
        best = key[i];
        at = i;
      }
    const K m = warp_max(best);
    if (m == 0) break;
    const int win = __ffs(__ballot_sync(kFull, best == m)) - 1;   // lanes hold ascending experts
    if (check) {
      const float value = key_value(static_cast<uint32_t>(m));
      if (j > 0 && prev - value <= 0x1p-20f * p_max + 0x1p-22f * (fabsf(value) + fabsf(prev))) close = true;
      prev = value;
    }
    const int id = __shfl_sync(kFull, lane * V + at, win);
    if (lane == j && j < top_k) my_id = id;
    if (lane == win) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (i == at) key[i] = 0;
    }
  }
  return my_id;
}

template <int V, bool kBf16>
__global__ void __launch_bounds__(kWarps * 32) route_kernel(const RouteParams p) {
  __shared__ double buf_all[kWarps][kMaxExperts];
  griddep_launch_dependents();
  griddep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = blockIdx.x * kWarps + warp;
  if (t >= p.tokens) return;
  const void* row = static_cast<const char*>(p.logits) + static_cast<int64_t>(t) * p.ld * (kBf16 ? 2 : 4);
  const bool sigmoid = (p.flags & SMB_ROUTE_SIGMOID) != 0;
  const bool renorm = (p.flags & SMB_ROUTE_RENORM) != 0;
  float l[V], bias[V];
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = lane * V + i;
    l[i] = e < p.experts ? clean_logit(load_logit<kBf16>(row, e)) : -INFINITY;
    bias[i] = (p.bias != nullptr && e < p.experts) ? p.bias[e] : 0.0f;
    top = fmaxf(top, l[i]);
  }
  top = warp_max_float(top);
  const bool by_group = p.top_groups < p.n_groups;
  const bool by_score = p.bias != nullptr;

  float s[V];
  float p_max = 0.0f;
  if (by_score || by_group) scores<V, float>(l, bias, sigmoid, top, s, p_max);
  uint32_t kept = kFull;
  if (by_group) {
    bool close = false;
    kept = choose_groups<V, float>(p, s, reinterpret_cast<float*>(buf_all[warp]), lane, p_max, close);
    if (close) {
      double d[V];
      float unused;
      scores<V, double>(l, bias, sigmoid, top, d, unused);
      kept = choose_groups<V, double>(p, d, buf_all[warp], lane, p_max, close);
    }
  }
  const int size = p.experts / p.n_groups;
  auto open = [&](int i) {
    return l[i] > -INFINITY && (!by_group || ((kept >> ((lane * V + i) / size)) & 1u));
  };
  uint32_t key[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const float v = by_score ? s[i] : l[i];
    key[i] = open(i) && v > -INFINITY ? order_key(v) : 0u;   // a bias of -inf closes an expert too
  }
  bool close = false;
  int id = choose_experts<V, uint32_t>(p.top_k, key, lane, by_score, p_max, close);
  if (close) {
    double d[V];
    float unused;
    scores<V, double>(l, bias, sigmoid, top, d, unused);
    unsigned long long wide[V];
#pragma unroll
    for (int i = 0; i < V; ++i) wide[i] = open(i) && d[i] > -INFINITY ? order_key(d[i]) : 0ull;
    id = choose_experts<V, unsigned long long>(p.top_k, wide, lane, false, p_max, close);
  }

  // Weights: lane j has choice j.
  const float lj = id >= 0 ? clean_logit(load_logit<kBf16>(row, id)) : -INFINITY;
  float w = 0.0f;
  if (sigmoid) {
    const float low = fminf(lj, 0.0f);
    const float ref = renorm ? warp_max_float(low) : 0.0f;
    if (id >= 0) w = expf(low - ref) / (1.0f + expf(-fabsf(lj)));
  } else if (renorm) {
    const float ref = warp_max_float(lj);
    if (id >= 0) w = expf(lj - ref);
  } else {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) sum += l[i] > -INFINITY ? expf(l[i] - top) : 0.0f;
    sum = warp_sum(sum);
    if (id >= 0) w = expf(lj - top) / sum;
  }
  if (renorm) {
    const float sum = warp_sum(w);
    w = id >= 0 ? w / sum : 0.0f;
  }
  if (lane < p.top_k) {
    p.ids[static_cast<int64_t>(t) * p.top_k + lane] = id;
    p.weights[static_cast<int64_t>(t) * p.top_k + lane] = w * p.scale;
  }
}

// Backward for fixed ids: with c = scale, g = dL/dweights, sums over the chosen j
//   softmax:         dl[e] = p[e] (sum_{id_j = e} c g_j - sum_j c g_j p_j)
//   softmax, renorm: dl[e] = sum_{id_j = e} q_j c (g_j - sum_i g_i q_i),  q = p / sum of the chosen p
//   sigmoid:         dl[e] = sum_{id_j = e} c g_j p_j (1 - p_j)
//   sigmoid, renorm: dl[e] = sum_{id_j = e} (1 - p_j) q_j c (g_j - sum_i g_i q_i)
struct RouteGradParams {
  const void* logits;
  int64_t ld;
  const int* ids;
  const float* grad_weights;
  int tokens, experts, top_k;
  unsigned flags;
  float scale;
  void* grad_logits;
  int64_t ld_grad;
};

template <int V, bool kBf16>
__global__ void __launch_bounds__(kWarps * 32) route_grad_kernel(const RouteGradParams p) {
  griddep_launch_dependents();
  griddep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t = blockIdx.x * kWarps + warp;
  if (t >= p.tokens) return;
  const void* row = static_cast<const char*>(p.logits) + static_cast<int64_t>(t) * p.ld * (kBf16 ? 2 : 4);
  const bool sigmoid = (p.flags & SMB_ROUTE_SIGMOID) != 0;
  const bool renorm = (p.flags & SMB_ROUTE_RENORM) != 0;
  int id = lane < p.top_k ? p.ids[static_cast<int64_t>(t) * p.top_k + lane] : -1;
  if (id >= p.experts) id = -1;
  float lj = -INFINITY, g = 0.0f;
  if (id >= 0) {
    lj = clean_logit(load_logit<kBf16>(row, id));
    g = p.grad_weights[static_cast<int64_t>(t) * p.top_k + lane] * p.scale;
  }
  const bool has = lj > -INFINITY;
  // Softmax over all experts is needed only where its sum is the denominator.
  float l[V], top = -INFINITY, inv_sum = 0.0f;
  const bool dense = !sigmoid && !renorm;
  if (dense) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = lane * V + i;
      l[i] = e < p.experts ? clean_logit(load_logit<kBf16>(row, e)) : -INFINITY;
      top = fmaxf(top, l[i]);
    }
    top = warp_max_float(top);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      l[i] = l[i] > -INFINITY ? expf(l[i] - top) : 0.0f;
      sum += l[i];
    }
    sum = warp_sum(sum);
    inv_sum = sum > 0.0f ? 1.0f / sum : 0.0f;
  }
  float part = 0.0f;   // this choice's own contribution to dl[id]
  float common = 0.0f;
  if (dense) {
    const float pj = has ? expf(lj - top) * inv_sum : 0.0f;
    common = warp_sum(has ? g * pj : 0.0f);
    part = has ? g * pj : 0.0f;
  } else if (sigmoid && !renorm) {
    const float e = expf(-fabsf(lj));   // p (1 - p) = e / (1 + e)^2 on either side of zero
    part = has ? g * (e / ((1.0f + e) * (1.0f + e))) : 0.0f;
  } else {
    float q = 0.0f, rest = 1.0f;
    if (sigmoid) {
      const float low = fminf(lj, 0.0f);
      const float ref = warp_max_float(low);
      const float e = expf(-fabsf(lj));
      if (has) {
        q = expf(low - ref) / (1.0f + e);
        rest = (lj >= 0.0f ? e : 1.0f) / (1.0f + e);   // 1 - p
      }
    } else {
      const float ref = warp_max_float(lj);
      if (has) q = expf(lj - ref);
    }
    const float sum = warp_sum(q);
    q = has ? q / sum : 0.0f;
    const float mean = warp_sum(has ? g * q : 0.0f);
    part = has ? rest * q * (g - mean) : 0.0f;
  }
  float out[V];
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = dense ? -l[i] * inv_sum * common : 0.0f;
  for (int j = 0; j < p.top_k; ++j) {
    const int e = __shfl_sync(kFull, id, j);
    const float v = __shfl_sync(kFull, part, j);
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (lane * V + i == e) out[i] += v;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = lane * V + i;
    if (e >= p.experts) continue;
    if (kBf16) {
      static_cast<uint16_t*>(p.grad_logits)[static_cast<int64_t>(t) * p.ld_grad + e] =
          static_cast<uint16_t>(pack_bf16x2(__float_as_uint(out[i]), 0u) & 0xFFFFu);
    } else {
      static_cast<float*>(p.grad_logits)[static_cast<int64_t>(t) * p.ld_grad + e] = out[i];
    }
  }
}

template <class P>
int launch_tokens(void (*kernel)(const P), const P& p, cudaStream_t st, const char* what) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((p.tokens + kWarps - 1) / kWarps), 1, 1);
  cfg.blockDim = dim3(kWarps * 32, 1, 1);
  cfg.stream = st;
  cudaLaunchAttribute pdl;
  pdl.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  pdl.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &pdl;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, p);
  if (e == cudaSuccess) e = cudaGetLastError();
  if (e != cudaSuccess) return set_cuda_error(e, what);
  return SMB_OK;
}

int check_route(const void* logits, int dtype, int64_t ld, int tokens, int experts, int top_k, unsigned flags,
                unsigned known) {
  if (tokens != 0 && logits == nullptr) return set_error(SMB_ERR_INVALID, "route: null logits");
  if (dtype != SMB_DTYPE_F32 && dtype != SMB_DTYPE_BF16)
    return set_error(SMB_ERR_UNSUPPORTED, "route: dtype %d is neither fp32 nor bf16", dtype);
  if (reinterpret_cast<uintptr_t>(logits) % (dtype == SMB_DTYPE_BF16 ? 2 : 4) != 0)
    return set_error(SMB_ERR_INVALID, "route: logits are not aligned to their type");
  if (tokens < 0) return set_error(SMB_ERR_INVALID, "route: negative token count");
  if (experts < 1 || experts > kMaxExperts)
    return set_error(SMB_ERR_UNSUPPORTED, "route: %d experts outside 1..%d", experts, kMaxExperts);
  if (top_k < 1 || top_k > kMaxTopK || top_k > experts)
    return set_error(SMB_ERR_INVALID, "route: top_k=%d outside 1..min(%d, experts)", top_k, kMaxTopK);
  if (ld < experts) return set_error(SMB_ERR_INVALID, "route: pitch smaller than the number of experts");
  if (flags & ~known) return set_error(SMB_ERR_UNSUPPORTED, "route: unknown flags 0x%x", flags & ~known);
  return SMB_OK;
}

template <template <int, bool> class Launch, class P>
int by_width(bool bf16, int experts, const P& p, cudaStream_t st) {
  const int v = (experts + 31) / 32;
  if (v <= 1) return bf16 ? Launch<1, true>::go(p, st) : Launch<1, false>::go(p, st);
  if (v <= 2) return bf16 ? Launch<2, true>::go(p, st) : Launch<2, false>::go(p, st);
  if (v <= 4) return bf16 ? Launch<4, true>::go(p, st) : Launch<4, false>::go(p, st);
  if (v <= 8) return bf16 ? Launch<8, true>::go(p, st) : Launch<8, false>::go(p, st);
  return bf16 ? Launch<16, true>::go(p, st) : Launch<16, false>::go(p, st);
}

template <int V, bool kBf16>
struct LaunchRoute {
  static int go(const RouteParams& p, cudaStream_t st) { return launch_tokens(route_kernel<V, kBf16>, p, st, "route launch"); }
};
template <int V, bool kBf16>
struct LaunchRouteGrad {
  static int go(const RouteGradParams& p, cudaStream_t st) {
    return launch_tokens(route_grad_kernel<V, kBf16>, p, st, "route backward launch");
  }
};

}  // namespace
}  // namespace smb

using namespace smb;

extern "C" int smb_moe_route_device(const void* logits, int dtype, int64_t ld, const float* bias, int tokens, int experts,
                                    int top_k, int n_groups, int top_groups, unsigned flags, float scale, int32_t* ids,
                                    float* weights, void* stream) {
  if (int rc = check_route(logits, dtype, ld, tokens, experts, top_k, flags,
                           SMB_ROUTE_SIGMOID | SMB_ROUTE_RENORM | SMB_ROUTE_GROUP_TOP2))
    return rc;
  if (tokens != 0 && (ids == nullptr || weights == nullptr)) return set_error(SMB_ERR_INVALID, "route: null output");
  if (n_groups < 1 || n_groups > kMaxRouteGroups || experts % n_groups != 0)
    return set_error(SMB_ERR_INVALID, "route: %d groups must divide %d experts and be at most %d", n_groups, experts,
                     kMaxRouteGroups);
  if (top_groups < 1 || top_groups > n_groups)
    return set_error(SMB_ERR_INVALID, "route: top_groups=%d outside 1..%d", top_groups, n_groups);
  if (top_k > experts / n_groups * top_groups)
    return set_error(SMB_ERR_INVALID, "route: top_k=%d above the %d experts of the open groups", top_k,
                     experts / n_groups * top_groups);
  if (tokens == 0) return SMB_OK;
  const RouteParams p = {logits, ld, bias, tokens, experts, top_k, n_groups, top_groups, flags, scale, ids, weights};
  return by_width<LaunchRoute>(dtype == SMB_DTYPE_BF16, experts, p, static_cast<cudaStream_t>(stream));
}

extern "C" int smb_moe_route_backward_device(const void* logits, int dtype, int64_t ld, const int32_t* ids,
                                             const float* grad_weights, int tokens, int experts, int top_k, unsigned flags,
                                             float scale, void* grad_logits, int64_t ld_grad, void* stream) {
  if (int rc = check_route(logits, dtype, ld, tokens, experts, top_k, flags,
                           SMB_ROUTE_SIGMOID | SMB_ROUTE_RENORM | SMB_ROUTE_GROUP_TOP2))
    return rc;
  if (tokens != 0 && (ids == nullptr || grad_weights == nullptr || grad_logits == nullptr))
    return set_error(SMB_ERR_INVALID, "route backward: null pointer");
  if (ld_grad < experts) return set_error(SMB_ERR_INVALID, "route backward: gradient pitch smaller than the number of experts");
  if (reinterpret_cast<uintptr_t>(grad_logits) % (dtype == SMB_DTYPE_BF16 ? 2 : 4) != 0)
    return set_error(SMB_ERR_INVALID, "route backward: gradient is not aligned to its type");
  if (tokens == 0) return SMB_OK;
  const RouteGradParams p = {logits, ld, ids, grad_weights, tokens, experts, top_k, flags, scale, grad_logits, ld_grad};
  return by_width<LaunchRouteGrad>(dtype == SMB_DTYPE_BF16, experts, p, static_cast<cudaStream_t>(stream));
}
