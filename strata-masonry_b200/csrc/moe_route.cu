// Routing of tokens to experts, forward and backward.
//
// Forward.  With a token's logits l[e]:
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
// closer together than the fp32 error of p, fp64 scores of the experts in question decide, so the ids
// are those of fp64 scores whatever fp32 makes of them.  (What fp64 cannot tell apart ties: softmax values more than
// 700 below the largest logit, sigmoid values above 37.)  Choices on bf16 logits need no such care.
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
  bool wide, bias_wide;   // rows of logits / the bias start on 16-byte boundaries
  int group_size;         // experts per group
  int group_lanes;        // a power of two of lanes hold a group each; 0: lanes take no account of groups
};

// Lane sl of a token's segment holds the experts from lane_first on, at most V and up to lane_end; lower lanes
// hold lower ones.  kSpread: groups are no whole numbers of full lanes, yet have lanes of their own.
template <int V, bool kSpread>
__device__ __forceinline__ int lane_first(const RouteParams& p, int sl) {
  if (!kSpread) return sl * V;
  const int shift = 31 - __clz(p.group_lanes);
  return (sl >> shift) * p.group_size + (sl & (p.group_lanes - 1)) * V;
}
template <bool kSpread>
__device__ __forceinline__ int lane_end(const RouteParams& p, int sl) {
  if (!kSpread) return p.experts;
  return min(p.experts, ((sl >> (31 - __clz(p.group_lanes))) + 1) * p.group_size);
}

// Bit patterns that order like the values.  Keys up to that of -inf stand for "closed".
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t b = __float_as_uint(v);
  return b ^ (static_cast<uint32_t>(static_cast<int>(b) >> 31) | 0x80000000u);
}
constexpr uint32_t kClosedKey = 0x007FFFFFu;
__device__ __forceinline__ unsigned long long order_key(double v) {
  const unsigned long long b = static_cast<unsigned long long>(__double_as_longlong(v));
  return b ^ ((b >> 63) ? ~0ull : 0x8000000000000000ull);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float(k ^ ((k >> 31) ? 0x80000000u : 0xFFFFFFFFu));
}
__device__ __forceinline__ unsigned long long warp_max(unsigned long long k) {
  const uint32_t hi = static_cast<uint32_t>(k >> 32);
  const uint32_t top = __reduce_max_sync(kFull, hi);
  const uint32_t low = __reduce_max_sync(kFull, hi == top ? static_cast<uint32_t>(k) : 0u);
  return (static_cast<unsigned long long>(top) << 32) | low;
}

template <class T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) v += __shfl_xor_sync(kFull, v, d);
  return v;
}
__device__ __forceinline__ float warp_max_float(float v) {
  return key_value(__reduce_max_sync(kFull, order_key(v)));
}

// The same over the L lanes that share a token.
template <int L>
__device__ __forceinline__ uint32_t seg_max(uint32_t v) {
  if (L == 32) return __reduce_max_sync(kFull, v);
#pragma unroll
  for (int d = L / 2; d > 0; d >>= 1) v = max(v, __shfl_xor_sync(kFull, v, d));
  return v;
}
template <int L>
__device__ __forceinline__ float seg_max_float(float v) {
  if (L == 32) return warp_max_float(v);
#pragma unroll
  for (int d = L / 2; d > 0; d >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, d));
  return v;
}
template <int L, class T>
__device__ __forceinline__ T seg_sum(T v) {
#pragma unroll
  for (int d = L / 2; d > 0; d >>= 1) v += __shfl_xor_sync(kFull, v, d);
  return v;
}
// Bit i: lane i of this lane's segment.
template <int L>
__device__ __forceinline__ unsigned seg_ballot(bool v, int lane) {
  const unsigned all = __ballot_sync(kFull, v);
  return L == 32 ? all : (all >> (lane & ~(L - 1))) & ((1u << (L & 31)) - 1u);
}

__device__ __forceinline__ float ex2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp_approx(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Logits as this file uses them: closed experts are -inf, +inf is the largest finite value, and zero has no
// sign (keys would put +0 above -0).
__device__ __forceinline__ float clean_logit(float l) { return fminf(fmaxf(l, -INFINITY), FLT_MAX) + 0.0f; }

template <bool kBf16>
__device__ __forceinline__ float load_logit(const void* row, int e) {
  if (kBf16) return __uint_as_float(static_cast<uint32_t>(static_cast<const uint16_t*>(row)[e]) << 16);
  return static_cast<const float*>(row)[e];
}

// V consecutive values from index e0 on, -inf from n on.  `wide`: the row starts on a 16-byte boundary.
template <int V, bool kBf16, bool kSpread = false>
__device__ __forceinline__ void load_run(const void* row, int e0, int n, bool wide, float (&v)[V]) {
  constexpr int kPer = kBf16 ? 8 : 4;   // values in 16 bytes
  if (kSpread) wide = wide && e0 % (V < kPer ? V : kPer) == 0;
  if (V % kPer == 0 && wide && e0 + V <= n) {
#pragma unroll
    for (int i = 0; i < V / kPer; ++i) {
      const uint4 q = reinterpret_cast<const uint4*>(static_cast<const char*>(row) + e0 * (kBf16 ? 2 : 4))[i];
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (kBf16) {
          v[i * kPer + 2 * j] = __uint_as_float(w[j] << 16);
          v[i * kPer + 2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
        } else {
          v[i * kPer + j] = __uint_as_float(w[j]);
        }
      }
    }
    return;
  }
  if (V == 4 && kBf16 && wide && e0 + V <= n) {
    const uint2 q = *reinterpret_cast<const uint2*>(static_cast<const char*>(row) + e0 * 2);
    v[0] = __uint_as_float(q.x << 16);
    v[1] = __uint_as_float(q.x & 0xFFFF0000u);
    v[2 % V] = __uint_as_float(q.y << 16);
    v[3 % V] = __uint_as_float(q.y & 0xFFFF0000u);
    return;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = e0 + i < n ? load_logit<kBf16>(row, e0 + i) : -INFINITY;
}

// Best and second best value of a set; two sets join.
template <class S>
struct Top2 {
  S best, second;
  __device__ __forceinline__ void add(S v) {
    second = fmax(second, fmin(best, v));
    best = fmax(best, v);
  }
  __device__ __forceinline__ void join(const Top2& o) {
    second = fmax(fmin(best, o.best), fmax(second, o.second));
    best = fmax(best, o.best);
  }
  // -inf: no expert of the group is open.
  __device__ __forceinline__ S value(bool top2) const {
    return top2 && second > S(-INFINITY) ? best + second : best;
  }
  // What the value is rounded by: its two scores may have opposite signs.
  __device__ __forceinline__ S size(bool top2) const {
    return top2 && second > S(-INFINITY) ? fabs(best) + fabs(second) : fabs(best);
  }
};

__device__ __forceinline__ float key_score(uint32_t k) { return k > kClosedKey ? key_value(k) : -INFINITY; }

// The whole choice on fp64 scores: for tokens with more experts closer together than fp32 can tell than
// their segment has lanes.
// `s` holds experts doubles of this warp.  Returns lane j's choice j.
template <bool kBf16>
__device__ __noinline__ int choose_in_fp64(const RouteParams& p, const void* row, double* s, int lane) {
  const bool sigmoid = (p.flags & SMB_ROUTE_SIGMOID) != 0;
  const int size = p.experts / p.n_groups;
  float top = -INFINITY;
  for (int e = lane; e < p.experts; e += 32) top = fmaxf(top, clean_logit(load_logit<kBf16>(row, e)));
  top = warp_max_float(top);
  double sum = 0.0;
#pragma unroll 4
  for (int e = lane; e < p.experts; e += 32) {
    const float l = clean_logit(load_logit<kBf16>(row, e));
    double v = 0.0;
    if (l > -INFINITY) v = sigmoid ? 1.0 / (1.0 + exp(-static_cast<double>(l))) : exp(static_cast<double>(l) - top);
    s[e] = v;
    sum += v;
  }
  sum = sigmoid ? 1.0 : warp_sum(sum);
#pragma unroll 4
  for (int e = lane; e < p.experts; e += 32) {
    const bool open = clean_logit(load_logit<kBf16>(row, e)) > -INFINITY;
    const double v = s[e] / sum + (p.bias != nullptr ? static_cast<double>(p.bias[e]) : 0.0);
    s[e] = open && v > -INFINITY ? v : -INFINITY;
  }
  __syncwarp();
  uint32_t kept = kFull;
  if (p.top_groups < p.n_groups) {
    Top2<double> best = {-INFINITY, -INFINITY};
    if (lane < p.n_groups)
      for (int i = 0; i < size; ++i) best.add(s[lane * size + i]);
    const double value = best.value((p.flags & SMB_ROUTE_GROUP_TOP2) != 0);
    unsigned long long key = value > -INFINITY ? order_key(value) : 0ull;
    kept = 0;
    for (int j = 0; j < p.top_groups; ++j) {
      const unsigned long long m = warp_max(key);
      if (m == 0) break;
      const int win = __ffs(__ballot_sync(kFull, key == m)) - 1;
      kept |= 1u << win;
      if (lane == win) key = 0;
    }
  }
  // Without a bias the logits are compared inside the kept groups.
  if (p.bias == nullptr)
    for (int e = lane; e < p.experts; e += 32) s[e] = clean_logit(load_logit<kBf16>(row, e));
  for (int e = lane; e < p.experts; e += 32)
    if (!((kept >> (e / size)) & 1u)) s[e] = -INFINITY;
  __syncwarp();
  int id = -1;
  for (int j = 0; j < p.top_k; ++j) {
    unsigned long long best = 0;
    int at = 0;
#pragma unroll 4
    for (int e = lane; e < p.experts; e += 32) {
      const unsigned long long k = s[e] > -INFINITY ? order_key(s[e]) : 0ull;
      if (k > best) {
        best = k;
        at = e;
      }
    }
    const unsigned long long m = warp_max(best);
    if (m == 0) break;
    const int e = __reduce_min_sync(kFull, best == m ? at : 0x7FFFFFFF);
    if (lane == j) id = e;
    if (lane == (e & 31)) s[e] = -INFINITY;
    __syncwarp();
  }
  return id;
}

// The open groups of the segments' tokens from fp64 scores.  The lane's V exponentials are independent of one
// another, which is what keeps this short: a token in a thousand needs it, and the last of them sets the
// kernel's end.
template <int V, int L, bool kBf16, bool kSpread>
__device__ __noinline__ uint32_t groups_in_fp64(const RouteParams& p, const void* row, bool valid, double* buf, int lane) {
  const bool sigmoid = (p.flags & SMB_ROUTE_SIGMOID) != 0;
  const int sl = lane & (L - 1);
  const int e0 = lane_first<V, kSpread>(p, sl), e_end = lane_end<kSpread>(p, sl);
  float l[V], b[V];
  load_run<V, kBf16, kSpread>(row, e0, valid ? e_end : 0, p.wide, l);
#pragma unroll
  for (int i = 0; i < V; ++i) b[i] = 0.0f;
  if (p.bias != nullptr) load_run<V, false, kSpread>(p.bias, e0, e_end, p.bias_wide, b);
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    l[i] = clean_logit(l[i]);
    top = fmaxf(top, l[i]);
  }
  top = fmaxf(seg_max_float<L>(top), -FLT_MAX);
  double s[V], sum = 0.0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const double e = exp(sigmoid ? -static_cast<double>(l[i]) : static_cast<double>(l[i]) - top);
    s[i] = sigmoid ? 1.0 / (1.0 + e) : e;
    sum += s[i];
  }
  if (!sigmoid) {
    sum = seg_sum<L>(sum);
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = sum > 0.0 ? s[i] / sum : 0.0;
  }
  Top2<double> best = {-INFINITY, -INFINITY};
#pragma unroll
  for (int i = 0; i < V; ++i) {
    s[i] += b[i];
    s[i] = l[i] > -INFINITY && s[i] > -INFINITY ? s[i] : -INFINITY;
  }
  const bool top2 = (p.flags & SMB_ROUTE_GROUP_TOP2) != 0;
  double value;
  if (p.group_lanes != 0) {
#pragma unroll
    for (int i = 0; i < V; ++i) best.add(s[i]);
    for (int d = 1; d < p.group_lanes; d <<= 1) {
      const Top2<double> o = {__shfl_xor_sync(kFull, best.best, d), __shfl_xor_sync(kFull, best.second, d)};
      best.join(o);
    }
    value = __shfl_sync(kFull, best.value(top2), sl * p.group_lanes, L);
  } else {
    buf += lane / L * (V * L);
#pragma unroll
    for (int i = 0; i < V; ++i) buf[e0 + i] = s[i];
    __syncwarp();
    if (sl < p.n_groups)
      for (int i = 0; i < p.group_size; ++i) best.add(buf[sl * p.group_size + i]);
    __syncwarp();
    value = best.value(top2);
  }
  int ahead = 0;
  for (int g = 0; g < p.n_groups; ++g) {
    const double other = __shfl_sync(kFull, value, g, L);
    ahead += other > value || (other == value && g < sl) ? 1 : 0;
  }
  return seg_ballot<L>(sl < p.n_groups && ahead < p.top_groups, lane);
}

// Lanes 0 .. n - 1 of a segment hold the ids of all experts that can be among the top_k of its token; their
// fp64 scores (logits without a bias) settle the order.  Returns lane j's choice j.
template <int L, bool kBf16>
__device__ __noinline__ int order_in_fp64(const RouteParams& p, const void* row, int id, int n, int lane) {
  const bool sigmoid = (p.flags & SMB_ROUTE_SIGMOID) != 0;
  const int sl = lane & (L - 1);
  const float l = id >= 0 ? clean_logit(load_logit<kBf16>(row, id)) : -INFINITY;
  double score = l;
  if (p.bias != nullptr) {
    double sum = 1.0, top = 0.0;
    if (!sigmoid) {
      float m = -INFINITY;
      if (n > 0)
        for (int e = sl; e < p.experts; e += L) m = fmaxf(m, clean_logit(load_logit<kBf16>(row, e)));
      top = seg_max_float<L>(m);
      sum = 0.0;
      if (n > 0) {
#pragma unroll 4
        for (int e = sl; e < p.experts; e += L) {
          const float v = clean_logit(load_logit<kBf16>(row, e));
          sum += v > -INFINITY ? exp(static_cast<double>(v) - top) : 0.0;
        }
      }
      sum = seg_sum<L>(sum);
    }
    if (id >= 0) {
      const double e = exp(sigmoid ? -score : score - top);
      score = (sigmoid ? 1.0 / (1.0 + e) : e / sum) + static_cast<double>(p.bias[id]);
    }
  }
  const int most = __reduce_max_sync(kFull, n);
  int rank = 0;
  for (int c = 0; c < most; ++c) {
    const double other = __shfl_sync(kFull, score, c, L);
    const int other_id = __shfl_sync(kFull, id, c, L);
    rank += c < n && (other > score || (other == score && other_id < id)) ? 1 : 0;
  }
  if (sl >= n) rank = L;
  int out = -1;
  for (int c = 0; c < most; ++c) {
    const int r = __shfl_sync(kFull, rank, c, L), other_id = __shfl_sync(kFull, id, c, L);
    if (r == sl) out = other_id;
  }
  return sl < p.top_k ? out : -1;
}

// Batcher's odd-even merge sort, largest first.
template <int V>
__device__ __forceinline__ void sort_down(uint32_t (&k)[V]) {
#pragma unroll
  for (int p = 1; p < V; p *= 2)
#pragma unroll
    for (int q = p; q >= 1; q /= 2)
#pragma unroll
      for (int lo = 0; lo < V; ++lo) {
        const int hi = lo + q;
        // q == p merges runs from their first elements on, smaller q the inner ones.
        const bool used = hi < V && lo / (2 * p) == hi / (2 * p) && (lo >= q % p) && ((lo - q % p) / q) % 2 == 0;
        if (used) {
          const uint32_t x = k[lo], y = k[hi];
          k[lo] = max(x, y);
          k[hi] = min(x, y);
        }
      }
}

// What bounds it: instructions, and the latency of a token.  A token of 256 experts is 1 KB to read (0.16 ns
// at the copy rate), but eight choices out of it are hundreds of warp instructions, most of them on the
// half-rate ALU pipe.  So L lanes share a token, as few as hold its experts (8 for up to 64: four tokens to
// a warp, 16 for 128, a whole warp above); every lane sorts its V scores once, with the position inside
// the lane in the low bits of the key (two instructions per compare-exchange), and a choice is then one
// maximum over the segment, one ballot and a shift of the winner's list.  The bits that the position covers
// are made good like the rounding of exp: neighbours closer than their worth are settled in fp64.
template <int V, int L, bool kBf16, bool kSpread>
__global__ void __launch_bounds__(kWarps * 32, V <= 8 ? 12 : 6) route_kernel(const RouteParams p) {
  constexpr int kTokens = 32 / L;   // per warp
  __shared__ double buf_all[kWarps][V * 32];
  griddep_launch_dependents();
  griddep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sl = lane & (L - 1);   // lane inside the segment
  const int t0 = (blockIdx.x * kWarps + warp) * kTokens;
  if (t0 >= p.tokens) return;
  const int t = t0 + lane / L;
  const bool valid = t < p.tokens;
  auto row_of = [&](int token) -> const void* {
    return static_cast<const char*>(p.logits) + static_cast<int64_t>(token) * p.ld * (kBf16 ? 2 : 4);
  };
  const void* row = row_of(t);
  const bool sigmoid = (p.flags & SMB_ROUTE_SIGMOID) != 0;
  const bool renorm = (p.flags & SMB_ROUTE_RENORM) != 0;
  const bool by_group = p.top_groups < p.n_groups;
  const bool by_score = p.bias != nullptr;
  const bool exact = kBf16 && !by_score;   // bf16 logits leave the low 16 bits of the key free
  constexpr uint32_t kPos = V <= 4 ? 3 : (V <= 8 ? 7 : 15);
  const int e0 = lane_first<V, kSpread>(p, sl), e_end = lane_end<kSpread>(p, sl);
  float l[V];
  load_run<V, kBf16, kSpread>(row, e0, valid ? e_end : 0, p.wide, l);
  float top = 0.0f;
  if (sigmoid) {
#pragma unroll
    for (int i = 0; i < V; ++i) l[i] += 0.0f;   // as clean_logit does
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) l[i] = clean_logit(l[i]);
    top = l[0];
#pragma unroll
    for (int i = 1; i < V; ++i) top = fmaxf(top, l[i]);
    top = seg_max_float<L>(top);
  }
  float denominator = 0.0f;   // of the plain softmax weights, before the logits are used up
  if (!sigmoid && !renorm) {
#pragma unroll
    for (int i = 0; i < V; ++i) denominator += l[i] > -INFINITY ? expf(l[i] - top) : 0.0f;
    denominator = seg_sum<L>(denominator);
  }

  uint32_t key[V];
  float p_max = 0.0f, slack = 0.0f;
  bool close = false;   // more experts tie than the segment has lanes: the whole choice once more in fp64
  if (by_score || by_group) {
    float s[V];
    constexpr float kLog2e = 1.4426950408889634f;
    // exp as one product and ex2.approx is off by (2 + 1.2 |argument|) u relative, u = 2^-24.
    // Sigmoid: that times (1 - p), and 1.5 u for the sum and the reciprocal; |l| p is largest at the
    // largest p, where |l| < 0.7 (number of binary places of p + 1).  Softmax: at most 2.2 u of the largest
    // p, and common factors (the sum over V values and five shuffles, its reciprocal) below 16 u.  So
    // `slack` bounds the error of the difference of two scores.
    if (sigmoid) {
#pragma unroll
      for (int i = 0; i < V; ++i) s[i] = rcp_approx(1.0f + ex2_approx(-l[i] * kLog2e));   // closed: 1 / (1 + inf) = 0
    } else {
      float sum = 0.0f;
      const float shift = fmaxf(top, -FLT_MAX);   // no open expert at all: (-inf) - (-FLT_MAX) gives 0
#pragma unroll
      for (int i = 0; i < V; ++i) {
        s[i] = ex2_approx((l[i] - shift) * kLog2e);
        sum += s[i];
      }
      sum = seg_sum<L>(sum);
      const float inv = sum > 0.0f ? rcp_approx(sum) : 0.0f;
#pragma unroll
      for (int i = 0; i < V; ++i) s[i] *= inv;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) p_max = fmaxf(p_max, s[i]);
    p_max = __uint_as_float(seg_max<L>(__float_as_uint(p_max)));   // p >= 0: bits order as they are
    const int places = 127 - static_cast<int>(__float_as_uint(p_max) >> 23);
    slack = 0x1p-23f * p_max * (sigmoid ? 6.0f + static_cast<float>(places) : 20.0f);
    if (by_score) {
      float b[V];
      load_run<V, false, kSpread>(p.bias, e0, e_end, p.bias_wide, b);
#pragma unroll
      for (int i = 0; i < V; ++i) s[i] += b[i];
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      s[i] = l[i] > -INFINITY ? fmaxf(s[i], -INFINITY) : -INFINITY;   // a bias of -inf or NaN closes an expert too
      key[i] = (order_key(by_score ? s[i] : fmaxf(l[i], -INFINITY)) & ~kPos) | (kPos - i);
    }
    sort_down<V>(key);
    if (by_group) {
      Top2<float> best = {-INFINITY, -INFINITY};
      const bool top2 = (p.flags & SMB_ROUTE_GROUP_TOP2) != 0;
      float value = -INFINITY, size = 0.0f;   // lane g of the segment: value of group g, and its scores' magnitude
      const int lanes = p.group_lanes;
      if (lanes != 0) {
        // A group has 2^n lanes of its own: join them by shuffles.  Keys of scores are sorted already.
        if (by_score) {
          best.best = key_score(key[0] & ~kPos);
          best.second = key_score(key[1] & ~kPos);
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) best.add(s[i]);
        }
        for (int d = 1; d < lanes; d <<= 1) {
          const Top2<float> o = {__shfl_xor_sync(kFull, best.best, d), __shfl_xor_sync(kFull, best.second, d)};
          best.join(o);
        }
        value = __shfl_sync(kFull, best.value(top2), sl * lanes, L);
        size = top2 && by_score ? __shfl_sync(kFull, best.size(true), sl * lanes, L) : fabsf(value);
      } else {
        // A padded copy (a word after every 32) for every token of the warp.
        constexpr int kStride = V * L + V * L / 32 + 1;
        static_assert(kTokens * kStride <= V * 64, "the copies fit the fp64 buffer");
        float* buf = reinterpret_cast<float*>(buf_all[warp]) + lane / L * kStride;
#pragma unroll
        for (int i = 0; i < V; ++i) buf[e0 + i + ((e0 + i) >> 5)] = s[i];
        __syncwarp();
        if (sl < p.n_groups)
          for (int i = 0; i < p.group_size; ++i) best.add(buf[sl * p.group_size + i + ((sl * p.group_size + i) >> 5)]);
        __syncwarp();
        value = best.value(top2);
        size = best.size(top2);
      }
      const uint32_t gkey = sl < p.n_groups ? order_key(value) : 0u;
      // A group stays open if fewer than top_groups come before it (higher value, or equal and lower index).
      int ahead = 0;
      for (int g = 0; g < p.n_groups; ++g) {
        const uint32_t other = __shfl_sync(kFull, gkey, g, L);
        ahead += other > gkey || (other == gkey && g < sl) ? 1 : 0;
      }
      const bool in = sl < p.n_groups && ahead < p.top_groups;
      uint32_t kept = seg_ballot<L>(in, lane);
      // Only the border matters: the lowest value that a kept group may have against the highest of one left out.
      // Values are sums of up to two scores, each with its rounding and hidden position bits.
      const float reach = slack + 0x1p-23f * (kPos + 3) * fminf(size, FLT_MAX);
      const float low = -seg_max_float<L>(in ? reach - value : -INFINITY);
      const float high = seg_max_float<L>(!in && sl < p.n_groups && value > -INFINITY ? value + reach : -INFINITY);
      const bool tie = high > -INFINITY && high >= low;
      if (__any_sync(kFull, tie)) kept = groups_in_fp64<V, L, kBf16, kSpread>(p, row, valid, buf_all[warp], lane);
      if (lanes != 0) {
        // A closed lane never wins, so its head alone keeps it out.
        if (!((kept >> ((sl >> (31 - __clz(lanes))) & 31)) & 1u)) key[0] = 0;
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const int g = (e0 + static_cast<int>(kPos - (key[i] & kPos))) / p.group_size;
          key[i] = ((kept >> (g & 31)) & 1u) ? key[i] : 0u;
        }
        sort_down<V>(key);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) key[i] = (order_key(fmaxf(l[i], -INFINITY)) & ~kPos) | (kPos - i);
    sort_down<V>(key);
  }

  uint2* won = reinterpret_cast<uint2*>(buf_all[warp]) + (lane & ~(L - 1));   // key and lane of the j-th best
  auto take = [&](int j, uint32_t m, bool open) {
    const int win = __ffs(seg_ballot<L>((key[0] & ~kPos) == m, lane)) - 1;   // lanes hold ascending experts
    const bool pop = open && sl == win;
    if (pop) won[j] = make_uint2(key[0], sl);
#pragma unroll
    for (int i = 0; i + 1 < V; ++i) key[i] = pop ? key[i + 1] : key[i];
    key[V - 1] = pop ? 0u : key[V - 1];
  };
  int n = 0;
  for (int j = 0; j < p.top_k; ++j) {
    const uint32_t m = seg_max<L>(key[0] & ~kPos);
    const bool open = m > kClosedKey;
    if (L == 32 && !open) break;
    take(j, m, open);
    n += open ? 1 : 0;
  }
  __syncwarp();
  uint32_t mine = sl < n ? won[sl].x : 0u;   // lane j of the segment: the j-th best
  int id = -1;
  if (!exact) {
    uint32_t border = seg_max<L>(key[0] & ~kPos);   // what the last choice won against
    const uint32_t have = mine & ~kPos;
    uint32_t next = __shfl_down_sync(kFull, have, 1, L);
    if (sl == p.top_k - 1) next = border;
    auto tied = [&](uint32_t hi, uint32_t lo) {
      const float v = key_value(hi), w = key_value(lo);
      // The rounding of p + bias, and the steps that the position bits hide.
      return by_score ? v - w <= slack + 0x1p-23f * (kPos + 2) * (fabsf(v) + fabsf(w)) : hi == lo;
    };
    const bool tie = seg_ballot<L>(sl < p.top_k && have > kClosedKey && next > kClosedKey && tied(have, next), lane) != 0;
    if (__any_sync(kFull, tie)) {
      // Everything that may belong to the top_k joins: what ties with the last choice.
      const uint32_t last = __shfl_sync(kFull, have, p.top_k - 1, L);
      while (true) {
        const bool more = tie && border > kClosedKey && tied(last, border);
        close = more && n == L;
        if (!__any_sync(kFull, more && n < L)) break;
        take(min(n, L - 1), border, more && n < L);
        n += more && n < L ? 1 : 0;
        border = seg_max<L>(key[0] & ~kPos);
      }
      __syncwarp();
      mine = sl < n ? won[sl].x : 0u;
      id = mine != 0 ? static_cast<int>(lane_first<V, kSpread>(p, won[sl].y) + kPos - (mine & kPos)) : -1;
      const int ordered = order_in_fp64<L, kBf16>(p, row, tie ? id : -1, tie ? n : 0, lane);
      if (tie) id = ordered;
      else if (sl >= p.top_k) id = -1;
      mine = 0;
    }
  }
  if (mine != 0) id = static_cast<int>(lane_first<V, kSpread>(p, won[sl].y) + kPos - (mine & kPos));
  const unsigned again = __ballot_sync(kFull, close);
  if (again != 0) {
    __syncwarp();
    for (int k = 0; k < kTokens; ++k) {
      if (!((again >> (k * L)) & 1u)) continue;
      const int chosen = choose_in_fp64<kBf16>(p, row_of(t0 + k), buf_all[warp], lane);
      const int mine_now = __shfl_sync(kFull, chosen, sl);
      if (lane / L == k) id = mine_now;
      __syncwarp();
    }
  }

  // Weights: lane j has choice j.
  const float lj = id >= 0 ? clean_logit(load_logit<kBf16>(row, id)) : -INFINITY;
  float w = 0.0f;
  if (sigmoid) {
    const float low = fminf(lj, 0.0f);
    const float ref = renorm ? seg_max_float<L>(low) : 0.0f;
    if (id >= 0) w = __fdividef(expf(low - ref), 1.0f + expf(-fabsf(lj)));
  } else if (renorm) {
    const float ref = seg_max_float<L>(lj);
    if (id >= 0) w = expf(lj - ref);
  } else {
    if (id >= 0) w = __fdividef(expf(lj - top), denominator);
  }
  if (renorm) {
    const float sum = seg_sum<L>(w);   // at least the largest choice's own 1 or 1/2
    w = id >= 0 ? __fdividef(w, sum) : 0.0f;
  }
  if (valid && sl < p.top_k) {
    p.ids[static_cast<int64_t>(t) * p.top_k + sl] = id;
    p.weights[static_cast<int64_t>(t) * p.top_k + sl] = w * p.scale;
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
  bool wide, grad_wide;   // rows of logits and gradient start on 16-byte boundaries
};

// L lanes share a token, as in the forward pass; lane j of them has choice j.
template <int V, int L, bool kBf16>
__global__ void __launch_bounds__(kWarps * 32) route_grad_kernel(const RouteGradParams p) {
  griddep_launch_dependents();
  griddep_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sl = lane & (L - 1);
  const int t0 = (blockIdx.x * kWarps + warp) * (32 / L);
  if (t0 >= p.tokens) return;
  const int t = t0 + lane / L;
  const bool valid = t < p.tokens;
  const void* row = static_cast<const char*>(p.logits) + static_cast<int64_t>(t) * p.ld * (kBf16 ? 2 : 4);
  const bool sigmoid = (p.flags & SMB_ROUTE_SIGMOID) != 0;
  const bool renorm = (p.flags & SMB_ROUTE_RENORM) != 0;
  const bool dense = !sigmoid && !renorm;   // softmax over all experts is the denominator
  const int e0 = sl * V;
  float l[V];
  if (dense) load_run<V, kBf16>(row, e0, valid ? p.experts : 0, p.wide, l);
  int id = valid && sl < p.top_k ? p.ids[static_cast<int64_t>(t) * p.top_k + sl] : -1;
  float g = valid && sl < p.top_k ? p.grad_weights[static_cast<int64_t>(t) * p.top_k + sl] * p.scale : 0.0f;
  if (id >= p.experts) id = -1;
  const float lj = id >= 0 ? clean_logit(load_logit<kBf16>(row, id)) : -INFINITY;
  const bool has = lj > -INFINITY;
  if (!has) g = 0.0f;
  float top = -INFINITY, inv_sum = 0.0f;
  if (dense) {
    float sum = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      l[i] = clean_logit(l[i]);
      top = fmaxf(top, l[i]);
    }
    top = seg_max_float<L>(top);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      l[i] = l[i] > -INFINITY ? expf(l[i] - top) : 0.0f;
      sum += l[i];
    }
    sum = seg_sum<L>(sum);
    inv_sum = sum > 0.0f ? 1.0f / sum : 0.0f;
  }
  float part = 0.0f;   // this choice's own contribution to dl[id]
  float common = 0.0f;
  if (dense) {
    part = has ? g * (expf(lj - top) * inv_sum) : 0.0f;
    common = seg_sum<L>(part) * inv_sum;
  } else if (sigmoid && !renorm) {
    const float e = expf(-fabsf(lj));   // p (1 - p) = e / (1 + e)^2 on either side of zero
    part = has ? g * (e / ((1.0f + e) * (1.0f + e))) : 0.0f;
  } else {
    float q = 0.0f, rest = 1.0f;
    if (sigmoid) {
      const float low = fminf(lj, 0.0f);
      const float ref = seg_max_float<L>(low);
      const float e = expf(-fabsf(lj));
      if (has) {
        q = expf(low - ref) / (1.0f + e);
        rest = (lj >= 0.0f ? e : 1.0f) / (1.0f + e);   // 1 - p
      }
    } else {
      const float ref = seg_max_float<L>(lj);
      if (has) q = expf(lj - ref);
    }
    const float sum = seg_sum<L>(q);
    q = has ? q / sum : 0.0f;
    const float mean = seg_sum<L>(g * q);
    part = has ? rest * q * (g - mean) : 0.0f;
  }
  float out[V];
#pragma unroll
  for (int i = 0; i < V; ++i) out[i] = dense ? -l[i] * common : 0.0f;
  for (int j = 0; j < p.top_k; ++j) {
    const int at = __shfl_sync(kFull, id, j, L) - e0;
    const float v = __shfl_sync(kFull, part, j, L);
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] += i == at ? v : 0.0f;
  }
  if (!valid) return;
  char* dst = static_cast<char*>(p.grad_logits) + static_cast<int64_t>(t) * p.ld_grad * (kBf16 ? 2 : 4);
  if (p.grad_wide && e0 + V <= p.experts) {
    if (kBf16) {
      uint32_t q[V / 2];
#pragma unroll
      for (int i = 0; i < V / 2; ++i) q[i] = pack_bf16x2(__float_as_uint(out[2 * i]), __float_as_uint(out[2 * i + 1]));
      if (V == 4) {
        *reinterpret_cast<uint2*>(dst + e0 * 2) = make_uint2(q[0], q[1]);
      } else {
#pragma unroll
        for (int i = 0; i + 3 < V / 2; i += 4)
          *reinterpret_cast<uint4*>(dst + e0 * 2 + i * 4) = make_uint4(q[i], q[i + 1], q[i + 2], q[i + 3]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; i += 4)
        *reinterpret_cast<float4*>(dst + (e0 + i) * 4) = make_float4(out[i], out[i + 1], out[i + 2], out[i + 3]);
    }
    return;
  }
#pragma unroll
  for (int i = 0; i < V; ++i) {
    if (e0 + i >= p.experts) continue;
    if (kBf16) reinterpret_cast<uint16_t*>(dst)[e0 + i] = static_cast<uint16_t>(pack_bf16x2(__float_as_uint(out[i]), 0u) & 0xFFFFu);
    else reinterpret_cast<float*>(dst)[e0 + i] = out[i];
  }
}

template <class P>
int launch_tokens(void (*kernel)(const P), const P& p, int tokens_per_warp, cudaStream_t st, const char* what) {
  const int per_cta = kWarps * tokens_per_warp;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>((static_cast<int64_t>(p.tokens) + per_cta - 1) / per_cta), 1, 1);
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

// Lanes of L with V experts each that a group gets if every group has a power of two of its own; 0: too few.
int group_lanes(int V, int L, int experts, int n_groups) {
  int lanes = 1;
  while (lanes * V < experts / n_groups) lanes *= 2;
  return lanes * n_groups <= L ? lanes : 0;
}

// Lanes per token: as few as hold the experts, the choices (and two more that tie with the last) and the
// groups.  16384 tokens of 64 experts (bf16, softmax, six choices), forward and backward: 16.6 us with a warp
// for every token, 9.5 with 8 lanes.  256 experts (sigmoid, bias, groups): 17.8 us with 32 lanes of 8, 20.0 with 16 lanes of 16.
template <template <int, int, bool> class Launch, class P>
int by_width(bool bf16, int experts, int lanes, int n_groups, const P& p, cudaStream_t st) {
  // Every group on lanes of its own if that is possible at some width (17 groups of 30 it is not).
  const bool whole = group_lanes(16, 32, experts, n_groups) != 0;
  auto fits = [&](int v, int l) {
    return experts <= v * l && lanes <= l && (n_groups == 1 || !whole || group_lanes(v, l, experts, n_groups) != 0);
  };
  if (fits(4, 8)) return bf16 ? Launch<4, 8, true>::go(p, st) : Launch<4, 8, false>::go(p, st);
  if (fits(8, 8)) return bf16 ? Launch<8, 8, true>::go(p, st) : Launch<8, 8, false>::go(p, st);
  if (fits(8, 16)) return bf16 ? Launch<8, 16, true>::go(p, st) : Launch<8, 16, false>::go(p, st);
  if (fits(8, 32)) return bf16 ? Launch<8, 32, true>::go(p, st) : Launch<8, 32, false>::go(p, st);
  return bf16 ? Launch<16, 32, true>::go(p, st) : Launch<16, 32, false>::go(p, st);
}

template <int V, int L, bool kBf16>
struct LaunchRoute {
  static int go(RouteParams p, cudaStream_t st) {
    p.group_lanes = p.top_groups < p.n_groups ? group_lanes(V, L, p.experts, p.n_groups) : 0;
    auto kernel = p.group_lanes != 0 && p.group_lanes * V != p.group_size ? route_kernel<V, L, kBf16, true>
                                                                          : route_kernel<V, L, kBf16, false>;
    return launch_tokens(kernel, p, 32 / L, st, "route launch");
  }
};
template <int V, int L, bool kBf16>
struct LaunchRouteGrad {
  static int go(const RouteGradParams& p, cudaStream_t st) {
    return launch_tokens(route_grad_kernel<V, L, kBf16>, p, 32 / L, st, "route backward launch");
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
  for (const void* q : {static_cast<const void*>(bias), static_cast<const void*>(ids), static_cast<const void*>(weights)})
    if (reinterpret_cast<uintptr_t>(q) % 4 != 0) return set_error(SMB_ERR_INVALID, "route: bias, ids and weights must be 4-byte aligned");
  if (n_groups < 1 || n_groups > kMaxRouteGroups || experts % n_groups != 0)
    return set_error(SMB_ERR_INVALID, "route: %d groups must divide %d experts and be at most %d", n_groups, experts,
                     kMaxRouteGroups);
  if (top_groups < 1 || top_groups > n_groups)
    return set_error(SMB_ERR_INVALID, "route: top_groups=%d outside 1..%d", top_groups, n_groups);
  if (top_k > experts / n_groups * top_groups)
    return set_error(SMB_ERR_INVALID, "route: top_k=%d above the %d experts of the open groups", top_k,
                     experts / n_groups * top_groups);
  if (tokens == 0) return SMB_OK;
  const int size = dtype == SMB_DTYPE_BF16 ? 2 : 4;
  const bool wide = reinterpret_cast<uintptr_t>(logits) % 16 == 0 && (ld * size) % 16 == 0;
  const RouteParams p = {logits, ld,    bias, tokens,  experts, top_k, n_groups, top_groups,
                         flags,  scale, ids,  weights, wide,    reinterpret_cast<uintptr_t>(bias) % 16 == 0,
                         experts / n_groups, 0};
  const int lanes = top_k + 2 > n_groups ? (top_k + 2 < 32 ? top_k + 2 : 32) : n_groups;
  return by_width<LaunchRoute>(dtype == SMB_DTYPE_BF16, experts, lanes, top_groups < n_groups ? n_groups : 1, p,
                               static_cast<cudaStream_t>(stream));
}

extern "C" int smb_moe_route_backward_device(const void* logits, int dtype, int64_t ld, const int32_t* ids,
                                             const float* grad_weights, int tokens, int experts, int top_k, unsigned flags,
                                             float scale, void* grad_logits, int64_t ld_grad, void* stream) {
  if (int rc = check_route(logits, dtype, ld, tokens, experts, top_k, flags,
                           SMB_ROUTE_SIGMOID | SMB_ROUTE_RENORM | SMB_ROUTE_GROUP_TOP2))
    return rc;
  if (tokens != 0 && (ids == nullptr || grad_weights == nullptr || grad_logits == nullptr))
    return set_error(SMB_ERR_INVALID, "route backward: null pointer");
  for (const void* q : {static_cast<const void*>(ids), static_cast<const void*>(grad_weights)})
    if (reinterpret_cast<uintptr_t>(q) % 4 != 0)
      return set_error(SMB_ERR_INVALID, "route backward: ids and gradients must be 4-byte aligned");
  if (ld_grad < experts) return set_error(SMB_ERR_INVALID, "route backward: gradient pitch smaller than the number of experts");
  if (reinterpret_cast<uintptr_t>(grad_logits) % (dtype == SMB_DTYPE_BF16 ? 2 : 4) != 0)
    return set_error(SMB_ERR_INVALID, "route backward: gradient is not aligned to its type");
  if (tokens == 0) return SMB_OK;
  const int size = dtype == SMB_DTYPE_BF16 ? 2 : 4;
  auto rows_at = [](const void* q, int64_t bytes, int n) { return reinterpret_cast<uintptr_t>(q) % n == 0 && bytes % n == 0; };
  const RouteGradParams p = {logits, ld, ids, grad_weights, tokens, experts, top_k, flags, scale, grad_logits, ld_grad,
                             rows_at(logits, ld * size, 16), rows_at(grad_logits, ld_grad * size, 16)};
  return by_width<LaunchRouteGrad>(dtype == SMB_DTYPE_BF16, experts, top_k, 1, p, static_cast<cudaStream_t>(stream));
}
