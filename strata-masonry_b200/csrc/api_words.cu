// The stream-ordered calls around the grouped products with their arguments as 64-bit words, for bindings that
// pay for every argument they convert.  A decode step makes several of these calls, each for a kernel of two
// microseconds: from Python a call of fourteen converted arguments takes 4 us, one of a packed string 1.1.
#include <cmath>
#include <cstring>
#include <tuple>
#include <type_traits>
#include <utility>

#include "gemm_common.cuh"

using namespace smb;

namespace {

// One word to the parameter's type; false where the value does not fit.
template <class T>
bool take(int64_t w, T& out) {
  if constexpr (std::is_pointer_v<T>) {
    out = reinterpret_cast<T>(static_cast<uintptr_t>(w));
  } else if constexpr (std::is_floating_point_v<T>) {
    double v;
    memcpy(&v, &w, 8);
    out = static_cast<T>(v);
    return std::isinf(out) == std::isinf(v);
  } else {
    out = static_cast<T>(w);
    return static_cast<int64_t>(out) == w;
  }
  return true;
}

template <class... A, size_t... I>
int spread(int (*call)(A...), const int64_t* words, std::index_sequence<I...>) {
  std::tuple<A...> args;
  if (!(take(words[I], std::get<I>(args)) && ...))
    return set_error(SMB_ERR_INVALID, "call by words: an argument does not fit its type");
  return call(std::get<I>(args)...);
}

template <class... A>
int unpack(int (*call)(A...), const int64_t* words, int count) {
  if (count != static_cast<int>(sizeof...(A)))
    return set_error(SMB_ERR_INVALID, "call by words: %d words for %d arguments", count, static_cast<int>(sizeof...(A)));
  return spread(call, words, std::index_sequence_for<A...>());
}

}  // namespace

extern "C" int smb_call_words(int call, const void* words, int count) {
  constexpr int kMaxWords = 14;
  int64_t w[kMaxWords];
  if (words == nullptr || count < 0 || count > kMaxWords) return set_error(SMB_ERR_INVALID, "call by words: no words");
  memcpy(w, words, sizeof(int64_t) * count);   // of any alignment
  switch (call) {
    case SMB_CALL_QUANTIZE_I8: return unpack(smb_quantize_i8_device, w, count);
    case SMB_CALL_QUANTIZE_I8_BF16: return unpack(smb_quantize_i8_bf16_device, w, count);
    case SMB_CALL_MOE_ROUTE: return unpack(smb_moe_route_device, w, count);
    case SMB_CALL_MOE_ROUTE_BACKWARD: return unpack(smb_moe_route_backward_device, w, count);
    case SMB_CALL_MOE_DISPATCH: return unpack(smb_moe_dispatch_device, w, count);
    case SMB_CALL_MOE_GATHER_BF16: return unpack(smb_moe_gather_bf16_device, w, count);
    case SMB_CALL_MOE_GATHER_I8: return unpack(smb_moe_gather_i8_device, w, count);
    case SMB_CALL_MOE_COMBINE: return unpack(smb_moe_combine_device, w, count);
    case SMB_CALL_MOE_COMBINE_BACKWARD: return unpack(smb_moe_combine_backward_device, w, count);
    default: return set_error(SMB_ERR_UNSUPPORTED, "call by words: unknown call %d", call);
  }
}
