// The entry points whose kernels are short enough for the cost of a foreign call to show,
// with their arguments as 8-byte words of one array (no kernels here).
#include <cstring>
#include <type_traits>
#include <utility>

#include "../../include/gdn_mi355x.h"

namespace {

template <class T>
T value(const char* word) {
  if constexpr (std::is_floating_point_v<T>) {
    double d;
    std::memcpy(&d, word, 8);
    return static_cast<T>(d);
  } else {
    int64_t w;
    std::memcpy(&w, word, 8);
    if constexpr (std::is_pointer_v<T>) return reinterpret_cast<T>(static_cast<uintptr_t>(w));
    else return static_cast<T>(w);
  }
}

// Whether an integer argument holds its word.
template <class T>
bool fits(const char* word) {
  if constexpr (std::is_integral_v<T>) return static_cast<int64_t>(value<T>(word)) == value<int64_t>(word);
  else return true;
}

template <class... A, size_t... I>
int spread(int (*entry)(A...), const char* words, std::index_sequence<I...>) {
  return (fits<A>(words + 8 * I) && ...) ? entry(value<A>(words + 8 * I)...) : GDN_ERR_INVALID_ARG;
}

template <class... A>
int call(int (*entry)(A...), const char* words, int64_t count) {
  return count == sizeof...(A) ? spread(entry, words, std::index_sequence_for<A...>{}) : GDN_ERR_INVALID_ARG;
}

// gdn_gemm_fp8's arguments, the part tables' own addresses left out, then each part's
// address, stride and end.
int gemm_fp8(const char* words, int64_t count) {
  constexpr int kFixed = 20, kParts = 16, kMost = 4;  // n_parts is word 16
  if (count < kFixed) return GDN_ERR_INVALID_ARG;
  const int64_t n = value<int64_t>(words + 8 * kParts);
  if (n < 1 || n > kMost || count != kFixed + 3 * n) return GDN_ERR_INVALID_ARG;
  uint16_t* c[kMost];
  int64_t ld[kMost];
  int end[kMost];
  for (int i = 0; i < n; ++i) {
    const char* part = words + 8 * (kFixed + 3 * i);
    if (!fits<int>(part + 16)) return GDN_ERR_INVALID_ARG;
    c[i] = value<uint16_t*>(part);
    ld[i] = value<int64_t>(part + 8);
    end[i] = value<int>(part + 16);
  }
  for (int i : {1, 12, 13, 14, 15})
    if (!fits<int>(words + 8 * i)) return GDN_ERR_INVALID_ARG;
  auto p = [&](int i) { return words + 8 * i; };
  return gdn_gemm_fp8(value<const void*>(p(0)), value<int>(p(1)), value<int64_t>(p(2)), value<const float*>(p(3)),
                      value<int64_t>(p(4)), value<int64_t>(p(5)), value<const uint8_t*>(p(6)), value<int64_t>(p(7)),
                      value<const float*>(p(8)), value<int64_t>(p(9)), value<const uint16_t*>(p(10)),
                      value<int64_t>(p(11)), value<int>(p(12)), value<int>(p(13)), value<int>(p(14)), value<int>(p(15)),
                      static_cast<int>(n), c, ld, end, value<void*>(p(17)), value<int64_t>(p(18)), value<void*>(p(19)));
}

}  // namespace

extern "C" int gdn_call_words(const void* words) {
  if (!words) return GDN_ERR_INVALID_ARG;
  const char* w = static_cast<const char*>(words);
  const int64_t head = value<int64_t>(w), count = head >> 32;
  w += 8;
  switch (static_cast<uint32_t>(head)) {
    case GDN_CALL_QUANTIZE_FP8: return call(gdn_quantize_fp8, w, count);
    case GDN_CALL_GEMM_FP8: return gemm_fp8(w, count);
    case GDN_CALL_RMSNORM_GATED_FP8: return call(gdn_rmsnorm_gated_fp8, w, count);
    case GDN_CALL_CONV_TREE: return call(gdn_conv_tree, w, count);
    case GDN_CALL_RULE_TREE: return call(gdn_rule_tree, w, count);
    case GDN_CALL_RULE_TREE_LAYER: return call(gdn_rule_tree_layer, w, count);
    case GDN_CALL_COMMIT_TREE: return call(gdn_commit_tree, w, count);
    default: return GDN_ERR_INVALID_ARG;
  }
}
