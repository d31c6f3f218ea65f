// Entry points that take their arguments as one array of 64-bit words. A binding
// like ctypes converts argument by argument, 0.12 us each: more than a launch for
// the calls of 20 to 48 arguments that a step makes per layer.
#include <cstdint>
#include <cstring>
#include <type_traits>
#include <utility>

#include "../../include/asrback_attn.h"

namespace asrback {
namespace {

template <typename T>
T argument(const int64_t* args, size_t i) {
  if constexpr (std::is_pointer_v<T>) {
    return reinterpret_cast<T>(static_cast<intptr_t>(args[i]));
  } else if constexpr (std::is_floating_point_v<T>) {
    double x;
    std::memcpy(&x, args + i, sizeof(x));
    return static_cast<T>(x);
  } else {
    return static_cast<T>(args[i]);
  }
}

template <typename... Args, size_t... I>
int apply(int (*entry)(Args...), const int64_t* args, std::index_sequence<I...>) {
  return entry(argument<Args>(args, I)...);
}

template <typename... Args>
int apply(int (*entry)(Args...), const int64_t* args) {
  return apply(entry, args, std::index_sequence_for<Args...>{});
}

}  // namespace
}  // namespace asrback

using asrback::apply;

extern "C" int asrback_draft_tree_packed(const int64_t* args) {
  return apply(asrback_draft_tree, args);
}
extern "C" int asrback_draft_tree_in_cache_packed(const int64_t* args) {
  return apply(asrback_draft_tree_in_cache, args);
}
extern "C" int asrback_tree_attention_packed(const int64_t* args) {
  return apply(asrback_tree_attention, args);
}
extern "C" int asrback_accept_tree_packed(const int64_t* args) {
  return apply(asrback_accept_tree, args);
}
extern "C" int asrback_commit_tree_packed(const int64_t* args) {
  return apply(asrback_commit_tree, args);
}
extern "C" int asrback_evict_packed(const int64_t* args) { return apply(asrback_evict, args); }
