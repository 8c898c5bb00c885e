// Entry points called with their arguments as 64-bit words: from Python one argument is converted then instead
// of up to 28, at 0.1 to 0.3 us each (qk_norm_rope of one token: 18.4 us a call with 28 of them, 15.5 with one).
#include <string.h>

#include <type_traits>
#include <utility>

#include "common.cuh"

namespace {

template <typename T>
T from_word(const int64_t* w) {
  if constexpr (std::is_floating_point_v<T>) {
    double d;
    memcpy(&d, w, sizeof d);
    return static_cast<T>(d);
  } else if constexpr (std::is_pointer_v<T>) {
    return reinterpret_cast<T>(static_cast<uintptr_t>(*w));
  } else {
    return static_cast<T>(*w);
  }
}

template <typename R, typename... A, size_t... I>
int64_t from_words(R (*f)(A...), const int64_t* w, std::index_sequence<I...>) {
  return f(from_word<A>(w + I)...);
}
template <typename R, typename... A>
int64_t from_words(R (*f)(A...), const int64_t* w) {
  return from_words(f, w, std::index_sequence_for<A...>());
}

constexpr int kCacheWords = sizeof(modiff_kv4_cache) / 8;

// the cache, by value, before the other arguments
template <typename R, typename... A, size_t... I>
int64_t with_cache(R (*f)(const modiff_kv4_cache*, A...), const int64_t* w, std::index_sequence<I...>) {
  return f(reinterpret_cast<const modiff_kv4_cache*>(w), from_word<A>(w + kCacheWords + I)...);
}
template <typename R, typename... A>
int64_t with_cache(R (*f)(const modiff_kv4_cache*, A...), const int64_t* w) {
  return with_cache(f, w, std::index_sequence_for<A...>());
}

int attention_cache_first(const modiff_kv4_cache* cache, const void* q, int64_t q_seq, int64_t q_token, int64_t q_head,
                          const int32_t* table, const int32_t* lengths, void* out, int batch, int count, int heads,
                          int max_pages, float scale, int causal, int window, int sinks, int dtype, void* workspace,
                          void* stream) {
  return modiff_kv4_attention(q, q_seq, q_token, q_head, cache, table, lengths, out, batch, count, heads, max_pages,
                              scale, causal, window, sinks, dtype, workspace, stream);
}

}  // namespace

extern "C" int64_t modiff_packed_call(int entry, const int64_t* words) {
  if (!words || (uintptr_t)words % 8) return modiff::set_error(MODIFF_ERR_INVALID, "NULL or misaligned words");
  switch (entry) {
    case 0: return from_words(modiff_fp8_quantize, words);
    case 1: return from_words(modiff_fp8_linear, words);
    case 2: return from_words(modiff_fp8_linear_x, words);
    case 3: return from_words(modiff_qk_norm_rope, words);
    case 4: return with_cache(modiff_kv4_append, words);
    case 5: return with_cache(modiff_kv4_read, words);
    case 6: return with_cache(attention_cache_first, words);
    case 7: return with_cache(modiff_kv4_attention_bytes, words);
    default: return modiff::set_error(MODIFF_ERR_INVALID, "unknown entry %d", entry);
  }
}
