// packed.cpp - entry points called through one block of 64-bit words (lc_call_packed), for
// bindings whose foreign calls cost by the argument. A Python call of lc_paged_decode_kv8
// takes 3.8 us like this and 9 us with 23 arguments converted one by one; a decode step's
// launches are 5 to 10 us of GPU work each.
#include <cstdint>
#include <cstring>
#include <tuple>
#include <type_traits>
#include <utility>

#include "../../../include/lucciola_attn.h"

namespace {

// A word as the parameter's type; `fits` is cleared where an int cannot hold it.
template <class T>
T from_word(const unsigned char *w, bool &fits) {
    if constexpr (std::is_floating_point_v<T>) {
        double d;
        std::memcpy(&d, w, 8);
        return (T)d;
    } else {
        uint64_t u;
        std::memcpy(&u, w, 8);
        if constexpr (std::is_pointer_v<T>) {
            return reinterpret_cast<T>((uintptr_t)u);
        } else {
            if (std::is_same_v<T, int> && (int64_t)u != (int)u) fits = false;
            return (T)u;
        }
    }
}

template <class... A, size_t... I>
int call(int (*f)(A...), const unsigned char *words, std::index_sequence<I...>) {
    bool fits = true;
    const std::tuple<A...> args{from_word<A>(words + 8 * I, fits)...};
    return fits ? std::apply(f, args) : LC_ERR_INVALID_ARGUMENT;
}

template <class... A>
int call(int (*f)(A...), const void *words, int num_words) {
    if (num_words != (int)sizeof...(A)) return LC_ERR_INVALID_ARGUMENT;
    return call(f, static_cast<const unsigned char *>(words), std::index_sequence_for<A...>());
}

}  // namespace

extern "C" int lc_call_packed(int entry, const void *words, int num_words) {
    if (!words) return LC_ERR_INVALID_ARGUMENT;
    switch (entry) {
        case LC_PACKED_QK_NORM_ROPE_APPEND_KV8:
            return call(lc_qk_norm_rope_append_kv8, words, num_words);
        case LC_PACKED_UNPACK_KV8: return call(lc_unpack_kv8, words, num_words);
        case LC_PACKED_PAGED_DECODE_KV8: return call(lc_paged_decode_kv8, words, num_words);
        case LC_PACKED_SAMPLE: return call(lc_sample, words, num_words);
        default: return LC_ERR_INVALID_ARGUMENT;
    }
}
