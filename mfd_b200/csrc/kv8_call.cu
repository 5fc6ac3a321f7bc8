// kv8_call.cu -- the operators of the 8-bit cache with their arguments in an array of words, for callers that pay for each
// argument of a foreign call (from Python, 47 of them take 4 us; packed into one array, under 1).
#include <cstring>
#include <utility>

#include "common.cuh"

namespace {

template <class T>
T word_as(uint64_t w) {
    if constexpr (std::is_pointer_v<T>) {
        return reinterpret_cast<T>(static_cast<uintptr_t>(w));
    } else if constexpr (std::is_floating_point_v<T>) {
        double d;
        memcpy(&d, &w, sizeof d);
        return static_cast<T>(d);
    } else {
        return static_cast<T>(static_cast<int64_t>(w));
    }
}

template <class... A, size_t... I>
int unpack(int (*f)(A...), const char* words, std::index_sequence<I...>) {
    uint64_t w[sizeof...(A)];
    memcpy(w, words, sizeof w);
    return f(word_as<A>(w[I])...);
}

template <class... A>
int call(int (*f)(A...), const void* words, int64_t count) {
    if (count != (int64_t)sizeof...(A)) {
        mfd::set_error("mfd_kv8_call: %lld words where the operator takes %d", (long long)count, (int)sizeof...(A));
        return MFD_ERR_INVALID;
    }
    return unpack(f, static_cast<const char*>(words), std::index_sequence_for<A...>());
}

}  // namespace

extern "C" int mfd_kv8_call(int op, const void* words, int64_t count) {
    if (!words) {
        mfd::set_error("mfd_kv8_call: null pointer");
        return MFD_ERR_INVALID;
    }
    switch (op) {
        case MFD_KV8_APPEND: return call(mfd_kv8_append, words, count);
        case MFD_KV8_ATTENTION: return call(mfd_kv8_attention, words, count);
        case MFD_KV8_PAGE_WEIGHTS: return call(mfd_kv8_page_weights, words, count);
        case MFD_KV8_EVICT: return call(mfd_kv8_evict, words, count);
    }
    mfd::set_error("mfd_kv8_call: no operator %d", op);
    return MFD_ERR_INVALID;
}
