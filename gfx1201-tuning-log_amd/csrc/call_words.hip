// fp8kv_call: entry points with many arguments, called with all of them in one array of 64-bit words.
//
// For bindings, which convert 35 arguments one by one otherwise (ctypes: 4.7 to 5.0 us a call with its launch, an array
// of words 3.7 to 3.9), and check here that every word fits its argument.
#include "fp8kv_common.h"
#include "fp8kv_status.h"

#include <cstring>
#include <limits>
#include <tuple>
#include <type_traits>
#include <utility>

namespace fp8kv {
namespace call_words {

template <typename T>
bool read(int64_t word, T& value)
{
    if constexpr (std::is_pointer_v<T>) {
        value = reinterpret_cast<T>(static_cast<uintptr_t>(word));
    } else if constexpr (std::is_same_v<T, float>) {
        const uint32_t bits = static_cast<uint32_t>(word);
        std::memcpy(&value, &bits, sizeof value);
    } else if constexpr (std::is_same_v<T, size_t>) {
        value = static_cast<size_t>(word);
        return word >= 0;
    } else {
        value = static_cast<T>(word);
        return word >= std::numeric_limits<T>::min() && word <= std::numeric_limits<T>::max();
    }
    return true;
}

template <typename... A, size_t... I>
int invoke(int (*entry)(A...), const int64_t* words, std::index_sequence<I...>)
{
    std::tuple<A...> a;
    return (read(words[I], std::get<I>(a)) && ...) ? entry(std::get<I>(a)...) : FP8KV_ERR_ARG;
}

template <auto Entry>
struct Words;
template <typename... A, int (*Entry)(A...)>
struct Words<Entry> {
    static constexpr int count = (int)sizeof...(A);
    static int call(const int64_t* words) { return invoke(Entry, words, std::index_sequence_for<A...>{}); }
};

struct Entry {
    const char* name;
    int count;
    int (*call)(const int64_t*);
};

#define FP8KV_ENTRY(f) {#f, Words<&f>::count, &Words<&f>::call}
constexpr Entry kEntries[] = {
    FP8KV_ENTRY(fp8kv_rope_append),           FP8KV_ENTRY(fp8kv_rope_append_bf16),
    FP8KV_ENTRY(fp8kv_rope_append_blk),       FP8KV_ENTRY(fp8kv_decode_attn_window),
    FP8KV_ENTRY(fp8kv_decode_attn_window_bf16), FP8KV_ENTRY(fp8kv_decode_attn_blk),
    FP8KV_ENTRY(fp8kv_prefill_attn_window),   FP8KV_ENTRY(fp8kv_prefill_attn_window_bf16),
    FP8KV_ENTRY(fp8kv_prefill_attn_blk)};
#undef FP8KV_ENTRY
constexpr int kNumEntries = sizeof(kEntries) / sizeof(kEntries[0]);

}  // namespace call_words
}  // namespace fp8kv

using namespace fp8kv::call_words;

extern "C" int fp8kv_call_entry(const char* name)
{
    for (int i = 0; name && i < kNumEntries; ++i)
        if (std::strcmp(kEntries[i].name, name) == 0) return i;
    return -1;
}

extern "C" int fp8kv_call(int entry, const int64_t* words, int count)
{
    if (entry < 0 || entry >= kNumEntries || !words || count != kEntries[entry].count) return FP8KV_ERR_ARG;
    return kEntries[entry].call(words);
}

extern "C" unsigned long long fp8kv_stream_capture(void* stream)
{
    if (!stream) return 0;                          // the null stream cannot be captured
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    unsigned long long id = 0;
    if (hipStreamGetCaptureInfo(reinterpret_cast<hipStream_t>(stream), &status, &id) != hipSuccess) return 0;
    return status == hipStreamCaptureStatusNone ? 0 : id + 1;
}
