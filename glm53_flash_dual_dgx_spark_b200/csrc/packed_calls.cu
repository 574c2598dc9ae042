// nvfp4kv_call_packed: the entries that a serving step calls, with their arguments in one block of
// memory.  A foreign call from Python converts its arguments one by one, 2 to 3 us for the 20 to 30
// of these entries, which is as long as their kernels run for a few tokens; packing them takes a
// third of it.
#include <string.h>

#include <tuple>
#include <utility>

#include "../../include/nvfp4kv_serving.h"
#include "abi_common.h"

namespace nvfp4kv {
namespace {

// Argument i as its type, or false: a pointer, a 64-bit number, a 32-bit one, a double.
template <typename T> bool take(const void* words, size_t i, T* out) {
    int64_t word;
    memcpy(&word, static_cast<const char*>(words) + 8 * i, 8);
    if constexpr (std::is_pointer_v<T>) {
        *out = reinterpret_cast<T>(static_cast<uintptr_t>(word));
    } else if constexpr (std::is_floating_point_v<T>) {
        double value;
        memcpy(&value, &word, 8);
        *out = static_cast<T>(value);
    } else {
        *out = static_cast<T>(word);
        return static_cast<int64_t>(*out) == word;
    }
    return true;
}

template <auto kEntry> struct Packed;
template <typename... A, int (*kEntry)(A...)> struct Packed<kEntry> {
    static constexpr int kNum = sizeof...(A);
    static int call(const void* words) { return call(words, std::index_sequence_for<A...>{}); }
    template <size_t... I> static int call(const void* words, std::index_sequence<I...>) {
        std::tuple<A...> args;
        size_t good = 0;      // arguments before the first that does not fit
        ((good += good == I && take(words, I, &std::get<I>(args))), ...);
        if (good < sizeof...(A)) return fail(NVFP4KV_EINVAL, "argument %d does not fit its type", static_cast<int>(good));
        return std::apply(kEntry, args);
    }
};

struct Entry {
    const char* name;
    int num;
    int (*call)(const void*);
};
#define PACKED(entry) {#entry, Packed<entry>::kNum, Packed<entry>::call}
const Entry kEntries[] = {
    PACKED(nvfp4kv_rope), PACKED(nvfp4kv_rope_axes), PACKED(nvfp4kv_append_rope_rotated), PACKED(nvfp4kv_append_rope_rotated_axes),
    PACKED(nvfp4kv_mla_prefill), PACKED(nvfp4kv_mla_prefill_window), PACKED(nvfp4kv_extend_pages), PACKED(nvfp4kv_trim_pages),
    PACKED(nvfp4kv_copy_pages), PACKED(nvfp4kv_free_pages), PACKED(nvfp4kv_fork_pages), PACKED(nvfp4kv_compact_pages)};
#undef PACKED
constexpr int kNumEntries = sizeof(kEntries) / sizeof(kEntries[0]);

}  // namespace
}  // namespace nvfp4kv

extern "C" int nvfp4kv_packed_entry(const char* name, int* entry, int* num_args) {
    using namespace nvfp4kv;
    if (!name || !entry || !num_args) return fail(NVFP4KV_EINVAL, "packed_entry: null pointer");
    for (int i = 0; i < kNumEntries; ++i) {
        if (strcmp(name, kEntries[i].name)) continue;
        *entry = i;
        *num_args = kEntries[i].num;
        return NVFP4KV_OK;
    }
    return fail(NVFP4KV_EINVAL, "packed_entry: no entry %s", name);
}

extern "C" int nvfp4kv_call_packed(int entry, int num_args, const void* args) {
    using namespace nvfp4kv;
    if (entry < 0 || entry >= kNumEntries) return fail(NVFP4KV_EINVAL, "call_packed: no entry %d", entry);
    if (num_args != kEntries[entry].num || !args)
        return fail(NVFP4KV_EINVAL, "call_packed: %s takes %d arguments, not %d", kEntries[entry].name, kEntries[entry].num, args ? num_args : 0);
    return kEntries[entry].call(args);
}
