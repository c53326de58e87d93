// Argument rules of the span attention and eviction entry points, on plain integers: the message of the first broken
// rule, or null. (No HIP types: they are tested on any host.)
#pragma once

#include <stddef.h>
#include <stdint.h>

namespace nd {

constexpr int kSpanMaxGroup = 16;  // query heads per kv head
constexpr int kMaxGrid = 65535;    // blocks in a grid's second and third dimension (and less than 2^32 threads in the first)

// seqs, kvheads: the cache's.
inline const char *check_heads(int seqs, int kvheads, int heads) {
    if (heads <= 0 || heads % kvheads) return "attention: heads must be a multiple of kvheads";
    if (heads / kvheads > kSpanMaxGroup) return "attention: at most 16 query heads per kv head";
    if (seqs > kMaxGrid || kvheads > kMaxGrid) return "attention: at most 65535 sequences and kv heads";
    if (int64_t(seqs) * heads > (int64_t(1) << 22)) return "attention: more than 2^22 query heads in the batch";
    return nullptr;
}

inline const char *check_window(int capacity, int seqs, int kvheads, int heads, int count, int sinks, int window) {
    if (const char *e = check_heads(seqs, kvheads, heads)) return e;
    if (count < 0) return "attention: count must be >= 0";
    if (sinks < 0) return "attention: sinks must be >= 0";
    if (window < 1) return "attention: window must be >= 1";
    if (int64_t(sinks) + window + (count > 0 ? count : 1) - 1 > capacity)
        return "attention: sinks + window + count - 1 exceeds the cache capacity";
    if (int64_t(seqs) * count * heads > (int64_t(1) << 25)) return "attention: more than 2^25 query rows";
    return nullptr;
}

inline const char *check_length(int capacity, int seqs, int kvheads, int heads, int length) {
    if (const char *e = check_heads(seqs, kvheads, heads)) return e;
    if (length < 0 || length > capacity) return "attention: length must be within the cache capacity";
    return nullptr;
}

inline const char *check_prefix(int kvheads, int head_dim, int p_capacity, int p_kvheads, int p_head_dim, int p_seqs,
                                int prefix_seq, int prefix_length) {
    if (p_kvheads != kvheads || p_head_dim != head_dim) return "attention: the prefix cache has another geometry";
    if (prefix_seq < 0 || prefix_seq >= p_seqs) return "attention: prefix sequence out of range";
    if (prefix_length < 0 || prefix_length > p_capacity) return "attention: prefix length must be within its cache's capacity";
    return nullptr;
}

inline const char *check_evict(int capacity, int seqs, int kvheads, int keep, int sinks, int recent) {
    if (keep < 1 || keep > capacity) return "eviction: keep must be within the cache capacity and at least 1";
    if (sinks < 0 || recent < 0) return "eviction: sinks and recent must be >= 0";
    if (int64_t(sinks) + recent > keep) return "eviction: sinks + recent exceeds keep";
    if (seqs > kMaxGrid || kvheads > kMaxGrid) return "eviction: at most 65535 sequences and kv heads";
    return nullptr;
}

}  // namespace nd
