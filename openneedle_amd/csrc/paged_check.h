// Argument rules of the paged cache's entry points and of the heads' norm and rotation, on plain integers: the message of
// the first broken rule, or null. (No HIP types: they are tested on any host.)
#pragma once

#include "span_check.h"

namespace nd {

constexpr int kMaxRequests = 8192;  // of a call: the tables' kernels hold three numbers of each in LDS
constexpr int kMaxTokens = 1 << 25;

inline const char *check_pages(int layers, int pages, int page_size, int kvheads, int head_dim) {
    if (layers <= 0 || pages <= 0 || kvheads <= 0) return "paged cache: sizes must be positive";
    if (page_size < 16 || page_size > 256 || (page_size & (page_size - 1)))
        return "paged cache: page_size must be 16, 32, 64, 128 or 256";
    if (head_dim != 32 && head_dim != 64 && head_dim != 128) return "paged cache: head_dim must be 32, 64 or 128";
    if (kvheads > kMaxGrid) return "paged cache: at most 65535 kv heads";
    if (int64_t(kvheads) * page_size * (2 * head_dim + 8) >= (int64_t(1) << 31))
        return "paged cache: the kv heads' rows of a page must be below 2^31 bytes";
    if (int64_t(pages) * page_size >= (int64_t(1) << 31)) return "paged cache: pages * page_size must be below 2^31";
    if (layers > (int64_t(1) << 46) / (int64_t(pages) * kvheads * page_size * (2 * head_dim + 8)))
        return "paged cache: more than 2^46 bytes";  // (and the sizes' products would wrap later)
    return nullptr;
}

inline const char *check_requests(int requests, int width, int page_size) {
    if (requests < 0 || requests > kMaxRequests) return "paged cache: 0 to 8192 requests a call";
    if (width < 1) return "paged cache: tables need a width of at least 1";
    if (int64_t(width) * page_size > (int64_t(1) << 30)) return "paged cache: width * page_size must be at most 2^30";
    return nullptr;
}

inline const char *check_tokens(int tokens) {
    if (tokens < 0 || tokens > kMaxTokens) return "paged cache: 0 to 2^25 tokens a call";
    return nullptr;
}

// A row of `heads` heads per token, `stride` values from one token to the next, as 16-byte pieces.
inline const char *check_rows(const void *p, int stride, int heads, int head_dim) {
    if (int64_t(stride) < int64_t(heads) * head_dim) return "heads: a row's stride is smaller than its heads";
    if (stride % 4 || reinterpret_cast<uintptr_t>(p) % 16) return "heads: rows must begin at multiples of 16 bytes";
    return nullptr;
}

inline const char *check_turn(int heads, int kvheads, int head_dim, int tokens, float eps, int rotary) {
    if (head_dim != 32 && head_dim != 64 && head_dim != 128) return "heads: head_dim must be 32, 64 or 128";
    if (heads < 0 || kvheads < 0 || heads > kMaxGrid || kvheads > kMaxGrid) return "heads: 0 to 65535 heads and kv heads";
    if (tokens < 0 || tokens > kMaxTokens) return "heads: 0 to 2^25 tokens a call";
    if (!(eps >= 0.0f && eps < 1e30f)) return "heads: eps must be finite and >= 0";
    if (rotary < 0 || rotary > head_dim || rotary % 2) return "heads: rotary must be even, 0 to head_dim";
    return nullptr;
}

inline const char *check_paged_attention(int kvheads, int heads, int requests, int tokens, int count, int length, int window) {
    if (heads <= 0 || heads % kvheads) return "attention: heads must be a multiple of kvheads";
    if (heads / kvheads > kSpanMaxGroup) return "attention: at most 16 query heads per kv head";
    if (count < 0 || count > tokens) return "attention: count must be within the tokens";
    if (length < 0) return "attention: length must be >= 0";
    if (window < 0) return "attention: window must be >= 0";
    if (int64_t(requests) * heads > (int64_t(1) << 22)) return "attention: more than 2^22 query heads in the batch";
    if (int64_t(tokens) * heads > (int64_t(1) << 25)) return "attention: more than 2^25 query rows";
    return nullptr;
}

}  // namespace nd
