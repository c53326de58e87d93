// How the paged attention's launch is cut, as arithmetic on plain integers (no HIP types: tested on any host), by the
// estimates of span_plan.h.
#pragma once

#include "span_plan.h"

namespace nd {

// Requests of at most `small` rows (tokens times query heads per kv head) are in `row_tiles` blocks of 16 rows each, others
// in blocks of 128 (`wide_blocks` of them at most).
struct PagedCut {
    int small = 0, row_tiles = 0, wide_blocks = 0;
    SpanCut rows, wide;
};

inline PagedCut cut_paged(int cus, int head_dim, int requests, int tokens, int count, int kvheads, int group, int length,
                          int window) {
    PagedCut c;
    const int64_t rows = int64_t(count) * group;
    const int keys = window > 0 ? static_cast<int>(std::min<int64_t>(length, int64_t(window) + count - 1)) : length;
    c.small = 1 << 30;
    c.row_tiles = static_cast<int>((rows + kSpanRows - 1) / kSpanRows);
    c.rows = cut_span(cus, head_dim, rows, int64_t(requests) * kvheads, keys, keys, 2, false, false);
    return c;
}

}  // namespace nd
