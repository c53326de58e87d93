// How the paged attention's launch is cut, as arithmetic on plain integers (no HIP types: tested on any host), by
// estimates as span_plan.h's.
#pragma once

#include "span_plan.h"

namespace nd {

// Of how many rows blocks of 16 turn a request's keys over faster than blocks of 128 with few rows in them, for rows of 128,
// 64 and 32 values: 64 requests of 2000 positions and 16, 32, 48 tokens of 4 rows each 188 against 205, 193 against 201, 191
// against 179 us; 24, 48, 64 tokens 273 against 233, 281 against 207, 255 against 248. (With fewer blocks than compute units
// up to twice as many rows.)
inline int paged_small(int head_dim) { return head_dim == 32 ? 192 : head_dim == 64 ? 128 : 64; }

// Requests that are put in the order of their lengths where there are more blocks than compute units, but not so many that
// the lengths even out (each looks for its request: 500 requests of 250 to 1000 positions, 4000 blocks, 163 us as they come
// and 188 in order; 200 of 750 to 3000, 1600 blocks, 166 and 160; 500 of up to 4000 and one kv head, 500 blocks, 86 and 75)
// and these are long enough (64 of up to 100 positions 11.4 and 13.1 us).
constexpr int kRanked = 512;
inline bool by_length(int cus, int requests, int64_t blocks, int length) {
    return requests > 1 && requests <= kRanked && blocks > cus && blocks <= 8 * int64_t(cus) && length >= 1024;
}

// Requests of at most `small` rows (tokens times query heads per kv head) are in `row_tiles` blocks of 16 rows each, others
// in blocks of 128 (`wide_blocks` of them at most).
struct PagedCut {
    int small = 0, row_tiles = 0, wide_blocks = 0;
    int round = 0;  // blocks of 16 rows by length (paged.h: PagedSpanArgs)
    SpanCut rows, wide;
    // rows that have rows.splits and wide.splits records each (0: one piece)
    int64_t few_records = 0, wide_records = 0;
};

// us that one piece more costs blocks of 16 rows (one request of 60000 positions, rows of 32 values: 32, 64 and 118 pieces
// 20.2, 17.7 and 17.0 us). At span_plan.h's 0.5 requests were cut too coarsely: one of 1500, 8000 and 30000 positions, rows
// of 64, took 13.1, 14.6 and 20.9 us and takes 10.5, 11.6 and 17.4; one of 4000, rows of 128, 16.4 and 13.3; but twelve of
// 600 there 14.1 and 15.3: one price for all of them, which gives these up for the others.
constexpr double kPiece = 0.03;

inline PagedCut cut_paged_blocks(int cus, int head_dim, int requests, int tokens, int count, int kvheads, int group, int length,
                          int window) {
    PagedCut c;
    const int64_t rows = int64_t(count) * group;
    const int h = head_dim == 32 ? 0 : head_dim == 64 ? 1 : 2;
    const double row = 2.0 * (head_dim + 4);
    static const SpanRate kFour[3] = {{4, 4, 5, 1.2, 1.6}, {4, 4, 5, 1.25, 2.4}, {4, 4, 5, 1.85, 4.1}};
    static const SpanRate kEight[3] = {{8, 8, 5.8, 1.2, 0}, {8, 8, 6, 1.25, 0}, {8, 8, 8, 1.85, 0}};
    const int keys = window > 0 ? static_cast<int>(std::min<int64_t>(length, int64_t(window) + count - 1)) : length;
    // (a grid holds 2^24 blocks of 256 threads)
    const int64_t most = std::max<int64_t>(1, (int64_t(1) << 22) / (int64_t(requests) * kvheads));
    c.small = static_cast<int>(std::min<int64_t>(paged_small(head_dim), most * kSpanRows));
    if (rows <= c.small) {
        c.row_tiles = static_cast<int>((rows + kSpanRows - 1) / kSpanRows);
        const int64_t pairs = int64_t(requests) * kvheads, tiled = c.row_tiles * pairs;
        const int tiles = std::max(1, span_tiles(keys) + (window > 0));
        const double record = double(rows) * pairs * head_dim * 8 / 3e6 + kPiece;
        best_cut(c.rows, cus, tiled, tiles, keys * row, kFour[h], record, 3.5);
        best_cut(c.rows, cus, tiled, tiles, keys * row, kEight[h], record, 3.5);
        const int64_t blocks = int64_t(requests) * kvheads * c.row_tiles * c.rows.splits;
        if (by_length(cus, requests, blocks, keys)) c.round = std::max(1, cus / kvheads);
        return c;
    }
    // Beside blocks of 128, at most four blocks of 16 a request, most of which have no rows (500 decoding requests and a
    // prompt piece, rows of 64 values: eight 112 us, four 96, two 90). With two, requests of 33 to 64 rows would be in blocks
    // of 128: 20, 100 and 250 requests of 36 to 48 rows beside a piece of 600 tokens, rows of 64, 48, 79, 130 us with four
    // and 65, 125, 248 with two; of 128 73, 114, 231 and 91, 160, 310.
    c.small = std::min(c.small, 64);
    static const SpanRate kWide[3] = {{4, 1, 6, 1.1, 1.27}, {4, 1, 6, 1.25, 1.45}, {4, 1, 6, 1.57, 2.2}};
    // the tokens' whole blocks, and one that is not filled for every request that may have more than `small` rows (every
    // one where they are found without their lengths, which costs: a piece of 300 tokens, rows of 64, 4 kv heads, contexts of
    // 4096, under a bound of 1, 512, 513, 2048, 8192 requests 27, 35, 113, 406, 1866 us)
    const int64_t whole = int64_t(tokens) * group / kWideRows, filled = std::max<int64_t>(1, whole);
    c.wide_blocks = static_cast<int>(whole + (requests > kRanked ? requests
                                                                 : std::min<int64_t>(requests, int64_t(tokens) * group / (c.small + 1) + 1)));
    const double record = double(tokens) * group * kvheads * head_dim * 8 / 3e6;
    best_cut(c.wide, cus, filled * kvheads, std::max(1, wide_tiles(keys)), keys * row, kWide[h], record, 3.5);
    if (requests == 1) {  // (whatever its tokens turn out to be)
        c.small = 0;
        return c;
    }
    c.row_tiles = c.small / kSpanRows;
    best_cut(c.rows, cus, int64_t(requests) * kvheads, std::max(1, span_tiles(keys)), keys * row, kFour[h], kPiece, 3.5);
    return c;
}

inline PagedCut cut_paged(int cus, int head_dim, int requests, int tokens, int count, int kvheads, int group, int length,
                          int window) {
    PagedCut c = cut_paged_blocks(cus, head_dim, requests, tokens, count, kvheads, group, length, window);
    if (c.row_tiles && c.rows.splits > 1) c.few_records = int64_t(requests) * kvheads * c.row_tiles * kSpanRows;
    if (c.wide_blocks && c.wide.splits > 1) c.wide_records = int64_t(tokens) * kvheads * group;
    return c;
}

}  // namespace nd
