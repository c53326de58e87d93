// How the span attention's launches are cut, as arithmetic on plain integers (no HIP types: tested on any host).
//
// By estimates (us) from measurements at 256 compute units. A round of a 16-row block (a tile of 64 keys per wave) takes
// 1.2 / 1.25 / 1.85 for rows of 32 / 64 / 128 values with at most one block per unit, of four or eight waves, and
// 1.6 / 2.4 / 4.1 with two of four; a tile of a wide block (32 keys) 1.15 / 1.15 / 1.2 and 1.5 / 1.7 / 2.3. Blocks start
// and end in 5 (eight waves 5.8, wide 6), a join launch takes 3.5, records are written and read at 3 TB/s, a piece of a
// 16-row block costs 0.5 more, and a unit takes its keys at 20 GB/s.
#pragma once

#include "span_geom.h"

#include <algorithm>

namespace nd {

constexpr int kSpanRows = 16;   // query rows of a block
constexpr int kWideRows = 128;  // of a wide block, in groups of 32

struct SpanRate {
    int waves;               // of a block
    int tiles;               // of a round
    double start, one, two;  // us a block, and a round with one block per compute unit and with two (0: never two)
};
// A launch: pieces of `per` tiles each, and the kernel (span.h: SpanArgs).
struct SpanCut {
    double us = 0;
    int splits = 1, per = 1, waves = 4;
    int groups = 0;     // of the wide kernel
    bool wide = false;
};

// The cheapest cut of blocks of `tiles` tiles and `bytes` each, `blocks` of them without pieces.
inline void best_cut(SpanCut &best, int cus, int64_t blocks, int tiles, double bytes, const SpanRate &r, double record,
                     double join) {
    const int room = r.two > 0 ? 2 * cus : cus;
    const int rounds = (tiles + r.tiles - 1) / r.tiles;
    const int most = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(rounds, room / blocks)));
    for (int s = 1;; s = std::min(most, s < 4 ? s + 1 : s + s / 3)) {
        const int64_t n = s * blocks;
        const int per = (rounds + s - 1) / s;
        const bool one = n <= cus;
        if (!one && r.two == 0) return;
        const double flights = one ? 1 : double((n + room - 1) / room);
        const double stream = blocks * bytes / (double(std::min<int64_t>(n, cus)) * 2e4);
        const double us = std::max(stream, flights * (r.start + per * (one ? r.one : r.two))) + (s > 1 ? join : 0) + s * record;
        if (best.us == 0 || us < best.us) {
            best = SpanCut();
            best.us = us;
            best.splits = (rounds + per - 1) / per;
            best.per = per * r.tiles;
            best.waves = r.waves;
        }
        if (s >= most) return;
    }
}

// `rows` query rows of each of `pairs` (unit, kv head)s. keys: at most so many per row tile of 16 (wide: of 128) rows, in
// `runs` runs; joined: a join follows in any case.
inline SpanCut cut_span(int cus, int head_dim, int64_t rows, int64_t pairs, int keys, int wide_keys, int runs, bool joined,
                        bool may_wide) {
    static const SpanRate kFour[3] = {{4, 4, 5, 1.2, 1.6}, {4, 4, 5, 1.25, 2.4}, {4, 4, 5, 1.85, 4.1}};
    static const SpanRate kEight[3] = {{8, 8, 5.8, 1.2, 0}, {8, 8, 5.8, 1.25, 0}, {8, 8, 5.8, 1.85, 0}};
    static const SpanRate kWide[3] = {{4, 1, 6, 1.15, 1.5}, {4, 1, 6, 1.15, 1.7}, {4, 1, 6, 1.2, 2.3}};
    const int h = head_dim == 32 ? 0 : head_dim == 64 ? 1 : 2;
    const double record = double(rows) * pairs * head_dim * 8 / 3e6, join = joined ? 0 : 3.5;
    const int64_t blocks = (rows + kSpanRows - 1) / kSpanRows * pairs;
    const int tiles = std::max(1, span_tiles(keys) + runs - 1);
    const double row = 2.0 * (head_dim + 4);
    SpanCut c;
    best_cut(c, cus, blocks, tiles, keys * row, kFour[h], record + 0.5, join);
    best_cut(c, cus, blocks, tiles, keys * row, kEight[h], record + 0.5, join);
    if (may_wide && rows > kSpanRows) {
        const int64_t row_blocks = (rows + kWideRows - 1) / kWideRows;
        SpanCut w;
        best_cut(w, cus, row_blocks * pairs, std::max(1, wide_tiles(wide_keys) + runs - 1), wide_keys * row, kWide[h], record,
                 join);
        if (w.us < c.us) {
            c = w;
            c.wide = true;
            c.groups = static_cast<int>(((rows + 31) / 32 + row_blocks - 1) / row_blocks);
        }
    }
    return c;
}

// Windows of `count` tokens a sequence; the ring form of the wide kernel has all of a block's groups.
inline SpanCut cut_window(int cus, int head_dim, int capacity, int seqs, int kvheads, int heads, int count, int sinks,
                          int window) {
    const int group = heads / kvheads;
    auto keys = [&](int rows) {  // of a block: its tokens' windows
        const int64_t tokens = (rows + group - 1) / group + 1;
        return static_cast<int>(
            std::min<int64_t>(sinks + int64_t(window) + std::min<int64_t>(count, tokens) - 1, capacity));
    };
    SpanCut c = cut_span(cus, head_dim, int64_t(count) * group, int64_t(seqs) * kvheads, keys(kSpanRows), keys(kWideRows), 2,
                         false, true);
    if (c.wide) c.groups = kWideRows / 32;
    return c;
}

// A prefix that `seqs` sequences share; the sequences' own slots (or any decode step), one token each.
inline SpanCut cut_prefix(int cus, int head_dim, int seqs, int kvheads, int heads, int length) {
    return cut_span(cus, head_dim, int64_t(seqs) * (heads / kvheads), kvheads, length, length, 1, true, true);
}
inline SpanCut cut_own(int cus, int head_dim, int seqs, int kvheads, int heads, int length, bool joined) {
    return cut_span(cus, head_dim, heads / kvheads, int64_t(seqs) * kvheads, length, 0, 1, joined, false);
}

}  // namespace nd
