// The paged int8 cache: device argument blocks and launchers (paged_tables.hip, heads_kernels.hip, paged_attn.hip).
#pragma once

#include "span.h"
#include "paged_check.h"
#include "paged_plan.h"

namespace nd {

// A layer of a paged cache. Page p of kv head kh is block p * kvheads + kh; a block of `page` positions holds their K codes
// [page][head_dim], V codes, K scales [page] and V scales, so that what a kernel reads of a page lies together.
struct PagePool {
    uint8_t *at;
    int pages, shift;  // page = 1 << shift positions
    int kvheads;
};
ND_BOTH uint32_t page_block_bytes(int shift, int head_dim) { return static_cast<uint32_t>(2 * head_dim + 8) << shift; }

// The free pages of a cache: stack[0 .. *top), the next one dealt last. *done: blocks of the running launch that are done.
struct PageStack {
    int *stack, *top, *done;
    int pages;
};

struct ExtendArgs {
    PageStack free;
    const int *counts;
    int *lengths, *tables, *starts, *firsts, *slots, *positions;
    int requests, tokens, width, shift;
};
struct TrimArgs {
    PageStack free;
    const int *keep;
    int *lengths, *tables;
    int requests, width, shift;
};
void launch_zero(int2 *at, size_t n, hipStream_t s);
void launch_pages_reset(const PageStack &f, hipStream_t s);
void launch_extend(const ExtendArgs &a, hipStream_t s);
void launch_trim(const TrimArgs &a, hipStream_t s);

// Rows of tokens: q (heads of them a token), k and v (kvheads each); a null input has none. q and k are normed where their
// gain is set, rotated where `half` > 0, and go to q_out and k_out where those are set; k and v into the cache's slots
// where `pool.at` is set.
struct HeadsArgs {
    const float *q, *k, *v;
    float *q_out, *k_out;
    int64_t q_stride, k_stride, v_stride, q_out_stride, k_out_stride;
    const float *q_gain, *k_gain;
    const double *freq;     // [half]: angle per position of dimensions j and j + half
    const int *positions;   // [tokens]; negative: the token is left out. Null: none is
    const int *slots;       // [tokens]; outside the cache: not stored
    PagePool pool;
    int tokens, heads, kvheads, half;
    float eps;
};
void launch_heads(const HeadsArgs &a, int head_dim, hipStream_t s);

// Attention of a ragged batch: request r (the unit) has the tokens starts[r] .. starts[r + 1] - 1 of q and out, at most
// `count` of them, the first at position positions[r]; its keys are the positions up to a token's own (the last `window` of
// them; 0: all) in the pages of tables[r][..]. Requests of at most `small` rows are in blocks of 16 rows, `row_tiles` of
// them a request; the others in blocks of 128. A request's tiles are cut into at most `splits` pieces of at least `per`
// tiles (wide_splits and wide_per: of those in blocks of 128).
struct PagedSpanArgs : SpanArgs {
    PagePool pool;
    const int *starts, *tables;
    int tokens, width;
    int small, row_tiles;
    // Not 0: the requests in blocks of 16 rows are taken by their lengths, the longest first, in rounds of so many of which
    // every other goes from the shortest up: blocks that share a compute unit, a round's and the next one's, then have
    // about as much to do as other pairs.
    int round;
    int wide_splits, wide_per;
    int wide_blocks;       // of 128 rows, an upper bound
    // Where there may be several pieces: how many records a row has, and its row of out; 0 before the call, and after the
    // join. Rows in blocks of 16, [units][kvheads][16 row_tiles], with rec_o, rec_ml and splits_total (= splits); those in
    // blocks of 128 as in q, with records of their own, wide_splits a row.
    int2 *some, *wide_some;
    float *wide_o;
    float2 *wide_ml;
};
// `waves` and the pieces by splits, per; wide: the blocks of 128 rows too
void launch_paged(const PagedSpanArgs &a, int head_dim, hipStream_t s);
// The records of `rows` rows: rec_o, rec_ml, splits_total and some of `a`.
void launch_paged_join(const PagedSpanArgs &a, int64_t rows, int head_dim, hipStream_t s);

}  // namespace nd
