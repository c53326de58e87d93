// Attention over spans of the int8 cache: device argument blocks and launchers (span_kernels.hip), and eviction
// (evict_kernels.hip).
#pragma once

#include "common.h"
#include "span_check.h"
#include "span_geom.h"
#include "span_plan.h"

namespace nd {

// Rows of one layer of a cache, [seq][kvh][capacity][head_dim] codes and [seq][kvh][capacity] scales.
struct SpanCache {
    int8_t *k8, *v8;
    float *ks, *vs;
    int capacity;
};

// Query row r (token i = r / group, head g = r % group of the kv head) of unit u and kv head kh is row
// (u * count + i) * heads + kh * group + g of q and out (fp32, head_dim each). A unit is a sequence with its own cache
// rows, or (shared prefix) the whole batch, its sequences as the tokens, over one sequence's rows.
struct SpanArgs {
    SpanCache c;
    const float *q;
    float *out;
    int units, kvheads, heads, group, count;
    // Keys. ring: token i of unit u is at position positions[u] + i and attends the last `window` positions up to its
    // own and those below `sinks`. Else every row attends slots [0, n), n = lengths[u] (null: length), at most length.
    const int *positions, *lengths;
    int length, sinks, window;
    // A unit's tiles (span_geom.h) are cut into `splits` pieces of `per` tiles; piece s leaves record split0 + s of a row's
    // splits_total. Without records (one piece) the rows are finished in place.
    int splits, per, split0, splits_total;
    int waves;             // of a block of 16 rows: 4 or 8
    int groups;            // row groups of 32 of a block of the wide kernel, 1 to 4
    float *rec_o;          // nullable, [rows][splits_total][head_dim]
    float2 *rec_ml;        // [rows][splits_total]: running maximum (of scores times log2 e) and sum
    float *scores;         // nullable: [unit][kvh][group][score_stride] scores times log2 e (count 1, no ring)
    int score_stride;      // a whole number of tiles
    float scale;           // log2(e) / sqrt(head_dim)
    // launch_span, at most 16 rows a unit: the tokens' own rows (null: stored already), [units][count][kvheads][head_dim],
    // stored at their ring slots, or (no ring, count 1) in the unit's last attended slot, before they are attended
    const float *new_k, *new_v;
};

// New tokens [seqs][count][kvheads][head_dim] into ring slots: token i of sequence s at position positions[s] + i
// (negative positions are not stored).
struct SpanStoreArgs {
    SpanCache c;
    const float *k, *v;
    const int *positions;
    int seqs, count, kvheads, head_dim, sinks;
};

// record[unit][kvh][slot] += the softmax weights of the kv head's rows, and the rows' outputs from their records.
struct SpanRecordArgs {
    SpanArgs a;
    float *record;         // [units][kvheads][capacity]
};

void launch_span_store(const SpanStoreArgs &a, hipStream_t s);
// Blocks of 16 query rows; and of 32 * groups, whose keys are turned into operands once for them all.
void launch_span(const SpanArgs &a, int head_dim, hipStream_t s);
void launch_span_wide(const SpanArgs &a, int head_dim, hipStream_t s);
// A shared prefix (one unit, no ring), as either of them, and the units' own keys (at most 16 rows each) in one launch.
void launch_span_two(const SpanArgs &far, const SpanArgs &own, int head_dim, hipStream_t s);
void launch_span_wide_own(const SpanArgs &far, const SpanArgs &own, int head_dim, hipStream_t s);
// out rows from all their records
void launch_span_join(const SpanArgs &a, int head_dim, hipStream_t s);
void launch_span_record(const SpanRecordArgs &a, int head_dim, hipStream_t s);

// Eviction of one layer: sequence s with n = lengths[s] slots (clamped to [0, capacity]) keeps, per kv head, all of them
// if n <= keep, else slots [0, sinks), [n - recent, n) and the keep - sinks - recent of the others with the largest
// weights. kept[seq][kvh][keep]: old slots in order, -1 past the last.
struct EvictArgs {
    SpanCache c;
    const float *weights;  // [seqs][kvheads][capacity]
    float *new_weights;    // may be `weights`
    const int *lengths;
    int *new_lengths;      // may be `lengths`
    int *kept;             // null only for one launch
    int *counts;           // [seqs], two launches: min(n, keep)
    int seqs, kvheads, head_dim, keep, sinks, recent;
};
// whether launch_evict needs `kept` and `counts` between two launches
bool evict_takes_two(const EvictArgs &a);
void launch_evict(const EvictArgs &a, hipStream_t s);

}  // namespace nd
