// C ABI of attention over spans of the int8 KV cache and of its eviction (additive exports): windows with pinned first
// positions, a shared prefix, decode attention that records the weights, and the cut by that record. The reference has
// one sequence at a time, its window as a slot list (needle2/csrc/engine.cpp:898-911), and no eviction.
#include "kv.h"
#include "span.h"

#include <algorithm>
#include <cmath>

namespace nd {

static void check_rule(const char *broken) {
    if (broken) throw Error(broken);
}

// The handle, which must be used where its memory is.
static KvHandle &kv_here(void *h) {
    KvHandle &kv = *kv_of(h);
    int device = 0;
    ND_HIP(hipGetDevice(&device));
    ND_CHECK(device == kv.device, "KV cache: made on another device than the current one");
    return kv;
}

static SpanCache layer_of(KvHandle &kv, int layer, int seq = 0) {
    const size_t row = (size_t(layer) * kv.seqs + seq) * kv.kvheads * kv.capacity;
    return SpanCache{kv.k8.p + row * kv.head_dim, kv.v8.p + row * kv.head_dim, kv.ks.p + row, kv.vs.p + row, kv.capacity};
}

static SpanArgs span_args(KvHandle &kv, const SpanCache &c, const float *d_q, float *d_out, int units, int heads, int count) {
    SpanArgs a{};
    a.c = c;
    a.q = d_q;
    a.out = d_out;
    a.units = units;
    a.kvheads = kv.kvheads;
    a.heads = heads;
    a.group = heads / kv.kvheads;
    a.count = count;
    a.scale = float(1.4426950408889634 / std::sqrt(double(kv.head_dim)));
    return a;
}

// How a launch is cut: `waves` 0 for the 16-row kernel, else the wide kernel's row groups of 32 per block.
struct SpanPlan {
    int waves = 0;
};

// Pieces of a unit's keys (at most `keys` in `runs` runs): two blocks per compute unit, of whole rounds of a block.
static SpanPlan cut(SpanArgs &a, int keys, int runs) {
    const int64_t rows = int64_t(a.count) * a.group;
    SpanPlan p;
    if (rows > kSpanRows) {
        double best = 0;
        for (int w = 4; w >= 1; --w) {
            const double cost = double((rows + 32 * w - 1) / (32 * w)) * (w + 0.6);
            if (!p.waves || cost < best) {
                best = cost;
                p.waves = w;
            }
        }
    }
    const int block_rows = p.waves ? 32 * p.waves : kSpanRows;
    const int64_t blocks = std::max<int64_t>(1, (rows + block_rows - 1) / block_rows * a.kvheads * a.units);
    const int round = p.waves ? 1 : 4;  // tiles of a block's round
    const int tiles = (p.waves ? wide_tiles(keys) : span_tiles(keys)) + runs - 1;
    const int rounds = std::max(1, (tiles + round - 1) / round);
    const int target = 2 * device_cus();
    const int want = static_cast<int>(std::min<int64_t>(rounds, std::max<int64_t>(1, target / blocks)));
    const int per_rounds = (rounds + want - 1) / want;
    a.per = round * per_rounds;
    a.splits = (rounds + per_rounds - 1) / per_rounds;
    return p;
}

static void launch(const SpanArgs &a, const SpanPlan &p, int head_dim, hipStream_t s) {
    if (p.waves) launch_span_wide(a, head_dim, p.waves, s);
    else launch_span(a, head_dim, s);
}

// Room for the records of `rows` rows.
static void reserve_records(KvHandle &kv, SpanArgs &a, int64_t rows) {
    const size_t n = size_t(rows) * a.splits_total;
    a.rec_o = kv.records.reserve(n * (kv.head_dim + 2));
    a.rec_ml = reinterpret_cast<float2 *>(a.rec_o + n * kv.head_dim);
}

static void check_new(const float *d_new_k, const float *d_new_v) {
    ND_CHECK(!d_new_k == !d_new_v, "attention: new K and V come together");
}

}  // namespace nd

using namespace nd;

extern "C" {

int needle2_gpu_attention_window(void *h, int layer, const float *d_q, float *d_out, int heads, int count,
                                 const int *d_positions, int sinks, int window, const float *d_new_k, const float *d_new_v,
                                 void *stream) {
    return guarded([&] {
        ND_CHECK(h != nullptr, "null KV cache handle");
        KvHandle &kv = kv_here(h);
        check_layer(kv, layer);
        check_rule(check_window(kv.capacity, kv.seqs, kv.kvheads, heads, count, sinks, window));
        if (count == 0) return;
        ND_CHECK(d_q && d_out && d_positions, "attention: null q, out or positions");
        check_new(d_new_k, d_new_v);
        hipStream_t s = static_cast<hipStream_t>(stream);
        SpanArgs a = span_args(kv, layer_of(kv, layer), d_q, d_out, kv.seqs, heads, count);
        a.positions = d_positions;
        a.sinks = sinks;
        a.window = window;
        // keys of a block: its tokens' windows
        const int most = int64_t(count) * a.group <= kSpanRows ? kSpanRows : 128;
        const int tokens = std::min(count, (most + a.group - 1) / a.group + 1);
        const SpanPlan plan = cut(a, sinks + window + tokens - 1, 2);
        a.splits_total = a.splits;
        if (a.splits_total > 1) reserve_records(kv, a, int64_t(kv.seqs) * count * heads);
        if (d_new_k && count == 1) {
            a.new_k = d_new_k;
            a.new_v = d_new_v;
        } else if (d_new_k) {
            SpanStoreArgs st{};
            st.c = a.c;
            st.k = d_new_k;
            st.v = d_new_v;
            st.positions = d_positions;
            st.seqs = kv.seqs;
            st.count = count;
            st.kvheads = kv.kvheads;
            st.head_dim = kv.head_dim;
            st.sinks = sinks;
            launch_span_store(st, s);
        }
        launch(a, plan, kv.head_dim, s);
        if (a.splits_total > 1) launch_span_join(a, kv.head_dim, s);
    });
}

int needle2_gpu_attention_shared(void *h, int layer, void *prefix, int prefix_seq, int prefix_length, const float *d_q,
                                 float *d_out, int heads, int length, const int *d_lengths, const float *d_new_k,
                                 const float *d_new_v, void *stream) {
    return guarded([&] {
        ND_CHECK(h != nullptr && prefix != nullptr, "null KV cache handle");
        ND_CHECK(h != prefix, "attention: the prefix must be in a cache of its own");
        KvHandle &kv = kv_here(h), &pre = kv_here(prefix);
        check_layer(kv, layer);
        check_layer(pre, layer);
        check_rule(check_length(kv.capacity, kv.seqs, kv.kvheads, heads, length));
        check_rule(check_prefix(kv.kvheads, kv.head_dim, pre.capacity, pre.kvheads, pre.head_dim, pre.seqs, prefix_seq,
                                prefix_length));
        ND_CHECK(d_q && d_out, "attention: null q or out");
        check_new(d_new_k, d_new_v);
        hipStream_t s = static_cast<hipStream_t>(stream);
        SpanArgs own = span_args(kv, layer_of(kv, layer), d_q, d_out, kv.seqs, heads, 1);
        own.length = length;
        own.lengths = d_lengths;
        own.new_k = d_new_k;
        own.new_v = d_new_v;
        const SpanPlan own_plan = cut(own, length, 1);
        SpanArgs far = span_args(kv, layer_of(pre, layer, prefix_seq), d_q, d_out, 1, heads, kv.seqs);
        far.length = prefix_length;
        const SpanPlan far_plan = cut(far, prefix_length, 1);
        if (prefix_length == 0) far.splits = 0;
        own.split0 = far.splits;
        own.splits_total = far.splits_total = far.splits + own.splits;
        if (own.splits_total > 1) {
            reserve_records(kv, own, int64_t(kv.seqs) * heads);
            far.rec_o = own.rec_o;
            far.rec_ml = own.rec_ml;
        }
        if (prefix_length > 0) launch(far, far_plan, kv.head_dim, s);
        launch(own, own_plan, kv.head_dim, s);
        if (own.splits_total > 1) launch_span_join(own, kv.head_dim, s);
    });
}

int needle2_gpu_attention_weights(void *h, int layer, const float *d_q, float *d_out, float *d_weights, int heads, int length,
                                  const int *d_lengths, const float *d_new_k, const float *d_new_v, void *stream) {
    return guarded([&] {
        ND_CHECK(h != nullptr, "null KV cache handle");
        KvHandle &kv = kv_here(h);
        check_layer(kv, layer);
        check_rule(check_length(kv.capacity, kv.seqs, kv.kvheads, heads, length));
        ND_CHECK(d_q && d_out && d_weights, "attention: null q, out or weights");
        check_new(d_new_k, d_new_v);
        hipStream_t s = static_cast<hipStream_t>(stream);
        SpanArgs a = span_args(kv, layer_of(kv, layer), d_q, d_out, kv.seqs, heads, 1);
        a.length = length;
        a.lengths = d_lengths;
        a.new_k = d_new_k;
        a.new_v = d_new_v;
        const int tiles = span_tiles(length);
        const SpanPlan plan = cut(a, length, 1);
        a.splits_total = a.splits;
        reserve_records(kv, a, int64_t(kv.seqs) * heads);  // for one piece too: the weights need the final sums
        a.score_stride = std::max(1, tiles) * kSpanTile;
        a.scores = kv.scores.reserve(size_t(kv.seqs) * heads * a.score_stride);
        SpanRecordArgs r{a, d_weights};
        launch(a, plan, kv.head_dim, s);
        launch_span_record(r, kv.head_dim, s);
    });
}

int needle2_gpu_kv_evict(void *h, int layer, const float *d_weights, const int *d_lengths, int keep, int sinks, int recent,
                         float *d_new_weights, int *d_new_lengths, int *d_kept, void *stream) {
    return guarded([&] {
        ND_CHECK(h != nullptr, "null KV cache handle");
        KvHandle &kv = kv_here(h);
        check_layer(kv, layer);
        check_rule(check_evict(kv.capacity, kv.seqs, kv.kvheads, keep, sinks, recent));
        ND_CHECK(d_weights && d_lengths && d_new_weights && d_new_lengths, "eviction: null weights or lengths");
        EvictArgs a{};
        a.c = layer_of(kv, layer);
        a.weights = d_weights;
        a.new_weights = d_new_weights;
        a.lengths = d_lengths;
        a.new_lengths = d_new_lengths;
        a.seqs = kv.seqs;
        a.kvheads = kv.kvheads;
        a.head_dim = kv.head_dim;
        a.keep = keep;
        a.sinks = sinks;
        a.recent = recent;
        const size_t rows = size_t(kv.seqs) * kv.kvheads * keep;
        a.counts = kv.kept.reserve(kv.seqs + (d_kept ? 0 : rows));
        a.kept = d_kept ? d_kept : a.counts + kv.seqs;
        launch_evict(a, static_cast<hipStream_t>(stream));
    });
}

int needle2_gpu_kv_layer(void *h, int layer, int8_t **d_k, int8_t **d_v, float **d_ks, float **d_vs) {
    return guarded([&] {
        KvHandle &kv = *kv_of(h);
        check_layer(kv, layer);
        ND_CHECK(d_k && d_v && d_ks && d_vs, "KV layer: null result");
        const SpanCache c = layer_of(kv, layer);
        *d_k = c.k8;
        *d_v = c.v8;
        *d_ks = c.ks;
        *d_vs = c.vs;
    });
}

}  // extern "C"
