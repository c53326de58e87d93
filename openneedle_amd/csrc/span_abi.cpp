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

static void use(SpanArgs &a, const SpanCut &c) {
    a.splits = c.splits;
    a.per = c.per;
    a.waves = c.waves;
    a.groups = c.groups;
}

static void launch(const SpanArgs &a, bool wide, int head_dim, hipStream_t s) {
    if (wide) launch_span_wide(a, head_dim, s);
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
        const SpanCut cut = cut_window(device_cus(), kv.head_dim, kv.capacity, kv.seqs, kv.kvheads, heads, count, sinks, window);
        use(a, cut);
        a.splits_total = a.splits;
        if (a.splits_total > 1) reserve_records(kv, a, int64_t(kv.seqs) * count * heads);
        if (d_new_k && int64_t(count) * a.group <= kSpanRows) {
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
        launch(a, cut.wide, kv.head_dim, s);
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
        SpanArgs far = span_args(kv, layer_of(pre, layer, prefix_seq), d_q, d_out, 1, heads, kv.seqs);
        far.length = prefix_length;
        const bool shared = prefix_length > 0;
        use(own, cut_own(device_cus(), kv.head_dim, kv.seqs, kv.kvheads, heads, length, shared));
        const SpanCut cut = cut_prefix(device_cus(), kv.head_dim, kv.seqs, kv.kvheads, heads, prefix_length);
        use(far, cut);
        if (!shared) far.splits = 0;
        own.split0 = far.splits;
        own.splits_total = far.splits_total = far.splits + own.splits;
        if (own.splits_total > 1) {
            reserve_records(kv, own, int64_t(kv.seqs) * heads);
            far.rec_o = own.rec_o;
            far.rec_ml = own.rec_ml;
        }
        if (!shared) {
            launch_span(own, kv.head_dim, s);
        } else if (cut.wide) {
            launch_span_wide_own(far, own, kv.head_dim, s);
        } else {
            // eight waves fill a compute unit, and the launch has the sequences' own blocks too
            const int64_t row_tiles = (int64_t(far.count) * far.group + kSpanRows - 1) / kSpanRows;
            if ((row_tiles * far.splits + int64_t(own.splits) * own.units) * own.kvheads > device_cus()) far.waves = 4;
            launch_span_two(far, own, kv.head_dim, s);
        }
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
        use(a, cut_own(device_cus(), kv.head_dim, kv.seqs, kv.kvheads, heads, length, true));
        a.splits_total = a.splits;
        reserve_records(kv, a, int64_t(kv.seqs) * heads);  // for one piece too: the weights need the final sums
        a.score_stride = std::max(1, span_tiles(length)) * kSpanTile;
        // for the whole capacity: a length that grows with every step must not grow the scratch with it
        a.scores = kv.scores.reserve(size_t(kv.seqs) * heads * span_tiles(kv.capacity) * kSpanTile);
        SpanRecordArgs r{a, d_weights};
        launch_span(a, kv.head_dim, s);
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
        a.kept = d_kept;
        if (evict_takes_two(a)) {
            a.counts = kv.kept.reserve(kv.seqs + (d_kept ? 0 : size_t(kv.seqs) * kv.kvheads * keep));
            if (!d_kept) a.kept = a.counts + kv.seqs;
        }
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
