// C ABI of the paged int8 cache (additive exports): pages dealt to requests on the GPU, heads normed, rotated and stored by
// slot, and attention of ragged new tokens. The reference has one sequence at a time in one run of slots
// (needle2/csrc/engine.cpp:433-449, 898-967) and norms and rotates the heads inside its step (engine.cpp:994-1021).
#include "kv.h"
#include "paged.h"

#include <algorithm>
#include <cmath>

namespace nd {

namespace {

struct PagedHandle {
    int layers = 0, pages = 0, shift = 0, kvheads = 0, head_dim = 0, device = 0;
    DevBuf<uint8_t> rows;
    DevBuf<int> stack, state;  // state: free pages; blocks of a running launch that are done
    KeptBuf<float> records;    // of the attention (span.h)
    KeptBuf<int2> some;
    const int2 *zeroed = nullptr;  // the last of `some`, once zeros have been written to it and not only captured

    size_t layer_bytes() const { return size_t(pages) * kvheads * page_block_bytes(shift, head_dim); }
    PageStack free() const { return PageStack{stack.p, state.p, state.p + 1, pages}; }
    PagePool pool(int layer) const { return PagePool{rows.p + layer * layer_bytes(), pages, shift, kvheads}; }
};

void check_rule(const char *broken) {
    if (broken) throw Error(broken);
}

// The handle, which must be used where its memory is.
PagedHandle &paged_here(void *h) {
    ND_CHECK(h != nullptr, "null paged cache handle");
    PagedHandle &p = *static_cast<PagedHandle *>(h);
    int device = 0;
    ND_HIP(hipGetDevice(&device));
    ND_CHECK(device == p.device, "paged cache: made on another device than the current one");
    return p;
}

void check_layer(const PagedHandle &p, int layer) {
    ND_CHECK(layer >= 0 && layer < p.layers, "paged cache: layer out of range");
}

}  // namespace

}  // namespace nd

using namespace nd;

extern "C" {

void *needle2_gpu_pages_create(int layers, int pages, int page_size, int kvheads, int head_dim) {
    PagedHandle *made = nullptr;
    if (guarded([&] {
            check_rule(check_pages(layers, pages, page_size, kvheads, head_dim));
            auto h = std::make_unique<PagedHandle>();
            h->layers = layers;
            h->pages = pages;
            while ((1 << h->shift) < page_size) ++h->shift;
            h->kvheads = kvheads;
            h->head_dim = head_dim;
            ND_HIP(hipGetDevice(&h->device));
            h->rows.reserve(h->layer_bytes() * layers);
            h->stack.reserve(pages);
            h->state.reserve(2);
            ND_HIP(hipMemset(h->rows.p, 0, h->layer_bytes() * layers));
            launch_pages_reset(h->free(), nullptr);
            ND_HIP(hipDeviceSynchronize());
            made = h.release();
        }))
        return nullptr;
    return made;
}

void needle2_gpu_pages_destroy(void *h) { delete static_cast<PagedHandle *>(h); }

size_t needle2_gpu_pages_storage_bytes(void *h) {
    if (!h) return 0;
    const PagedHandle &p = *static_cast<PagedHandle *>(h);
    return p.layer_bytes() * p.layers;
}

int needle2_gpu_pages_layer(void *h, int layer, uint8_t **d_rows) {
    return guarded([&] {
        ND_CHECK(h != nullptr, "null paged cache handle");
        const PagedHandle &p = *static_cast<PagedHandle *>(h);
        check_layer(p, layer);
        ND_CHECK(d_rows, "paged cache: null result");
        *d_rows = p.pool(layer).at;
    });
}

int needle2_gpu_pages_free(void *h, int *count, void *stream) {
    return guarded([&] {
        PagedHandle &p = paged_here(h);
        ND_CHECK(count, "paged cache: null result");
        hipStream_t s = static_cast<hipStream_t>(stream);
        ND_HIP(hipMemcpyAsync(count, p.state.p, sizeof(int), hipMemcpyDeviceToHost, s));
        ND_HIP(hipStreamSynchronize(s));
    });
}

int needle2_gpu_pages_reset(void *h, void *stream) {
    return guarded([&] { launch_pages_reset(paged_here(h).free(), static_cast<hipStream_t>(stream)); });
}

int needle2_gpu_pages_extend(void *h, int requests, const int *d_counts, int tokens, int *d_lengths, int *d_tables, int width,
                             int *d_starts, int *d_firsts, int *d_slots, int *d_positions, void *stream) {
    return guarded([&] {
        PagedHandle &p = paged_here(h);
        check_rule(check_requests(requests, width, 1 << p.shift));
        check_rule(check_tokens(tokens));
        ND_CHECK(d_starts && (requests == 0 || (d_counts && d_lengths && d_tables && d_firsts)) &&
                     (tokens == 0 || (d_slots && d_positions)),
                 "paged cache: null counts, lengths, tables or results");
        launch_extend(ExtendArgs{p.free(), d_counts, d_lengths, d_tables, d_starts, d_firsts, d_slots, d_positions, requests,
                                 tokens, width, p.shift},
                      static_cast<hipStream_t>(stream));
    });
}

int needle2_gpu_pages_trim(void *h, int requests, const int *d_keep, int *d_lengths, int *d_tables, int width, void *stream) {
    return guarded([&] {
        PagedHandle &p = paged_here(h);
        check_rule(check_requests(requests, width, 1 << p.shift));
        if (requests == 0) return;
        ND_CHECK(d_keep && d_lengths && d_tables, "paged cache: null keep, lengths or tables");
        launch_trim(TrimArgs{p.free(), d_keep, d_lengths, d_tables, requests, width, p.shift},
                    static_cast<hipStream_t>(stream));
    });
}

int needle2_gpu_pages_store(void *h, int layer, const float *d_k, int k_stride, const float *d_v, int v_stride, int tokens,
                            const int *d_slots, void *stream) {
    return guarded([&] {
        PagedHandle &p = paged_here(h);
        check_layer(p, layer);
        check_rule(check_tokens(tokens));
        if (tokens == 0) return;
        ND_CHECK(d_k && d_v && d_slots, "paged cache: null k, v or slots");
        check_rule(check_rows(d_k, k_stride, p.kvheads, p.head_dim));
        check_rule(check_rows(d_v, v_stride, p.kvheads, p.head_dim));
        HeadsArgs a{};
        a.k = d_k;
        a.v = d_v;
        a.k_stride = k_stride;
        a.v_stride = v_stride;
        a.slots = d_slots;
        a.pool = p.pool(layer);
        a.tokens = tokens;
        a.kvheads = p.kvheads;
        launch_heads(a, p.head_dim, static_cast<hipStream_t>(stream));
    });
}

// What heads and heads_store share.
static HeadsArgs heads_args(const float *d_q, int q_stride, float *d_q_out, int q_out_stride, int heads, const float *d_k,
                            int k_stride, float *d_k_out, int k_out_stride, int kvheads, int head_dim, int tokens,
                            const int *d_positions, const float *d_q_gain, const float *d_k_gain, float eps,
                            const double *d_freq, int rotary) {
    check_rule(check_turn(heads, kvheads, head_dim, tokens, eps, rotary));
    ND_CHECK(!heads || !tokens || (d_q && d_q_out), "heads: null q or its output");
    ND_CHECK(!kvheads || !tokens || d_k, "heads: null k");
    ND_CHECK(!rotary || !tokens || (d_freq && d_positions), "heads: a rotation needs positions and frequencies");
    if (tokens > 0 && heads) {
        check_rule(check_rows(d_q, q_stride, heads, head_dim));
        check_rule(check_rows(d_q_out, q_out_stride, heads, head_dim));
    }
    if (tokens > 0 && kvheads) {
        check_rule(check_rows(d_k, k_stride, kvheads, head_dim));
        if (d_k_out) check_rule(check_rows(d_k_out, k_out_stride, kvheads, head_dim));
    }
    ND_CHECK((!heads || d_q != d_q_out || q_stride == q_out_stride) && (!kvheads || d_k != d_k_out || k_stride == k_out_stride),
             "heads: rows in place have one stride");
    for (const float *g : {d_q_gain, d_k_gain})
        ND_CHECK(reinterpret_cast<uintptr_t>(g) % 16 == 0, "heads: gains must begin at multiples of 16 bytes");
    HeadsArgs a{};
    a.q = heads ? d_q : nullptr;
    a.k = kvheads ? d_k : nullptr;
    a.q_out = d_q_out;
    a.k_out = d_k_out;
    a.q_stride = q_stride;
    a.k_stride = k_stride;
    a.q_out_stride = q_out_stride;
    a.k_out_stride = k_out_stride;
    a.q_gain = d_q_gain;
    a.k_gain = d_k_gain;
    a.freq = d_freq;
    a.positions = d_positions;
    a.tokens = tokens;
    a.heads = heads;
    a.kvheads = kvheads;
    a.half = rotary / 2;
    a.eps = eps;
    return a;
}

int needle2_gpu_heads(const float *d_q, int q_stride, float *d_q_out, int q_out_stride, int heads, const float *d_k,
                      int k_stride, float *d_k_out, int k_out_stride, int kvheads, int head_dim, int tokens,
                      const int *d_positions, const float *d_q_gain, const float *d_k_gain, float eps, const double *d_freq,
                      int rotary, void *stream) {
    return guarded([&] {
        ND_CHECK(!kvheads || !tokens || d_k_out, "heads: null output of k");
        const HeadsArgs a = heads_args(d_q, q_stride, d_q_out, q_out_stride, heads, d_k, k_stride, d_k_out, k_out_stride,
                                       kvheads, head_dim, tokens, d_positions, d_q_gain, d_k_gain, eps, d_freq, rotary);
        launch_heads(a, head_dim, static_cast<hipStream_t>(stream));
    });
}

int needle2_gpu_heads_store(void *h, int layer, const float *d_q, int q_stride, float *d_q_out, int q_out_stride, int heads,
                            const float *d_k, int k_stride, float *d_k_out, int k_out_stride, const float *d_v, int v_stride,
                            int tokens, const int *d_positions, const int *d_slots, const float *d_q_gain,
                            const float *d_k_gain, float eps, const double *d_freq, int rotary, void *stream) {
    return guarded([&] {
        PagedHandle &p = paged_here(h);
        check_layer(p, layer);
        HeadsArgs a = heads_args(d_q, q_stride, d_q_out, q_out_stride, heads, d_k, k_stride, d_k_out, k_out_stride, p.kvheads,
                                 p.head_dim, tokens, d_positions, d_q_gain, d_k_gain, eps, d_freq, rotary);
        if (tokens == 0) return;
        ND_CHECK(d_v && d_slots, "paged cache: null v or slots");
        check_rule(check_rows(d_v, v_stride, p.kvheads, p.head_dim));
        a.v = d_v;
        a.v_stride = v_stride;
        a.slots = d_slots;
        a.pool = p.pool(layer);
        launch_heads(a, p.head_dim, static_cast<hipStream_t>(stream));
    });
}

int needle2_gpu_pages_attention(void *h, int layer, const float *d_q, float *d_out, int heads, int requests, int tokens,
                                int count, const int *d_starts, const int *d_firsts, const int *d_tables, int width,
                                int length, int window, void *stream) {
    return guarded([&] {
        PagedHandle &p = paged_here(h);
        check_layer(p, layer);
        check_rule(check_requests(requests, width, 1 << p.shift));
        check_rule(check_tokens(tokens));
        check_rule(check_paged_attention(p.kvheads, heads, requests, tokens, count, length, window));
        if (requests == 0 || count == 0) return;
        ND_CHECK(d_q && d_out && d_starts && d_firsts && d_tables, "attention: null q, out, starts, firsts or tables");
        check_rule(check_rows(d_q, heads * p.head_dim, heads, p.head_dim));
        check_rule(check_rows(d_out, heads * p.head_dim, heads, p.head_dim));
        hipStream_t s = static_cast<hipStream_t>(stream);
        PagedSpanArgs a{};
        a.q = d_q;
        a.out = d_out;
        a.units = requests;
        a.kvheads = p.kvheads;
        a.heads = heads;
        a.group = heads / p.kvheads;
        a.count = count;
        a.scale = float(1.4426950408889634 / std::sqrt(double(p.head_dim)));
        a.positions = d_firsts;
        a.window = window;
        a.pool = p.pool(layer);
        a.starts = d_starts;
        a.tables = d_tables;
        a.tokens = tokens;
        a.width = width;
        const int most = length > 0 ? std::min(length, width << p.shift) : width << p.shift;
        const PagedCut cut = cut_paged(device_cus(), p.head_dim, requests, tokens, count, p.kvheads, a.group, most, window);
        a.small = cut.small;
        a.row_tiles = cut.row_tiles;
        a.round = cut.round;
        a.splits = cut.rows.splits;
        a.per = cut.rows.per;
        a.waves = cut.rows.waves;
        a.wide_blocks = cut.wide_blocks;
        a.wide_splits = cut.wide.splits;
        a.wide_per = cut.wide.per;
        a.splits_total = a.splits;
        if (length == 0) {  // cut for the tables' width: requests that are far shorter have pieces of their own size
            a.per = std::min(a.per, 2 * a.waves);
            a.wide_per = std::min(a.wide_per, 16);
        }
        const size_t few = size_t(cut.few_records), many = size_t(cut.wide_records);
        if (few + many) {
            const size_t n = few * a.splits, m = many * a.wide_splits;
            a.rec_o = p.records.reserve((n + m) * (p.head_dim + 2));
            a.wide_o = a.rec_o + n * p.head_dim;
            a.rec_ml = reinterpret_cast<float2 *>(a.wide_o + m * p.head_dim);
            a.wide_ml = a.rec_ml + n;
            a.some = p.some.reserve(few + many);
            a.wide_some = a.some + few;
            if (a.some != p.zeroed) {
                launch_zero(a.some, p.some.bufs.back()->n, s);
                hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
                ND_HIP(hipStreamIsCapturing(s, &capture));
                if (capture == hipStreamCaptureStatusNone) p.zeroed = a.some;
            }
        }
        launch_paged(a, p.head_dim, s);
        if (few) launch_paged_join(a, int64_t(few), p.head_dim, s);
        if (many) {
            PagedSpanArgs w = a;
            w.rec_o = a.wide_o;
            w.rec_ml = a.wide_ml;
            w.some = a.wide_some;
            w.splits_total = a.wide_splits;
            launch_paged_join(w, int64_t(many), p.head_dim, s);
        }
    });
}

}  // extern "C"
