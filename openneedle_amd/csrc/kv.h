// The int8 KV cache behind a C handle (kv_abi.cpp, span_abi.cpp).
#pragma once

#include "abi_internal.h"

#include <algorithm>
#include <memory>
#include <vector>

namespace nd {

// Device scratch of a handle that only grows and never moves under a captured graph: what it outgrows stays allocated
// until the handle is destroyed, so a graph captured with the smaller buffer may still be replayed. It at least doubles,
// so that all of it together is at most twice the last.
template <class T>
struct KeptBuf {
    std::vector<std::unique_ptr<DevBuf<T>>> bufs;
    T *reserve(size_t count) {
        if (bufs.empty() || bufs.back()->n < count) {
            auto b = std::make_unique<DevBuf<T>>();
            b->reserve(bufs.empty() ? count : std::max(count, 2 * bufs.back()->n));
            bufs.push_back(std::move(b));
        }
        return bufs.back()->p;
    }
};

struct KvHandle {
    int layers = 0, capacity = 0, kvheads = 0, head_dim = 0, seqs = 0, device = 0;
    DevBuf<int8_t> k8, v8;
    DevBuf<float> ks, vs;
    DevBuf<float> part;
    DevBuf<int> first;    // per-sequence first slot of a store
    HostBuf<int> hfirst;  // pinned staging for `first`
    hipEvent_t first_copied = nullptr;
    KeptBuf<float> records, scores;  // the span kernels' (span.h)
    KeptBuf<int> kept;               // eviction's

    size_t layer_codes() const { return size_t(seqs) * kvheads * capacity * head_dim; }
    size_t layer_scales() const { return size_t(seqs) * kvheads * capacity; }
    ~KvHandle() {
        if (first_copied) (void)hipEventDestroy(first_copied);
    }
};

inline KvHandle *kv_of(void *h) {
    ND_CHECK(h != nullptr, "null KV cache handle");
    return static_cast<KvHandle *>(h);
}

inline void check_layer(const KvHandle &kv, int layer) {
    ND_CHECK(layer >= 0 && layer < kv.layers, "KV cache: layer out of range");
}

}  // namespace nd
