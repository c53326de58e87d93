// Which cache slots a query attends, as arithmetic on plain integers (host and device; no HIP types).
#pragma once

#include <stddef.h>
#include <stdint.h>

#ifdef __HIPCC__
#define ND_BOTH __host__ __device__ __forceinline__
#else
#define ND_BOTH inline
#endif

namespace nd {

// A cache with `sinks` pinned positions and a ring: position p lies in slot p while p < sinks, then in
// sinks + (p - sinks) mod (capacity - sinks). capacity > sinks, p >= 0.
ND_BOTH int ring_slot(int p, int sinks, int capacity) {
    return p < sinks ? p : sinks + static_cast<int>(static_cast<uint32_t>(p - sinks) % static_cast<uint32_t>(capacity - sinks));
}

// The keys of consecutive queries at positions first .. last as two runs of consecutive slots: [0, n0) and
// [begin1, begin1 + n1). A slot j below `pinned` holds position j; any other slot of run 0 holds position j + shift0, one
// of run 1 holds j + shift1. Together they hold [0, min(sinks, last + 1)) and every position from
// max(sinks, first - window + 1) to last, each once.
struct KeyRuns {
    int n0, begin1, n1, pinned, shift0, shift1;
};

// Queries at negative positions attend nothing. Needs last - first + window <= capacity - sinks, so that no two of the
// positions share a slot.
ND_BOTH KeyRuns ring_runs(int first, int last, int sinks, int window, int capacity) {
    KeyRuns r = {0, 0, 0, 0, 0, 0};
    if (last < 0) return r;
    r.pinned = last < sinks ? last + 1 : sinks;
    r.n0 = r.pinned;
    if (last < sinks) return r;
    int low = first < 0 ? 0 : first;
    low = low >= window ? low - window + 1 : 0;
    low = low > sinks ? low : sinks;
    const int a = ring_slot(low, sinks, capacity), b = ring_slot(last, sinks, capacity);
    r.begin1 = a;
    r.shift1 = low - a;
    if (a <= b) {
        r.n1 = b - a + 1;
    } else {  // the positions wrap: slots [sinks, b] hold the newest of them, right behind the pinned ones
        r.n1 = capacity - a;
        r.n0 = b + 1;
        r.shift0 = last - b;
    }
    return r;
}

constexpr int kSpanTile = 64;  // keys of a tile; a tile lies in one run

constexpr int kWideTile = 32;  // where many query rows share them

ND_BOTH int span_tiles(int n) { return (n + kSpanTile - 1) / kSpanTile; }
ND_BOTH int wide_tiles(int n) { return (n + kWideTile - 1) / kWideTile; }

}  // namespace nd
