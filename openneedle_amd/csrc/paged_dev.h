// What the attention kernels read through a page table.
#pragma once

#include "paged.h"

namespace nd {

// Memory that no kernel of the running launch writes, read through the scalar cache where the address is uniform.
#define ND_CONST __attribute__((address_space(4)))

// The kernel's arguments, as the first of which it has `a`, read again where this is called instead of held in registers.
template <class A>
__device__ __forceinline__ const ND_CONST A &late(const PagedSpanArgs &) {
    auto p = (const ND_CONST A *)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *p;
}
template <class A>
__device__ __forceinline__ const A &late(const SpanArgs &a) { return a; }

// A request's tokens: the first one's row of q and its position, and how many. A request that does not lie in its table (or
// at a negative position) attends nothing.
struct Request {
    int token, count, first;
};
__device__ __forceinline__ Request request(const PagedSpanArgs &a, int r) {
    const ND_CONST int *starts = (const ND_CONST int *)(a.starts), *firsts = (const ND_CONST int *)(a.positions);
    const int t0 = max(0, min(starts[r], a.tokens)), t1 = max(t0, min(starts[r + 1], a.tokens));
    Request q = {t0, min(t1 - t0, a.count), firsts[r]};
    if (q.first < 0 || q.first > (a.width << a.pool.shift) - q.count) q.first = -1;
    return q;
}

// Block b of 128 rows: request r has those from starts[r] * group / 128 + r on, at least as many as it has row tiles (of two
// requests' whole and cut tiles, one more than the rows before them fill). 64 of the requests are looked at at a time.
struct WideBlock {
    int unit, row;
};
__device__ __forceinline__ WideBlock wide_block(const PagedSpanArgs &a, int b, int lane) {
    auto from = [&](int r) { return max(0, min(a.starts[r], a.tokens)) * a.group / kWideRows + r; };
    int low = 0, n = a.units;
    while (n > 1) {
        const int step = (n + 63) / 64, i = lane * step;
        const bool before = i == 0 || (i < n && from(low + i) <= b);
        const int at = (__popcll(__ballot(before)) - 1) * step;
        low += at;
        n = min(step, n - at);
    }
    low = __builtin_amdgcn_readfirstlane(low);
    return WideBlock{low, max(0, b - __builtin_amdgcn_readfirstlane(from(low))) * kWideRows};
}

// The same for at most kRanked requests, those in blocks of 128 rows by the length of their keys, the longest first, and of
// each the last row tile, which attends the most, first: what takes longest does not begin last, and no block has a request
// of fewer rows. In wide_block's order and this one (contexts of 4000): 20 pieces of up to 300 tokens, rows of 64 values, 8
// kv heads of 4 heads 358 and 341 us, 4 of 2 171 and 179; two of up to 800 beside 200 decoding requests 185 and 187, 107
// and 107; three of up to 1024 beside 48, rows of 128, 256 and 256, 129 and 129. But every block looks at every request
// that is in blocks of 128, one after the other: of up to 8 tokens with 16 heads (rows of 128, 4 kv heads, contexts of 1000)
// 64, 128, 256, 512 requests 61, 78, 150, 271 us in wide_block's and 68, 98, 260, 775 in this. row -1: there is no such
// block.
__device__ __forceinline__ WideBlock ranked_block(const PagedSpanArgs &a, int b, int lane) {
    constexpr int kEach = kRanked / 64;
    const ND_GLOBAL int *starts = (const ND_GLOBAL int *)(a.starts), *firsts = (const ND_GLOBAL int *)(a.positions);
    int tiles[kEach], length[kEach], before[kEach];  // tiles: 0 where the rows are in blocks of 16
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        tiles[i] = length[i] = before[i] = 0;
        if (i * 64 < a.units) {
            const int r = min(i * 64 + lane, a.units - 1);
            const int t0 = max(0, min(starts[r], a.tokens)), t1 = max(t0, min(starts[r + 1], a.tokens));
            const int count = min(t1 - t0, a.count), rows = count * a.group;
            length[i] = max(0, min(firsts[r], 1 << 30)) + count;
            tiles[i] = i * 64 + lane < a.units && rows > a.small ? (rows + kWideRows - 1) / kWideRows : 0;
        }
    }
#pragma unroll
    for (int j = 0; j < kEach; ++j)
        for (uint64_t some = __ballot(tiles[j] > 0); some; some &= some - 1) {
            const int l = __builtin_ctzll(some);
            const int its = __builtin_amdgcn_readlane(tiles[j], l), far = __builtin_amdgcn_readlane(length[j], l);
#pragma unroll
            for (int i = 0; i < kEach; ++i)
                before[i] += far > length[i] || (far == length[i] && j * 64 + l < i * 64 + lane) ? its : 0;
        }
    WideBlock found = {0, -1};
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const uint64_t it = __ballot(b >= before[i] && b < before[i] + tiles[i]);
        if (!it) continue;
        const int l = __builtin_ctzll(it);
        found.unit = i * 64 + l;
        found.row = (__builtin_amdgcn_readlane(before[i], l) + __builtin_amdgcn_readlane(tiles[i], l) - 1 - b) * kWideRows;
    }
    return found;
}

// The request with the k-th most positions before its tokens (of equal ones in a fixed order), by one wave, of at most
// kRanked requests: a search for that number of positions, bit by bit, by counting the requests that reach it.
__device__ __forceinline__ int ranked_request(const PagedSpanArgs &a, int k, int lane) {
    constexpr int kEach = kRanked / 64;
    const ND_GLOBAL int *firsts = (const ND_GLOBAL int *)(a.positions);
    const int most = a.width << a.pool.shift;
    int past[kEach];  // one more than it has; -1: no request
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const int r = i * 64 + lane;
        past[i] = -1;
        if (i * 64 < a.units) past[i] = r < a.units ? max(min(firsts[min(r, a.units - 1)], most), -1) + 1 : -1;
    }
    auto reach = [&](int limit) {
        int n = 0;
#pragma unroll
        for (int i = 0; i < kEach; ++i)
            if (i * 64 < a.units) n += __popcll(__ballot(past[i] >= limit));
        return n;
    };
    int value = 0;  // the largest that more than k of them reach
    for (int bit = 31 - __builtin_clz(most + 1); bit >= 0; --bit)
        if (reach(value + (1 << bit)) > k) value += 1 << bit;
    k -= reach(value + 1);
    int found = 0;
#pragma unroll
    for (int i = 0; i < kEach; ++i) {
        const uint64_t equal = __ballot(past[i] == value);
        const int before = __builtin_amdgcn_mbcnt_hi(static_cast<uint32_t>(equal >> 32),
                                                     __builtin_amdgcn_mbcnt_lo(static_cast<uint32_t>(equal), 0));
        const uint64_t it = __ballot(past[i] == value && before == k);
        if (it) found = i * 64 + __builtin_ctzll(it);
        k -= __popcll(equal);
    }
    return __builtin_amdgcn_readfirstlane(found);
}

// The pages of a request and kv head. A page outside the cache is none (-1): its rows read as zeros and are masked.
template <int HD>
struct PageReader {
    const ND_CONST int *table;
    const uint8_t *at;
    uint32_t page_bytes;  // of all kv heads
    int width, pages, shift;
    __device__ __forceinline__ PageReader() = default;
    __device__ __forceinline__ PageReader(const PagedSpanArgs &a, int unit, int kh)
        : table((const ND_CONST int *)(a.tables + static_cast<size_t>(unit) * a.width)),
          at(a.pool.at + static_cast<size_t>(kh) * page_block_bytes(a.pool.shift, HD)),
          page_bytes(a.pool.kvheads * page_block_bytes(a.pool.shift, HD)), width(a.width),
          pages(a.pool.pages), shift(a.pool.shift) {}
    // The table's entry for a position (the same for all lanes, or of every lane's own), loaded ahead of its use, and the
    // page that it says.
    __device__ __forceinline__ int entry(int position) const { return table[min(position >> shift, width - 1)]; }
    __device__ __forceinline__ int entry_of_lane(int position) const {
        return ((const ND_GLOBAL int *)(uintptr_t)table)[min(position >> shift, width - 1)];
    }
    __device__ __forceinline__ int page(int entry, int position) const {
        return position >> shift < width && static_cast<unsigned>(entry) < static_cast<unsigned>(pages) ? entry : -1;
    }
    __device__ __forceinline__ const uint8_t *block(int id) const { return at + static_cast<uint64_t>(static_cast<uint32_t>(max(id, 0))) * page_bytes; }
    __device__ __forceinline__ int off(int position) const { return position & ((1 << shift) - 1); }
    // 16 rows from a position on (a multiple of 16); past them, and of no page, zeros
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t k_codes(int id, int position) const {
        return buffer_rsrc(block(id) + off(position) * HD, id >= 0 ? 16 * HD : 0);
    }
    __device__ __forceinline__ __amdgpu_buffer_rsrc_t v_codes(int id, int position) const {
        return buffer_rsrc(block(id) + (HD << shift) + off(position) * HD, id >= 0 ? 16 * HD : 0);
    }
    // their K scales; the V scales are 1 << shift further
    __device__ __forceinline__ const float *k_scales(int id, int position) const {
        return reinterpret_cast<const float *>(block(id) + (2 * HD << shift)) + off(position);
    }
};

}  // namespace nd
