// gfx950 kernels that cut the int8 cache to the slots with the largest recorded attention weights.
//
// For a (sequence, kv head) with n > keep slots and weights w: kept are [0, sinks), [n - recent, n) and the
// keep - sinks - recent slots j of the middle that come first in the order (w_j descending, j ascending). The last of
// them has the rank-th largest key; a radix select over order-preserving 32-bit keys finds that key and how many of the
// slots that share it are kept, the lowest first. Rows then move to slot 0 .. keep - 1 in their order, in place.
// The selection is bound by its passes' latencies (256 pairs of up to 8192 slots, a block each: 14 us), the move by memory.
#include "span.h"
#include "wave.h"

namespace nd {

namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kBins = 2 * kThreads;
constexpr int kChunk = 4 * kThreads;  // slots of one step: four consecutive ones a thread
constexpr int kHeld = 2;              // steps whose weights stay in registers (8192 slots)

// Larger weights have larger keys; NaN ranks below every number, and -0 with 0.
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0;
    const uint32_t b = __builtin_bit_cast(uint32_t, w + 0.0f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// Sums of v over lanes 0 .. lane of the wave.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const uint32_t o = __shfl_up(v, d);
        v += lane >= d ? o : 0u;
    }
    return v;
}

struct SelectLds {
    uint32_t hist[kBins];
    uint32_t waves[2][kWaves];
    uint32_t found[3][3];
};

// Exclusive prefix sums of v over the block's threads, and the total; one barrier (callers alternate `half`).
__device__ __forceinline__ uint32_t block_scan(uint32_t v, int t, uint32_t (&waves)[kWaves], uint32_t &total) {
    const int lane = t & 63, wave = t >> 6;
    const uint32_t incl = wave_scan(v, lane);
    if (lane == 63) waves[wave] = incl;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        const uint32_t s = waves[w];
        before += w < wave ? s : 0u;
        all += s;
    }
    total = all;
    return before + incl - v;
}

// Four consecutive weights from slot j on; those from n on are 0.
struct Four {
    float x[4];
};
__device__ __forceinline__ Four read_four(const float *w, int j, int n) {
    Four r;
#pragma unroll
    for (int u = 0; u < 4; ++u) r.x[u] = 0.0f;
    if (j + 3 < n) {
        typedef float unaligned4 __attribute__((ext_vector_type(4), aligned(4)));
        const unaligned4 v = *reinterpret_cast<const unaligned4 *>(w + j);
#pragma unroll
        for (int u = 0; u < 4; ++u) r.x[u] = v[u];
    } else {
#pragma unroll
        for (int u = 0; u < 3; ++u)
            if (j + u < n) r.x[u] = w[j + u];
    }
    return r;
}

// put(new slot, old slot, weight) for the kept slots of n > 0, by a block of kThreads. A step's weights are read by every
// thread before any of its puts, and kept slots only move down, so put may write the weights over themselves.
template <class Put>
__device__ __forceinline__ void select_kept(SelectLds &lds, const float *w, int n, int keep, int sinks, int recent, Put &&put) {
    const int t = threadIdx.x;
    const int lo = sinks, hi = n - recent;  // the middle, if anything goes
    Four held[kHeld];
#pragma unroll
    for (int c = 0; c < kHeld; ++c) held[c] = read_four(w, c * kChunk + 4 * t, n);

    uint32_t bar = 0, ties = 0;  // keys above `bar` are kept, and the first `ties` of those equal to it
    if (n > keep) {
        uint32_t rank = keep - sinks - recent;  // of the middle to keep
        if (rank == 0) {
            bar = 0xFFFFFFFFu;
        } else {
            uint32_t mask = 0;
            constexpr int kShift[3] = {21, 10, 0};
            lds.hist[t] = 0;
            lds.hist[t + kThreads] = 0;
            __syncthreads();
#pragma unroll 1
            for (int pass = 0; pass < 3; ++pass) {
                const int shift = kShift[pass];
                const uint32_t bins = pass == 2 ? 1024 : 2048;
                auto count = [&](const Four &f, int j) {
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const uint32_t key = weight_key(f.x[u]);
                        if (j + u >= lo && j + u < hi && (key & mask) == bar) atomicAdd(&lds.hist[key >> shift & (bins - 1)], 1u);
                    }
                };
#pragma unroll
                for (int c = 0; c < kHeld; ++c) count(held[c], c * kChunk + 4 * t);
                for (int j = kHeld * kChunk + 4 * t; j < hi; j += kChunk) count(read_four(w, j, n), j);
                __syncthreads();
                // from the largest bin down: thread t has the bins 2047 - 2 t and 2046 - 2 t, and clears them for the next pass
                const int b0 = kBins - 1 - 2 * t, b1 = b0 - 1;
                const uint32_t h0 = lds.hist[b0], h1 = lds.hist[b1];
                lds.hist[b0] = 0;
                lds.hist[b1] = 0;
                uint32_t total;
                const uint32_t above = block_scan(h0 + h1, t, lds.waves[pass & 1], total);
                if (above < rank && rank <= above + h0 + h1) {
                    const bool first = rank <= above + h0;
                    lds.found[pass][0] = first ? b0 : b1;
                    lds.found[pass][1] = rank - above - (first ? 0u : h0);
                    lds.found[pass][2] = first ? h0 : h1;
                }
                __syncthreads();
                bar |= lds.found[pass][0] << shift;
                rank = lds.found[pass][1];
                mask |= (bins - 1) << shift;
                ties = rank;
                if (rank == lds.found[pass][2]) {  // all of the bin are kept: no need to tell them apart
                    bar -= 1;  // (not below 0: a bin with the key 0 that is kept whole would be the last of the whole middle)
                    ties = 0;
                    break;
                }
            }
        }
    }

    uint32_t done = 0, tied = 0;
    int half = 0;
    auto step = [&](const Four &f, int j) {
        bool sure[4], tie[4];
        uint32_t count = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const uint32_t key = weight_key(f.x[u]);
            const bool always = n <= keep || j + u < lo || j + u >= hi;
            sure[u] = j + u < n && (always || key > bar);
            tie[u] = j + u < n && !always && key == bar && ties > 0;
            count += sure[u] ? 1u : 0u;
            count += tie[u] ? 0x10000u : 0u;
        }
        uint32_t total;
        const uint32_t before = block_scan(count, t, lds.waves[half], total);  // (waits for every read of the step)
        half ^= 1;
        uint32_t e = tied + (before >> 16);
        uint32_t at = done + (before & 0xFFFFu) + min(e, ties) - min(tied, ties);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (sure[u] || (tie[u] && e < ties)) put(static_cast<int>(at++), j + u, f.x[u]);
            e += tie[u] ? 1u : 0u;
        }
        const uint32_t tied_now = tied + (total >> 16);
        done += (total & 0xFFFFu) + min(tied_now, ties) - min(tied, ties);
        tied = tied_now;
    };
    __syncthreads();  // (the last pass's use of lds.waves)
#pragma unroll
    for (int c = 0; c < kHeld; ++c)
        if (c * kChunk < n) step(held[c], c * kChunk + 4 * t);
    for (int j0 = kHeld * kChunk; j0 < n; j0 += kChunk) step(read_four(w, j0 + 4 * t, n), j0 + 4 * t);
    __syncthreads();  // every put is made, and no weight is read any more
}

// A pair's weights and list behind its `left` kept slots.
__device__ __forceinline__ void clear_rest(const EvictArgs &a, size_t pair, int left) {
    for (int j = left + threadIdx.x; j < a.keep; j += kThreads)
        if (a.kept) a.kept[pair * a.keep + j] = -1;
    for (int j = left + threadIdx.x; j < a.c.capacity; j += kThreads) a.new_weights[pair * a.c.capacity + j] = 0.0f;
}

__device__ __forceinline__ int slots_of(const EvictArgs &a, int seq) { return max(0, min(a.lengths[seq], a.c.capacity)); }

// Block (kv head, sequence): the kept slots and their weights.
__global__ __launch_bounds__(kThreads) void evict_select_kernel(EvictArgs a) {
    __shared__ SelectLds lds;
    const int kh = blockIdx.x, seq = blockIdx.y;
    const size_t pair = static_cast<size_t>(seq) * a.kvheads + kh;
    const int n = slots_of(a, seq), left = min(n, a.keep);
    if (kh == 0 && threadIdx.x == 0) a.counts[seq] = left;
    int *kept = a.kept + pair * a.keep;
    float *out = a.new_weights + pair * a.c.capacity;
    select_kept(lds, a.weights + pair * a.c.capacity, n, a.keep, a.sinks, a.recent, [&](int to, int from, float w) {
        kept[to] = from;
        out[to] = w;
    });
    clear_rest(a, pair, left);
}

// A part of the kept rows' bytes (slice `part` of K, then of V) to slots 0 .. left - 1, by a block. A slot's row only
// moves down, and rows are read in order before the block writes over them, so nothing is lost in place; the slices are
// different bytes and their blocks need no order. `kept`: the old slots. Memory bounds it: 256 pairs of rows of 128, 4001
// of up to 8192 kept, 541 MB read and written: 95-104 us (5.2-5.7 TB/s) with whole rows, 127-139 with slices of 64 bytes,
// which spread few pairs over more units.
constexpr int kMoveRows = 4;  // rows in flight per thread
template <int HD, int SLICE>
__device__ __forceinline__ void move_rows(const EvictArgs &a, size_t pair, int part, int left, const int *kept) {
    constexpr int kSlices = HD / SLICE, kLanes = SLICE / 16, kRows = kThreads / kLanes;
    const int t = threadIdx.x, slice = part % kSlices;
    const bool values = part >= kSlices;
    int8_t *rows = (values ? a.c.v8 : a.c.k8) + pair * a.c.capacity * HD + slice * SLICE + t % kLanes * 16;
    float *scales = (values ? a.c.vs : a.c.ks) + pair * a.c.capacity;
    const bool scaled = slice == 0 && t % kLanes == 0;
    for (int j0 = 0; j0 < left; j0 += kRows * kMoveRows) {
        u32x4 x[kMoveRows];
        float s[kMoveRows];
        int from[kMoveRows];
#pragma unroll
        for (int u = 0; u < kMoveRows; ++u) {
            const int j = j0 + u * kRows + t / kLanes;
            from[u] = j < left ? kept[j] : j;
        }
#pragma unroll
        for (int u = 0; u < kMoveRows; ++u) {
            const int j = j0 + u * kRows + t / kLanes;
            if (from[u] != j) {
                x[u] = *reinterpret_cast<const u32x4 *>(rows + static_cast<size_t>(from[u]) * HD);
                if (scaled) s[u] = scales[from[u]];
            }
        }
        // every wave has what it moves before any of them writes
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
#pragma unroll
        for (int u = 0; u < kMoveRows; ++u) {
            const int j = j0 + u * kRows + t / kLanes;
            if (from[u] != j) {
                *reinterpret_cast<u32x4 *>(rows + static_cast<size_t>(j) * HD) = x[u];
                if (scaled) scales[j] = s[u];
            }
        }
    }
}

// Block (part, kv head, sequence), after the selection.
template <int HD, int SLICE>
__global__ __launch_bounds__(kThreads) void evict_move_kernel(EvictArgs a) {
    const int kh = blockIdx.y, seq = blockIdx.z;
    const size_t pair = static_cast<size_t>(seq) * a.kvheads + kh;
    const int left = a.counts[seq];
    if (blockIdx.x == 0 && kh == 0 && threadIdx.x == 0) a.new_lengths[seq] = left;
    move_rows<HD, SLICE>(a, pair, blockIdx.x, left, a.kept + pair * a.keep);
}

// Both in one launch: every part's block selects for itself, its list in LDS, and the first part's writes the results. Only
// where the results are not the inputs, which another part's block may still read.
constexpr int kListMax = 12288;
template <int HD, int SLICE>
__global__ __launch_bounds__(kThreads) void evict_kernel(EvictArgs a) {
    __shared__ SelectLds lds;
    extern __shared__ int list[];
    const int kh = blockIdx.y, seq = blockIdx.z, part = blockIdx.x;
    const size_t pair = static_cast<size_t>(seq) * a.kvheads + kh;
    const int n = slots_of(a, seq), left = min(n, a.keep);
    const float *w = a.weights + pair * a.c.capacity;
    float *out = a.new_weights + pair * a.c.capacity;
    select_kept(lds, w, n, a.keep, a.sinks, a.recent, [&](int to, int from, float x) {
        list[to] = from;
        if (part == 0) {
            out[to] = x;
            if (a.kept) a.kept[pair * a.keep + to] = from;
        }
    });
    move_rows<HD, SLICE>(a, pair, part, left, list);
    if (part == 0) {
        clear_rest(a, pair, left);
        if (kh == 0 && threadIdx.x == 0) a.new_lengths[seq] = left;
    }
}

template <int HD, int SLICE>
void launch_two_hd(const EvictArgs &a, hipStream_t s) {
    hipLaunchKernelGGL(evict_select_kernel, dim3(a.kvheads, a.seqs), dim3(kThreads), 0, s, a);
    ND_HIP(hipGetLastError());
    hipLaunchKernelGGL((evict_move_kernel<HD, SLICE>), dim3(2 * (HD / SLICE), a.kvheads, a.seqs), dim3(kThreads), 0, s, a);
    ND_HIP(hipGetLastError());
}

template <int HD, int SLICE>
void launch_one_hd(const EvictArgs &a, hipStream_t s) {
    hipLaunchKernelGGL((evict_kernel<HD, SLICE>), dim3(2 * (HD / SLICE), a.kvheads, a.seqs), dim3(kThreads),
                       a.keep * sizeof(int), s, a);
    ND_HIP(hipGetLastError());
}

}  // namespace

// One launch where its blocks, each of which repeats the selection, leave compute units free (8 pairs, 1024 of up to 2048
// slots kept: 12.5 -> 9.1 us).
bool evict_takes_two(const EvictArgs &a) {
    const int64_t blocks = static_cast<int64_t>(a.seqs) * a.kvheads * (a.head_dim == 128 ? 4 : 2);
    return blocks > device_cus() || a.keep > kListMax || a.new_weights == a.weights || a.new_lengths == a.lengths;
}

void launch_evict(const EvictArgs &a, hipStream_t s) {
    const bool two = evict_takes_two(a);
    switch (a.head_dim) {
    case 32:
        if (two) launch_two_hd<32, 32>(a, s);
        else launch_one_hd<32, 32>(a, s);
        break;
    case 64:
        if (two) launch_two_hd<64, 64>(a, s);
        else launch_one_hd<64, 64>(a, s);
        break;
    default:
        if (two) launch_two_hd<128, 128>(a, s);
        else launch_one_hd<128, 64>(a, s);
    }
}

}  // namespace nd
