// gfx950 kernels that cut the int8 cache to the slots with the largest recorded attention weights.
//
// For a (sequence, kv head) with n > keep slots and weights w: kept are [0, sinks), [n - recent, n) and the
// keep - sinks - recent slots j of the middle that come first in the order (w_j descending, j ascending). The last of
// them has the rank-th largest key; a radix select over order-preserving 32-bit keys finds that key and how many of the
// slots that share it are kept, the lowest first. Rows then move to slot 0 .. keep - 1 in their order, in place.
#include "span.h"
#include "wave.h"

namespace nd {

namespace {

constexpr int kSelectThreads = 1024;
constexpr int kBins = 2048;

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

// Exclusive prefix sums of v over the block's threads, and the total; two barriers.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, int t, uint32_t (&waves)[kSelectThreads / 64 + 1], uint32_t &total) {
    const int lane = t & 63, wave = t >> 6;
    const uint32_t incl = wave_scan(v, lane);
    if (lane == 63) waves[wave] = incl;
    __syncthreads();
    uint32_t before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < kSelectThreads / 64; ++w) {
        const uint32_t s = waves[w];
        before += w < wave ? s : 0u;
        all += s;
    }
    __syncthreads();
    total = all;
    return before + incl - v;
}

// Block (kv head, sequence): the kept slots and their weights.
__global__ __launch_bounds__(kSelectThreads) void evict_select_kernel(EvictArgs a) {
    __shared__ uint32_t hist[kBins];
    __shared__ uint32_t waves[kSelectThreads / 64 + 1];
    __shared__ uint32_t found[2];
    const int t = threadIdx.x, kh = blockIdx.x, seq = blockIdx.y;
    const int cap = a.c.capacity;
    const size_t pair = static_cast<size_t>(seq) * a.kvheads + kh;
    const float *w = a.weights + pair * cap;
    float *out = a.new_weights + pair * cap;
    int *kept = a.kept + pair * a.keep;
    const int n = max(0, min(a.lengths[seq], cap));
    const int left = min(n, a.keep);
    if (kh == 0 && t == 0) a.counts[seq] = left;
    const int lo = a.sinks, hi = n - a.recent;  // the middle, if anything goes

    uint32_t bar = 0, ties = 0;  // keys above `bar` are kept, and the first `ties` of those equal to it
    if (n > a.keep) {
        uint32_t rank = a.keep - a.sinks - a.recent;  // of the middle to keep
        if (rank == 0) {
            bar = 0xFFFFFFFFu;
        } else {
            uint32_t mask = 0;
            constexpr int kShift[3] = {21, 10, 0};
#pragma unroll 1
            for (int pass = 0; pass < 3; ++pass) {
                const int shift = kShift[pass];
                const uint32_t bins = pass == 2 ? 1024 : 2048;
                for (int i = t; i < kBins; i += kSelectThreads) hist[i] = 0;
                __syncthreads();
                for (int j = lo + t; j < hi; j += kSelectThreads) {
                    const uint32_t key = weight_key(w[j]);
                    if ((key & mask) == bar) atomicAdd(&hist[key >> shift & (bins - 1)], 1u);
                }
                __syncthreads();
                // from the largest bin down: thread t has the bins 2047 - 2 t and 2046 - 2 t
                const uint32_t h0 = hist[kBins - 1 - 2 * t], h1 = hist[kBins - 2 - 2 * t];
                uint32_t total;
                const uint32_t above = block_scan(h0 + h1, t, waves, total);
                if (above < rank && rank <= above + h0 + h1) {
                    const bool first = rank <= above + h0;
                    found[0] = first ? kBins - 1 - 2 * t : kBins - 2 - 2 * t;
                    found[1] = rank - above - (first ? 0u : h0);
                }
                __syncthreads();
                bar |= found[0] << shift;
                rank = found[1];
                mask |= (bins - 1) << shift;
                __syncthreads();
            }
            ties = rank;
        }
    }

    // the kept slots in order, four consecutive slots a thread; a chunk's weights are read before any of it is written,
    // and kept ones only move down, so the weights may be compacted in place
    uint32_t done = 0, tied = 0;
    for (int j0 = 0; j0 < n; j0 += 4 * kSelectThreads) {
        float x[4];
        bool sure[4], tie[4];
        uint32_t count = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int j = j0 + 4 * t + u;
            x[u] = j < n ? w[j] : 0.0f;
            const uint32_t key = weight_key(x[u]);
            const bool always = n <= a.keep || j < lo || j >= hi;
            sure[u] = j < n && (always || key > bar);
            tie[u] = j < n && !always && key == bar && ties > 0;
            count += sure[u] ? 1u : 0u;
            count += tie[u] ? 0x10000u : 0u;
        }
        uint32_t total;
        const uint32_t before = block_scan(count, t, waves, total);  // (waits for every load of the chunk)
        uint32_t k = before & 0xFFFFu, e = tied + (before >> 16);
        uint32_t at = done + k + min(e, ties) - min(tied, ties);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const bool in = sure[u] || (tie[u] && e < ties);
            if (in) {
                kept[at] = j0 + 4 * t + u;
                out[at] = x[u];
                ++at;
            }
            e += tie[u] ? 1u : 0u;
        }
        const uint32_t tied_now = tied + (total >> 16);
        done += (total & 0xFFFFu) + min(tied_now, ties) - min(tied, ties);
        tied = tied_now;
    }
    __syncthreads();  // the last chunk is read and written before the rest of its slots are cleared
    for (int j = left + t; j < a.keep; j += kSelectThreads) kept[j] = -1;
    for (int j = left + t; j < cap; j += kSelectThreads) out[j] = 0.0f;
}

// Block (K or V and slice of 64 bytes of a row, kv head, sequence): the kept rows' slice to slots 0 .. A slot's row only
// moves down, and rows are read in order before the block writes over them, so nothing is lost in place; the slices of a
// row are different bytes and their blocks need no order.
constexpr int kMoveRows = 4;  // rows in flight per thread
template <int HD>
__global__ __launch_bounds__(1024) void evict_move_kernel(EvictArgs a) {
    constexpr int kSlice = HD < 64 ? HD : 64, kSlices = HD / kSlice, kLanes = kSlice / 16, kRows = 1024 / kLanes;
    const int t = threadIdx.x, kh = blockIdx.y, seq = blockIdx.z;
    const int slice = blockIdx.x % kSlices;
    const bool values = blockIdx.x >= kSlices;
    const size_t pair = static_cast<size_t>(seq) * a.kvheads + kh;
    const int left = a.counts[seq];
    if (blockIdx.x == 0 && kh == 0 && t == 0) a.new_lengths[seq] = left;
    int8_t *rows = (values ? a.c.v8 : a.c.k8) + pair * a.c.capacity * HD + slice * kSlice + t % kLanes * 16;
    float *scales = (values ? a.c.vs : a.c.ks) + pair * a.c.capacity;
    const bool scaled = slice == 0 && t % kLanes == 0;
    const int *kept = a.kept + pair * a.keep;
    for (int j0 = 0; j0 < left; j0 += kRows * kMoveRows) {
        u32x4 x[kMoveRows];
        float s[kMoveRows];
        int from[kMoveRows];
#pragma unroll
        for (int u = 0; u < kMoveRows; ++u) {
            const int j = j0 + u * kRows + t / kLanes;
            from[u] = j < left ? kept[j] : j;
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

}  // namespace

void launch_evict(const EvictArgs &a, hipStream_t s) {
    hipLaunchKernelGGL(evict_select_kernel, dim3(a.kvheads, a.seqs), dim3(kSelectThreads), 0, s, a);
    ND_HIP(hipGetLastError());
    const dim3 grid(a.head_dim == 128 ? 4 : 2, a.kvheads, a.seqs);
    switch (a.head_dim) {
    case 32: hipLaunchKernelGGL((evict_move_kernel<32>), grid, dim3(1024), 0, s, a); break;
    case 64: hipLaunchKernelGGL((evict_move_kernel<64>), grid, dim3(1024), 0, s, a); break;
    default: hipLaunchKernelGGL((evict_move_kernel<128>), grid, dim3(1024), 0, s, a); break;
    }
    ND_HIP(hipGetLastError());
}

}  // namespace nd
