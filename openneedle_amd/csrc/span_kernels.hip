// gfx950 kernels of attention over spans of the int8 cache: windows with pinned first positions, a shared prefix, and
// decode attention that records the weights.
//
// For a query row q and the keys j that it attends,
//   x_j = (q . kc_j) * ks_j * log2(e) / sqrt(HD),   p_j = 2^(x_j - m),   l = sum p_j,   out = sum (p_j vs_j) vc_j / l
// with int8 codes kc, vc and fp32 scales ks, vs; m, l and out are running values over tiles of 64 keys (m the largest
// x so far; l and out rescaled by 2^(m_old - m_new) when it moves). Pieces of the keys, and a prefix and a sequence's own
// keys, are joined through records (m, l, unnormalised out).
//
// Both products run on v_mfma_f32_16x16x32_bf16. The codes are bfloat16 numbers as they are; q and p * vs are three
// bfloat16 terms each (8 + 8 + 8 bits: the fp32 value exactly, at any magnitude), so only the sums round, in fp32.
#include "span_join.h"
#include "span_rows.h"

#include <cmath>
#include <type_traits>

namespace nd {

namespace {

// A K or V row per HD / 4 lanes, four values each (the cache's quantiser, as quantise_row): a wave has the K and V rows of
// 128 / HD (sequence, token, kv head)s (6 x 999 tokens of 8 kv heads of 128: 29 us with a wave per row -> 22 us).
template <int HD>
__global__ __launch_bounds__(256) void span_store_kernel(SpanStoreArgs a) {
    constexpr int kLanes = HD / 4;
    const uint32_t t = blockIdx.x * 256 + threadIdx.x;  // (at most 2^25 query rows, so below 2^31)
    const int lane = threadIdx.x & 63, part = threadIdx.x % kLanes;
    const bool values = t / kLanes % 2;
    const uint32_t item = t / (2 * kLanes), kvheads = a.kvheads, count = a.count;
    const bool in = item < a.seqs * count * kvheads;
    const uint32_t token = in ? item / kvheads : 0;
    const int kh = in ? item - token * kvheads : 0;
    const int seq = token / count, i = token - seq * count;
    const int p = at_position(a.positions[seq], i);
    const int slot = !in || p < 0 ? -1 : ring_slot(p, a.sinks, a.c.capacity);
    float4 x = make_float4(0, 0, 0, 0);
    if (in) x = *reinterpret_cast<const float4 *>((values ? a.v : a.k) + static_cast<size_t>(item) * HD + part * 4);
    const float top = group_max<kLanes>(fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w))), lane);
    if (slot < 0) return;
    const float inv = top > 0 ? 127.0f / top : 0.0f;
    auto quantised = [&](float v) {
        return static_cast<uint32_t>(static_cast<int>(fmaxf(-127.0f, fminf(127.0f, rintf(v * inv))))) & 0xFFu;
    };
    const size_t row = (static_cast<size_t>(seq) * a.kvheads + kh) * a.c.capacity + slot;
    *reinterpret_cast<uint32_t *>((values ? a.c.v8 : a.c.k8) + row * HD + part * 4) =
        quantised(x.x) | quantised(x.y) << 8 | quantised(x.z) << 16 | quantised(x.w) << 24;
    if (part == 0) (values ? a.c.vs : a.c.ks)[row] = top > 0 ? top / 127.0f : 1.0f;
}

template <int HD, int NW, Keys K>
__global__ __launch_bounds__(64 * NW, 2) void span_kernel(SpanArgs a) {
    span_block<HD, NW, K>(a, blockIdx.x);
}

// A shared prefix and the units' own keys in one launch: the first `far_blocks` blocks have the prefix.
template <int HD, int NW>
__global__ __launch_bounds__(64 * NW, 2) void span_two_kernel(SpanArgs far, SpanArgs own, int far_blocks) {
    const int b = blockIdx.x;
    if (b < far_blocks) span_block<HD, NW, Keys::Flat>(far, b);
    else span_block<HD, NW, Keys::Flat>(own, b - far_blocks);
}

template <int HD, int G>
__global__ __launch_bounds__(256) void span_join_kernel(SpanArgs a, int64_t rows) {
    constexpr int kRows = 256 / (G * (HD / 4));
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kRows;
    join_rows<HD, G>(a, row0, static_cast<int>(min(static_cast<int64_t>(kRows), rows - row0)));
}

// Block (kRecordSlots slots, kv head, unit); the first block of x joins the kv head's rows instead. The scores are on
// their way while the rows' sums are joined (16 sequences x 8 kv heads x 4 heads, up to 8192 slots: 9.1 -> 6.3 us).
constexpr int kRecordSlots = 512, kAhead = 8;  // heads whose scores are loaded ahead
template <int HD, int G>
__global__ __launch_bounds__(256) void span_record_kernel(SpanRecordArgs r) {
    const SpanArgs &a = r.a;
    const int kh = blockIdx.y, unit = blockIdx.z, t = threadIdx.x;
    const size_t row0 = static_cast<size_t>(unit) * a.heads + kh * a.group;
    if (blockIdx.x == 0) {
        join_rows<HD, G>(a, row0, a.group);
        return;
    }
    __shared__ float2 all[kSpanMaxGroup];
    const int n = min(a.lengths ? a.lengths[unit] : a.length, a.length);
    const int slot = (blockIdx.x - 1) * kRecordSlots + t;
    if (static_cast<int>(blockIdx.x - 1) * kRecordSlots >= n) return;
    const bool in[2] = {slot < n, slot + 256 < n};
    const float *x = a.scores + row0 * a.score_stride + slot;
    float *record = r.record + (static_cast<size_t>(unit) * a.kvheads + kh) * a.c.capacity + slot;
    float ahead[kAhead][2], sum[2] = {0.0f, 0.0f}, old[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
        old[u] = in[u] ? record[256 * u] : 0.0f;
#pragma unroll
        for (int g = 0; g < kAhead; ++g)
            ahead[g][u] = in[u] && g < a.group ? x[static_cast<size_t>(g) * a.score_stride + 256 * u] : 0.0f;
    }
    for (int g = t >> 6; g < a.group; g += 4) {
        const float2 v = join_sums(a, row0 + g, a.splits_total, t & 63, nullptr);
        if ((t & 63) == 0) all[g] = v;
    }
    __syncthreads();
    auto add = [&](int g, float s0, float s1) {
        const float2 v = all[g];
        if (!(v.y > 0)) return;  // no softmax
        const float inv = 1.0f / v.y;
        sum[0] += __builtin_amdgcn_exp2f(s0 - v.x) * inv;
        sum[1] += __builtin_amdgcn_exp2f(s1 - v.x) * inv;
    };
#pragma unroll
    for (int g = 0; g < kAhead; ++g)
        if (g < a.group) add(g, ahead[g][0], ahead[g][1]);
    for (int g = kAhead; g < a.group; ++g) {
        const float *s = x + static_cast<size_t>(g) * a.score_stride;
        add(g, in[0] ? s[0] : 0.0f, in[1] ? s[256] : 0.0f);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u)
        if (in[u]) record[256 * u] = old[u] + sum[u];
}

// f(head_dim, waves of a block)
template <class F>
void with_rows(int head_dim, int waves, F &&f) {
    auto by_waves = [&](auto hd) {
        if (waves == 4) f(hd, std::integral_constant<int, 4>{});
        else f(hd, std::integral_constant<int, 8>{});
    };
    switch (head_dim) {
    case 32: by_waves(std::integral_constant<int, 32>{}); break;
    case 64: by_waves(std::integral_constant<int, 64>{}); break;
    default: by_waves(std::integral_constant<int, 128>{}); break;
    }
}

int64_t row_tiles(const SpanArgs &a) { return (static_cast<int64_t>(a.count) * a.group + kSpanRows - 1) / kSpanRows; }

}  // namespace

void launch_span_store(const SpanStoreArgs &a, hipStream_t s) {
    const int64_t threads = static_cast<int64_t>(a.seqs) * a.count * a.kvheads * (a.head_dim / 2);
    if (threads <= 0) return;
    const dim3 grid(static_cast<unsigned>((threads + 255) / 256));
    switch (a.head_dim) {
    case 32: hipLaunchKernelGGL((span_store_kernel<32>), grid, dim3(256), 0, s, a); break;
    case 64: hipLaunchKernelGGL((span_store_kernel<64>), grid, dim3(256), 0, s, a); break;
    default: hipLaunchKernelGGL((span_store_kernel<128>), grid, dim3(256), 0, s, a); break;
    }
    ND_HIP(hipGetLastError());
}

void launch_span_two(const SpanArgs &far, const SpanArgs &own, int head_dim, hipStream_t s) {
    const int64_t far_blocks = row_tiles(far) * far.splits * far.kvheads;
    const dim3 grid(static_cast<unsigned>(far_blocks + static_cast<int64_t>(own.splits) * own.units * own.kvheads));
    with_rows(head_dim, far.waves, [&](auto hd, auto waves) {
        constexpr int HD = decltype(hd)::value, NW = decltype(waves)::value;
        hipLaunchKernelGGL((span_two_kernel<HD, NW>), grid, dim3(64 * NW), 0, s, far, own, static_cast<int>(far_blocks));
    });
    ND_HIP(hipGetLastError());
}

void launch_span(const SpanArgs &a, int head_dim, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(a.splits * row_tiles(a) * a.kvheads * a.units));
    with_rows(head_dim, a.waves, [&](auto hd, auto waves) {
        constexpr int HD = decltype(hd)::value, NW = decltype(waves)::value;
        if (a.positions) hipLaunchKernelGGL((span_kernel<HD, NW, Keys::Ring>), grid, dim3(64 * NW), 0, s, a);
        else hipLaunchKernelGGL((span_kernel<HD, NW, Keys::Flat>), grid, dim3(64 * NW), 0, s, a);
    });
    ND_HIP(hipGetLastError());
}

void launch_span_join(const SpanArgs &a, int head_dim, hipStream_t s) {
    ND_CHECK(a.splits_total <= kJoinMax, "attention: too many pieces");
    const int64_t rows = static_cast<int64_t>(a.units) * a.count * a.heads;
    with_join(head_dim, a.splits_total, [&](auto hd, auto groups) {
        constexpr int HD = decltype(hd)::value, G = decltype(groups)::value;
        constexpr int kRows = 256 / (G * (HD / 4));
        hipLaunchKernelGGL((span_join_kernel<HD, G>), dim3(static_cast<unsigned>((rows + kRows - 1) / kRows)), dim3(256), 0, s,
                           a, rows);
    });
    ND_HIP(hipGetLastError());
}

void launch_span_record(const SpanRecordArgs &r, int head_dim, hipStream_t s) {
    ND_CHECK(r.a.splits_total <= kJoinMax, "attention: too many pieces");
    const dim3 grid((r.a.length + kRecordSlots - 1) / kRecordSlots + 1, r.a.kvheads, r.a.units);
    with_join(head_dim, r.a.splits_total, [&](auto hd, auto groups) {
        hipLaunchKernelGGL((span_record_kernel<decltype(hd)::value, decltype(groups)::value>), grid, dim3(256), 0, s, r);
    });
    ND_HIP(hipGetLastError());
}

}  // namespace nd
