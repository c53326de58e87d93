// gfx950 kernel of span attention with many query rows over the same keys: prompt pieces, and a batch over its shared
// prefix. The mathematics and the records are span_kernels.hip's; both products run on v_mfma_f32_32x32x16_bf16.
#include "span_dev.h"

namespace nd {

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ f32x16 mfma32(const u32x4 &a, const u32x4 &b, const f32x16 &c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// A wave's running maximum moves only when a score is this much above it (powers of two): weights up to 2^kSlack are as
// exact as weights up to 1, and most tiles leave the outputs unscaled.
constexpr float kSlack = 16.0f;

constexpr int kFrag = 66;  // 16-byte lanes of an operand in LDS: 32, one of padding (the halves in different banks), 32, 1
__device__ __forceinline__ int frag_lane(int m, int half) { return m + 33 * half; }

// Block (W row groups of 32 and piece, with unit and kv head): W waves over the same tiles of 32 keys, which the block
// turns into bfloat16 operands in LDS once, the next tile's codes in flight meanwhile (two buffers, one barrier a tile).
//   Scores: operand A is 32 keys' codes, operand B the wave's 32 rows of q. Lane l holds row l % 32 and of each 32 keys
//   8 (i / 4) + 4 (l / 32) + i % 4, i < 16.
//   Values: operand B is p * vs straight from those registers, operand A the V codes in the same order of keys. Result t
//   of lane l is row l % 32, dimensions DT * (8 (i / 4) + 4 (l / 32) + i % 4) + t (DT = HD / 32 results).
template <int HD, int W, bool RING>
__global__ __launch_bounds__(64 * W, 2) void span_wide_kernel(SpanArgs a) {
    constexpr int KS = HD / 16;                     // steps of the score product's depth
    constexpr int DT = HD / 32;                     // results of 32 dimensions
    constexpr int T = 64 * W;
    constexpr int kChunks = 2 * HD;                 // of a tile's K codes, 16 bytes each; and pieces of V, 4 keys x 4 dimensions
    constexpr int C = (kChunks + T - 1) / T;        // of each per thread
    __shared__ u32x4 kf[2][KS][kFrag];
    __shared__ u32x4 vf[2][2][DT][kFrag];
    __shared__ __attribute__((aligned(16))) float sc[2][2][kWideTile];  // K (times scale) and V scales

    const int t = threadIdx.x, lane = t & 63, col = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int pairs = a.units * a.kvheads;
    const int pair = blockIdx.x % pairs, rest = blockIdx.x / pairs;
    const int unit = pair / a.kvheads, kh = pair % a.kvheads;
    const int piece = rest % a.splits, tile_rows = rest / a.splits * (32 * W);
    const int rows = a.count * a.group;
    const int last_row = min(rows, tile_rows + 32 * W) - 1;
    const int row = tile_rows + wave * 32 + col;
    const bool live = row < rows;
    const int cap = a.c.capacity;

    KeyRuns runs = {0, 0, 0, 0, 0, 0};
    int own = 0, full_low = 0, full_high = 0;  // as in span_kernel
    if constexpr (RING) {
        const int first = a.positions[unit];
        const int p0 = at_position(first, tile_rows / a.group), p1 = at_position(first, last_row / a.group);
        runs = ring_runs(p0, p1, a.sinks, a.window, cap);
        own = at_position(first, (live ? row : last_row) / a.group);
        full_low = p1 >= a.window ? p1 - a.window : -1;
        full_high = p0;
    } else {
        const int n = min(a.lengths ? a.lengths[unit] : a.length, a.length);
        runs.n0 = runs.pinned = n > 0 ? n : 0;
    }
    const int tiles0 = wide_tiles(runs.n0), tiles = tiles0 + wide_tiles(runs.n1);
    const int begin = piece * a.per, end = min(begin + a.per, tiles);
    auto slot0 = [&](int tile) { return tile < tiles0 ? tile * kWideTile : runs.begin1 + (tile - tiles0) * kWideTile; };
    auto stop = [&](int tile) { return tile < tiles0 ? runs.n0 : runs.begin1 + runs.n1; };

    const size_t row0 = (static_cast<size_t>(unit) * a.kvheads + kh) * cap;
    const auto rk = buffer_rsrc(a.c.k8 + row0 * HD, static_cast<uint32_t>(cap) * HD);
    const auto rv = buffer_rsrc(a.c.v8 + row0 * HD, static_cast<uint32_t>(cap) * HD);
    const auto rks = buffer_rsrc(a.c.ks + row0, static_cast<uint32_t>(cap) * 4u);
    const auto rvs = buffer_rsrc(a.c.vs + row0, static_cast<uint32_t>(cap) * 4u);

    // A tile's codes on their way to LDS: K as 16 dimensions of a key, V as 8 dimensions of 4 keys. Loads past the
    // cache's rows read zero.
    struct Raw {
        u32x4 k[C];
        uint32_t v[C][4];
        float s[2];  // K and V scale of key `col`
    };
    auto fetch = [&](Raw &r, int tile) {
        const uint32_t s0 = static_cast<uint32_t>(slot0(tile));
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const int c = t + i * T, keys = c / (HD / 4), dims = c % (HD / 4);
            r.k[i] = __builtin_amdgcn_raw_buffer_load_b128(rk, s0 * HD + c * 16, 0, 0);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                r.v[i][j] = __builtin_amdgcn_raw_buffer_load_b32(rv, (s0 + 4 * keys + j) * HD + dims * 4, 0, 0);
        }
        const uint32_t at = (s0 + col) * 4u;
        r.s[0] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rks, at, 0, 0));
        r.s[1] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rvs, at, 0, 0));
    };
    auto place = [&](const Raw &r, int buf) {
#pragma unroll
        for (int i = 0; i < C; ++i) {
            const int c = t + i * T;
            if (kChunks % T != 0 && c >= kChunks) break;
            const int key = c / KS, step = c % KS;
            kf[buf][step][frag_lane(key, 0)] = widen(r.k[i].x, r.k[i].y);
            kf[buf][step][frag_lane(key, 1)] = widen(r.k[i].z, r.k[i].w);
            const int keys = c / (HD / 4), dims = c % (HD / 4);  // 4 keys: half and quarter of a step's depth
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                float f[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) f[j] = code(r.v[i][j], b);
                const int d = dims * 4 + b;
                u32x2 *to = reinterpret_cast<u32x2 *>(&vf[buf][keys / 4][d % DT][frag_lane(d / DT, keys & 1)]);
                to[(keys >> 1) & 1] = u32x2{upper_halves(f[0], f[1]), upper_halves(f[2], f[3])};
            }
        }
        if (wave == 0) sc[buf][half][col] = half ? r.s[1] : r.s[0] * a.scale;
    };

    Raw raw;
    fetch(raw, begin);

    // q as operand B: lane (row col, half) holds dimensions 16 c + 8 half .. of step c
    const size_t orow = (static_cast<size_t>(unit) * a.count + (live ? row : 0) / a.group) * a.heads + kh * a.group +
                        (live ? row : 0) % a.group;
    Terms q[KS];
    {
        const float4 *src = reinterpret_cast<const float4 *>(a.q + orow * HD + half * 8);
#pragma unroll
        for (int c = 0; c < KS; ++c) {
            const float4 u = src[4 * c], w = src[4 * c + 1];
            const float both[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) x[j] = live ? both[j] : 0.0f;
            q[c] = split8(x);
        }
    }

    float m = -INFINITY, l = 0.0f;
    f32x16 acc[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[i][j] = 0.0f;

    auto compute = [&](int buf, int tile) {
        const int s0 = slot0(tile), behind = stop(tile);
        f32x16 x;
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = 0.0f;
#pragma unroll
        for (int c = 0; c < KS; ++c) {
            const u32x4 k = kf[buf][c][frag_lane(col, half)];
            x = mfma32(k, q[c].t[2], x);
            x = mfma32(k, q[c].t[1], x);
            x = mfma32(k, q[c].t[0], x);
        }
        const bool odd = __any(!(fabsf(sc[buf][1][col]) < INFINITY));  // an infinite or NaN V scale
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float4 ks = *reinterpret_cast<const float4 *>(&sc[buf][0][8 * g + 4 * half]);
            x[4 * g] *= ks.x;
            x[4 * g + 1] *= ks.y;
            x[4 * g + 2] *= ks.z;
            x[4 * g + 3] *= ks.w;
        }
        bool masked = s0 + kWideTile > behind;
        if constexpr (RING) {
            const int shift = tile < tiles0 ? runs.shift0 : runs.shift1;
            const bool all_pinned = s0 + kWideTile <= runs.pinned;
            masked |= all_pinned ? s0 + kWideTile - 1 > full_high
                                 : s0 < runs.pinned || s0 + shift <= full_low || s0 + kWideTile - 1 + shift > full_high;
        }
        uint32_t gone = 0;  // this lane's keys that the row does not attend
        if (masked) {
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const int slot = s0 + 8 * (j / 4) + 4 * half + j % 4;
                bool ok = slot < behind;
                if constexpr (RING) {
                    const bool pin = tile < tiles0 && slot < runs.pinned;
                    const int p = pin ? slot : slot + (tile < tiles0 ? runs.shift0 : runs.shift1);
                    ok = ok && p <= own && (pin || own - p < a.window);
                }
                x[j] = ok ? x[j] : -INFINITY;
                gone |= ok ? 0u : 1u << j;
            }
        }
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 16; ++j) top = fmaxf(top, x[j]);
        top = fmaxf(top, butterfly_partner<32>(top, lane));
        if (__any(top > m + kSlack)) {  // (m = -inf: the first scores)
            const float mn = fmaxf(m, top);
            const float alpha = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int i = 0; i < DT; ++i) acc[i] *= alpha;
        }
        const float base = m == -INFINITY ? 0.0f : m;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float4 v4 = *reinterpret_cast<const float4 *>(&sc[buf][1][8 * g + 4 * half]);
            const float vs[4] = {v4.x, v4.y, v4.z, v4.w};
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const float p = __builtin_amdgcn_exp2f(x[4 * g + u] - base);
                l += p;
                x[4 * g + u] = p * vs[u];
            }
        }
        if (masked) {  // whatever scale a masked slot has
#pragma unroll
            for (int j = 0; j < 16; ++j) x[j] = gone >> j & 1u ? 0.0f : x[j];
        }
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
            float w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) w[j] = x[8 * ks + j];
            const Terms p = odd ? split8_any(w) : split8(w);
#pragma unroll
            for (int i = 0; i < DT; ++i) {
                const u32x4 v = vf[buf][ks][i][frag_lane(col, half)];
                acc[i] = mfma32(v, p.t[2], acc[i]);
                acc[i] = mfma32(v, p.t[1], acc[i]);
                acc[i] = mfma32(v, p.t[0], acc[i]);
            }
        }
    };

    int buf = 0;
    place(raw, buf);
    __syncthreads();
    for (int tile = begin; tile < end; ++tile) {
        fetch(raw, tile + 1);
        asm volatile("" ::: "memory");
        compute(buf, tile);
        buf ^= 1;
        place(raw, buf);
        __syncthreads();
    }

    l += butterfly_partner<32>(l, lane);
    if (!live) return;
    const bool finish = !a.rec_o;
    const size_t rec = orow * a.splits_total + a.split0 + piece;
    float *to = finish ? a.out + orow * HD : a.rec_o + rec * HD;
    const float inv = !finish ? 1.0f : l > 0 ? 1.0f / l : 0.0f;
    const bool none = finish && !(l > 0);  // nothing attended, or no softmax
    if (!finish && half == 0) a.rec_ml[rec] = make_float2(m, l);
#pragma unroll
    for (int j = 0; j < 16; ++j) {
        const int d = DT * (8 * (j / 4) + 4 * half + j % 4);
        float o[DT];
#pragma unroll
        for (int i = 0; i < DT; ++i) o[i] = none ? 0.0f : acc[i][j] * inv;
        if constexpr (DT == 4) *reinterpret_cast<float4 *>(to + d) = make_float4(o[0], o[1], o[2], o[3]);
        else if constexpr (DT == 2) *reinterpret_cast<float2 *>(to + d) = make_float2(o[0], o[1]);
        else to[d] = o[0];
    }
}

template <int HD, int W>
void launch_wide_hd(const SpanArgs &a, hipStream_t s) {
    const int64_t tiles = (static_cast<int64_t>(a.count) * a.group + 32 * W - 1) / (32 * W);
    const dim3 grid(static_cast<unsigned>(tiles * a.splits * a.units * a.kvheads));
    if (a.positions) hipLaunchKernelGGL((span_wide_kernel<HD, W, true>), grid, dim3(64 * W), 0, s, a);
    else hipLaunchKernelGGL((span_wide_kernel<HD, W, false>), grid, dim3(64 * W), 0, s, a);
    ND_HIP(hipGetLastError());
}

template <int HD>
void launch_wide_w(const SpanArgs &a, int waves, hipStream_t s) {
    switch (waves) {
    case 1: launch_wide_hd<HD, 1>(a, s); break;
    case 2: launch_wide_hd<HD, 2>(a, s); break;
    case 3: launch_wide_hd<HD, 3>(a, s); break;
    default: launch_wide_hd<HD, 4>(a, s); break;
    }
}

}  // namespace

void launch_span_wide(const SpanArgs &a, int head_dim, int waves, hipStream_t s) {
    switch (head_dim) {
    case 32: launch_wide_w<32>(a, waves, s); break;
    case 64: launch_wide_w<64>(a, waves, s); break;
    default: launch_wide_w<128>(a, waves, s); break;
    }
}

}  // namespace nd
