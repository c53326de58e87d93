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
#include "span_dev.h"

#include <cmath>
#include <type_traits>

namespace nd {

namespace {

__device__ __forceinline__ f32x4 mfma(const u32x4 &a, const u32x4 &b, const f32x4 &c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// One K or V row of HD values into codes and scale, by one wave (the cache's quantiser: top = max|x|, scale = top / 127 or
// 1, codes round(x * (127 / top))).
__device__ __forceinline__ void quantise_row(const float *x, int HD, int lane, int8_t *codes, float *scale) {
    float v[2];
    float top = 0.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        v[i] = lane + 64 * i < HD ? x[lane + 64 * i] : 0.0f;
        top = fmaxf(top, fabsf(v[i]));
    }
    top = wave_max(top, lane);
    const float inv = top > 0 ? 127.0f / top : 0.0f;
    if (lane == 0) *scale = top > 0 ? top / 127.0f : 1.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (lane + 64 * i < HD)
            codes[lane + 64 * i] = static_cast<int8_t>(fmaxf(-127.0f, fminf(127.0f, rintf(v[i] * inv))));
}

__device__ __forceinline__ void store_token(const SpanCache &c, const float *k, const float *v, size_t row, int HD, int lane) {
    quantise_row(k, HD, lane, c.k8 + row * HD, c.ks + row);
    quantise_row(v, HD, lane, c.v8 + row * HD, c.vs + row);
}

// One wave per (sequence, token, kv head).
__global__ __launch_bounds__(256) void span_store_kernel(SpanStoreArgs a) {
    const int64_t wave = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) >> 6;
    const int lane = threadIdx.x & 63;
    if (wave >= static_cast<int64_t>(a.seqs) * a.count * a.kvheads) return;
    const int kh = static_cast<int>(wave % a.kvheads);
    const int i = static_cast<int>((wave / a.kvheads) % a.count);
    const int seq = static_cast<int>(wave / (static_cast<int64_t>(a.kvheads) * a.count));
    int slot;
    if (a.positions) {
        const int p = at_position(a.positions[seq], i);
        slot = p < 0 ? -1 : ring_slot(p, a.sinks, a.c.capacity);
    } else {
        slot = min(a.lengths ? a.lengths[seq] : a.length, a.length) - 1;
    }
    if (slot < 0) return;
    const size_t src = static_cast<size_t>(wave) * a.head_dim;
    store_token(a.c, a.k + src, a.v + src, (static_cast<size_t>(seq) * a.kvheads + kh) * a.c.capacity + slot, a.head_dim, lane);
}

// Block (piece and row tile, kv head, unit): up to 16 query rows (the columns of both products' results), four waves
// with every fourth tile of 64 keys each, joined at the end.
//   Scores: operand A is 16 keys' codes, operand B the rows' q. Lane l holds row l % 16 and keys 16 t + 4 (l / 16) + i.
//   Values: operand B is p * vs straight from those registers (the contraction runs over the keys in their order:
//   depth 8 (l / 16) + j is key 32 u + 4 (l / 16) + j, and from j = 4 on 32 u + 16 + 4 (l / 16) + j - 4), operand A the V
//   codes of dimensions HD / 16 * (l % 16) + t. Result t of lane l is row l % 16, dimensions HD / 16 * (4 (l / 16) + i) + t.
template <int HD, bool RING>
__global__ __launch_bounds__(256, 2) void span_kernel(SpanArgs a) {
    constexpr int kSteps = HD / 32;        // of the score product's depth
    constexpr int kBytes = HD / 4;         // of a K row per lane
    constexpr int VB = HD / 16;            // bytes of a V row per lane
    __shared__ __attribute__((aligned(16))) float sc[4][2][kSpanTile];  // K (times scale) and V scales of a wave's tile
    __shared__ __attribute__((aligned(16))) float so[4][kSpanRows][HD + 4];
    __shared__ float sm[4][kSpanRows], sl[4][kSpanRows];

    const int t = threadIdx.x, lane = t & 63, col = lane & 15, quad = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int kh = blockIdx.y, unit = blockIdx.z;
    const int piece = blockIdx.x % a.splits, tile0 = blockIdx.x / a.splits;
    const int rows = a.count * a.group;
    const int row = tile0 * kSpanRows + col;
    const int last_row = min(rows, (tile0 + 1) * kSpanRows) - 1;
    const bool live = row < rows;
    const int cap = a.c.capacity;

    KeyRuns runs = {0, 0, 0, 0, 0, 0};
    int own = 0;           // the row's position
    int full_low = 0, full_high = 0;  // positions that every row of the block attends: (full_low, full_high]
    if constexpr (RING) {
        const int first = a.positions[unit];
        const int p0 = at_position(first, tile0 * kSpanRows / a.group), p1 = at_position(first, last_row / a.group);
        runs = ring_runs(p0, p1, a.sinks, a.window, cap);
        own = at_position(first, (live ? row : last_row) / a.group);
        full_low = p1 >= a.window ? p1 - a.window : -1;
        full_high = p0;
    } else {
        const int n = min(a.lengths ? a.lengths[unit] : a.length, a.length);
        runs.n0 = runs.pinned = n > 0 ? n : 0;
    }
    const int tiles0 = span_tiles(runs.n0), tiles = tiles0 + span_tiles(runs.n1);
    const int begin = piece * a.per, end = min(begin + a.per, tiles);

    const size_t row0 = (static_cast<size_t>(unit) * a.kvheads + kh) * cap;
    if (a.new_k && tiles > 0) {
        // the newest token's slot is the last of run 1, or of run 0 where that is empty or wraps
        const bool in1 = runs.n1 > 0 && !(RING && runs.n0 > runs.pinned);
        const int slot = in1 ? runs.begin1 + runs.n1 - 1 : runs.n0 - 1;
        const int in_tile = in1 ? tiles - 1 : tiles0 - 1;
        if (in_tile >= begin && in_tile < end) {
            if (wave == 0) {
                const size_t src = (static_cast<size_t>(unit) * a.kvheads + kh) * HD;
                store_token(a.c, a.new_k + src, a.new_v + src, row0 + slot, HD, lane);
            }
            __syncthreads();
        }
    }
    const auto rk = buffer_rsrc(a.c.k8 + row0 * HD, static_cast<uint32_t>(cap) * HD);
    const auto rv = buffer_rsrc(a.c.v8 + row0 * HD, static_cast<uint32_t>(cap) * HD);
    const auto rks = buffer_rsrc(a.c.ks + row0, static_cast<uint32_t>(cap) * 4u);
    const auto rvs = buffer_rsrc(a.c.vs + row0, static_cast<uint32_t>(cap) * 4u);

    // first slot of a tile, and the first slot behind its run
    auto slot0 = [&](int tile) { return tile < tiles0 ? tile * kSpanTile : runs.begin1 + (tile - tiles0) * kSpanTile; };
    auto stop = [&](int tile) { return tile < tiles0 ? runs.n0 : runs.begin1 + runs.n1; };

    struct Tile {
        uint32_t k[4][kSteps][2];
        uint32_t v[4][4][(VB + 3) / 4];
        float ks, vs;
    };
    // Loads past the cache's rows read zero; slots of a tile behind its run are masked in compute.
    auto load = [&](Tile &T, int tile) {
        const uint32_t s0 = static_cast<uint32_t>(slot0(tile));
        const uint32_t kb = (s0 + col) * HD + quad * kBytes;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (HD == 32) {
                const auto w = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rk, kb + i * 16 * HD, 0, 0));
                T.k[i][0][0] = w.x;
                T.k[i][0][1] = w.y;
            } else {
#pragma unroll
                for (int h = 0; h < kSteps / 2; ++h) {
                    const u32x4 w = __builtin_amdgcn_raw_buffer_load_b128(rk, kb + i * 16 * HD + h * 16, 0, 0);
                    T.k[i][2 * h][0] = w.x;
                    T.k[i][2 * h][1] = w.y;
                    T.k[i][2 * h + 1][0] = w.z;
                    T.k[i][2 * h + 1][1] = w.w;
                }
            }
        }
        T.ks = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rks, (s0 + lane) * 4u, 0, 0));
        T.vs = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rvs, (s0 + lane) * 4u, 0, 0));
        const uint32_t vb = (s0 + 4 * quad) * HD + col * VB;
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const uint32_t at = vb + (16 * i + u) * HD;
                if constexpr (VB == 8) {
                    const auto w = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(rv, at, 0, 0));
                    T.v[i][u][0] = w.x;
                    T.v[i][u][1] = w.y;
                } else if constexpr (VB == 4) {
                    T.v[i][u][0] = __builtin_amdgcn_raw_buffer_load_b32(rv, at, 0, 0);
                } else {
                    T.v[i][u][0] = static_cast<uint16_t>(__builtin_amdgcn_raw_buffer_load_b16(rv, at, 0, 0));
                }
            }
    };

    // q as operand B: lane (row col, quad) holds dimensions quad * HD / 4 .. in steps of eight
    const size_t orow = (static_cast<size_t>(unit) * a.count + (live ? row : 0) / a.group) * a.heads + kh * a.group +
                        (live ? row : 0) % a.group;
    Terms q[kSteps];
    {
        float x[kSteps][8];
#pragma unroll
        for (int c = 0; c < kSteps; ++c) {
            const float4 *src = reinterpret_cast<const float4 *>(a.q + orow * HD + quad * kBytes + c * 8);
            const float4 u = src[0], w = src[1];
            const float both[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
#pragma unroll
            for (int j = 0; j < 8; ++j) x[c][j] = live ? both[j] : 0.0f;
        }
#pragma unroll
        for (int c = 0; c < kSteps; ++c) q[c] = split8(x[c]);
    }

    float m = -INFINITY, l = 0.0f;
    f32x4 acc[VB];
#pragma unroll
    for (int i = 0; i < VB; ++i) acc[i] = f32x4{0, 0, 0, 0};

    auto compute = [&](const Tile &T, int tile) {
        const int s0 = slot0(tile), behind = stop(tile);
        // LDS operations of one wave complete in order; the fences only keep the compiler from reordering them
        sc[wave][0][lane] = T.ks * a.scale;
        sc[wave][1][lane] = T.vs;
        __builtin_amdgcn_wave_barrier();
        asm volatile("" ::: "memory");
        float x[4][4], vs[4][4];
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f32x4 d = {0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < kSteps; ++c) {
                const u32x4 k = widen(T.k[i][c][0], T.k[i][c][1]);
                d = mfma(k, q[c].t[2], d);
                d = mfma(k, q[c].t[1], d);
                d = mfma(k, q[c].t[0], d);
            }
            const float4 ks = *reinterpret_cast<const float4 *>(&sc[wave][0][16 * i + 4 * quad]);
            const float4 v4 = *reinterpret_cast<const float4 *>(&sc[wave][1][16 * i + 4 * quad]);
            const float ksv[4] = {ks.x, ks.y, ks.z, ks.w}, vsv[4] = {v4.x, v4.y, v4.z, v4.w};
            const float dv[4] = {d.x, d.y, d.z, d.w};
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                x[i][u] = dv[u] * ksv[u];
                vs[i][u] = vsv[u];
            }
        }
        __builtin_amdgcn_wave_barrier();
        asm volatile("" ::: "memory");
        bool masked = s0 + kSpanTile > behind;
        if constexpr (RING) {
            const int shift = tile < tiles0 ? runs.shift0 : runs.shift1;
            const bool all_pinned = s0 + kSpanTile <= runs.pinned;
            // pinned ones are seen by every row from their position on
            masked |= all_pinned ? s0 + kSpanTile - 1 > full_high
                                 : s0 < runs.pinned || s0 + shift <= full_low || s0 + kSpanTile - 1 + shift > full_high;
        }
        if (masked) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const int slot = s0 + 16 * i + 4 * quad + u;
                    bool ok = slot < behind;
                    if constexpr (RING) {
                        const bool pin = tile < tiles0 && slot < runs.pinned;
                        const int p = pin ? slot : slot + (tile < tiles0 ? runs.shift0 : runs.shift1);
                        ok = ok && p <= own && (pin || own - p < a.window);
                    }
                    x[i][u] = ok ? x[i][u] : -INFINITY;
                    vs[i][u] = ok ? vs[i][u] : 0.0f;
                }
        }
        if (a.scores && live) {
            float *to = a.scores + (static_cast<size_t>(unit) * a.kvheads * a.group + kh * a.group + row) * a.score_stride + s0;
#pragma unroll
            for (int i = 0; i < 4; ++i)
                *reinterpret_cast<float4 *>(to + 16 * i + 4 * quad) = make_float4(x[i][0], x[i][1], x[i][2], x[i][3]);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int u = 0; u < 4; ++u) top = fmaxf(top, x[i][u]);
        top = fmaxf(top, butterfly_partner<16>(top, lane));
        top = fmaxf(top, butterfly_partner<32>(top, lane));
        const float mn = fmaxf(m, top);
        const float base = mn == -INFINITY ? 0.0f : mn;  // nothing attended yet: every power is 0
        const float alpha = __builtin_amdgcn_exp2f(m - base);
        m = mn;
        float sum = 0.0f;
        float w[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const float p = __builtin_amdgcn_exp2f(x[i][u] - base);
                sum += p;
                w[i][u] = p * vs[i][u];
            }
        l = __builtin_fmaf(l, alpha, sum);
#pragma unroll
        for (int i = 0; i < VB; ++i) acc[i] *= alpha;
        const bool odd = __any(!(fabsf(T.vs) < INFINITY));  // an infinite or NaN V scale
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float both[8];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                both[j] = w[2 * u][j];
                both[4 + j] = w[2 * u + 1][j];
            }
            const Terms p = odd ? split8_any(both) : split8(both);
#pragma unroll
            for (int i = 0; i < VB; ++i) {
                float f[8];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    f[j] = code(T.v[2 * u][j][i / 4], i % 4);
                    f[4 + j] = code(T.v[2 * u + 1][j][i / 4], i % 4);
                }
                const u32x4 v = {upper_halves(f[0], f[1]), upper_halves(f[2], f[3]), upper_halves(f[4], f[5]),
                                 upper_halves(f[6], f[7])};
                acc[i] = mfma(v, p.t[2], acc[i]);
                acc[i] = mfma(v, p.t[1], acc[i]);
                acc[i] = mfma(v, p.t[0], acc[i]);
            }
        }
    };

    // the next tile is loaded before this one is computed
    Tile cur, nxt;
    int tile = begin + wave;
    load(cur, tile);
    for (; tile < end; tile += 4) {
        load(nxt, tile + 4);
        asm volatile("" ::: "memory");
        compute(cur, tile);
        cur = nxt;
    }

    // the waves' results over their own maxima
    l += butterfly_partner<16>(l, lane);
    l += butterfly_partner<32>(l, lane);
    if (quad == 0) {
        sm[wave][col] = m;
        sl[wave][col] = l;
    }
#pragma unroll
    for (int i = 0; i < VB; ++i) {
        const float d4[4] = {acc[i].x, acc[i].y, acc[i].z, acc[i].w};
#pragma unroll
        for (int u = 0; u < 4; ++u) so[wave][col][VB * (4 * quad + u) + i] = d4[u];
    }
    __syncthreads();
    for (int i = t; i < kSpanRows * HD / 4; i += 256) {
        const int r = i / (HD / 4), d = i % (HD / 4) * 4;
        const int grow = tile0 * kSpanRows + r;
        if (grow >= rows) break;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) M = fmaxf(M, sm[w][r]);
        const float base = M == -INFINITY ? 0.0f : M;
        float L = 0.0f, o[4] = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            if (sm[w][r] == -INFINITY && sl[w][r] == 0.0f) continue;  // nothing attended
            const float f = __builtin_amdgcn_exp2f(sm[w][r] - base);
            L = __builtin_fmaf(f, sl[w][r], L);
            const float4 p = *reinterpret_cast<const float4 *>(&so[w][r][d]);
            o[0] = __builtin_fmaf(f, p.x, o[0]);
            o[1] = __builtin_fmaf(f, p.y, o[1]);
            o[2] = __builtin_fmaf(f, p.z, o[2]);
            o[3] = __builtin_fmaf(f, p.w, o[3]);
        }
        const size_t at = (static_cast<size_t>(unit) * a.count + grow / a.group) * a.heads + kh * a.group + grow % a.group;
        if (!a.rec_o) {
            const float inv = L > 0 ? 1.0f / L : 0.0f;
            *reinterpret_cast<float4 *>(a.out + at * HD + d) =
                L > 0 ? make_float4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv) : make_float4(0, 0, 0, 0);
        } else {
            const size_t rec = at * a.splits_total + a.split0 + piece;
            *reinterpret_cast<float4 *>(a.rec_o + rec * HD + d) = make_float4(o[0], o[1], o[2], o[3]);
            if (d == 0) a.rec_ml[rec] = make_float2(M, L);
        }
    }
}

// A row's maximum and sum over its records, by one wave; the records' factors 2^(m - maximum) to `factor` if that is set.
__device__ __forceinline__ float2 join_sums(const SpanArgs &a, size_t row, int lane, float *factor) {
    const float2 *ml = a.rec_ml + row * a.splits_total;
    float2 mine = make_float2(-INFINITY, 0.0f);  // of this lane's first record: most rows have no second
    float M = -INFINITY;
    for (int s = lane; s < a.splits_total; s += 64) {
        const float2 v = ml[s];
        if (s == lane) mine = v;
        M = fmaxf(M, v.x);
    }
    M = wave_max(M, lane);
    const float base = M == -INFINITY ? 0.0f : M;
    float L = 0.0f;
    for (int s = lane; s < a.splits_total; s += 64) {
        const float2 v = s == lane ? mine : ml[s];
        const bool empty = v.x == -INFINITY && v.y == 0.0f;
        const float f = empty ? 0.0f : __builtin_amdgcn_exp2f(v.x - base);
        if (factor) factor[s] = f;
        L += empty ? 0.0f : f * v.y;
    }
    return make_float2(base, wave_sum(L, lane));
}

// Rows row0 .. row0 + count - 1 from their records, by a block of 256: G groups of HD / 4 lanes share a row's records
// (every G-th each), whose loads do not wait for each other; 256 / (G * HD / 4) rows at a time. The sums' order depends
// on the number of records only.
constexpr int kJoinMax = 1024;  // records of a row
template <int HD, int G>
__device__ __forceinline__ void join_rows(const SpanArgs &a, size_t row0, int count) {
    constexpr int kLanes = HD / 4, kRows = 256 / (G * kLanes);
    constexpr int kFactors = kRows * (G == 8 ? kJoinMax : G);
    __shared__ float factor[kFactors];
    __shared__ float total[kRows];
    __shared__ __attribute__((aligned(16))) float part[G > 1 ? G : 1][kRows][HD];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int splits = a.splits_total;
    const int d = t % kLanes * 4, g = t / kLanes % G, r = t / (kLanes * G);
    for (int i0 = 0; i0 < count; i0 += kRows) {
        for (int i = wave; i < kRows && i0 + i < count; i += 4) {
            const float2 all = join_sums(a, row0 + i0 + i, lane, factor + i * splits);
            if (lane == 0) total[i] = all.y;
        }
        __syncthreads();
        const bool live = i0 + r < count;
        float4 o = make_float4(0, 0, 0, 0);
        if (live) {
            const float *rec = a.rec_o + (row0 + i0 + r) * splits * HD + d;
#pragma unroll 4
            for (int s = g; s < splits; s += G) {
                const float f = factor[r * splits + s];
                const float4 p = *reinterpret_cast<const float4 *>(rec + static_cast<size_t>(s) * HD);
                if (f == 0.0f) continue;  // an empty piece, or weights that vanish beside the rest
                o.x = __builtin_fmaf(f, p.x, o.x);
                o.y = __builtin_fmaf(f, p.y, o.y);
                o.z = __builtin_fmaf(f, p.z, o.z);
                o.w = __builtin_fmaf(f, p.w, o.w);
            }
        }
        if constexpr (G > 1) {
            *reinterpret_cast<float4 *>(&part[g][r][d]) = o;
            __syncthreads();
            if (g == 0) {
#pragma unroll
                for (int k = 1; k < G; ++k) {
                    const float4 p = *reinterpret_cast<const float4 *>(&part[k][r][d]);
                    o.x += p.x;
                    o.y += p.y;
                    o.z += p.z;
                    o.w += p.w;
                }
            }
        }
        if (live && g == 0) {
            const float L = total[r], inv = 1.0f / L;
            *reinterpret_cast<float4 *>(a.out + (row0 + i0 + r) * HD + d) =
                L > 0 ? make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv) : make_float4(0, 0, 0, 0);
        }
        __syncthreads();
    }
}

template <int HD, int G>
__global__ __launch_bounds__(256) void span_join_kernel(SpanArgs a, int64_t rows) {
    constexpr int kRows = 256 / (G * (HD / 4));
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kRows;
    join_rows<HD, G>(a, row0, static_cast<int>(min(static_cast<int64_t>(kRows), rows - row0)));
}

// Block (256 slots, kv head, unit); the first block of x joins the kv head's rows instead.
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
    if (static_cast<int>(blockIdx.x - 1) * 256 >= n) return;
    for (int g = t >> 6; g < a.group; g += 4) {
        const float2 v = join_sums(a, row0 + g, t & 63, nullptr);
        if ((t & 63) == 0) all[g] = v;
    }
    __syncthreads();
    const int slot = (blockIdx.x - 1) * 256 + t;
    if (slot >= n) return;
    const float *x = a.scores + row0 * a.score_stride + slot;
    float sum = 0.0f;
    for (int g = 0; g < a.group; ++g) {
        const float2 v = all[g];
        if (v.y > 0) sum += __builtin_amdgcn_exp2f(x[static_cast<size_t>(g) * a.score_stride] - v.x) * (1.0f / v.y);
    }
    r.record[(static_cast<size_t>(unit) * a.kvheads + kh) * a.c.capacity + slot] += sum;
}

template <int HD>
void launch_span_hd(const SpanArgs &a, hipStream_t s) {
    const int64_t tiles = (static_cast<int64_t>(a.count) * a.group + kSpanRows - 1) / kSpanRows;
    const dim3 grid(static_cast<unsigned>(a.splits * tiles), a.kvheads, a.units);
    if (a.positions) hipLaunchKernelGGL((span_kernel<HD, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((span_kernel<HD, false>), grid, dim3(256), 0, s, a);
    ND_HIP(hipGetLastError());
}

}  // namespace

void launch_span_store(const SpanStoreArgs &a, hipStream_t s) {
    const int64_t waves = static_cast<int64_t>(a.seqs) * a.count * a.kvheads;
    if (waves <= 0) return;
    hipLaunchKernelGGL(span_store_kernel, dim3(static_cast<unsigned>((waves + 3) / 4)), dim3(256), 0, s, a);
    ND_HIP(hipGetLastError());
}

void launch_span(const SpanArgs &a, int head_dim, hipStream_t s) {
    switch (head_dim) {
    case 32: launch_span_hd<32>(a, s); break;
    case 64: launch_span_hd<64>(a, s); break;
    default: launch_span_hd<128>(a, s); break;
    }
}

namespace {

// F(head_dim, groups that share a row's records)
template <class F>
void with_join(int head_dim, int splits, F &&f) {
    auto groups = [&](auto hd) {
        if (splits <= 1) f(hd, std::integral_constant<int, 1>{});
        else if (splits <= 2) f(hd, std::integral_constant<int, 2>{});
        else if (splits <= 4) f(hd, std::integral_constant<int, 4>{});
        else f(hd, std::integral_constant<int, 8>{});
    };
    switch (head_dim) {
    case 32: groups(std::integral_constant<int, 32>{}); break;
    case 64: groups(std::integral_constant<int, 64>{}); break;
    default: groups(std::integral_constant<int, 128>{}); break;
    }
}

}  // namespace

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
    const dim3 grid((r.a.length + 255) / 256 + 1, r.a.kvheads, r.a.units);
    with_join(head_dim, r.a.splits_total, [&](auto hd, auto groups) {
        hipLaunchKernelGGL((span_record_kernel<decltype(hd)::value, decltype(groups)::value>), grid, dim3(256), 0, s, r);
    });
    ND_HIP(hipGetLastError());
}

}  // namespace nd
