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
#include "span.h"
#include "wave.h"

#include <cmath>

namespace nd {

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float code(uint32_t w, int c) {
    return static_cast<float>(static_cast<int8_t>((w >> (8 * c)) & 0xffu));
}

// bfloat16 pair of the upper halves of two fp32 values (the low half from a).
__device__ __forceinline__ uint32_t upper_halves(float a, float b) {
    return __builtin_amdgcn_perm(__builtin_bit_cast(uint32_t, b), __builtin_bit_cast(uint32_t, a), 0x07060302u);
}
__device__ __forceinline__ float cut(float x) {
    return __builtin_bit_cast(float, __builtin_bit_cast(uint32_t, x) & 0xFFFF0000u);
}

struct Terms {
    u32x4 t[3];  // eight values as three bfloat16 terms, the largest first
};

// The three terms of values 2 i and 2 i + 1. Exact for finite values: every cut leaves 8 bits less.
__device__ __forceinline__ void split_pair(float a, float b, uint32_t &t0, uint32_t &t1, uint32_t &t2) {
    t0 = upper_halves(a, b);
    a -= cut(a);
    b -= cut(b);
    t1 = upper_halves(a, b);
    a -= cut(a);
    b -= cut(b);
    t2 = upper_halves(a, b);
}
__device__ __forceinline__ Terms split8(const float (&x)[8]) {
    uint32_t t[3][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) split_pair(x[2 * i], x[2 * i + 1], t[0][i], t[1][i], t[2][i]);
    Terms r;
#pragma unroll
    for (int k = 0; k < 3; ++k) r.t[k] = u32x4{t[k][0], t[k][1], t[k][2], t[k][3]};
    return r;
}

// The same where values may be infinite or NaN: those are their first term alone.
__device__ __forceinline__ Terms split8_any(const float (&x)[8]) {
    float y[8];
    bool odd[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        odd[i] = !(fabsf(x[i]) < INFINITY);
        y[i] = odd[i] ? 0.0f : x[i];
    }
    Terms r = split8(y);
#pragma unroll
    for (int i = 0; i < 8; ++i) y[i] = odd[i] ? x[i] : y[i];
    r.t[0] = u32x4{upper_halves(y[0], y[1]), upper_halves(y[2], y[3]), upper_halves(y[4], y[5]), upper_halves(y[6], y[7])};
    return r;
}

// Eight codes of two dwords as bfloat16.
__device__ __forceinline__ u32x4 widen(uint32_t a, uint32_t b) {
    return u32x4{upper_halves(code(a, 0), code(a, 1)), upper_halves(code(a, 2), code(a, 3)),
                 upper_halves(code(b, 0), code(b, 1)), upper_halves(code(b, 2), code(b, 3))};
}

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

__device__ __forceinline__ int at_position(int first, int i) {
    return static_cast<int>(static_cast<uint32_t>(first) + static_cast<uint32_t>(i));
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

// The row's maximum and sum over its records (empty ones skipped), by one thread.
__device__ __forceinline__ float2 join_ml(const float2 *ml, int splits) {
    float M = -INFINITY, L = 0.0f;
    for (int s = 0; s < splits; ++s) M = fmaxf(M, ml[s].x);
    const float base = M == -INFINITY ? 0.0f : M;
    for (int s = 0; s < splits; ++s) {
        const float2 v = ml[s];
        if (v.x == -INFINITY && v.y == 0.0f) continue;
        L = __builtin_fmaf(__builtin_amdgcn_exp2f(v.x - base), v.y, L);
    }
    return make_float2(base, L);
}

// Output d .. d + 3 of one row from its records, in their order.
__device__ __forceinline__ void join_row(const SpanArgs &a, int HD, size_t row, int d) {
    const float2 *ml = a.rec_ml + row * a.splits_total;
    const float2 all = join_ml(ml, a.splits_total);
    float o[4] = {0, 0, 0, 0};
    for (int s = 0; s < a.splits_total; ++s) {
        const float2 v = ml[s];
        if (v.x == -INFINITY && v.y == 0.0f) continue;
        const float f = __builtin_amdgcn_exp2f(v.x - all.x);
        const float4 p = *reinterpret_cast<const float4 *>(a.rec_o + (row * a.splits_total + s) * HD + d);
        o[0] = __builtin_fmaf(f, p.x, o[0]);
        o[1] = __builtin_fmaf(f, p.y, o[1]);
        o[2] = __builtin_fmaf(f, p.z, o[2]);
        o[3] = __builtin_fmaf(f, p.w, o[3]);
    }
    const float inv = 1.0f / all.y;
    *reinterpret_cast<float4 *>(a.out + row * HD + d) =
        all.y > 0 ? make_float4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv) : make_float4(0, 0, 0, 0);
}

__global__ __launch_bounds__(256) void span_join_kernel(SpanArgs a, int HD, int64_t rows) {
    const int per = HD / 4;
    const int64_t row = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) / per;
    if (row < rows) join_row(a, HD, row, threadIdx.x % per * 4);
}

// Block (256 slots, kv head, unit); the last block of x joins the kv head's rows instead.
__global__ __launch_bounds__(256) void span_record_kernel(SpanRecordArgs r, int HD) {
    const SpanArgs &a = r.a;
    const int kh = blockIdx.y, unit = blockIdx.z, t = threadIdx.x;
    const size_t row0 = static_cast<size_t>(unit) * a.heads + kh * a.group;
    if (blockIdx.x == gridDim.x - 1) {
        const int per = HD / 4;
        for (int i = t; i < a.group * per; i += 256) join_row(a, HD, row0 + i / per, i % per * 4);
        return;
    }
    __shared__ float2 all[kSpanMaxGroup];
    if (t < a.group) all[t] = join_ml(a.rec_ml + (row0 + t) * a.splits_total, a.splits_total);
    __syncthreads();
    const int n = min(a.lengths ? a.lengths[unit] : a.length, a.length);
    const int slot = blockIdx.x * 256 + t;
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

void launch_span_join(const SpanArgs &a, int head_dim, hipStream_t s) {
    const int64_t rows = static_cast<int64_t>(a.units) * a.count * a.heads;
    const int per = 256 / (head_dim / 4);
    hipLaunchKernelGGL(span_join_kernel, dim3(static_cast<unsigned>((rows + per - 1) / per)), dim3(256), 0, s, a, head_dim, rows);
    ND_HIP(hipGetLastError());
}

void launch_span_record(const SpanRecordArgs &r, int head_dim, hipStream_t s) {
    const dim3 grid((r.a.length + 255) / 256 + 1, r.a.kvheads, r.a.units);
    hipLaunchKernelGGL(span_record_kernel, grid, dim3(256), 0, s, r, head_dim);
    ND_HIP(hipGetLastError());
}

}  // namespace nd
