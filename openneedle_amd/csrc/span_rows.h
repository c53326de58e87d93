// Attention of up to 16 query rows by a block of four or eight waves over parts of the keys (span_kernels.hip has the
// mathematics).
#pragma once

#include "span_dev.h"

namespace nd {

namespace {

__device__ __forceinline__ f32x4 mfma(const u32x4 &a, const u32x4 &b, const f32x4 &c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Block (piece and row tile, kv head, unit): up to 16 query rows (the columns of both products' results), NW waves with
// every NW-th tile of 64 keys each, joined at the end. Eight waves where there is at most one block per compute unit: a
// block's rounds then bound the launch (one conversation of 272 keys 8.7 -> 6.8 us, 35 blocks of 1006 keys of
// 32 values 13.8 -> 11.0). With many blocks the cache's rows bound it, read once, each lane its operands' bytes straight
// from memory: 64 sequences x 8 kv heads x 4100 keys of 128 values, 101 us (5.5 TB/s). Three terms cost matrix work that
// stays below that time at 16 rows a block.
//   Scores: operand A is 16 keys' codes, operand B the rows' q. Lane l holds row l % 16 and keys 16 t + 4 (l / 16) + i.
//   Values: operand B is p * vs straight from those registers (the contraction runs over the keys in their order:
//   depth 8 (l / 16) + j is key 32 u + 4 (l / 16) + j, and from j = 4 on 32 u + 16 + 4 (l / 16) + j - 4), operand A the V
//   codes of dimensions HD / 16 * (l % 16) + t. Result t of lane l is row l % 16, dimensions HD / 16 * (4 (l / 16) + i) + t.
template <int HD, int NW, bool RING>
__device__ __forceinline__ void span_rows(const SpanArgs &a, int bx, int kh, int unit) {
    constexpr int kSteps = HD / 32;        // of the score product's depth
    constexpr int kBytes = HD / 4;         // of a K row per lane
    constexpr int VB = HD / 16;            // bytes of a V row per lane
    __shared__ __attribute__((aligned(16))) float sc[NW][2][kSpanTile];  // K (times scale) and V scales of a wave's tile
    __shared__ __attribute__((aligned(16))) float so[NW][kSpanRows][HD + 4];
    __shared__ float sm[NW][kSpanRows], sl[NW][kSpanRows];

    const int t = threadIdx.x, lane = t & 63, col = lane & 15, quad = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int tiles_of_rows = (a.count * a.group + kSpanRows - 1) / kSpanRows;
    const int tile0 = bx % tiles_of_rows, piece = bx / tiles_of_rows;
    const int rows = a.count * a.group;
    const int row = tile0 * kSpanRows + col;
    const int last_row = min(rows, (tile0 + 1) * kSpanRows) - 1;
    const bool live = row < rows;
    const int cap = a.c.capacity;

    // New tokens (at most one row tile, so at most 16): token wave + NW i's rows, ahead of everything that waits for the
    // unit's position or length.
    NewRow fresh[kSpanRows / NW];
    if (a.new_k) {
#pragma unroll
        for (int i = 0; i < kSpanRows / NW; ++i) {
            if (wave + NW * i >= a.count) break;
            const size_t src = ((static_cast<size_t>(unit) * a.count + wave + NW * i) * a.kvheads + kh) * HD;
            fresh[i] = read_row(a.new_k + src, a.new_v + src, HD, lane);
        }
    }
    KeyRuns runs = {0, 0, 0, 0, 0, 0};
    int own = 0;           // the row's position
    bool alone = true;     // every row attends all keys of the runs (those of one token)
    int full_low = 0, full_high = 0;  // positions that every row of the block attends: (full_low, full_high]
    if constexpr (RING) {
        const int first = a.positions[unit];
        const int p0 = at_position(first, tile0 * kSpanRows / a.group), p1 = at_position(first, last_row / a.group);
        runs = ring_runs(p0, p1, a.sinks, a.window, cap);
        own = at_position(first, (live ? row : last_row) / a.group);
        full_low = p1 >= a.window ? p1 - a.window : -1;
        full_high = p0;
        alone = p0 == p1;
    } else {
        const int n = min(a.lengths ? a.lengths[unit] : a.length, a.length);
        runs.n0 = runs.pinned = n > 0 ? n : 0;
    }
    const int tiles0 = span_tiles(runs.n0), tiles = tiles0 + span_tiles(runs.n1);
    const int begin = piece * a.per, end = min(begin + a.per, tiles);

    const size_t row0 = (static_cast<size_t>(unit) * a.kvheads + kh) * cap;
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

    // A new token's slot; -1: not in this block's tiles. Its tile in `in`.
    auto new_slot = [&](int i, int &in) {
        const int p = RING ? at_position(a.positions[unit], i) : runs.n0 - 1;
        if (p < 0) return -1;
        const int slot = RING ? ring_slot(p, a.sinks, cap) : p;
        in = slot < runs.n0 ? slot / kSpanTile : tiles0 + (slot - runs.begin1) / kSpanTile;
        return in >= begin && in < end ? slot : -1;
    };
    // The first tile is on its way before the new tokens are stored, unless it holds one of them; the next tile is loaded
    // before a tile is computed.
    Tile cur, nxt;
    int tile = begin + wave;
    bool wait = false;
    if (a.new_k) {
        for (int i = 0; i < a.count; ++i) {
            int in = -1;
            wait = wait || (new_slot(i, in) >= 0 && in == tile);
        }
    }
    if (!wait) load(cur, tile);

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

    if (a.new_k) {
#pragma unroll
        for (int i = 0; i < kSpanRows / NW; ++i) {
            if (wave + NW * i >= a.count) break;
            int in;
            const int slot = new_slot(wave + NW * i, in);
            if (slot >= 0) store_row(a.c, fresh[i], row0 + slot, HD, lane);
        }
        __syncthreads();  // (and the block's stores before its loads of those rows)
    }
    if (wait) load(cur, tile);

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
            masked |= !alone && (all_pinned ? s0 + kSpanTile - 1 > full_high
                                            : s0 < runs.pinned || s0 + shift <= full_low || s0 + kSpanTile - 1 + shift > full_high);
        }
        if (masked) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int u = 0; u < 4; ++u) {
                    const bool ok = s0 + 16 * i + 4 * quad + u < behind;
                    x[i][u] = ok ? x[i][u] : -INFINITY;
                    vs[i][u] = ok ? vs[i][u] : 0.0f;
                }
            if (RING && !alone) {
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int u = 0; u < 4; ++u) {
                        const int slot = s0 + 16 * i + 4 * quad + u;
                        const bool pin = tile < tiles0 && slot < runs.pinned;
                        const int p = pin ? slot : slot + (tile < tiles0 ? runs.shift0 : runs.shift1);
                        const bool ok = p <= own && (pin || own - p < a.window);
                        x[i][u] = ok ? x[i][u] : -INFINITY;
                        vs[i][u] = ok ? vs[i][u] : 0.0f;
                    }
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

    for (; tile < end; tile += NW) {
        load(nxt, tile + NW);
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
    for (int i = t; i < kSpanRows * HD / 4; i += 64 * NW) {
        const int r = i / (HD / 4), d = i % (HD / 4) * 4;
        const int grow = tile0 * kSpanRows + r;
        if (grow >= rows) break;
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < NW; ++w) M = fmaxf(M, sm[w][r]);
        const float base = M == -INFINITY ? 0.0f : M;
        float L = 0.0f, o[4] = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < NW; ++w) {
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

// Block `b` of a launch of all units, kv heads, row tiles and pieces. The pieces are slowest: those behind the end of a
// short sequence come last, and the others spread over the compute units.
template <int HD, int NW, bool RING>
__device__ __forceinline__ void span_block(const SpanArgs &a, int b) {
    const int rest = b / a.kvheads;
    span_rows<HD, NW, RING>(a, rest / a.units, b % a.kvheads, rest % a.units);
}

}  // namespace

}  // namespace nd
