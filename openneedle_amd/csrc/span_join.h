// The joining of records (running maximum, sum, unnormalised output) of pieces of a row's keys.
#pragma once

#include "span_dev.h"

#include <type_traits>

namespace nd {

namespace {

// A row's maximum and sum over its n records, by one wave; the records' factors 2^(m - maximum) to `factor` if that is set.
__device__ __forceinline__ float2 join_sums(const SpanArgs &a, size_t row, int n, int lane, float *factor) {
    const float2 *ml = a.rec_ml + row * a.splits_total;
    float2 mine = make_float2(-INFINITY, 0.0f);  // of this lane's first record: most rows have no second
    float M = -INFINITY;
    for (int s = lane; s < n; s += 64) {
        const float2 v = ml[s];
        if (s == lane) mine = v;
        M = fmaxf(M, v.x);
    }
    M = wave_max(M, lane);
    const float base = M == -INFINITY ? 0.0f : M;
    float L = 0.0f;
    for (int s = lane; s < n; s += 64) {
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
// on the number of records only. Latency bounds it: 64 x 32 rows of 128 values 5 us, a long prefix's many records 7.
constexpr int kJoinMax = 1024;  // records of a row
// SOME: row r has some[r].x of them, from 2 on, and is row some[r].y of the output; of 0 there is nothing to join. What is
// read is 0 again for the next call.
template <int HD, int G, bool SOME = false>
__device__ __forceinline__ void join_rows(const SpanArgs &a, size_t row0, int count, int2 *some = nullptr) {
    constexpr int kLanes = HD / 4, kRows = 256 / (G * kLanes);
    constexpr int kFactors = kRows * (G == 8 ? kJoinMax : G);
    __shared__ float factor[kFactors];
    __shared__ float total[kRows];
    __shared__ __attribute__((aligned(16))) float part[G > 1 ? G : 1][kRows][HD];
    const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const int splits = a.splits_total;
    __shared__ int2 number[SOME ? kRows : 1];
    const int d = t % kLanes * 4, g = t / kLanes % G, r = t / (kLanes * G);
    for (int i0 = 0; i0 < count; i0 += kRows) {
        for (int i = wave; i < kRows && i0 + i < count; i += 4) {
            int n = splits;
            if constexpr (SOME) {
                const int2 its = some[row0 + i0 + i];
                n = min(__builtin_amdgcn_readfirstlane(its.x), splits);
                if (lane == 0) number[i] = make_int2(n, its.y);
                if (n == 0) continue;
                if (lane == 0) some[row0 + i0 + i].x = 0;
            }
            const float2 all = join_sums(a, row0 + i0 + i, n, lane, factor + i * splits);
            if (lane == 0) total[i] = all.y;
        }
        __syncthreads();
        bool live = i0 + r < count;
        int n = splits;
        size_t to = row0 + i0 + r;
        if constexpr (SOME) {
            n = live ? number[r].x : 0;
            live = n > 0;
            if (live) to = number[r].y;
        }
        float4 o = make_float4(0, 0, 0, 0);
        if (live) {
            const float *rec = a.rec_o + (row0 + i0 + r) * splits * HD + d;
#pragma unroll 4
            for (int s = g; s < n; s += G) {
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
            *reinterpret_cast<float4 *>(a.out + to * HD + d) =
                L > 0 ? make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv) : make_float4(0, 0, 0, 0);
        }
        __syncthreads();
    }
}

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

}  // namespace nd
