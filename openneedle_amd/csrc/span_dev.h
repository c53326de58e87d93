// What the span kernels share: codes and fp32 values as bfloat16 matrix operands.
#pragma once

#include "span.h"
#include "wave.h"

namespace nd {

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

// A new token's K and V rows of HD values in a wave's registers, two values each a lane.
struct NewRow {
    float k[2], v[2];
};
__device__ __forceinline__ NewRow read_row(const float *k, const float *v, int HD, int lane) {
    NewRow r;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const bool in = lane + 64 * i < HD;
        r.k[i] = in ? k[lane + 64 * i] : 0.0f;
        r.v[i] = in ? v[lane + 64 * i] : 0.0f;
    }
    return r;
}

// One row into codes and scale, by one wave (the cache's quantiser: top = max|x|, scale = top / 127 or 1, codes
// round(x * (127 / top))).
__device__ __forceinline__ void quantise_row(const float (&x)[2], int HD, int lane, int8_t *codes, float *scale) {
    const float top = wave_max(fmaxf(fabsf(x[0]), fabsf(x[1])), lane);
    const float inv = top > 0 ? 127.0f / top : 0.0f;
    if (lane == 0) *scale = top > 0 ? top / 127.0f : 1.0f;
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (lane + 64 * i < HD)
            codes[lane + 64 * i] = static_cast<int8_t>(fmaxf(-127.0f, fminf(127.0f, rintf(x[i] * inv))));
}

__device__ __forceinline__ void store_row(const SpanCache &c, const NewRow &r, size_t row, int HD, int lane) {
    quantise_row(r.k, HD, lane, c.k8 + row * HD, c.ks + row);
    quantise_row(r.v, HD, lane, c.v8 + row * HD, c.vs + row);
}

__device__ __forceinline__ int at_position(int first, int i) {
    return static_cast<int>(static_cast<uint32_t>(first) + static_cast<uint32_t>(i));
}

}  // namespace nd
