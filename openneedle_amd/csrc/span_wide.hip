// gfx950 kernel of span attention with many query rows over the same keys: prompt pieces, and a batch over its shared
// prefix. The mathematics and the records are span_kernels.hip's. The matrix instructions bound this kernel, so both
// products run on v_mfma_f32_32x32x16_f16 with q and p * vs as two float16 terms (the codes are float16 numbers as they
// are) instead of three bfloat16 ones: 22 bits of a value, and of small values what lies above 2^-25 of the term's unit.
//   q is scaled by a power of two, 2^kMostLift at most, so that the row's largest |q| is in [2^14, 2^15). Of a value the
//   terms leave at most 2^-23 (the last bit of a quarter of them; the sums round by as much), of a small one at most 2^-25,
//   together 2^-25 * 127 HD * |ks| in a score; where that could pass 2^-24 (of a score times log2 e, whose own rounding is
//   2^-24 of its size) the tile's scores get the rest of q in further terms, until nothing is left.
//   p * vs is scaled by one power of two a row, 2^(kLift - M), that follows the largest score and the largest V scale, and of
//   it the terms leave at most 2^-23, of a small one 2^-25: 2^-26 of the row's largest in the tile, where that is at least 2
//   (an fp32 sum of the 32 rounds by 2^-24 of its largest term). Where it is not (the largest V scale is another key's, or
//   one's that the row does not attend; or the scores are far below the row's largest), the tile is added with a power of
//   two of its own a row, whose largest is then in [2^9, 2^10). V rows of zeros as the cache stores them (scale 1) count
//   for none of this. Held in fp32 before that, a weight below 2^-119 of the row's largest V scale may be lost.
// 6 x 999 tokens, 32 heads of 128 values, window 2048, rows stored before: 435 us a call, 428 GFLOP of matrix work at
// 0.98 PFLOP/s (a large bfloat16 product of the library reaches 1.2); rows of 64 305 us, of 32 197. The matrix unit is busy
// 45% of the cycles; the rest is the softmax and the making of terms, 256 vector instructions a wave and tile next to its 32
// matrix instructions. Tiles with powers of two of their own: peaky scores (three times these) 510 us, rows of 64 345.
// Two blocks a compute unit: with rows of 128 up to 10 registers are kept in memory around the loop over tiles, none in it.
#include "span_rows.h"

namespace nd {

namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x16 mfma32(const u32x4 &a, const u32x4 &b, const f32x16 &c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// x - h of the lower or upper float16 of a pair (exact where h is x rounded).
__device__ __forceinline__ float less_low(uint32_t h, float x) {
    float r;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(x));
    return r;
}
__device__ __forceinline__ float less_high(uint32_t h, float x) {
    float r;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(r) : "v"(h), "v"(x));
    return r;
}
__device__ __forceinline__ uint32_t round_pair(float a, float b) {
    const f16x2 h = {static_cast<_Float16>(a), static_cast<_Float16>(b)};
    return __builtin_bit_cast(uint32_t, h);
}

// Two float16 terms of eight values.
struct Halves {
    u32x4 hi, lo;
};
__device__ __forceinline__ Halves halve8(const float (&x)[8]) {
    uint32_t h[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        h[i] = round_pair(x[2 * i], x[2 * i + 1]);
        l[i] = round_pair(less_low(h[i], x[2 * i]), less_high(h[i], x[2 * i + 1]));
    }
    return Halves{u32x4{h[0], h[1], h[2], h[3]}, u32x4{l[0], l[1], l[2], l[3]}};
}
// and what they leave, exactly
__device__ __forceinline__ Halves take8(float (&x)[8]) {
    const Halves t = halve8(x);
    const uint32_t h[4] = {t.hi.x, t.hi.y, t.hi.z, t.hi.w}, l[4] = {t.lo.x, t.lo.y, t.lo.z, t.lo.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[2 * i] = less_low(l[i], less_low(h[i], x[2 * i]));
        x[2 * i + 1] = less_high(l[i], less_high(h[i], x[2 * i + 1]));
    }
    return t;
}
// The same where values may be infinite or NaN: those are their first term alone.
__device__ __forceinline__ Halves halve8_any(const float (&x)[8]) {
    float y[8], z[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const bool odd = !(fabsf(x[i]) < INFINITY);
        y[i] = odd ? 0.0f : x[i];
        z[i] = odd ? x[i] : y[i];
    }
    return Halves{halve8(z).hi, halve8(y).lo};
}

// Two codes as float16 (exact).
__device__ __forceinline__ uint32_t half_pair(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(a, b));
}
// Eight codes of two dwords as float16: a byte b = code + 128 under the exponent of 1024 is 1024 + b.
__device__ __forceinline__ u32x4 widen_half(uint32_t a, uint32_t b) {
    const uint32_t w[2] = {a ^ 0x80808080u, b ^ 0x80808080u};
    const f16x2 off = {static_cast<_Float16>(-1152.0f), static_cast<_Float16>(-1152.0f)};
    uint32_t r[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const uint32_t p = __builtin_amdgcn_perm(w[i / 2], 0x64646464u, i % 2 ? 0x00070006u : 0x00050004u);
        r[i] = __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2, p) + off);
    }
    return u32x4{r[0], r[1], r[2], r[3]};
}

// The row's outputs and sum are held times 2^(kLift - M): M is a whole number, at least the largest score (times log2 e)
// plus the exponent of its tile's largest V scale, less kSlack (so it moves, and the outputs are rescaled, in few tiles).
// While a tile is added that lies kDrop or more below M, or whose weights are small for another reason, its weights and the
// outputs are held times another power of two, at most 2^kMostUp: the outputs, below 2^48 (2^21 tiles of 32 weights below
// 2^15 times 127), stay finite.
constexpr float kLift = 10.0f, kSlack = 5.0f, kDrop = 7.0f;
constexpr int kMostExp = 50;  // of a V scale that M follows: the sum, which M scales too, stays far from underflow
constexpr int kMostUp = 76;
// of q: scores, held times 2^lift, stay finite up to 2^97 (smaller q lie below the terms; where their scores could matter
// they are taken in further ones)
constexpr int kMostLift = 30;
constexpr int kOddTile = 1024;

constexpr int kFrag = 66;  // 16-byte lanes of an operand in LDS: 32, one of padding (the halves in different banks), 32, 1
__device__ __forceinline__ int frag_lane(int m, int half) { return m + 33 * half; }

// Block (up to four row groups of 32 and piece, with unit and kv head): four waves over the same tiles of 32 keys, which
// the block turns into float16 operands in LDS once; a wave without rows only helps with that (a window's blocks have
// four groups but for the last). A wave forms the next tile's scores while it does this tile's softmax and
// values, so that the matrix unit and the vector unit of a SIMD work at once: K is in LDS two tiles ahead of its values,
// codes are a tile further ahead in registers, and there is one barrier a tile.
//   Scores: operand A is 32 keys' codes, operand B the wave's 32 rows of q. Lane l holds row l % 32 and of each 32 keys
//   8 (i / 4) + 4 (l / 32) + i % 4, i < 16.
//   Values: operand B is p * vs straight from those registers, operand A the V codes in the same order of keys. Result t
//   of lane l is row l % 32, dimensions DT * (8 (i / 4) + 4 (l / 32) + i % 4) + t (DT = HD / 32 results).
template <int HD, bool RING>
__device__ __forceinline__ void span_wide(const SpanArgs &a, int bx) {
    constexpr int KS = HD / 16;                     // steps of the score product's depth
    constexpr int DT = HD / 32;                     // results of 32 dimensions
    constexpr int T = 256;
    // A tile's K codes are 2 HD chunks of 16 bytes, its V codes as many pieces of 4 keys x 4 dimensions: one of each a
    // thread (HD = 128), or K's on the first waves and V's on the next.
    constexpr int kChunks = 2 * HD;
    constexpr bool kBoth = kChunks == T;
    constexpr int kRoleWaves = kChunks / 64;
    constexpr int kScaleWave = HD == 32 ? 2 : 0;    // it brings the scales too
    static_assert(kBoth || 2 * kChunks <= T, "roles of the waves");
    __shared__ u32x4 kf[2][KS][kFrag];
    __shared__ u32x4 vf[2][2][DT][kFrag];
    __shared__ __attribute__((aligned(16))) float sc[4][2][kWideTile];  // K (times scale) and V scales, by tile modulo 4
    // of the tile's slots in its run: the exponent of the largest finite V scale, plus kOddTile where one is infinite or
    // NaN; and the largest |K scale|
    __shared__ int2 about[4];

    const int t = threadIdx.x, lane = t & 63, col = lane & 31, half = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int pairs = a.units * a.kvheads;
    const int pair = bx % pairs, rest = bx / pairs;
    const int unit = pair / a.kvheads, kh = pair % a.kvheads;
    const int piece = rest % a.splits, tile_rows = rest / a.splits * (32 * a.groups);
    const int rows = a.count * a.group;
    const int last_row = min(rows, tile_rows + 32 * a.groups) - 1;
    const bool works = wave < a.groups;
    const int row = tile_rows + wave * 32 + col;
    const bool live = works && row < rows;
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

    // Codes on their way to LDS: K as 16 dimensions of a key, V as 4 dimensions of 4 keys. Loads past the cache's rows
    // read zero.
    constexpr uint32_t kNone = 0x80000000u;  // past every buffer: no request
    const bool k_role = kBoth || wave < kRoleWaves, v_role = kBoth || (wave >= kRoleWaves && wave < 2 * kRoleWaves);
    const int kc = t, vc = kBoth ? t : t - kChunks;  // chunk, piece
    const int v_keys = vc / (HD / 4), v_dims = vc % (HD / 4);
    struct RawK {
        u32x4 k;
        float s[2];  // K and V scale of key `col`
    };
    struct RawV {
        uint32_t v[4];
    };
    auto fetch_k = [&](RawK &r, int tile) {
        const uint32_t s0 = static_cast<uint32_t>(slot0(tile));
        r.k = __builtin_amdgcn_raw_buffer_load_b128(rk, k_role ? s0 * HD + kc * 16 : kNone, 0, 0);
        const uint32_t at = wave == kScaleWave ? (s0 + col) * 4u : kNone;
        r.s[0] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rks, at, 0, 0));
        r.s[1] = __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(rvs, at, 0, 0));
    };
    auto fetch_v = [&](RawV &r, int tile) {
        const uint32_t s0 = static_cast<uint32_t>(slot0(tile));
        const uint32_t at = v_role ? (s0 + 4 * v_keys) * HD + v_dims * 4 : kNone;
#pragma unroll
        for (int j = 0; j < 4; ++j) r.v[j] = __builtin_amdgcn_raw_buffer_load_b32(rv, at + j * HD, 0, 0);
    };
    auto place_k = [&](const RawK &r, int tile) {
        const int buf = (tile - begin) & 1, sb = (tile - begin) & 3;
        if (k_role) {
            const int key = kc / KS, step = kc % KS;
            kf[buf][step][frag_lane(key, 0)] = widen_half(r.k.x, r.k.y);
            kf[buf][step][frag_lane(key, 1)] = widen_half(r.k.z, r.k.w);
        }
        if (wave == kScaleWave) {
            const bool in = slot0(tile) + col < stop(tile);
            const float ks = in ? r.s[0] * a.scale : 0.0f;
            float vs = in ? r.s[1] : 0.0f;
            // A V row of zeros, whose scale the quantiser makes 1, adds nothing: scale 0, so that neither M nor a row's
            // largest weight is taken from it.
            if (__builtin_expect(__any(vs == 1.0f), 0)) {
                uint32_t codes = 0;  // of a half of the row
#pragma unroll
                for (int c = 0; c < HD / 2; c += 4)
                    codes |= __builtin_amdgcn_raw_buffer_load_b32(
                        rv, (static_cast<uint32_t>(slot0(tile)) + col) * HD + half * (HD / 2) + c, 0, 0);
                const float mine = codes != 0 ? 1.0f : 0.0f, other = butterfly_partner<32>(mine, lane);
                if (vs == 1.0f && mine + other == 0.0f) vs = 0.0f;
            }
            sc[sb][half][col] = half ? vs : ks;
            const float v = fabsf(vs);
            const bool odd = !(v < INFINITY);
            const float most = group_max<32>(half ? odd ? 0.0f : v : fabsf(ks), lane);
            const float v_most = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, most), 32));
            const int ve = (v_most > 0 ? __builtin_amdgcn_frexp_expf(v_most) : 0) + (__any(odd) ? kOddTile : 0);
            if (lane == 0) about[sb] = make_int2(ve, __builtin_bit_cast(int, most));
        }
    };
    auto place_v = [&](const RawV &r, int tile) {
        if (!v_role) return;
        const int buf = (tile - begin) & 1;
#pragma unroll
        for (int b = 0; b < 4; ++b) {
            float f[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j] = code(r.v[j], b);
            const int d = v_dims * 4 + b;
            // 4 keys: half and quarter of a step's depth
            u32x2 *to = reinterpret_cast<u32x2 *>(&vf[buf][v_keys / 4][d % DT][frag_lane(d / DT, v_keys & 1)]);
            to[(v_keys >> 1) & 1] = u32x2{half_pair(f[0], f[1]), half_pair(f[2], f[3])};
        }
    };

    RawK rk_next, rk_first;
    RawV rv_next;
    fetch_k(rk_first, begin);
    fetch_k(rk_next, begin + 1);
    fetch_v(rv_next, begin);
    if (!RING && !works) {
        place_k(rk_first, begin);
        place_k(rk_next, begin + 1);
        place_v(rv_next, begin);
        fetch_k(rk_next, begin + 2);
        fetch_v(rv_next, begin + 1);
        __syncthreads();
        __syncthreads();
        for (int tile = begin; tile < end; ++tile) {
            place_v(rv_next, tile + 1);
            place_k(rk_next, tile + 2);
            fetch_k(rk_next, tile + 3);
            fetch_v(rv_next, tile + 2);
            __syncthreads();
        }
        return;
    }

    // q as operand B: lane (row col, half) holds dimensions 16 c + 8 half .. of step c
    const size_t orow = (static_cast<size_t>(unit) * a.count + (live ? row : 0) / a.group) * a.heads + kh * a.group +
                        (live ? row : 0) % a.group;
    const float4 *src = reinterpret_cast<const float4 *>(a.q + orow * HD + half * 8);
    Halves q[KS];
    int lift;     // q is held times 2^lift
    float down;   // 2^-lift; NaN for a row with an infinity or NaN, whose scores it makes NaN
    float worst;  // a tile whose |K scale| (times a.scale) is above 1 / worst takes further terms of q
    {
        float x[KS][8];
        float most = 0.0f;
        bool finite = true;
#pragma unroll
        for (int c = 0; c < KS; ++c) {
            const float4 u = src[4 * c], w = src[4 * c + 1];
            const float both[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                x[c][j] = live ? both[j] : 0.0f;
                finite = finite && fabsf(x[c][j]) < INFINITY;
                most = fmaxf(most, fabsf(x[c][j]));
            }
        }
        most = fmaxf(most, butterfly_partner<32>(most, lane));
        finite = butterfly_partner<32>(finite ? 1.0f : 0.0f, lane) != 0.0f && finite;
        lift = finite && most > 0 ? min(15 - __builtin_amdgcn_frexp_expf(most), kMostLift) : 0;
        down = finite ? ldexpf(1.0f, -lift) : __builtin_nanf("");
        worst = wave_max(finite && most > 0 ? down : 0.0f, lane) * (127.0f * HD * 0.5f);
#pragma unroll
        for (int c = 0; c < KS; ++c) {
#pragma unroll
            for (int j = 0; j < 8; ++j) x[c][j] = finite ? ldexpf(x[c][j], lift) : 0.0f;
            q[c] = halve8(x[c]);
        }
    }

    float M = -INFINITY, l = 0.0f;
    f32x16 acc[DT];
#pragma unroll
    for (int i = 0; i < DT; ++i)
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[i][j] = 0.0f;

    // q times a tile's K codes, both terms (times 2^lift)
    auto product = [&](int tile) {
        const int buf = (tile - begin) & 1;
        f32x16 x;
#pragma unroll
        for (int j = 0; j < 16; ++j) x[j] = 0.0f;
#pragma unroll
        for (int c = 0; c < KS; ++c) {
            const u32x4 k = kf[buf][c][frag_lane(col, half)];
            x = mfma32(k, q[c].lo, x);
            x = mfma32(k, q[c].hi, x);
        }
        return x;
    };
    // and the rest of q where it could matter
    auto finish_product = [&](f32x16 &x, int tile) {
        if (!(__builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(about[(tile - begin) & 3].y)) * worst > 1.0f)) return;
        bool left = true;
#pragma unroll 1
        for (int round = 1; __any(left); ++round) {
            left = false;
            f32x16 e;
#pragma unroll
            for (int j = 0; j < 16; ++j) e[j] = 0.0f;
#pragma unroll 1
            for (int c = 0; c < KS; ++c) {
                const float4 u = src[4 * c], w = src[4 * c + 1];
                float r[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w};
#pragma unroll
                for (int j = 0; j < 8; ++j) r[j] = live && down == down ? ldexpf(r[j], lift) : 0.0f;
#pragma unroll 1
                for (int i = 0; i < round; ++i) {  // what the terms before leave
                    take8(r);
#pragma unroll
                    for (int j = 0; j < 8; ++j) r[j] *= 0x1p24f;
                }
                const Halves h = take8(r);
                const u32x4 k = kf[(tile - begin) & 1][c][frag_lane(col, half)];
                e = mfma32(k, h.lo, e);
                e = mfma32(k, h.hi, e);
#pragma unroll
                for (int j = 0; j < 8; ++j) left = left || r[j] != 0.0f;
            }
            const float unit = ldexpf(1.0f, -24 * round);
#pragma unroll
            for (int j = 0; j < 16; ++j) x[j] = __builtin_fmaf(e[j], unit, x[j]);
        }
    };

    // A tile of weights w too small for float16, too large, or not finite: w, and the outputs while it is added, are held
    // times the row's own power of two 2^-unit (next to the 2^up that they are held times already).
    bool wide_range = false;  // a V scale above 2^kMostExp has been met: the outputs' size has to be looked at
    auto rescale = [&](f32x16 &w, uint32_t gone, bool far, float up) {
        wide_range = wide_range || far;
        float most = 0.0f;
        int least = static_cast<int>(up) - kMostUp;
        if (__builtin_expect(wide_range, 0)) {
            float reach = 0.0f;
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                w[j] = gone >> j & 1u ? 0.0f : w[j];  // (0 times a scale that is no number)
                most = fmaxf(most, fabsf(w[j]) < INFINITY ? fabsf(w[j]) : 0.0f);
            }
#pragma unroll
            for (int i = 0; i < DT; ++i)
#pragma unroll
                for (int j = 0; j < 16; ++j) reach = fmaxf(reach, fabsf(acc[i][j]) < INFINITY ? fabsf(acc[i][j]) : 0.0f);
            reach = fmaxf(reach, butterfly_partner<32>(reach, lane));
            least = static_cast<int>(up) - 126;
            if (reach > 0) least = max(least, __builtin_amdgcn_frexp_expf(reach) - 125);
        } else {
#pragma unroll
            for (int j = 0; j < 16; ++j) most = fmaxf(most, fabsf(w[j]));
        }
        most = fmaxf(most, butterfly_partner<32>(most, lane));
        const int unit = max(least, most > 0 ? __builtin_amdgcn_frexp_expf(most) - 10 : 0);
        const float to = ldexpf(1.0f, -unit);
#pragma unroll
        for (int j = 0; j < 16; ++j) w[j] *= to;
#pragma unroll
        for (int i = 0; i < DT; ++i) acc[i] *= to;
        return unit;
    };

    place_k(rk_first, begin);
    place_k(rk_next, begin + 1);
    place_v(rv_next, begin);
    fetch_k(rk_next, begin + 2);
    fetch_v(rv_next, begin + 1);
    __syncthreads();
    f32x16 next = product(begin);
    finish_product(next, begin);
    __syncthreads();  // every wave has its first scores before K's buffer is written again
    for (int tile = begin; tile < end; ++tile) {
        const int vb = (tile - begin) & 1, sb = (tile - begin) & 3;
        const int s0 = slot0(tile), behind = stop(tile);
        const int code = __builtin_amdgcn_readfirstlane(about[sb].x);
        const int ve = code > kOddTile / 2 ? code - kOddTile : code;
        f32x16 x;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float4 ks = *reinterpret_cast<const float4 *>(&sc[sb][0][8 * g + 4 * half]);
            x[4 * g] = next[4 * g] * ks.x;
            x[4 * g + 1] = next[4 * g + 1] * ks.y;
            x[4 * g + 2] = next[4 * g + 2] * ks.z;
            x[4 * g + 3] = next[4 * g + 3] * ks.w;
        }
        bool masked = s0 + kWideTile > behind;
        if constexpr (RING) {
            const int shift = tile < tiles0 ? runs.shift0 : runs.shift1;
            const bool all_pinned = s0 + kWideTile <= runs.pinned;
            masked |= all_pinned ? s0 + kWideTile - 1 > full_high
                                 : s0 < runs.pinned || s0 + shift <= full_low || s0 + kWideTile - 1 + shift > full_high;
        }
        uint32_t gone = 0;  // this lane's keys that the row does not attend
        uint32_t idle = 0;  // rows that attend none of the tile's
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
            const uint64_t none = __ballot(gone == 0xFFFFu);
            idle = static_cast<uint32_t>(none) & static_cast<uint32_t>(none >> 32);
        }
        float top = -INFINITY;
#pragma unroll
        for (int j = 0; j < 16; ++j) top = fmaxf(top, x[j]);
        top = fmaxf(top, butterfly_partner<32>(top, lane)) * down;
        const int follow = max(-kMostExp, min(kMostExp, ve));
        const float high = ceilf(top) + static_cast<float>(max(-kMostExp, min(kMostExp, ve)));
        float up = 0.0f;
        bool low = false;
        // (M = -inf: the first scores; rows that attend none of the tile are here too)
        if (__any(fabsf(high - M + 0.5f * (kDrop - kSlack)) > 0.5f * (kDrop + kSlack))) {
            const float most = fmaxf(M, high);
            const float alpha = M == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(M - most);
            M = most;
            const bool below = high < M - kDrop && high > -INFINITY && !wide_range;
            low = __any(below);
            up = below ? fminf(M - high, static_cast<float>(kMostUp)) : 0.0f;
            const float grow = alpha * __builtin_amdgcn_exp2f(up);
            l *= grow;
#pragma unroll
            for (int i = 0; i < DT; ++i) acc[i] *= grow;
        }
        const float lifted = M > -INFINITY ? kLift + up - M : 0.0f;  // nothing attended yet: every power is 0
        // the next tile's product beside this tile's weights (ahead of the other block's wave: 466 -> 456 us where the
        // matrix unit is the bound)
        __builtin_amdgcn_s_setprio(1);
        next = product(tile + 1);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float4 v4 = *reinterpret_cast<const float4 *>(&sc[sb][1][8 * g + 4 * half]);
            const float vs[4] = {v4.x, v4.y, v4.z, v4.w};
            float p[4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                p[u] = __builtin_amdgcn_exp2f(__builtin_fmaf(x[4 * g + u], down, lifted));
                x[4 * g + u] = p[u] * vs[u];
            }
            l += (p[0] + p[1]) + (p[2] + p[3]);
        }
        Halves p[2];
        auto halve = [&] {
#pragma unroll
            for (int ks = 0; ks < 2; ++ks) {
                float w[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) w[j] = x[8 * ks + j];
                p[ks] = halve8(w);
            }
        };
        halve();
        // a row none of whose weights reaches 2 (the first bit of a float16 exponent), though it attends some of the keys
        const uint32_t bits = (p[0].hi.x | p[0].hi.y | p[0].hi.z | p[0].hi.w) | (p[1].hi.x | p[1].hi.y | p[1].hi.z | p[1].hi.w);
        const uint64_t held = __ballot((bits & 0x40004000u) != 0);
        const bool far = code > kMostExp;
        const bool apart = far || (static_cast<uint32_t>(held) | static_cast<uint32_t>(held >> 32) | idle) != ~0u;
        int back = static_cast<int>(-up);
        if (__builtin_expect(apart, 0)) {
            back += rescale(x, gone, far, up);
            halve();
            if (__builtin_expect(far, 0)) {
#pragma unroll
                for (int ks = 0; ks < 2; ++ks) {
                    float w[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) w[j] = x[8 * ks + j];
                    p[ks] = halve8_any(w);
                }
            }
        }
        // this tile's values beside the operands of the tiles to come
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
            for (int i = 0; i < DT; ++i) acc[i] = mfma32(vf[vb][ks][i][frag_lane(col, half)], p[ks].lo, acc[i]);
#pragma unroll
            for (int i = 0; i < DT; ++i) acc[i] = mfma32(vf[vb][ks][i][frag_lane(col, half)], p[ks].hi, acc[i]);
        }
        place_v(rv_next, tile + 1);
        place_k(rk_next, tile + 2);
        __builtin_amdgcn_s_setprio(0);
        if (__builtin_expect(apart || low, 0)) {
            l *= __builtin_amdgcn_exp2f(-up);
            const float from = ldexpf(1.0f, back);
#pragma unroll
            for (int i = 0; i < DT; ++i) acc[i] *= from;
        }
        finish_product(next, tile + 1);
        fetch_k(rk_next, tile + 3);
        fetch_v(rv_next, tile + 2);
        __syncthreads();
    }

    l += butterfly_partner<32>(l, lane);
    if (!live) return;
    const bool finish = !a.rec_o;
    const size_t rec = orow * a.splits_total + a.split0 + piece;
    float *to = finish ? a.out + orow * HD : a.rec_o + rec * HD;
    const float inv = !finish ? 1.0f : l > 0 ? 1.0f / l : 0.0f;
    const bool none = finish && !(l > 0);  // nothing attended, or no softmax
    if (!finish && half == 0) a.rec_ml[rec] = make_float2(M - kLift, l);
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

template <int HD, bool RING>
__global__ __launch_bounds__(256, 2) void span_wide_kernel(SpanArgs a) {
    span_wide<HD, RING>(a, blockIdx.x);
}

// A shared prefix and the units' own keys in one launch: the first `far_blocks` blocks have the prefix.
template <int HD>
__global__ __launch_bounds__(256, 2) void span_wide_own_kernel(SpanArgs far, SpanArgs own, int far_blocks) {
    if (static_cast<int>(blockIdx.x) < far_blocks) span_wide<HD, false>(far, blockIdx.x);
    else span_block<HD, 4, false>(own, blockIdx.x - far_blocks);
}

int64_t wide_blocks(const SpanArgs &a) {
    const int64_t rows = static_cast<int64_t>(a.count) * a.group, block = 32 * a.groups;
    return (rows + block - 1) / block * a.splits * a.units * a.kvheads;
}

template <int HD>
void launch_wide_hd(const SpanArgs &a, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(wide_blocks(a)));
    if (a.positions) hipLaunchKernelGGL((span_wide_kernel<HD, true>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((span_wide_kernel<HD, false>), grid, dim3(256), 0, s, a);
    ND_HIP(hipGetLastError());
}

}  // namespace

void launch_span_wide(const SpanArgs &a, int head_dim, hipStream_t s) {
    switch (head_dim) {
    case 32: launch_wide_hd<32>(a, s); break;
    case 64: launch_wide_hd<64>(a, s); break;
    default: launch_wide_hd<128>(a, s); break;
    }
}

void launch_span_wide_own(const SpanArgs &far, const SpanArgs &own, int head_dim, hipStream_t s) {
    const int64_t far_blocks = wide_blocks(far);
    const dim3 grid(static_cast<unsigned>(far_blocks + static_cast<int64_t>(own.splits) * own.kvheads * own.units));
    const int n = static_cast<int>(far_blocks);
    switch (head_dim) {
    case 32: hipLaunchKernelGGL((span_wide_own_kernel<32>), grid, dim3(256), 0, s, far, own, n); break;
    case 64: hipLaunchKernelGGL((span_wide_own_kernel<64>), grid, dim3(256), 0, s, far, own, n); break;
    default: hipLaunchKernelGGL((span_wide_own_kernel<128>), grid, dim3(256), 0, s, far, own, n); break;
    }
    ND_HIP(hipGetLastError());
}

}  // namespace nd
