// gfx950 kernel of what happens to q, k and v between a projection and the attention: norms of every head of q and k, their
// rotation by position, and the store of k and v in the paged cache, in one pass over the rows.
//
//   y = x / sqrt(sum x^2 / HD + eps) * (1 + gain);  (y_j, y_{j + h}) -> (y_j cos t - y_{j + h} sin t, y_{j + h} cos t +
//   y_j sin t) for j < h = rotary / 2, t = position * freq_j;  stored rows as the cache's quantiser has them.
//
// t is formed in 64 bits (a position of a million times a frequency in 32 would be off by 0.06), reduced there to an eighth
// of a turn, and only the rest is rounded: sin and cos are within 2^-23 of t's (which 64 bits hold to 2^-53 of its size).
// Everything else is fp32, every result rounded once or twice. Where a row's squares pass the fp32 range, or they and eps are
// so small that the squares lose bits (below 2^-126), the row and eps are taken times a power of two, which is exact.
//
// Memory bounds many tokens, latency few. A row is one 16-byte piece a lane (HD / 4 lanes); a lane's angles are those of
// all of a token's rows, so HD / 4 lanes take four of a token's rows, all of them loaded first (8191 tokens, 40 rows of 128
// values: 66.4 us, 5.05 TB/s; with two or eight rows 72.7 and 69.9), and two where nothing is rotated (8191 tokens' K and V
// rows of 8 heads of 128 into slots: 19.7 us, 4.3 TB/s; four or eight rows 20.6 and 21.9). Half of each of the 40 rows
// rotated, through LDS: 70 us; 32 rows of q, 8 of k and 8 of v, those of k and v into slots: 74.4, 4.7 TB/s, and 79 with half
// of each rotated (in a graph, where the 40 whole rows take 64).
#include "paged.h"
#include "span_dev.h"

namespace nd {

namespace {

// Sine and cosine of an angle: the rest of it behind whole quarter turns, |x| <= pi / 4, by the first terms of their series
// (what they leave out is below 2^-29).
__device__ __forceinline__ void sin_cos(double angle, float &sine, float &cosine) {
    const double quarters = angle * 0.63661977236758134308;  // 2 / pi
    const double whole = rint(quarters);
    const float x = static_cast<float>((quarters - whole) * 1.57079632679489661923), y = x * x;
    float s = __builtin_fmaf(y, -1.0f / 39916800.0f, 1.0f / 362880.0f);
    s = __builtin_fmaf(s, y, -1.0f / 5040.0f);
    s = __builtin_fmaf(s, y, 1.0f / 120.0f);
    s = __builtin_fmaf(s, y, -1.0f / 6.0f);
    s = __builtin_fmaf(s * y, x, x);
    float c = __builtin_fmaf(y, -1.0f / 3628800.0f, 1.0f / 40320.0f);
    c = __builtin_fmaf(c, y, -1.0f / 720.0f);
    c = __builtin_fmaf(c, y, 1.0f / 24.0f);
    c = __builtin_fmaf(c, y, -0.5f);
    c = __builtin_fmaf(c, y, 1.0f);
    // whole modulo 4, exactly: |whole| can pass the integers
    const int turn = static_cast<int>(whole - 4.0 * floor(whole * 0.25));
    const float a = turn & 1 ? c : s, b = turn & 1 ? s : c;
    sine = turn & 2 ? -a : a;
    cosine = (turn + 1) & 2 ? -b : b;
}

template <int L, int H = 1>
__device__ __forceinline__ float group_sum(float v, int t) {
    if constexpr (H < L) return group_sum<L, H * 2>(v + butterfly_partner<H>(v, t), t);
    else return v;
}

// e of |v| in [2^(e - 1), 2^e); far below every other's for 0.
__device__ __forceinline__ int exponent(float v) { return v > 0 ? __builtin_amdgcn_frexp_expf(v) : -1000; }

// ROT: 0 none, 1 the whole row (partners half a row apart: HD / 8 lanes), 2 any even number of dimensions (through LDS).
template <int HD, int ROWS, int ROT>
__global__ __launch_bounds__(256) void heads_kernel(HeadsArgs a, int parts) {
    constexpr int L = HD / 4;
    __shared__ __attribute__((aligned(16))) float rows[ROT == 2 ? 256 / L : 1][HD];
    const int t = threadIdx.x, lane = t & 63, part = t % L, d = part * 4;
    const uint32_t item = blockIdx.x * (256 / L) + t / L;
    const int token = item / static_cast<uint32_t>(parts), row0 = item % static_cast<uint32_t>(parts) * ROWS;
    const int nq = a.q ? a.heads : 0, nk = a.k ? a.kvheads : 0, nv = a.v ? a.kvheads : 0, all = nq + nk + nv;
    bool in = token < a.tokens;
    const int position = in && a.positions ? a.positions[token] : 0;
    const int slot = in && a.slots ? a.slots[token] : -1;
    in = in && position >= 0;

    float4 x[ROWS];
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int row = row0 + i;
        const float *src = row < nq        ? a.q + token * a.q_stride + row * HD
                           : row < nq + nk ? a.k + token * a.k_stride + (row - nq) * HD
                                           : a.v + token * a.v_stride + (row - nq - nk) * HD;
        x[i] = in && row < all ? *reinterpret_cast<const float4 *>(src + d) : make_float4(0, 0, 0, 0);
    }
    float sine[4], cosine[4];
    const bool turned = ROT != 0 && row0 < nq + nk;
    if (turned) {
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int e = d + c, j = e < a.half ? e : e - a.half;
            sine[c] = 0.0f;
            cosine[c] = 1.0f;
            if (ROT == 1 || e < 2 * a.half) {
                sin_cos(static_cast<double>(position) * a.freq[j], sine[c], cosine[c]);
                if (e < a.half) sine[c] = -sine[c];
            }
        }
    }

#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const int row = row0 + i;
        if (row >= all) break;  // (of all lanes of the row, whose exchanges stay among themselves)
        const bool is_q = row < nq, is_v = row >= nq + nk;
        float y[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
        const float *gain = is_q ? a.q_gain : is_v ? nullptr : a.k_gain;
        if (gain) {
            auto squares = [&] { return group_sum<L>((y[0] * y[0] + y[1] * y[1]) + (y[2] * y[2] + y[3] * y[3]), lane); };
            const float sum = squares();
            float mean = sum / HD + a.eps;
            if (__builtin_expect(!(sum < INFINITY && mean >= 0x1p-100f), 0)) {
                const float top = group_max<L>(fmaxf(fmaxf(fabsf(y[0]), fabsf(y[1])), fmaxf(fabsf(y[2]), fabsf(y[3]))), lane);
                // the row's largest value, or the root of eps where that is larger, to 2^59 .. 2^60: the sum of 128 squares is
                // below 2^127, and what becomes smaller than a normal number has a result of zero
                const int up = top < INFINITY ? 60 - max(exponent(top), (exponent(a.eps) + 1) >> 1) : 0;
#pragma unroll
                for (int c = 0; c < 4; ++c) y[c] = ldexpf(y[c], up);
                mean = squares() / HD + ldexpf(a.eps, 2 * up);
            }
            const float r = 1.0f / sqrtf(mean);
            const float4 g = *reinterpret_cast<const float4 *>(gain + d);
            const float gs[4] = {g.x, g.y, g.z, g.w};
#pragma unroll
            for (int c = 0; c < 4; ++c) y[c] = y[c] * r * (1.0f + gs[c]);
        }
        if (ROT == 1 && !is_v) {
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const float o = butterfly_partner<L / 2>(y[c], lane);
                y[c] = __builtin_fmaf(o, sine[c], y[c] * cosine[c]);
            }
        } else if (ROT == 2 && !is_v) {
            float *mine = rows[t / L];
            *reinterpret_cast<float4 *>(mine + d) = make_float4(y[0], y[1], y[2], y[3]);
            __builtin_amdgcn_wave_barrier();  // LDS operations of one wave complete in order
            asm volatile("" ::: "memory");
#pragma unroll
            for (int c = 0; c < 4; ++c) {
                const int e = d + c, other = e < a.half ? e + a.half : e - a.half;
                const float o = e < 2 * a.half ? mine[other] : 0.0f;
                y[c] = e < 2 * a.half ? __builtin_fmaf(o, sine[c], y[c] * cosine[c]) : y[c];
            }
            __builtin_amdgcn_wave_barrier();
            asm volatile("" ::: "memory");
        }
        if (!is_v) {
            float *out = is_q ? a.q_out : a.k_out;
            if (out && in)
                *reinterpret_cast<float4 *>(out + token * (is_q ? a.q_out_stride : a.k_out_stride) +
                                            (is_q ? row : row - nq) * HD + d) = make_float4(y[0], y[1], y[2], y[3]);
        }
        if (!is_q && a.pool.at) {
            const float top = group_max<L>(fmaxf(fmaxf(fabsf(y[0]), fabsf(y[1])), fmaxf(fabsf(y[2]), fabsf(y[3]))), lane);
            const int id = slot >> a.pool.shift;
            if (!in || slot < 0 || id >= a.pool.pages) continue;
            const float inv = top > 0 ? 127.0f / top : 0.0f;
            auto code = [&](float v) {
                return static_cast<uint32_t>(static_cast<int>(fmaxf(-127.0f, fminf(127.0f, rintf(v * inv))))) & 0xFFu;
            };
            const int kh = is_v ? row - nq - nk : row - nq, off = slot & ((1 << a.pool.shift) - 1);
            uint8_t *block = a.pool.at + (static_cast<size_t>(id) * a.pool.kvheads + kh) * page_block_bytes(a.pool.shift, HD);
            uint8_t *codes = block + ((is_v ? HD : 0) << a.pool.shift) + off * HD + d;
            *reinterpret_cast<uint32_t *>(codes) = code(y[0]) | code(y[1]) << 8 | code(y[2]) << 16 | code(y[3]) << 24;
            if (part == 0)
                reinterpret_cast<float *>(block + (2 * HD << a.pool.shift))[(is_v ? 1 << a.pool.shift : 0) + off] =
                    top > 0 ? top / 127.0f : 1.0f;
        }
    }
}

template <int HD, int ROWS, int ROT>
void launch_rows(const HeadsArgs &a, int all, hipStream_t s) {
    const int parts = (all + ROWS - 1) / ROWS, per_block = 256 / (HD / 4);
    const int64_t items = static_cast<int64_t>(a.tokens) * parts;
    ND_CHECK(items * (HD / 4) < (int64_t(1) << 32) - 256, "heads: more rows than a grid holds");
    hipLaunchKernelGGL((heads_kernel<HD, ROWS, ROT>), dim3(static_cast<unsigned>((items + per_block - 1) / per_block)),
                       dim3(256), 0, s, a, parts);
    ND_HIP(hipGetLastError());
}

template <int HD, int ROWS, int STILL>
void launch_rot(const HeadsArgs &a, int all, hipStream_t s) {
    if (a.half == 0) launch_rows<HD, STILL, 0>(a, all, s);
    else if (a.half == HD / 2) launch_rows<HD, ROWS, 1>(a, all, s);
    else launch_rows<HD, ROWS, 2>(a, all, s);
}

template <int HD>
void launch_hd(const HeadsArgs &a, hipStream_t s) {
    const int all = (a.q ? a.heads : 0) + (a.k ? a.kvheads : 0) + (a.v ? a.kvheads : 0);
    if (all == 0 || a.tokens == 0) return;
    // a row a lane group while that leaves every compute unit fewer than eight waves
    if (static_cast<int64_t>(a.tokens) * all * (HD / 4) < int64_t(512) * device_cus()) launch_rot<HD, 1, 1>(a, all, s);
    else launch_rot<HD, 4, 2>(a, all, s);
}

}  // namespace

void launch_heads(const HeadsArgs &a, int head_dim, hipStream_t s) {
    switch (head_dim) {
    case 32: launch_hd<32>(a, s); break;
    case 64: launch_hd<64>(a, s); break;
    default: launch_hd<128>(a, s); break;
    }
}

}  // namespace nd
