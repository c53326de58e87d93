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
#include "span_wide.h"

namespace nd {

namespace {

template <int HD, Keys K>
__global__ __launch_bounds__(256, 2) void span_wide_kernel(SpanArgs a) {
    span_wide<HD, K>(a, blockIdx.x);
}

// A shared prefix and the units' own keys in one launch: the first `far_blocks` blocks have the prefix.
template <int HD>
__global__ __launch_bounds__(256, 2) void span_wide_own_kernel(SpanArgs far, SpanArgs own, int far_blocks) {
    if (static_cast<int>(blockIdx.x) < far_blocks) span_wide<HD, Keys::Flat>(far, blockIdx.x);
    else span_block<HD, 4, Keys::Flat>(own, blockIdx.x - far_blocks);
}

int64_t wide_blocks(const SpanArgs &a) {
    const int64_t rows = static_cast<int64_t>(a.count) * a.group, block = 32 * a.groups;
    return (rows + block - 1) / block * a.splits * a.units * a.kvheads;
}

template <int HD>
void launch_wide_hd(const SpanArgs &a, hipStream_t s) {
    const dim3 grid(static_cast<unsigned>(wide_blocks(a)));
    if (a.positions) hipLaunchKernelGGL((span_wide_kernel<HD, Keys::Ring>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((span_wide_kernel<HD, Keys::Flat>), grid, dim3(256), 0, s, a);
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
