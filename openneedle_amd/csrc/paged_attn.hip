// gfx950 kernels of attention over the paged cache: new tokens of many requests, one, a draft or a prompt piece each. The
// mathematics, the operands and the records are span_kernels.hip's; a tile's pages are looked up ahead of its loads.
#include "paged.h"
#include "span_join.h"
#include "span_wide.h"

namespace nd {

namespace {

// Block b of 16 rows. The order of the requests (64 of 2048 to 8192 positions, 8 kv heads of 128 values, 512 blocks of which
// two share a compute unit: as they come 159 us, the longest first 148, every other round from the shortest 138; 40 of them
// 144, 112, 111) takes about a microsecond to find, so it is not looked for where every block has a unit of its own.
template <int HD, int NW>
__device__ __forceinline__ void paged_rows(const PagedSpanArgs &a, int b) {
    const int kh = b % a.kvheads, rest = b / a.kvheads;
    int unit = rest % a.units;
    if (a.round) {
        const int round = unit / a.round, in = unit - round * a.round;
        if (round & 1) unit = min(a.units, (round + 1) * a.round) - 1 - in;
        unit = ranked_request(a, unit, threadIdx.x & 63);
    }
    span_rows<HD, NW, Keys::Paged>(a, rest / a.units, kh, unit);
}

template <int HD, int NW>
__global__ __launch_bounds__(64 * NW, 2) void paged_kernel(PagedSpanArgs a) {
    paged_rows<HD, NW>(a, blockIdx.x);
}

// The blocks of 128 rows first: they take the longest. With rows of 128 values 23 registers a lane are kept in memory, one of
// them read in the loop over tiles.
template <int HD>
__global__ __launch_bounds__(256, 2) void paged_wide_kernel(PagedSpanArgs a, int blocks) {
    if (static_cast<int>(blockIdx.x) < blocks) span_wide<HD, Keys::Paged>(a, blockIdx.x);
    else paged_rows<HD, 4>(a, blockIdx.x - blocks);
}

template <int HD, int G>
__global__ __launch_bounds__(256) void paged_join_kernel(PagedSpanArgs a, int64_t rows) {
    constexpr int kRows = 256 / (G * (HD / 4));
    const int64_t row0 = static_cast<int64_t>(blockIdx.x) * kRows;
    join_rows<HD, G, true>(a, row0, static_cast<int>(min(static_cast<int64_t>(kRows), rows - row0)), a.some);
}

template <int HD>
void launch_hd(const PagedSpanArgs &a, hipStream_t s) {
    const int64_t wide = static_cast<int64_t>(a.wide_blocks) * a.wide_splits * a.kvheads;
    const dim3 grid(static_cast<unsigned>(wide + static_cast<int64_t>(a.splits) * a.row_tiles * a.kvheads * a.units));
    if (wide > 0) {
        hipLaunchKernelGGL((paged_wide_kernel<HD>), grid, dim3(256), 0, s, a, static_cast<int>(wide));
        ND_HIP(hipGetLastError());
        return;
    }
    if (a.waves == 4) hipLaunchKernelGGL((paged_kernel<HD, 4>), grid, dim3(256), 0, s, a);
    else hipLaunchKernelGGL((paged_kernel<HD, 8>), grid, dim3(512), 0, s, a);
    ND_HIP(hipGetLastError());
}

}  // namespace

void launch_paged(const PagedSpanArgs &a, int head_dim, hipStream_t s) {
    switch (head_dim) {
    case 32: launch_hd<32>(a, s); break;
    case 64: launch_hd<64>(a, s); break;
    default: launch_hd<128>(a, s); break;
    }
}

void launch_paged_join(const PagedSpanArgs &a, int64_t rows, int head_dim, hipStream_t s) {
    ND_CHECK(a.splits_total <= kJoinMax, "attention: too many pieces");
    with_join(head_dim, a.splits_total, [&](auto hd, auto groups) {
        constexpr int HD = decltype(hd)::value, G = decltype(groups)::value;
        constexpr int kRows = 256 / (G * (HD / 4));
        hipLaunchKernelGGL((paged_join_kernel<HD, G>), dim3(static_cast<unsigned>((rows + kRows - 1) / kRows)), dim3(256), 0,
                           s, a, rows);
    });
    ND_HIP(hipGetLastError());
}

}  // namespace nd
