// gfx950 kernels of the paged cache's tables: pages dealt to requests for their new tokens, with every token's position and
// slot, and taken back.
//
// Request r holds n = lengths[r] positions and gets c = counts[r] more. Its new pages are ceil((n + c) / page) -
// ceil(n / page); the sums of c and of the new pages over the requests before it say where its tokens begin and which of the
// free pages are its own. Page ceil(n / page) + i begins with one of the request's new tokens, so the token at a multiple
// of `page` writes the table's entry, and a pass over the tokens does all.
//
// Latency bounds both kernels: loads, a scan, a search, a page's load and the stores, each after the other (an extension and
// its trim, 32 requests or 500 with 11000 tokens: 14.6 us). So there is one launch each, in which every block of 1024 tokens
// scans all requests for itself (16 waves, a request a thread up to 1024 of them), which costs less than a second launch
// behind the first one's end. Sums saturate instead of growing past 32 bits.
#include "paged.h"

namespace nd {

namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;

__device__ __forceinline__ int capped(int a, int b, int cap) { return min(a + b, cap); }  // a, b <= cap <= 2^30

// Sums (capped) over the threads before this one, and of all.
struct Sums {
    int tokens, pages;
};
__device__ __forceinline__ Sums scan(Sums mine, int token_cap, int page_cap, Sums &all) {
    __shared__ Sums waves[kWaves];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    Sums s = mine;
#pragma unroll
    for (int d = 1; d < 64; d *= 2) {
        const int t = __shfl_up(s.tokens, d), p = __shfl_up(s.pages, d);
        if (lane >= d) {
            s.tokens = capped(s.tokens, t, token_cap);
            s.pages = capped(s.pages, p, page_cap);
        }
    }
    if (lane == 63) waves[wave] = s;
    const int before_t = __shfl_up(s.tokens, 1), before_p = __shfl_up(s.pages, 1);
    __syncthreads();
    Sums before = {lane ? before_t : 0, lane ? before_p : 0};
    all = {0, 0};
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        const Sums v = waves[w];
        if (w < wave) {
            before.tokens = capped(before.tokens, v.tokens, token_cap);
            before.pages = capped(before.pages, v.pages, page_cap);
        }
        all.tokens = capped(all.tokens, v.tokens, token_cap);
        all.pages = capped(all.pages, v.pages, page_cap);
    }
    return before;
}

// The last r in [0, n) with begin[r] <= t (begin[0] <= t).
__device__ __forceinline__ int holder(const int *begin, int n, int t) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (begin[mid] <= t) lo = mid;
        else hi = mid - 1;
    }
    return lo;
}

// True in the one block that ends last (alone: at once), where everything that the others read may be changed.
__device__ __forceinline__ bool ends_last(int *done) {
    __shared__ bool last;
    __syncthreads();
    if (gridDim.x == 1) return true;
    if (threadIdx.x == 0) {
        __threadfence();
        last = atomicAdd(done, 1) == static_cast<int>(gridDim.x) - 1;
        if (last) atomicExch(done, 0);
    }
    __syncthreads();
    return last;
}

__global__ __launch_bounds__(256) void zero_kernel(int2 *at, size_t n) {
    const size_t i = static_cast<size_t>(blockIdx.x) * 256 + threadIdx.x;
    if (i < n) at[i] = make_int2(0, 0);
}

__global__ __launch_bounds__(256) void pages_reset_kernel(PageStack f) {
    const int i = blockIdx.x * 256 + threadIdx.x;
    if (i < f.pages) f.stack[i] = f.pages - 1 - i;
    if (i == 0) {
        *f.top = f.pages;
        *f.done = 0;
    }
}

__global__ __launch_bounds__(kThreads) void extend_kernel(ExtendArgs a) {
    extern __shared__ int lds[];
    int *begin = lds, *deal = lds + a.requests, *held = lds + 2 * a.requests;  // a refused request's deal: -1
    const int t = threadIdx.x, page = 1 << a.shift;
    const int token_cap = a.tokens + 1, page_cap = a.free.pages + 1;
    const int top = *a.free.top;
    const int most = a.width << a.shift;  // positions of a table
    const int each = (a.requests + kThreads - 1) / kThreads;
    const int r0 = min(t * each, a.requests), r1 = min(r0 + each, a.requests);
    // n, c, new pages of a request; a request past its table, or with a negative length, takes none
    auto wants = [&](int r, int &n, int &c, bool &fits) {
        n = a.lengths[r];
        const int asked = max(a.counts[r], 0);
        c = min(asked, token_cap);
        fits = n >= 0 && n <= most && asked <= most - n;
        return fits ? ((n + asked + page - 1) >> a.shift) - ((n + page - 1) >> a.shift) : 0;
    };
    Sums mine = {0, 0};
    for (int r = r0; r < r1; ++r) {
        int n, c;
        bool fits;
        const int p = wants(r, n, c, fits);
        mine.tokens = capped(mine.tokens, c, token_cap);
        mine.pages = capped(mine.pages, min(p, page_cap), page_cap);
    }
    Sums all;
    Sums at = scan(mine, token_cap, page_cap, all);
    int dealt = 0;  // pages taken up to the last of this thread's requests that got any
    for (int r = r0; r < r1; ++r) {
        int n, c;
        bool fits;
        const int p = wants(r, n, c, fits);
        const int pages = capped(at.pages, min(p, page_cap), page_cap), tokens = capped(at.tokens, c, token_cap);
        const bool granted = fits && tokens <= a.tokens && (p == 0 || pages <= top);
        begin[r] = min(at.tokens, a.tokens);
        deal[r] = granted ? at.pages : -1;
        held[r] = n;
        if (granted && p) dealt = pages;
        if (blockIdx.x == 0) {
            a.starts[r] = min(at.tokens, a.tokens);
            a.firsts[r] = granted ? n : -1;
        }
        at = {tokens, pages};
    }
    const int total = min(all.tokens, a.tokens);
    if (blockIdx.x == 0 && t == 0) a.starts[a.requests] = total;
    __syncthreads();

    const int token = blockIdx.x * kThreads + t;
    if (token < a.tokens) {
        int slot = -1, position = -1;
        if (token < total) {
            const int r = holder(begin, a.requests, token);
            if (deal[r] >= 0) {
                const int n = held[r], p = n + token - begin[r];
                const int i = p >> a.shift, old = (n + page - 1) >> a.shift;
                int *entry = a.tables + static_cast<size_t>(r) * a.width + i;
                const int id = i < old ? *entry : a.free.stack[top - 1 - (deal[r] + i - old)];
                if (i >= old && (p & (page - 1)) == 0) *entry = id;
                position = p;
                if (static_cast<unsigned>(id) < static_cast<unsigned>(a.free.pages)) slot = (id << a.shift) + (p & (page - 1));
            }
        }
        a.slots[token] = slot;
        a.positions[token] = position;
    }

    if (!ends_last(a.free.done)) return;
    __shared__ int taken;
    if (t == 0) taken = 0;
    __syncthreads();
    if (dealt) atomicMax(&taken, dealt);  // (of a whole number: any order)
    for (int r = t; r < a.requests; r += kThreads)
        if (deal[r] >= 0) a.lengths[r] = held[r] + max(a.counts[r], 0);
    __syncthreads();
    if (t == 0) *a.free.top = top - taken;
}

// The pages of the positions from keep[r] on go back (negative: none does), the last one first, so that what an extension
// took lies in the stack as before it.
__global__ __launch_bounds__(kThreads) void trim_kernel(TrimArgs a) {
    extern __shared__ int lds[];
    int *begin = lds, *left = lds + a.requests;  // pages that go back before r's; pages that r keeps
    const int t = threadIdx.x, page = 1 << a.shift;
    const int page_cap = a.free.pages + 1, most = a.width << a.shift;
    const int top = *a.free.top;
    const int each = (a.requests + kThreads - 1) / kThreads;
    const int r0 = min(t * each, a.requests), r1 = min(r0 + each, a.requests);
    // n and what is kept of it, both within the table; true where the length is lowered
    auto kept = [&](int r, int &n, int &k) {
        const int length = a.lengths[r], keep = a.keep[r];
        n = min(max(length, 0), most);
        k = keep < 0 ? n : min(keep, n);
        return keep >= 0 && length > keep;
    };
    Sums mine = {0, 0};
    for (int r = r0; r < r1; ++r) {
        int n, k;
        kept(r, n, k);
        mine.pages = capped(mine.pages, min(((n + page - 1) >> a.shift) - ((k + page - 1) >> a.shift), page_cap), page_cap);
    }
    Sums all;
    Sums at = scan(mine, 0, page_cap, all);
    for (int r = r0; r < r1; ++r) {
        int n, k;
        kept(r, n, k);
        begin[r] = at.pages;
        left[r] = (k + page - 1) >> a.shift;
        at.pages = capped(at.pages, min(((n + page - 1) >> a.shift) - left[r], page_cap), page_cap);
    }
    __syncthreads();
    const int total = min(all.pages, a.free.pages - top);  // (more only in tables that were not dealt here)
    for (int j = blockIdx.x * kThreads + t; j < total; j += gridDim.x * kThreads) {
        const int r = holder(begin, a.requests, j);
        int *entry = a.tables + static_cast<size_t>(r) * a.width + left[r] + j - begin[r];
        a.free.stack[top + total - 1 - j] = *entry;
        *entry = -1;
    }
    if (!ends_last(a.free.done)) return;
    for (int r = t; r < a.requests; r += kThreads) {
        int n, k;
        if (kept(r, n, k)) a.lengths[r] = a.keep[r];
    }
    if (t == 0) *a.free.top = top + total;
}

}  // namespace

void launch_zero(int2 *at, size_t n, hipStream_t s) {
    hipLaunchKernelGGL(zero_kernel, dim3(static_cast<unsigned>((n + 255) / 256)), dim3(256), 0, s, at, n);
    ND_HIP(hipGetLastError());
}

void launch_pages_reset(const PageStack &f, hipStream_t s) {
    hipLaunchKernelGGL(pages_reset_kernel, dim3((f.pages + 255) / 256), dim3(256), 0, s, f);
    ND_HIP(hipGetLastError());
}

void launch_extend(const ExtendArgs &a, hipStream_t s) {
    const int blocks = a.tokens > kThreads ? (a.tokens + kThreads - 1) / kThreads : 1;
    hipLaunchKernelGGL(extend_kernel, dim3(blocks), dim3(kThreads), 3 * sizeof(int) * a.requests, s, a);
    ND_HIP(hipGetLastError());
}

// One block has room for the pages of most calls; more where whole long requests may go back at once.
void launch_trim(const TrimArgs &a, hipStream_t s) {
    const int64_t entries = static_cast<int64_t>(a.requests) * a.width;
    const int blocks = entries > 16 * kThreads ? 16 : 1;
    hipLaunchKernelGGL(trim_kernel, dim3(blocks), dim3(kThreads), 2 * sizeof(int) * a.requests, s, a);
    ND_HIP(hipGetLastError());
}

}  // namespace nd
