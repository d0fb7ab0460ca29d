// Block tables, token slots and offsets of a step built from the requests'
// lengths, and the way back (lengths cut, pages returned).
//
// With len_b the tokens held, n_b the new ones and ps the page size, request b
// holds have_b = ceil(len_b / ps) pages and needs need_b = ceil((len_b + n_b)
// / ps); its need_b - have_b fresh pages are the next ones from the top of the
// stack of free pages, requests in row order. Token i of the step belongs to
// the request with cu_b <= i < cu_{b+1} (cu the running sum of n), stands at
// position p = len_b + i - cu_b, and its slot is page(p / ps) * ps + p % ps.
//
// Everything hangs on two running sums over the rows. They are cheap (4096
// rows at most), so every CTA makes them for itself in shared memory and none
// waits for another; each thread then finds its tokens' row by bisection. One
// launch, and it is bound by that launch: a decode step of 32 rows reads and
// writes under 1 KB (2.8 us a captured call), 512 rows with 71,000 tokens 0.9 MB
// (6.1 us: the sums over the rows, a bisection and a chain of three loads a token).
#include "kvq_paged.h"

namespace kvq {
namespace paged {

constexpr int THREADS = 512;
constexpr int WARPS = THREADS / 32;
// Tokens (or returned pages) per CTA before another CTA is launched.
constexpr uint32_t PER_CTA = 2048;

__device__ __forceinline__ uint64_t pages_of(int64_t tokens, uint32_t shift) {
    return (uint64_t)((tokens + (1ll << shift) - 1) >> shift);
}

__device__ __forceinline__ uint64_t warp_inclusive(uint64_t v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    return v;
}

// Exclusive running sums of (a, b) over the block's threads, and the totals.
__device__ void block_scan(uint64_t& a, uint64_t& b, uint64_t& total_a, uint64_t& total_b,
                           uint64_t (*scratch)[WARPS]) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint64_t ia = warp_inclusive(a, lane), ib = warp_inclusive(b, lane);
    if (lane == 31) {
        scratch[0][warp] = ia;
        scratch[1][warp] = ib;
    }
    __syncthreads();
    uint64_t base_a = 0, base_b = 0;
    total_a = total_b = 0;
    for (int w = 0; w < WARPS; ++w) {
        const uint64_t x = scratch[0][w], y = scratch[1][w];
        if (w < warp) {
            base_a += x;
            base_b += y;
        }
        total_a += x;
        total_b += y;
    }
    a = base_a + ia - a;
    b = base_b + ib - b;
}

// The last row whose offset is <= i (empty rows share their offset with the
// next one and are passed over).
__device__ __forceinline__ uint32_t row_of(const uint32_t* offsets, uint32_t rows, uint32_t i) {
    uint32_t lo = 0, hi = rows;            // offsets[lo] <= i < offsets[hi]
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (offsets[mid] <= i) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(THREADS) build_tables_kernel(Tables t) {
    extern __shared__ uint32_t sh[];
    __shared__ uint64_t scratch[2][WARPS];
    uint32_t* cu = sh;                     // [rows + 1]
    uint32_t* fresh = sh + t.rows + 1;     // [rows + 1]
    const uint32_t per = (t.rows + THREADS - 1) / THREADS;
    const uint32_t r0 = min(t.rows, threadIdx.x * per), r1 = min(t.rows, r0 + per);

    uint64_t tokens = 0, pages = 0;
    int wide = 0;
    for (uint32_t r = r0; r < r1; ++r) {
        const int64_t len = max(t.lens[r], 0), n = max(t.step[r], 0);
        const uint64_t need = pages_of(len + n, t.page_shift);
        wide |= need > t.width;
        tokens += (uint64_t)n;
        pages += need - pages_of(len, t.page_shift);
    }
    uint64_t at_tok = tokens, at_page = pages, all_tok, all_page;
    block_scan(at_tok, at_page, all_tok, all_page, scratch);
    const uint32_t stack = (uint32_t)min(max(*t.n_free, 0), (int)t.pool);
    const int status = (all_page > stack ? 1 : 0) | (__syncthreads_or(wide) ? 2 : 0) |
                       (all_tok > t.max_tokens ? 4 : 0);
    // a step that does not fit takes nothing
    const bool fits = status == 0;
    for (uint32_t r = r0; r < r1; ++r) {
        const int64_t len = max(t.lens[r], 0), n = max(t.step[r], 0);
        cu[r] = fits ? (uint32_t)at_tok : 0;
        fresh[r] = fits ? (uint32_t)at_page : 0;
        at_tok += (uint64_t)n;
        at_page += pages_of(len + n, t.page_shift) - pages_of(len, t.page_shift);
        if (blockIdx.x == 0) {
            t.cu_new[r] = (int32_t)cu[r];
            t.lens_out[r] = fits ? (int32_t)(len + n) : (int32_t)len;
        }
    }
    const uint32_t live = fits ? (uint32_t)all_tok : 0;
    if (threadIdx.x == 0) {
        cu[t.rows] = live;
        if (blockIdx.x == 0) {
            t.cu_new[t.rows] = (int32_t)live;
            *t.n_free_out = (int32_t)(stack - (fits ? (uint32_t)all_page : 0));
            *t.status = status;
        }
    }
    __syncthreads();
    for (uint32_t i = blockIdx.x * THREADS + threadIdx.x; i < t.max_tokens; i += gridDim.x * THREADS) {
        int64_t slot = -1;
        int32_t pos = 0;
        if (i < live) {
            const uint32_t r = row_of(cu, t.rows, i);
            const int32_t len = max(t.lens[r], 0);
            pos = len + (int32_t)(i - cu[r]);
            const uint32_t col = (uint32_t)pos >> t.page_shift;
            const uint32_t have = (uint32_t)pages_of(len, t.page_shift);
            int32_t* entry = t.block_tables + (size_t)r * t.width + col;
            int32_t page;
            if (col >= have) {
                page = t.free_pages[stack - 1 - (fresh[r] + (col - have))];
                if (((uint32_t)pos & ((1u << t.page_shift) - 1)) == 0) *entry = page;
            } else {
                page = *entry;
            }
            slot = ((int64_t)page << t.page_shift) + (pos & ((1 << t.page_shift) - 1));
        }
        t.slots[i] = slot;
        t.positions[i] = pos;
    }
}

// Requests cut to min(len, keep): the pages behind it go on the stack in row
// order, each row's in table order.
__global__ void __launch_bounds__(THREADS) truncate_kernel(Tables t) {
    extern __shared__ uint32_t sh[];
    __shared__ uint64_t scratch[2][WARPS];
    uint32_t* off = sh;                    // [rows + 1]
    const uint32_t per = (t.rows + THREADS - 1) / THREADS;
    const uint32_t r0 = min(t.rows, threadIdx.x * per), r1 = min(t.rows, r0 + per);
    const auto held = [&](int32_t n) { return min((uint32_t)pages_of(n, t.page_shift), t.width); };
    uint64_t pages = 0, none = 0;
    for (uint32_t r = r0; r < r1; ++r) {
        const int32_t len = max(t.lens[r], 0);
        pages += held(len) - held(min(len, max(t.step[r], 0)));
    }
    uint64_t at = pages, all, all_none;
    block_scan(at, none, all, all_none, scratch);
    for (uint32_t r = r0; r < r1; ++r) {
        const int32_t len = max(t.lens[r], 0), keep = min(len, max(t.step[r], 0));
        off[r] = (uint32_t)at;
        at += held(len) - held(keep);
        if (blockIdx.x == 0) t.lens_out[r] = keep;
    }
    const uint32_t stack = (uint32_t)min(max(*t.n_free, 0), (int)t.pool);
    const uint32_t room = t.pool - stack;
    const uint32_t back = all < room ? (uint32_t)all : room;
    if (threadIdx.x == 0) {
        off[t.rows] = (uint32_t)all;
        if (blockIdx.x == 0) *t.n_free_out = (int32_t)(stack + back);
    }
    __syncthreads();
    for (uint32_t e = blockIdx.x * THREADS + threadIdx.x; e < back; e += gridDim.x * THREADS) {
        const uint32_t r = row_of(off, t.rows, e);
        const int32_t len = max(t.lens[r], 0);
        const uint32_t col = held(min(len, max(t.step[r], 0))) + (e - off[r]);
        t.free_pages[stack + e] = t.block_tables[(size_t)r * t.width + col];
    }
}

static unsigned ctas_for(uint64_t work) {
    const uint64_t n = (work + PER_CTA - 1) / PER_CTA;
    return (unsigned)(n < 1 ? 1 : (n > 148 ? 148 : n));
}

cudaError_t launch_build_tables(const Tables& t, cudaStream_t stream) {
    const size_t smem = 2 * ((size_t)t.rows + 1) * sizeof(uint32_t);
    build_tables_kernel<<<ctas_for(t.max_tokens), THREADS, smem, stream>>>(t);
    return cudaGetLastError();
}

cudaError_t launch_truncate(const Tables& t, cudaStream_t stream) {
    const size_t smem = ((size_t)t.rows + 1) * sizeof(uint32_t);
    truncate_kernel<<<ctas_for((uint64_t)t.rows * t.width), THREADS, smem, stream>>>(t);
    return cudaGetLastError();
}

}  // namespace paged
}  // namespace kvq
