// How the paged attention kernels divide a ragged step among their CTAs.
//
// The step is a list of units (request, cache head, tile of query columns),
// each a run of key tiles. Only the device knows the lengths, so every CTA
// makes the running sum of the requests' tiles in shared memory and takes an
// equal, contiguous share of the whole list: no CTA has more than one share
// whatever the lengths, and none waits for another. (The few-token kernel's
// tiles are the cached ones; a unit's own entries come with its first tile and
// are not counted.) A unit that lies in one share is finished there. Of the
// others, a CTA leaves at most two partial results -- of the unit that began
// before its share (slot 0), and of the one that goes on after it (slot 1) --
// and the merge kernel joins a unit's parts, which are those of consecutive
// CTAs, in their order (results do not depend on timing).
#pragma once

#include <atomic>

#include "kvq_common.cuh"
#include "kvq_paged.h"

namespace kvq {
namespace paged {

// What the CTA in whose share a split unit begins leaves for the merge: the
// unit spans this CTA and the parts - 1 that follow. parts = 0: none.
struct Split {
    uint32_t parts, token0, hk, col0, cols;
};

// Partials live in the workspace as [grid] Split, then per (CTA, slot) m[cols],
// l[cols], O[cols][DH]; all of it is written before it is read.
__host__ __device__ inline size_t split_bytes(uint32_t grid) { return ((size_t)grid * sizeof(Split) + 255) / 256 * 256; }
__host__ __device__ inline size_t slot_floats(uint32_t cols, uint32_t dh) { return (size_t)cols * (dh + 2); }

// The request's tokens in this step, cut to the bounds the caller gave.
struct Request {
    uint32_t ctx, token0, n;
};
__device__ __forceinline__ Request request_of(const Attend& a, uint32_t b) {
    Request r;
    r.ctx = min((uint32_t)max(a.ctx_lens[b], 0), a.max_ctx);
    r.token0 = min((uint32_t)max(a.cu_new[b], 0), a.tokens);
    const uint32_t end = min((uint32_t)max(a.cu_new[b + 1], 0), a.tokens);
    r.n = end > r.token0 ? min(end - r.token0, a.max_new) : 0;
    return r;
}

// before[b] = tiles of the requests in front of b, before[rows] the total:
// tiles_of(b) summed over the rows by all THREADS threads of the block. Sums
// stop at TOO_MANY (the host refuses steps that can have as many, so only
// offsets that are no running sum get there): returned as a total of 0, and
// the step is left undone.
constexpr uint64_t TOO_MANY = 0x7FFFFFFFull;
template <int THREADS, typename F>
__device__ uint32_t sum_tiles(uint32_t* before, uint32_t rows, F&& tiles_of) {
    __shared__ uint64_t scratch[THREADS / 32];
    const uint32_t tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const uint32_t per = (rows + THREADS - 1) / THREADS;
    const uint32_t r0 = min(rows, tid * per), r1 = min(rows, r0 + per);
    uint64_t own = 0;
    for (uint32_t r = r0; r < r1; ++r) {
        const uint64_t t = min((uint64_t)tiles_of(r), TOO_MANY);
        if (per > 1) before[r] = (uint32_t)t;
        own += t;
    }
    uint64_t incl = own;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint64_t u = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= (uint32_t)o) incl += u;
    }
    if (lane == 31) scratch[warp] = incl;
    __syncthreads();
    uint64_t at = incl - own, total = 0;
    for (uint32_t w = 0; w < THREADS / 32; ++w) {
        if (w < warp) at += scratch[w];
        total += scratch[w];
    }
    if (per == 1) {
        if (r0 < r1) before[r0] = (uint32_t)at;
    } else {
        for (uint32_t r = r0; r < r1; ++r) {
            const uint32_t t = before[r];
            before[r] = (uint32_t)at;
            at += t;
        }
    }
    if (tid == THREADS - 1) before[rows] = (uint32_t)total;
    __syncthreads();
    return total < TOO_MANY ? (uint32_t)total : 0;
}

// The last request in front of which at most x tiles lie.
__device__ __forceinline__ uint32_t row_of_tile(const uint32_t* before, uint32_t rows, uint32_t x) {
    uint32_t lo = 0, hi = rows;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (before[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

// A block per (CTA of the split kernel, JOIN_COLS columns): the unit's parts
// joined, out = sum_p O_p 2^(m_p - m) / sum_p l_p 2^(m_p - m), m = max_p m_p in
// log2. A column's parts are shared out among several warps, whose loads do not
// wait for the weights: a long sequence's unit has about 20 parts, and one warp
// that walked them took 12 us.
constexpr int JOIN_WARPS = 8;
template <typename T, int DH, int COLS>
__global__ void __launch_bounds__(32 * JOIN_WARPS) join_kernel(Attend a, const unsigned char* ws) {
    constexpr int V = DH / 32;             // dims per lane
    constexpr int PW = COLS > 32 ? 1 : 4;  // warps per column
    constexpr int JC = JOIN_WARPS / PW;    // columns per block
    constexpr int AHEAD = 5;               // parts a warp has in flight
    constexpr size_t SLOT = (size_t)COLS * (DH + 2);
    using Vec = typename std::conditional<V == 4, float4, float2>::type;
    __shared__ Vec sum_o[JOIN_WARPS][32];
    __shared__ float sum_m[JOIN_WARPS], sum_l[JOIN_WARPS];
    pdl_wait();
    const uint32_t cta = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = warp % PW;
    const uint32_t col = blockIdx.y * JC + warp / PW;
    // this grid may have been launched while the one that wrote the parts still ran:
    // they are read through L2, past lines an SM may have cached
    Split u;
    {
        const uint32_t* s = reinterpret_cast<const uint32_t*>(reinterpret_cast<const Split*>(ws) + cta);
        u = {__ldcg(s), __ldcg(s + 1), __ldcg(s + 2), __ldcg(s + 3), __ldcg(s + 4)};
    }
    if (u.parts == 0 || blockIdx.y * JC >= u.cols) return;
    const float* slots = reinterpret_cast<const float*>(ws + split_bytes(gridDim.x));
    // part 0 is this CTA's slot 1, part p > 0 CTA cta + p's slot 0
    const auto part = [&](uint32_t p) { return slots + (2 * (size_t)(cta + p) + (p == 0 ? 1 : 0)) * SLOT; };
    float o[V], l = 0.0f, m = -INFINITY;
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = 0.0f;
    if (col < u.cols)
        for (uint32_t p0 = sub; p0 < u.parts; p0 += PW * AHEAD) {
            Vec v[AHEAD];
            float pm[AHEAD], pl[AHEAD], top = m;
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const uint32_t p = p0 + i * PW;
                pm[i] = -INFINITY;
                if (p < u.parts) {
                    const float* s = part(p);
                    pm[i] = __ldcg(s + col);
                    pl[i] = __ldcg(s + COLS + col);
                    v[i] = __ldcg(reinterpret_cast<const Vec*>(s + 2 * COLS + (size_t)col * DH + lane * V));
                }
            }
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) top = fmaxf(top, pm[i]);
            const float keep = m == top ? 1.0f : exp2f(m - top);
            m = top;
            l *= keep;
#pragma unroll
            for (int d = 0; d < V; ++d) o[d] *= keep;
#pragma unroll
            for (int i = 0; i < AHEAD; ++i)
                if (p0 + i * PW < u.parts) {
                    const float f = exp2f(pm[i] - m);
                    const float* x = reinterpret_cast<const float*>(&v[i]);
                    l += f * pl[i];
#pragma unroll
                    for (int d = 0; d < V; ++d) o[d] += f * x[d];
                }
        }
    if constexpr (PW > 1) {
        sum_o[warp][lane] = *reinterpret_cast<const Vec*>(o);
        if (lane == 0) {
            sum_m[warp] = m;
            sum_l[warp] = l;
        }
        __syncthreads();
        if (sub != 0) return;
        float top = m;
#pragma unroll
        for (int w = 1; w < PW; ++w) top = fmaxf(top, sum_m[warp + w]);
        const float keep = exp2f(m - top);
        l *= keep;
#pragma unroll
        for (int d = 0; d < V; ++d) o[d] *= keep;
#pragma unroll
        for (int w = 1; w < PW; ++w) {
            const float f = exp2f(sum_m[warp + w] - top);
            const Vec v = sum_o[warp + w][lane];
            const float* x = reinterpret_cast<const float*>(&v);
            l += f * sum_l[warp + w];
#pragma unroll
            for (int d = 0; d < V; ++d) o[d] += f * x[d];
        }
    }
    if (col >= u.cols) return;
    const uint32_t c = u.col0 + col, tok = u.token0 + c / a.r, head = u.hk * a.r + c % a.r;
    T* out = static_cast<T*>(a.out) + ((size_t)tok * a.n_heads + head) * DH + lane * V;
#pragma unroll
    for (int i = 0; i < V; ++i) out[i] = from_f32<T>(o[i] / l);
}

// A kernel's dynamic shared memory limit, set once per device (`done` is the
// kernel's own), so that later launches, captured ones included, make no
// attribute calls.
template <typename K>
cudaError_t allow_smem(K kernel, size_t bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return e;
    const uint64_t bit = dev >= 0 && dev < 64 ? 1ull << dev : 0;
    if (bit && (done.load(std::memory_order_acquire) & bit)) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e != cudaSuccess) return e;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributePreferredSharedMemoryCarveout, cudaSharedmemCarveoutMaxShared);
    if (e == cudaSuccess) done.fetch_or(bit, std::memory_order_acq_rel);
    return e;
}

template <typename T, int DH, int COLS>
cudaError_t launch_join(const Attend& a, uint32_t grid, const unsigned char* ws, cudaStream_t stream) {
    cudaLaunchConfig_t cfg{};
    constexpr int per_block = COLS > 32 ? JOIN_WARPS : JOIN_WARPS / 4;
    cfg.gridDim = dim3(grid, (COLS + per_block - 1) / per_block);
    cfg.blockDim = dim3(32 * JOIN_WARPS);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, join_kernel<T, DH, COLS>, a, ws);
}

}  // namespace paged
}  // namespace kvq
