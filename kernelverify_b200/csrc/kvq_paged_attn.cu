// Attention of a step's tokens over the pages of a 4-bit cache and over the
// step's own keys and values. The simplest form: a CTA per (token, query
// head), a thread per position of a 128-position tile for the scores, a thread
// per dim for the combine, an online softmax across the tiles.
#include "kvq_common.cuh"
#include "kvq_paged.h"

namespace kvq {
namespace paged {

constexpr int TILE = 128;

template <typename T, int DH, int GROUP>
__global__ void __launch_bounds__(TILE) attend_kernel(Attend a) {
    __shared__ float q[DH], p[TILE], red[TILE / 32];
    __shared__ uint64_t rowbase[TILE / 16];
    __shared__ int bad;
    const uint32_t tok = blockIdx.x, head = blockIdx.y, hk = head / a.r;
    const int tid = threadIdx.x;
    // the request that brings this token
    uint32_t lo = 0, hi = a.rows;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if ((uint32_t)max(a.cu_new[mid], 0) <= tok) lo = mid;
        else hi = mid;
    }
    const uint32_t b = lo, c0 = max(a.cu_new[b], 0), c1 = max(a.cu_new[b + 1], 0);
    if (tok < c0 || tok >= c1) return;               // behind the last request
    const uint32_t ctx = min((uint32_t)max(a.ctx_lens[b], 0), a.max_ctx);
    const uint32_t n_pos = ctx + (tok - c0) + 1;
    for (int d = tid; d < DH; d += TILE)
        q[d] = to_f32(static_cast<const T*>(a.q)[tok * a.q_token + head * a.q_head + d]);
    float m = -INFINITY, l = 0.0f, o = 0.0f;
    for (uint32_t t0 = 0; t0 < n_pos; t0 += TILE) {
        __syncthreads();
        if (tid == 0) bad = 0;
        __syncthreads();
        if (tid < TILE / 16) {                       // a run of 16 positions lies in one page
            const uint32_t pos = t0 + tid * 16;
            if (pos < ctx) {
                uint32_t page = (uint32_t)a.block_tables[(size_t)b * a.width + (pos >> a.page_shift)];
                if (page >= a.pages) { bad = 1; page = 0; }
                rowbase[tid] = (((uint64_t)page * a.n_kv_heads + hk) << a.page_shift) + (pos & ((1u << a.page_shift) - 1));
            }
        }
        __syncthreads();
        const uint32_t pos = t0 + tid;
        float s = -INFINITY;
        if (pos < ctx) {
            const uint64_t row = rowbase[tid / 16] + tid % 16;
            s = 0.0f;
            for (int w = 0; w < DH / 8; ++w) {
                const uint32_t word = a.k.words[row * (DH / 8) + w];
                const uint64_t g = row * (DH / GROUP) + w * 8 / GROUP;
                const float sc = to_f32(static_cast<const T*>(a.k.scales)[g]);
                const float bi = to_f32(static_cast<const T*>(a.k.biases)[g]);
                for (int i = 0; i < 8; ++i) s += q[w * 8 + i] * dequant(sc, (word >> (4 * i)) & 15u, bi);
            }
        } else if (pos < n_pos) {
            const T* k = static_cast<const T*>(a.new_k) + (c0 + pos - ctx) * a.k_token + hk * a.k_head;
            s = 0.0f;
            for (int d = 0; d < DH; ++d) s += q[d] * to_f32(k[d]);
        }
        s *= a.scale;
        if (bad) s = NAN;
        float top = warp_max(s);
        if ((tid & 31) == 0) red[tid >> 5] = top;
        __syncthreads();
        top = m;
        for (int w = 0; w < TILE / 32; ++w) top = fmaxf(top, red[w]);
        const float e = expf(s - top), keep = expf(m - top);
        p[tid] = e;
        float sum = warp_sum(e);
        __syncthreads();
        if ((tid & 31) == 0) red[tid >> 5] = sum;
        __syncthreads();
        l *= keep;
        for (int w = 0; w < TILE / 32; ++w) l += red[w];
        m = top;
        if (tid < DH) {
            o *= keep;
            const uint32_t n = min((uint32_t)TILE, n_pos - t0);
            for (uint32_t j = 0; j < n; ++j) {
                float v;
                if (t0 + j < ctx) {
                    const uint64_t row = rowbase[j / 16] + j % 16, g = row * (DH / GROUP) + tid / GROUP;
                    v = dequant(to_f32(static_cast<const T*>(a.v.scales)[g]),
                                (a.v.words[row * (DH / 8) + tid / 8] >> (4 * (tid % 8))) & 15u,
                                to_f32(static_cast<const T*>(a.v.biases)[g]));
                } else {
                    v = to_f32(static_cast<const T*>(a.new_v)[(c0 + t0 + j - ctx) * a.v_token + hk * a.v_head + tid]);
                }
                o += p[j] * v;
            }
        }
    }
    if (tid < DH)
        static_cast<T*>(a.out)[((size_t)tok * a.n_heads + head) * DH + tid] = from_f32<T>(o / l);
}

template <typename T, int DH, int GROUP>
static cudaError_t one(const Attend& a, cudaStream_t s) {
    attend_kernel<T, DH, GROUP><<<dim3(a.tokens, a.n_heads), TILE, 0, s>>>(a);
    return cudaGetLastError();
}
template <typename T>
static cudaError_t typed(const Attend& a, cudaStream_t s) {
    switch (a.head_dim * 1000 + a.group) {
        case 64032: return one<T, 64, 32>(a, s);
        case 64064: return one<T, 64, 64>(a, s);
        case 128032: return one<T, 128, 32>(a, s);
        case 128064: return one<T, 128, 64>(a, s);
        case 128128: return one<T, 128, 128>(a, s);
    }
    return cudaErrorInvalidValue;
}

size_t attend_workspace(const Attend&) { return 0; }
cudaError_t launch_attend(const Attend& a, void*, cudaStream_t s) {
    return a.dtype == KVQ_F16 ? typed<__half>(a, s) : typed<float>(a, s);
}

}  // namespace paged
}  // namespace kvq
