// Rows of the paged 4-bit cache by slot: keys and values quantized into their
// slots (append), and slots read back as values (gather).
//
// A slot s is position s % ps of page s / ps; cache head h's row there is row
// ((s / ps) * HKV + h) * ps + s % ps of the pool. A thread holds 8 codes (one
// packed word) of a row, so a group's minimum and maximum are shuffles over
// GROUP / 8 lanes and a row is read and written once, whole sectors at a time.
// The CTA's warps take consecutive tokens of one cache head, which lie side by
// side in a page. Bound by the bytes moved once the step is long, by the launch
// for a few tokens.
#include "kvq_common.cuh"
#include "kvq_paged.h"

namespace kvq {
namespace paged {

constexpr int THREADS = 256;

// the quantizer's rounding: sign(x) * floor(|x| + 0.5), the add in fp32
__device__ __forceinline__ float half_away(float x) {
    return copysignf(floorf(__fadd_rn(fabsf(x), 0.5f)), x);
}

// min(half_away(x / step), 15) as the canonical quantizer has it, mostly
// without its division. y = x * (1 / step) with both factors rounded is within
// 3 * 2^-24 of the rounded quotient relatively, so within 2^-18 below 16, and
// the rounded sum with 0.5 adds 2^-21 at most: where |y| + 0.5 stands further
// than 2^-17 from a whole number (from 16 up every value gives 15), the
// quotient's floor is the same. The rest, about one value in 2^16 of smooth
// data, divides; so do NaN and infinities, which fail the comparison.
__device__ __forceinline__ uint32_t code_of(float x, float step, float inv) {
    const float y = __fmul_rn(x, inv);
    const float s = __fadd_rn(fabsf(y), 0.5f);
    const float f = floorf(s), d = s - f;
    if (d > 7.62939453125e-6f && d < 1.0f - 7.62939453125e-6f) return (uint32_t)fminf(copysignf(f, y) + 0.0f, 15.0f);
    return (uint32_t)(int)fminf(half_away(__fdiv_rn(x, step)), 15.0f);
}

template <typename T>
__device__ __forceinline__ void load8(const T* p, bool vec, float (&x)[8]) {
    if (vec) {
        constexpr int N = 8 * sizeof(T) / 16;
        uint4 raw[N];
#pragma unroll
        for (int i = 0; i < N; ++i) raw[i] = reinterpret_cast<const uint4*>(p)[i];
        const T* v = reinterpret_cast<const T*>(raw);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f32(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f32(p[i]);
    }
}

template <typename T, int DH, int GROUP>
__global__ void __launch_bounds__(THREADS) append_kernel(Rows r) {
    constexpr int LANES = DH / 8;                  // lanes of a row
    constexpr int GL = GROUP / 8;                  // lanes of a group
    constexpr int ROWS = THREADS / LANES;
    const uint32_t lane = threadIdx.x % LANES;
    const uint32_t tok = blockIdx.x * ROWS + threadIdx.x / LANES;
    const uint32_t head = blockIdx.y >> 1, side = blockIdx.y & 1;
    const int64_t slot = tok < r.tokens ? r.slots[tok] : -1;
    // a warp's rows leave together only when none is written, so the shuffles
    // below always have all their lanes
    const bool live = slot >= 0 && (uint64_t)slot < r.slots_end;
    if (!__any_sync(0xffffffffu, live)) return;

    float x[8];
    if (live)
        load8(static_cast<const T*>(r.src[side]) + tok * r.token_stride[side] +
                  head * r.head_stride[side] + lane * 8, r.vec, x);
    else
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = 0.0f;
    float lo = INFINITY, hi = -INFINITY;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        lo = fminf(lo, x[i]);
        hi = fmaxf(hi, x[i]);
    }
#pragma unroll
    for (int o = GL / 2; o > 0; o >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
    hi = fmaxf(hi, 0.0f);
    float step = fmaxf(__fdiv_rn(__fsub_rn(hi, lo), 15.0f), 1e-7f);
    const bool low_side = fabsf(lo) > fabsf(hi);
    step = low_side ? step : -step;
    const float edge = low_side ? lo : hi;
    const float n_edge = half_away(__fdiv_rn(edge, step));
    const bool degenerate = n_edge == 0.0f;
    if (!degenerate) step = __fdiv_rn(edge, n_edge);
    const float bias = degenerate ? 0.0f : edge;

    const float inv = __frcp_rn(step);
    uint32_t word = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) word |= code_of(__fsub_rn(x[i], bias), step, inv) << (4 * i);
    if (!live) return;
    const uint64_t page = (uint64_t)slot >> r.page_shift;
    const uint64_t row = ((page * r.heads + head) << r.page_shift) + ((uint64_t)slot & ((1u << r.page_shift) - 1));
    const Pool& p = r.pool[side];
    p.words[row * LANES + lane] = word;
    if (lane % GL == 0) {
        const uint64_t g = row * (DH / GROUP) + lane / GL;
        static_cast<T*>(p.scales)[g] = from_f32<T>(step);
        static_cast<T*>(p.biases)[g] = from_f32<T>(bias);
    }
}

// Values scale * code + bias (a rounded multiply, a rounded add, then the
// output type's rounding); zeros for a slot that is not in the pool.
template <typename T, typename TO>
__global__ void __launch_bounds__(THREADS) gather_kernel(Rows r) {
    const uint32_t lanes = r.head_dim / 8, rows = THREADS / lanes;
    const uint32_t lane = threadIdx.x % lanes;
    const uint32_t tok = blockIdx.x * rows + threadIdx.x / lanes;
    const uint32_t head = blockIdx.y >> 1, side = blockIdx.y & 1;
    if (tok >= r.tokens) return;
    const int64_t slot = r.slots[tok];
    alignas(16) TO v[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = from_f32<TO>(0.0f);
    if (slot >= 0 && (uint64_t)slot < r.slots_end) {
        const uint64_t page = (uint64_t)slot >> r.page_shift;
        const uint64_t row = ((page * r.heads + head) << r.page_shift) + ((uint64_t)slot & ((1u << r.page_shift) - 1));
        const Pool& p = r.pool[side];
        const uint64_t g = row * (r.head_dim / r.group) + lane * 8 / r.group;
        const uint32_t w = p.words[row * lanes + lane];
        const float s = to_f32(static_cast<const T*>(p.scales)[g]);
        const float b = to_f32(static_cast<const T*>(p.biases)[g]);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = from_f32<TO>(dequant(s, (w >> (4 * i)) & 15u, b));
    }
    TO* out = static_cast<TO*>(r.dst[side]) + ((uint64_t)tok * r.heads + head) * r.head_dim + lane * 8;
#pragma unroll
    for (int i = 0; i < (int)(8 * sizeof(TO) / 16); ++i)
        reinterpret_cast<uint4*>(out)[i] = reinterpret_cast<const uint4*>(v)[i];
}

template <typename T, int DH, int GROUP>
static cudaError_t append_one(const Rows& r, cudaStream_t stream) {
    constexpr uint32_t ROWS = THREADS / (DH / 8);
    append_kernel<T, DH, GROUP><<<dim3((r.tokens + ROWS - 1) / ROWS, 2 * r.heads), THREADS, 0, stream>>>(r);
    return cudaGetLastError();
}

template <typename T>
static cudaError_t append_typed(const Rows& r, cudaStream_t stream) {
    switch (r.head_dim * 1000 + r.group) {
        case 64032: return append_one<T, 64, 32>(r, stream);
        case 64064: return append_one<T, 64, 64>(r, stream);
        case 128032: return append_one<T, 128, 32>(r, stream);
        case 128064: return append_one<T, 128, 64>(r, stream);
        case 128128: return append_one<T, 128, 128>(r, stream);
    }
    return cudaErrorInvalidValue;
}

cudaError_t launch_append(const Rows& r, cudaStream_t stream) {
    return r.dtype == KVQ_F16 ? append_typed<__half>(r, stream) : append_typed<float>(r, stream);
}

cudaError_t launch_gather(const Rows& r, cudaStream_t stream) {
    const uint32_t rows = THREADS / (r.head_dim / 8);
    const dim3 grid((r.tokens + rows - 1) / rows, 2 * r.heads);
    if (r.dtype == KVQ_F32)
        gather_kernel<float, float><<<grid, THREADS, 0, stream>>>(r);
    else if (r.out_dtype == KVQ_F32)
        gather_kernel<__half, float><<<grid, THREADS, 0, stream>>>(r);
    else
        gather_kernel<__half, __half><<<grid, THREADS, 0, stream>>>(r);
    return cudaGetLastError();
}

}  // namespace paged
}  // namespace kvq
