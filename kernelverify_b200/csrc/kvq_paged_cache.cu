// Rows of the paged 4-bit cache by slot: keys and values quantized into their
// slots (append), and slots read back as values (gather).
//
// A slot s is position s % ps of page s / ps; cache head h's row there is row
// ((s / ps) * HKV + h) * ps + s % ps of the pool. A thread holds 8 codes (one
// packed word) of a row, so a group's minimum and maximum are shuffles over
// GROUP / 8 lanes and a row is read and written once, whole sectors at a time.
// The CTA's warps take consecutive tokens of one cache head, which lie side by
// side in a page. Bound by instructions once the step is long (so the arithmetic
// below is what it is), by the launch for a few tokens. Four tokens per lane,
// loaded ahead, were slower: 33 us against 25 for 8192 tokens of 8 heads.
#include "kvq_common.cuh"
#include "kvq_paged.h"

namespace kvq {
namespace paged {

constexpr int THREADS = 256;

// the quantizer's rounding: sign(x) * floor(|x| + 0.5), the add in fp32
__device__ __forceinline__ float half_away(float x) {
    return copysignf(floorf(__fadd_rn(fabsf(x), 0.5f)), x);
}

// The codes min(half_away((x - bias) / step), 15) of eight values as the
// canonical quantizer has them, mostly without its division. y = (x - bias) *
// (1 / step) with the last two rounded is within 3 * 2^-24 of the rounded
// quotient relatively, so within 2^-18 below 16, and the rounded sum with 0.5
// adds 2^-21 at most: where s = |y| + 0.5 stands further than 2^-17 from a whole
// number, the quotient's floor is the same (from 15.75 up every value gives 15,
// and so does NaN, here as there). If one of the eight stands nearer, about one
// lane in 2^13 of smooth data, all of them divide. The floor is the low bits of
// s + 2^23 rounded down, and the eight are put together in one word with those
// of 2^23, whose sum is taken off at the end.
__device__ __forceinline__ uint32_t codes_of(const float (&x)[8], float bias, float step) {
    const float inv = __frcp_rn(step);
    uint32_t word = 0;
    float worst = 0.0f;
#pragma unroll
    for (int i = 7; i >= 0; --i) {
        const float s = fminf(__fadd_rn(fabsf(__fmul_rn(__fsub_rn(x[i], bias), inv)), 0.5f), 15.75f);
        const float t = __fadd_rd(s, 8388608.0f);
        worst = fmaxf(worst, fabsf(__fsub_rn(__fsub_rn(s, 0.5f), __fsub_rn(t, 8388608.0f))));
        word = word * 16u + __float_as_uint(t);
    }
    word -= 0x4B000000u * 0x11111111u;
    if (worst < 0.5f - 7.62939453125e-6f) return word;
    word = 0;
#pragma unroll 1
    for (int i = 7; i >= 0; --i)
        word = word * 16u + (uint32_t)(int)fminf(half_away(__fdiv_rn(__fsub_rn(x[i], bias), step)), 15.0f);
    return word;
}

template <bool VEC, typename T>
__device__ __forceinline__ void load8(const T* p, float (&x)[8]) {
    if constexpr (VEC) {
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

template <typename T, int DH, int GROUP, bool VEC>
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
        load8<VEC>(static_cast<const T*>(r.src[side]) + tok * r.token_stride[side] +
                       head * r.head_stride[side] + lane * 8, x);
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

    const uint32_t word = codes_of(x, bias, step);
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
template <typename T, typename TO, int DH, int GROUP>
__global__ void __launch_bounds__(THREADS) gather_kernel(Rows r) {
    constexpr uint32_t lanes = DH / 8, rows = THREADS / lanes;
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
        const uint64_t g = row * (DH / GROUP) + lane * 8 / GROUP;
        const uint32_t w = p.words[row * lanes + lane];
        const float s = to_f32(static_cast<const T*>(p.scales)[g]);
        const float b = to_f32(static_cast<const T*>(p.biases)[g]);
        // codes i and i + 4 as fp16 1024 + c (even i) or 1024 + 16 c; s * c is one
        // rounded multiply-add of that, as 1024 s and s / 16 are exact
        const float s16 = s * 0.0625f, m1024 = s * -1024.0f, m64 = s * -64.0f;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t h = ((i & 2 ? w >> 8 : w) & (i & 1 ? 0x00F000F0u : 0x000F000Fu)) | 0x64006400u;
            const float2 c = __half22float2(*reinterpret_cast<const __half2*>(&h));
            v[i] = from_f32<TO>(__fadd_rn(i & 1 ? fmaf(c.x, s16, m64) : fmaf(c.x, s, m1024), b));
            v[i + 4] = from_f32<TO>(__fadd_rn(i & 1 ? fmaf(c.y, s16, m64) : fmaf(c.y, s, m1024), b));
        }
    }
    TO* out = static_cast<TO*>(r.dst[side]) + ((uint64_t)tok * r.heads + head) * DH + lane * 8;
#pragma unroll
    for (int i = 0; i < (int)(8 * sizeof(TO) / 16); ++i)
        reinterpret_cast<uint4*>(out)[i] = reinterpret_cast<const uint4*>(v)[i];
}

// f(head_dim, group) as constants
template <typename F>
static cudaError_t by_format(const Rows& r, F&& f) {
    using std::integral_constant;
    switch (r.head_dim * 1000 + r.group) {
        case 64032: return f(integral_constant<int, 64>{}, integral_constant<int, 32>{});
        case 64064: return f(integral_constant<int, 64>{}, integral_constant<int, 64>{});
        case 128032: return f(integral_constant<int, 128>{}, integral_constant<int, 32>{});
        case 128064: return f(integral_constant<int, 128>{}, integral_constant<int, 64>{});
        case 128128: return f(integral_constant<int, 128>{}, integral_constant<int, 128>{});
    }
    return cudaErrorInvalidValue;
}

static dim3 grid_of(const Rows& r) {
    const uint32_t rows = THREADS / (r.head_dim / 8);
    return dim3((r.tokens + rows - 1) / rows, 2 * r.heads);
}

template <typename T>
static cudaError_t append_typed(const Rows& r, cudaStream_t stream) {
    return by_format(r, [&](auto dh, auto group) {
        if (r.vec) append_kernel<T, dh.value, group.value, true><<<grid_of(r), THREADS, 0, stream>>>(r);
        else append_kernel<T, dh.value, group.value, false><<<grid_of(r), THREADS, 0, stream>>>(r);
        return cudaGetLastError();
    });
}

template <typename T, typename TO>
static cudaError_t gather_typed(const Rows& r, cudaStream_t stream) {
    return by_format(r, [&](auto dh, auto group) {
        gather_kernel<T, TO, dh.value, group.value><<<grid_of(r), THREADS, 0, stream>>>(r);
        return cudaGetLastError();
    });
}

cudaError_t launch_append(const Rows& r, cudaStream_t stream) {
    return r.dtype == KVQ_F16 ? append_typed<__half>(r, stream) : append_typed<float>(r, stream);
}

cudaError_t launch_gather(const Rows& r, cudaStream_t stream) {
    if (r.dtype == KVQ_F32) return gather_typed<float, float>(r, stream);
    return r.out_dtype == KVQ_F32 ? gather_typed<__half, float>(r, stream) : gather_typed<__half, __half>(r, stream);
}

}  // namespace paged
}  // namespace kvq
