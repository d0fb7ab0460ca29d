// Rows of the paged 4-bit cache by slot: keys and values quantized into their
// slots (append), and slots read back as values (gather).
//
// A slot s is position s % ps of page s / ps; cache head h's row there is row
// ((s / ps) * HKV + h) * ps + s % ps of the pool. A thread holds 16 codes (two
// packed words) of a row, so a group's minimum and maximum are shuffles over
// GROUP / 16 lanes and a row is read and written once, whole sectors at a time.
// The CTA's warps take consecutive tokens of one cache head, which lie side by
// side in a page. Bound by instructions once the step is long (so the arithmetic
// below is what it is), by the launch for a few tokens. 8192 fp16 tokens of 8 heads
// of 128, groups of 64: append 14.3 us (43 MB; with 8 codes a thread, whose group
// arithmetic is then done twice as often, 24), read-back 8.9 us (43 MB; 11).
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
// canonical quantizer has them, mostly without its division. With d = x - bias
// and 1 / step rounded, d * (1 / step) is within 2^-23 of the rounded quotient
// relatively, so within 2^-19 below 16, and the two additions of 0.5 round by
// 2^-21 at most: where s = d * (1 / step) + 0.5 stands further than 2^-17 from a
// whole number, the quotient's floor is the same (from 15.75 up every value gives
// 15, and so does NaN, here as there). If one of the eight stands nearer, about
// one lane in 2^13 of smooth data, all of them divide. The floor is the low bits
// of s + 2^23 rounded down, and the eight are put together in one word with those
// of 2^23, whose sum is taken off at the end.
__device__ __forceinline__ uint32_t codes_of(const float2 (&x)[4], float bias, float step, float inv) {
    const auto both = [](float f) { return make_float2(f, f); };
    uint32_t word = 0;
    float worst = 0.0f;
#pragma unroll
    for (int i = 3; i >= 0; --i) {
        float2 s = __ffma2_rn(__fadd2_rn(x[i], both(-bias)), both(inv), both(0.5f));
        s.x = fminf(fabsf(s.x), 15.75f);
        s.y = fminf(fabsf(s.y), 15.75f);
        const float2 t = __fadd2_rd(s, both(8388608.0f));
        // s - floor(s) - 0.5
        const float2 off = __fadd2_rn(__fadd2_rn(s, __ffma2_rn(t, both(-1.0f), both(8388608.0f))), both(-0.5f));
        worst = fmaxf(fmaxf(worst, fabsf(off.x)), fabsf(off.y));
        word = (word * 16u + __float_as_uint(t.y)) * 16u + __float_as_uint(t.x);
    }
    word -= 0x4B000000u * 0x11111111u;
    if (worst < 0.5f - 7.62939453125e-6f) return word;
    word = 0;
#pragma unroll
    for (int i = 7; i >= 0; --i) {
        const float v = i & 1 ? x[i / 2].y : x[i / 2].x;
        word = word * 16u + (uint32_t)(int)fminf(half_away(__fdiv_rn(__fsub_rn(v, bias), step)), 15.0f);
    }
    return word;
}

constexpr int E = 16;                              // a thread's values of a row

// min and max over a thread's values and its group's lanes (NaNs are passed over)
template <int LANES>
__device__ __forceinline__ void range_of(const __half2 (&x)[E / 2], float& lo, float& hi) {
    const __half2 inf = __half2half2(__ushort_as_half(0x7C00));
    __half2 a = inf, b = __hneg2(inf);
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
        a = __hmin2(a, x[i]);
        b = __hmax2(b, x[i]);
    }
    b = __hneg2(b);
    __half2 m = __hmin2(__lows2half2(a, b), __highs2half2(a, b));         // (min, -max)
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) m = __hmin2(m, __shfl_xor_sync(0xffffffffu, m, o));
    lo = __low2float(m);
    hi = -__high2float(m);
}
template <int LANES>
__device__ __forceinline__ void range_of(const float2 (&x)[E / 2], float& lo, float& hi) {
    lo = INFINITY;
    hi = -INFINITY;
#pragma unroll
    for (int i = 0; i < E / 2; ++i) {
        lo = fminf(fminf(lo, x[i].x), x[i].y);
        hi = fmaxf(fmaxf(hi, x[i].x), x[i].y);
    }
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) {
        lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
        hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
    }
}
__device__ __forceinline__ float2 floats_of(__half2 x) { return __half22float2(x); }
__device__ __forceinline__ float2 floats_of(float2 x) { return x; }

template <typename T, int DH, int GROUP, bool VEC>
__global__ void __launch_bounds__(THREADS) append_kernel(Rows r) {
    using Two = typename std::conditional<sizeof(T) == 2, __half2, float2>::type;
    constexpr int LANES = DH / E;                  // lanes of a row
    constexpr int GL = GROUP / E;                  // lanes of a group
    constexpr int ROWS = THREADS / LANES;
    const uint32_t lane = threadIdx.x % LANES;
    const uint32_t tok = blockIdx.x * ROWS + threadIdx.x / LANES;
    const uint32_t head = blockIdx.y >> 1, side = blockIdx.y & 1;
    const int64_t slot = tok < r.tokens ? r.slots[tok] : -1;
    // a warp's rows leave together only when none is written, so the shuffles
    // below always have all their lanes
    const bool live = slot >= 0 && (uint64_t)slot < r.slots_end;
    if (!__any_sync(0xffffffffu, live)) return;

    alignas(16) Two x[E / 2];
    if (live) {
        const T* src = static_cast<const T*>(r.src[side]) + tok * r.token_stride[side] + head * r.head_stride[side] + lane * E;
        if constexpr (VEC) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(x) / 16; ++i)
                reinterpret_cast<uint4*>(x)[i] = reinterpret_cast<const uint4*>(src)[i];
        } else {
#pragma unroll
            for (int i = 0; i < E; ++i) reinterpret_cast<T*>(x)[i] = src[i];
        }
    } else {
#pragma unroll
        for (int i = 0; i < (int)sizeof(x) / 16; ++i) reinterpret_cast<uint4*>(x)[i] = make_uint4(0u, 0u, 0u, 0u);
    }
    float lo, hi;
    range_of<GL>(x, lo, hi);
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

    uint32_t word[E / 8];
#pragma unroll
    for (int w = 0; w < E / 8; ++w) {
        const float2 v[4] = {floats_of(x[4 * w]), floats_of(x[4 * w + 1]), floats_of(x[4 * w + 2]), floats_of(x[4 * w + 3])};
        word[w] = codes_of(v, bias, step, inv);
    }
    if (!live) return;
    // the pool has fewer than 2^32 rows
    const uint32_t page = (uint32_t)((uint64_t)slot >> r.page_shift);
    const uint32_t row = ((page * r.heads + head) << r.page_shift) + ((uint32_t)slot & ((1u << r.page_shift) - 1));
    const Pool& p = r.pool[side];
    reinterpret_cast<uint2*>(p.words)[(uint64_t)row * LANES + lane] = make_uint2(word[0], word[1]);
    if (lane % GL == 0) {
        const uint64_t g = (uint64_t)row * (DH / GROUP) + lane / GL;
        static_cast<T*>(p.scales)[g] = from_f32<T>(step);
        static_cast<T*>(p.biases)[g] = from_f32<T>(bias);
    }
}

// Values scale * code + bias (a rounded multiply, a rounded add, then the
// output type's rounding); zeros for a slot that is not in the pool.
template <typename T, typename TO, int DH, int GROUP>
__global__ void __launch_bounds__(THREADS) gather_kernel(Rows r) {
    constexpr uint32_t lanes = DH / E, rows = THREADS / lanes;
    const uint32_t lane = threadIdx.x % lanes;
    const uint32_t tok = blockIdx.x * rows + threadIdx.x / lanes;
    const uint32_t head = blockIdx.y >> 1, side = blockIdx.y & 1;
    if (tok >= r.tokens) return;
    const int64_t slot = r.slots[tok];
    alignas(16) TO v[E];
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = from_f32<TO>(0.0f);
    if (slot >= 0 && (uint64_t)slot < r.slots_end) {
        const uint32_t page = (uint32_t)((uint64_t)slot >> r.page_shift);
        const uint32_t row = ((page * r.heads + head) << r.page_shift) + ((uint32_t)slot & ((1u << r.page_shift) - 1));
        const Pool& p = r.pool[side];
        const uint64_t g = (uint64_t)row * (DH / GROUP) + lane * E / GROUP;
        const uint2 two = reinterpret_cast<const uint2*>(p.words)[(uint64_t)row * lanes + lane];
        const float s = to_f32(static_cast<const T*>(p.scales)[g]);
        const float b = to_f32(static_cast<const T*>(p.biases)[g]);
        // codes i and i + 4 as fp16 1024 + c (even i) or 1024 + 16 c; for fp16 scales s * c
        // is one rounded multiply-add of that, as 1024 s and s / 16 are exact. (For fp32 ones
        // they may be infinite or subnormal: the code first, exactly.)
        const float s16 = s * 0.0625f, m1024 = s * -1024.0f, m64 = s * -64.0f;
#pragma unroll
        for (int j = 0; j < E / 8; ++j) {
            const uint32_t w = j ? two.y : two.x;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t h = ((i & 2 ? w >> 8 : w) & (i & 1 ? 0x00F000F0u : 0x000F000Fu)) | 0x64006400u;
                const float2 c = __half22float2(*reinterpret_cast<const __half2*>(&h));
                const auto both = [&](float odd, float even) { return i & 1 ? make_float2(odd, odd) : make_float2(even, even); };
                float2 y;
                if constexpr (sizeof(T) == 2) {
                    y = __fadd2_rn(__ffma2_rn(c, both(s16, s), both(m64, m1024)), both(b, b));
                } else {
                    // (scalar: a packed product and sum come out as one fused operation)
                    const float2 code = __ffma2_rn(c, both(0.0625f, 1.0f), both(-64.0f, -1024.0f));
                    y = make_float2(__fadd_rn(__fmul_rn(code.x, s), b), __fadd_rn(__fmul_rn(code.y, s), b));
                }
                v[8 * j + i] = from_f32<TO>(y.x);
                v[8 * j + i + 4] = from_f32<TO>(y.y);
            }
        }
    }
    TO* out = static_cast<TO*>(r.dst[side]) + ((uint64_t)tok * r.heads + head) * DH + lane * E;
#pragma unroll
    for (int i = 0; i < (int)(E * sizeof(TO) / 16); ++i)
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
    const uint32_t rows = THREADS / (r.head_dim / E);
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
