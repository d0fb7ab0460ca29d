// Paged attention for requests with many new tokens (prompt chunks), fp16, on
// the 5th-generation tensor cores.
//
// A unit is up to 256 query rows of one (request, cache head): two M tiles of
// 128 rows, a row being one (token, query head), the R heads of a token side
// by side, so the R heads share every key they read. Keys come in tiles of
// 128: the cached positions first, dequantized to fp16, then the step's own
// entries under the causal mask. They are worked off in steps of 64 keys, and both
// products are tcgen05.mma kind::f16:
//
//   S_i = Q_i K^T   (both operands in shared memory, fp32 S in tensor memory)
//   O_i += P_i V    (P_i fp16 in tensor memory over its S_i's columns)
//
// Sixteen warps in four warpgroups:
//   0, 1  softmax of M tile 0 and 1, a thread per row: S from tensor memory,
//         an online softmax whose reference moves (and rescales O) only when
//         the row's maximum passed it by 2^14, P back to tensor memory; at the
//         end O / l to the output, or the unit's part to the workspace
//   2     loads: cached rows a thread per key, the next tile's words on their way
//         while this one's become fp16; tiles of own entries that every row sees by
//         tensor copies, the others by 16-byte asynchronous copies; all with the
//         128-byte swizzle the MMAs read
//   3     a warp per M tile whose elected lane issues its MMAs (one warp for both
//         spent 2,400 cycles on a step of 64 keys, waiting and issuing in turn)
// Each M tile has two S buffers, so that the scores of a step are there before
// the softmax is done with the one in front. K and V tiles have the same layout,
// rows of keys: K is read as a K-major operand, V as an MN-major one.
//
// 4096 tokens over 8192 cached ones, 32 heads over 8 of 128: 700 us, 980 TFLOP/s (756
// in a long run, under the power limit); a first chunk of 8192: 582 us, 945 TFLOP/s
// (630 to 640); 64 tokens of 64 requests over 8192: 580 us, 950 TFLOP/s (655). A step of
// 64 keys takes 2,200 cycles for both M tiles, of which the tensor pipe is busy for at
// least 1,024 (1,536 if, as it seems, MMAs 64 columns wide take as long as those of
// 128: without softmax and dequantizing it comes to 1,470 TFLOP/s), the special-function
// unit for 1,024 and each scheduler's issue slot for 1,100; what is left is their waiting
// for one another, which bounds the kernel. Half of the exponentials' share on the FMA
// pipe, more registers for the softmax and copies further ahead changed nothing. Steps of
// 128 keys with one score buffer per query tile fill the tensor memory just as well; they
// were slower (872 us against 842 for the 4096 tokens) while the maximum still was a pass
// of its own, and have not been tried since. At 128 registers a thread groups of 128
// spill 104 bytes, groups of 64 four.
//
// Rounded to fp16: the dequantized K and V (as a cache held in fp16 would be)
// and the weights P; everything else is fp32. P is at most 2^14 and its sum is
// taken before the rounding. (Root mean square error of an output over that of its own
// rounding, chunks of 64: 1.18 with an empty cache, 1.52 over 16 positions, 1.27 over 256,
// 1.10 over 1024, 1.02 over 8192.)
#pragma once

#include <cuda.h>

#include <atomic>

#include "kvq_paged_attn.h"
#include "kvq_paged_work.cuh"
#include "kvq_umma.cuh"

namespace kvq {
namespace paged {
namespace many {

using mma4::and_or;
using mma4::ex2;
using mma4::mbar_arrive;
using mma4::mbar_init;
using mma4::mbar_try_wait;
using umma::fence_async_smem;
using umma::idesc;
using umma::tc_fence_after;
using umma::tc_fence_before;
using umma::tmem_alloc;
using umma::tmem_dealloc;
using umma::tmem_relinquish;
using umma::tmem_wait_ld;
using umma::tmem_wait_st;
using umma::umma;
using umma::umma_commit;

constexpr int THREADS = 512;
constexpr int KT = 128;                    // keys per tile in shared memory
constexpr int KS = 64;                     // keys per step
constexpr int ROWS = 128;                  // query rows per M tile
constexpr int COLS = 2 * ROWS;             // query rows per unit
constexpr int STAGES = 2;                  // K and V tiles in shared memory, each
constexpr float RAISE = 14.0f, START = 4.0f;   // log2 room above the reference
constexpr long long WAIT_CYCLES = 2000000000ll;      // about a second

template <int DH>
struct Cfg {
    static constexpr int PANELS = DH / 64;             // 64 dims: 128-byte rows
    static constexpr int PANEL = KT * 128;
    static constexpr int TILE = PANELS * PANEL;        // a 128-row operand
    static constexpr int Q = 0;
    static constexpr int K = 2 * TILE;
    static constexpr int V = K + STAGES * TILE;
    static constexpr int BAR = V + STAGES * TILE;
    // q_full[2], s_full[2][2], p_full[2][2] (M tile, buffer), o_done[2], then k_full,
    // k_empty, v_full, v_empty [STAGES] each, and the MMA warps' last ones
    static constexpr int NBAR = 12 + 4 * STAGES + 2;
    static constexpr int MISC = BAR + NBAR * 8;        // TMEM address, error flag
    static constexpr int BEFORE = MISC + 16;           // uint32 [rows + 1]
    static constexpr uint32_t S0 = 0, O0 = 256;        // TMEM columns: S_i's buffer b at 128 i + 64 b, O_i at 256 + 128 i
    static_assert(PANEL % 1024 == 0, "swizzle atoms are 1024-byte aligned");
};

// ---- PTX wrappers ------------------------------------------------------------
__device__ __forceinline__ void ld32(uint32_t taddr, uint32_t* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,"
        "%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]),
          "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]),
          "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]),
          "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr));
}
__device__ __forceinline__ void st32(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
        "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]),
        "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]),
        "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
        : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem]
__device__ __forceinline__ void umma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(id), "r"(accumulate)
        : "memory");
}
// true in one lane of a converged warp
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred q;\n\telect.sync _|q, 0xffffffff;\n\tselp.u32 %0, 1, 0, q;\n\t}" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ float max_nan(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
// Descriptor of an operand with the 128-byte swizzle: rows of 128 bytes, eight
// to a 1024-byte atom. K-major (Q, K): the rows are M or N, atoms along them
// 1024 bytes apart. MN-major (V): the rows are K, atoms along them 1024 bytes
// apart (stride offset), the next 64 of N a panel apart (leading offset).
__device__ __forceinline__ uint64_t desc128(uint32_t saddr, uint32_t leading) {
    return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)((leading >> 4) & 0x3FFFu) << 16) |
           ((uint64_t)(1024u >> 4) << 32) | (1ull << 46) | (2ull << 61);
}
// byte offset of 16-byte chunk c (eight dims) of row r in a panel
__device__ __forceinline__ uint32_t swizzled(uint32_t r, uint32_t c) { return r * 128 + ((c ^ (r & 7)) << 4); }

// Every wait ends: after WAIT_CYCLES, or once another wait gave up. The rows of a
// CTA that gave up are NaN.
template <bool SLACK = false>
__device__ __forceinline__ void wait(uint64_t* bar, uint32_t parity, volatile int* err) {
    if (mbar_try_wait(bar, parity)) return;
    const long long t0 = clock64();
    do {
        // a role that is tiles ahead leaves the issue slots to the others
        if (SLACK) __nanosleep(100);
        if (mbar_try_wait(bar, parity) || *err) return;
    } while (clock64() - t0 < WAIT_CYCLES);
    *err = 1;
}

// a word's eight codes -> fp16 scale * code + bias, rounded once. A byte in both
// halves gives codes 2k and 2k + 1 as 1024 + c and 1024 + 16 c', exact, one
// HFMA2 makes them c and c', exact, and another the values.
__device__ __forceinline__ uint4 values_of(uint32_t w, __half2 s, __half2 z) {
    const __half2 mul = __halves2half2(__ushort_as_half(0x3C00), __ushort_as_half(0x2C00));    // 1, 1/16
    const __half2 sub = __halves2half2(__ushort_as_half(0xE400), __ushort_as_half(0xD400));    // -1024, -64
    uint32_t x[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const uint32_t b = and_or<0x00F0000Fu, 0x64006400u>(__byte_perm(w, 0, k * 0x0101));
        const __half2 v = __hfma2(__hfma2(*reinterpret_cast<const __half2*>(&b), mul, sub), s, z);
        x[k] = *reinterpret_cast<const uint32_t*>(&v);
    }
    return make_uint4(x[0], x[1], x[2], x[3]);
}
// 16 bytes to shared memory, or 16 zeros
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool live) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(live ? 16 : 0) : "memory");
}

// 64 dims of a head's 128 consecutive tokens, swizzled, to a panel
__device__ __forceinline__ void load_panel(uint32_t dst, const CUtensorMap& map, uint32_t dim, uint32_t head, uint32_t token, uint64_t* bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
                 "l"(&map), "r"(dim), "r"(head), "r"(token), "r"(mma4::s_addr(bar))
                 : "memory");
}

// sum_{i=1}^{n} ceil(i t / m) modulo 2^32, for n t < 2^32: lattice points under a line,
// counted by columns, then by rows, and so on, the slope being turned over each time as
// in Euclid's algorithm. With t < m (whole slopes are triangles, n (n + 1) / 2 points),
//   sum_{i=1}^{n} ceil(i t / m)  = n J - sum_{j=1}^{J-1} floor(j m / t),   J = ceil(n t / m):
//     row j < J has the i with i t > j m, which are n - floor(j m / t) many;
//   sum_{j=1}^{n} floor(j t / m) = (n + 1) K - sum_{k=1}^{K} ceil(k m / t),   K = floor(n t / m):
//     row k <= K has the j with j t >= k m, which are n + 1 - ceil(k m / t) many.
__device__ __forceinline__ uint32_t ceil_sum(uint32_t n, uint32_t t, uint32_t m) {
    uint32_t points = 0, sign = 1;
    for (bool up = true; n > 0; up = !up) {
        const uint32_t slope = t / m, rest = t - slope * m;
        points += sign * slope * (n & 1 ? (n + 1) / 2 * n : n / 2 * (n + 1));
        if (rest == 0) break;
        const uint32_t height = (n * rest + (up ? m - 1 : 0)) / m;
        points += sign * height * (up ? n : n + 1);
        n = up ? height - 1 : height;
        t = m;
        m = rest;
        sign = 0u - sign;
    }
    return points;
}

// A request's units and their key tiles. Unit i brings tokens [i tu, (i + 1)
// tu) and needs the cached tiles and the own tiles up to its last token. It counts
// MANY_UNIT tiles more, in front of its own, for what it costs besides them (queries,
// the masked tile, its result), so that a share of many short units is no longer
// than one of a few long ones (a first chunk of 8192: 588 us, counted by tiles alone
// 739).
struct Shape {
    Request rq;
    uint32_t tu, units, past;          // tokens per unit, units per cache head, cached tiles
    __device__ __forceinline__ uint32_t tiles(uint32_t i) const { return past + (min((i + 1) * tu, rq.n) + KT - 1) / KT; }
    // what the units in front of unit i count
    __device__ __forceinline__ uint32_t in_front(uint32_t i) const {
        const uint32_t full = i < units ? i : units - 1;
        const uint32_t s = full * (past + MANY_UNIT) + ceil_sum(full, tu, KT);
        return i < units ? s : s + tiles(full) + MANY_UNIT;
    }
    // the unit in which position x of a cache head's list lies: the root of in_front's
    // mean (a parabola in i), put right by steps that double and then by bisection, so
    // that any first guess ends at the same unit. (By bisection alone, each step of it
    // a sum by Euclid's algorithm, a first chunk of 4096 took 197 us, so 186 to 194.)
    __device__ __forceinline__ uint32_t unit_at(uint32_t x) const {
        const float a = tu * (1.0f / (2 * KT)), b = past + MANY_UNIT + 0.5f + a, y = (float)x;
        const float root = 2.0f * y / (b + sqrtf(b * b + 4.0f * a * y));
        const uint32_t guess = min((uint32_t)root, units - 1);
        uint32_t lo = 0, hi = units, step = 1;
        if (in_front(guess) <= x) {
            for (lo = guess; lo + step < hi; step *= 2) {
                if (in_front(lo + step) > x) {
                    hi = lo + step;
                    break;
                }
                lo += step;
            }
        } else {
            for (hi = guess; hi > step; step *= 2) {
                if (in_front(hi - step) <= x) {
                    lo = hi - step;
                    break;
                }
                hi -= step;
            }
        }
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) >> 1;
            if (in_front(mid) <= x) lo = mid;
            else hi = mid;
        }
        return lo;
    }
};
__device__ __forceinline__ Shape shape_of(const Attend& a, uint32_t b, uint32_t least_new) {
    Shape s;
    s.rq = request_of(a, b);
    s.tu = 2 * (ROWS / a.r);
    s.past = (s.rq.ctx + KT - 1) / KT;
    s.units = s.rq.n >= least_new ? (s.rq.n + s.tu - 1) / s.tu : 0;
    return s;
}

// The part [lo, hi) (counted over the whole step) of a unit's tiles [u0, u1) in a
// CTA's share.
struct Part {
    Shape s;
    uint32_t b, hk, unit, u0, u1, lo, hi;
    uint32_t tok0, n_tok;              // the unit's tokens
    bool second;                       // its second M tile has any
    __device__ __forceinline__ void settle(uint32_t end) {
        u1 = u0 + s.tiles(unit);
        hi = min(end, u1);
        tok0 = unit * s.tu;
        n_tok = min(s.tu, s.rq.n - tok0);
        second = n_tok > s.tu / 2;
    }
    // the part behind this one; false if the share has none
    __device__ __forceinline__ bool next(const Attend& a, const uint32_t* before, uint32_t least_new, uint32_t end) {
        if (u1 + MANY_UNIT >= end) return false;
        if (++unit == s.units) {
            unit = 0;
            if (++hk == a.n_kv_heads) {
                hk = 0;
                do ++b;
                while (before[b + 1] == u1);       // requests without a unit
                s = shape_of(a, b, least_new);
            }
        }
        lo = u0 = u1 + MANY_UNIT;
        settle(end);
        return true;
    }
};
// The part in which the share begins: found once (the arithmetic of the search
// is worth several tiles), the others follow from it.
__device__ __forceinline__ Part first_part(const Attend& a, const uint32_t* before, uint32_t least_new, uint32_t at, uint32_t end) {
    Part p;
    p.b = row_of_tile(before, a.rows, at);
    p.s = shape_of(a, p.b, least_new);
    const uint32_t per_head = p.s.in_front(p.s.units);
    const uint32_t rem = at - before[p.b];
    p.hk = rem / per_head;
    const uint32_t x = rem - p.hk * per_head;
    p.unit = p.s.unit_at(x);
    p.u0 = before[p.b] + p.hk * per_head + p.s.in_front(p.unit) + MANY_UNIT;
    p.lo = max(at, p.u0);
    p.settle(end);
    return p;
}

template <int DH, int GROUP>
__global__ void __launch_bounds__(THREADS, 1)
many_kernel(Attend a, uint32_t least_new, bool vec, bool maps, unsigned char* __restrict__ ws,
            const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map) {
    using C = Cfg<DH>;
    constexpr int G = DH / GROUP, W = DH / 8;
    extern __shared__ unsigned char smem_raw[];
    unsigned char* smem = smem_raw + ((1024u - (mma4::s_addr(smem_raw) & 1023u)) & 1023u);
    uint64_t* bar = reinterpret_cast<uint64_t*>(smem + C::BAR);
    uint64_t *q_full = bar, *s_full = bar + 2, *p_full = bar + 6, *o_done = bar + 10;
    uint64_t *k_full = bar + 12, *k_empty = k_full + STAGES, *v_full = k_empty + STAGES, *v_empty = v_full + STAGES;
    uint64_t* drained = v_empty + STAGES;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(smem + C::MISC);
    volatile int* err = reinterpret_cast<volatile int*>(smem + C::MISC + 4);
    uint32_t* before = reinterpret_cast<uint32_t*>(smem + C::BEFORE);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, wg = warp >> 2;

    if (tid == 0) {
        for (int i = 0; i < 2; ++i) {
            mbar_init(&q_full[i], 4);
            mbar_init(&o_done[i], 1);
        }
        for (int i = 0; i < 4; ++i) {
            mbar_init(&s_full[i], 1);
            mbar_init(&p_full[i], 4);
        }
        for (int i = 0; i < STAGES; ++i) {
            mbar_init(&k_full[i], 4);
            mbar_init(&k_empty[i], 2);
            mbar_init(&v_full[i], 4);
            mbar_init(&v_empty[i], 2);
        }
        mbar_init(&drained[0], 1);
        mbar_init(&drained[1], 1);
        *err = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        reinterpret_cast<Split*>(ws)[blockIdx.x].parts = 0;
    }
    const uint32_t total = sum_tiles<THREADS>(before, a.rows, [&](uint32_t b) {
        const Shape s = shape_of(a, b, least_new);
        return s.units ? (uint64_t)s.in_front(s.units) * a.n_kv_heads : 0ull;
    });
    const uint32_t share = (total + gridDim.x - 1) / gridDim.x;
    const uint64_t start64 = (uint64_t)blockIdx.x * share;
    if (start64 >= total) return;
    const uint32_t start = (uint32_t)start64, end = min(total, start + share);

    Part p = first_part(a, before, least_new, start, end);
    if (p.lo >= end) return;                       // none of its tiles
    if (warp == 12) {
        tmem_alloc(tmem_slot, 512);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;

    if (wg < 2) {
        // ---------------------------- softmax ------------------------------------
        const int mt = wg, row = tid & 127;
        const uint32_t tokm = ROWS / a.r;
        // x / R by a multiplication: exact for x < 128, R <= 128 (the excess stays below
        // 128 / 65536 < 1 / R)
        const uint32_t inv_r = (65536u + a.r - 1) / a.r;
        const auto token_of = [&](uint32_t x) { return x * inv_r >> 16; };
        const uint32_t rt = token_of(row);                           // the row's token of the M tile
        const uint32_t lanes = (uint32_t)(warp & 3) << 21;           // TMEM lane 32 (warp % 4), bits 16 up
        const uint32_t s_at = tmem + lanes + C::S0 + 128 * mt, o_at = tmem + lanes + C::O0 + 128 * mt;
        const float scale2 = a.scale * 1.4426950408889634f;
        // rows go in and out in whole lines: W lanes a row, RPW of the warp's 32 rows at once
        constexpr int RPW = 32 / W;
        const uint32_t r0 = (warp & 3) * 32 + lane / W, c0 = lane % W;
        uint32_t done = 0;                                           // steps
        do {
            if (mt == 1 && !p.second) continue;
            const uint32_t tok = p.tok0 + mt * tokm + rt;           // of the request
            const bool live = rt < tokm && tok < p.s.rq.n;
            // this M tile's queries (the last MMA that read the buffer is done: its
            // scores have been read)
            unsigned char* q_tile = smem + C::Q + mt * C::TILE;
            __syncwarp();
#pragma unroll 4
            for (int i = 0; i < 32 / RPW; ++i) {
                const uint32_t r = r0 + RPW * i, t = token_of(r), h = r - t * a.r, of = p.tok0 + mt * tokm + t;
                const bool has = t < tokm && of < p.s.rq.n;
                const __half* from = static_cast<const __half*>(a.q) +
                                     (has ? (p.s.rq.token0 + of) * a.q_token + (p.hk * a.r + h) * a.q_head + 8 * c0 : 0);
                unsigned char* to = q_tile + (c0 >> 3) * C::PANEL + swizzled(r, c0 & 7);
                if (vec) {
                    copy16(mma4::s_addr(to), from, has);
                } else {
                    __half x[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) x[e] = has ? from[e] : __ushort_as_half(0);
                    *reinterpret_cast<uint4*>(to) = *reinterpret_cast<const uint4*>(x);
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(&q_full[mt]);
            float ref = -INFINITY, l = 0.0f;
            const uint32_t steps = (p.hi - p.lo) * (KT / KS);
            for (uint32_t q = 0; q < steps; ++q, ++done) {
                const uint32_t buf = done & 1, s_buf = s_at + KS * buf;
                wait(&s_full[2 * mt + buf], (done >> 1) & 1, err);
                __syncwarp();
                tc_fence_after();
                // visible keys of the step: the cached ones up to the length, of the step's
                // own those up to the row's token
                const uint32_t tile = p.lo - p.u0 + q / 2, key = (tile < p.s.past ? tile : tile - p.s.past) * KT + (q & 1) * KS;
                const int lim = tile < p.s.past ? (int)p.s.rq.ctx - (int)key : (int)tok - (int)key + 1;
                const bool masked = __any_sync(0xffffffffu, lim < KS);
                uint32_t s[KS];
                float top;
                float2 sum[2];
                // The weights relative to the reference there is, and the maximum beside them
                // (in front of them it was 500 of 2,300 cycles of a step). Where it turns out
                // too far above the reference, which is rare, the step is done once more.
                for (;;) {
                    ld32(s_buf, s);
                    ld32(s_buf + 32, s + 32);
                    tmem_wait_ld();
                    if (masked) {
#pragma unroll
                        for (int c = 0; c < KS; ++c)
                            if (c >= lim) s[c] = 0xff800000u;
                    }
                    float tops[2] = {-INFINITY, -INFINITY};
                    sum[0] = sum[1] = make_float2(0.0f, 0.0f);
                    const float sub = ref == -INFINITY ? 0.0f : ref;
                    const float2 mul2 = make_float2(scale2, scale2), sub2 = make_float2(-sub, -sub);
#pragma unroll
                    for (int c = 0; c < KS; c += 2) {
                        tops[c / 2 % 2] = max_nan(tops[c / 2 % 2], __uint_as_float(s[c]), __uint_as_float(s[c + 1]));
                        float2 x = __ffma2_rn(make_float2(__uint_as_float(s[c]), __uint_as_float(s[c + 1])), mul2, sub2);
                        x.x = ex2(x.x);
                        x.y = ex2(x.y);
                        sum[(c >> 1) & 1] = __fadd2_rn(sum[(c >> 1) & 1], x);
                        const __half2 h = __floats2half2_rn(x.x, x.y);
                        s[c >> 1] = *reinterpret_cast<const uint32_t*>(&h);
                    }
                    top = max_nan(tops[0], tops[1], tops[1]) * scale2;
                    const bool over = top - ref > RAISE;
                    if (!__any_sync(0xffffffffu, over)) break;
                    const float to = over ? top - START : ref;
                    // a row that has seen nothing yet has nothing to rescale
                    const float f = ref == -INFINITY ? 0.0f : ex2(ref - to);
                    ref = to;
                    l *= f;
                    if (q > 0) {
                        // the combine in front is done: the next scores are issued behind it
                        if (q + 1 < steps) wait(&s_full[2 * mt + (buf ^ 1)], ((done + 1) >> 1) & 1, err);
                        else wait(&o_done[mt], 0, err);
                        __syncwarp();
                        tc_fence_after();
#pragma unroll
                        for (int c = 0; c < DH; c += 16) {
                            uint32_t o[16];
                            umma::tmem_ld16(o_at + c, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                            umma::tmem_st16(o_at + c, o);
                        }
                    }
                }
                if (!(top < INFINITY)) l = NAN;        // a NaN or an infinity among the scores it sees: the row is NaN
                st32(s_buf, s);
                l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
                tmem_wait_st();
                tc_fence_before();
                // the part's two phases of o_done are waited for in turn: a parity tells only
                // neighbouring ones apart
                if (q + 1 == steps) wait(&o_done[mt], 0, err);
                __syncwarp();
                if (lane == 0) mbar_arrive(&p_full[2 * mt + buf]);
            }
            // ---- the part's result ------------------------------------------------
            wait(&o_done[mt], 1, err);
            __syncwarp();
            tc_fence_after();
            const bool whole = p.u0 >= start && p.u1 <= end;
            const uint32_t col = mt * tokm * a.r + row;                 // row of the unit
            float* slot = reinterpret_cast<float*>(ws + split_bytes(gridDim.x)) +
                          (2 * (size_t)blockIdx.x + (p.u0 >= start ? 1 : 0)) * slot_floats(COLS, DH);
            const float inv = *err ? NAN : (whole ? 1.0f / l : 1.0f);
            // through this M tile's query buffer, whose MMAs are done, as rows of 2 DH bytes:
            // the fp16 result, or the two halves of an fp32 part one after the other. Each
            // warp uses the rows that it loads queries into: others may be at the next part.
#pragma unroll 1
            for (int half = 0; half < (whole ? 1 : 2); ++half) {
                __syncwarp();
#pragma unroll
                for (int c = 0; c < DH; c += 32) {
                    if (!whole && c / (DH / 2) != half) continue;
                    uint32_t o[32];
                    ld32(o_at + c, o);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * inv);
                    if (whole) {
#pragma unroll
                        for (int i = 0; i < 32; i += 2) {
                            const __half2 h = __floats2half2_rn(__uint_as_float(o[i]), __uint_as_float(o[i + 1]));
                            o[i / 2] = *reinterpret_cast<const uint32_t*>(&h);
                        }
                    }
                    const int first = whole ? c / 8 : (c % (DH / 2)) / 4;        // 16-byte chunk of the row
#pragma unroll
                    for (int i = 0; i < 8; ++i)
                        if (!whole || i < 4)
                            *reinterpret_cast<uint4*>(q_tile + ((first + i) >> 3) * C::PANEL + swizzled(row, (first + i) & 7)) =
                                make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                }
                __syncwarp();
#pragma unroll 4
                for (int i = 0; i < 32 / RPW; ++i) {
                    const uint32_t r = r0 + RPW * i, t = token_of(r), h = r - t * a.r, of = p.tok0 + mt * tokm + t;
                    if (t >= tokm || of >= p.s.rq.n) continue;
                    const uint4 x = *reinterpret_cast<const uint4*>(q_tile + (c0 >> 3) * C::PANEL + swizzled(r, c0 & 7));
                    if (whole)
                        *reinterpret_cast<uint4*>(static_cast<__half*>(a.out) +
                                                  ((size_t)(p.s.rq.token0 + of) * a.n_heads + p.hk * a.r + h) * DH + 8 * c0) = x;
                    else
                        *reinterpret_cast<uint4*>(slot + 2 * COLS + (size_t)(mt * tokm * a.r + r) * DH + half * (DH / 2) + 4 * c0) = x;
                }
            }
            if (!whole && live) {
                slot[col] = ref;
                slot[COLS + col] = l;
            }
            if (tid == 0 && p.u0 >= start && p.u1 > end)
                reinterpret_cast<Split*>(ws)[blockIdx.x] = {(p.u1 - 1) / share - blockIdx.x + 1, p.s.rq.token0, p.hk,
                                                            p.tok0 * a.r, p.n_tok * a.r};
            tc_fence_before();
        } while (p.next(a, before, least_new, end));
    } else if (wg == 2) {
        // ------------------------------ loads -------------------------------------
        const uint32_t row = tid & 127;
        const auto filled = [&](uint64_t* bar) {
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(bar);
        };
        // a whole tile of own entries by one thread's tensor copies, which the phase waits for
        const auto fetch = [&](uint64_t* bar, const CUtensorMap& map, uint32_t to, uint32_t head, uint32_t token) {
            if (warp == 8 && lane == 0) {
                mma4::mbar_expect_tx(bar, C::TILE);
#pragma unroll
                for (int i = 0; i < C::PANELS; ++i) load_panel(to + i * C::PANEL, map, 64 * i, head, token, bar);
            } else if (lane == 0) {
                mbar_arrive(bar);
            }
        };
        uint32_t done = 0;
        do {
            // ---- cached tiles: this thread's key of each -----------------------------
            const uint32_t t0 = p.lo - p.u0, tn = min(p.hi - p.u0, p.s.past);      // tiles [t0, tn)
            const int32_t* table = a.block_tables + (size_t)p.b * a.width;
            const auto page_of = [&](uint32_t tile) {                      // 0 past the length: not used
                const uint32_t pos = tile * KT + row;
                return tile < tn && pos < p.s.rq.ctx ? (uint32_t)table[pos >> a.page_shift] : 0u;
            };
            // a key's packed row, and whether there is one (0 none, 1 a row, 2 a page id
            // outside the pool)
            uint4 kw[W / 4], vw[W / 4];
            __half ks[G], kz[G], vs[G], vz[G];
            const auto row_of = [&](uint32_t tile, uint32_t page, uint32_t& kind) {
                const uint32_t pos = tile * KT + row;
                kind = tile < tn && pos < p.s.rq.ctx ? (page < a.pages ? 1 : 2) : 0;
                return (((kind == 1 ? page : 0u) * a.n_kv_heads + p.hk) << a.page_shift) + (pos & ((1u << a.page_shift) - 1));
            };
            const auto read = [&](uint32_t kind, uint64_t r, const Pool& pool, uint4 (&w)[W / 4], __half (&s)[G], __half (&z)[G]) {
                // keys past the length: zeros, which the mask (K) and the zero weights (V)
                // leave without effect
#pragma unroll
                for (int i = 0; i < W / 4; ++i) w[i] = kind ? reinterpret_cast<const uint4*>(pool.words + r * W)[i] : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
                for (int i = 0; i < G; ++i) {
                    s[i] = kind ? static_cast<const __half*>(pool.scales)[r * G + i] : __ushort_as_half(0);
                    z[i] = kind ? static_cast<const __half*>(pool.biases)[r * G + i] : __ushort_as_half(0);
                }
            };
            const auto put = [&](unsigned char* d, const uint4 (&w)[W / 4], const __half (&s)[G], const __half (&z)[G]) {
#pragma unroll
                for (int c = 0; c < W; ++c) {
                    const uint32_t word = c % 4 == 0 ? w[c / 4].x : c % 4 == 1 ? w[c / 4].y : c % 4 == 2 ? w[c / 4].z : w[c / 4].w;
                    *reinterpret_cast<uint4*>(d + (c >> 3) * C::PANEL + swizzled(row, c & 7)) =
                        values_of(word, __half2half2(s[c * 8 / GROUP]), __half2half2(z[c * 8 / GROUP]));
                }
            };
            uint32_t kind, page = page_of(t0);
            uint32_t r = row_of(t0, page, kind);
            page = page_of(t0 + 1);
            read(kind, r, a.k, kw, ks, kz);
            read(kind, r, a.v, vw, vs, vz);
            for (uint32_t tile = t0; tile < tn; ++tile, ++done) {
                const uint32_t st = done % STAGES, use = done / STAGES;
                if (kind == 2) {
#pragma unroll
                    for (int i = 0; i < G; ++i) kz[i] = __ushort_as_half(0x7FFF);
                }
                if (use) wait<true>(&k_empty[st], (use - 1) & 1, err);
                put(smem + C::K + st * C::TILE, kw, ks, kz);
                filled(&k_full[st]);
                r = row_of(tile + 1, page, kind);
                read(kind, r, a.k, kw, ks, kz);
                page = page_of(tile + 2);
                if (use) wait<true>(&v_empty[st], (use - 1) & 1, err);
                put(smem + C::V + st * C::TILE, vw, vs, vz);
                filled(&v_full[st]);
                read(kind, r, a.v, vw, vs, vz);
            }
            // ---- own entries: W lanes copy a row, a warp RPW rows at a time ---------------
            // (A thread per row left each load of a warp in 32 lines: 18,000 cycles a tile. All
            // tiles so: 5,000 cycles a tile for the copies alone, 886 us for a first chunk of 8192
            // where the tensor copies take 739.)
            constexpr int RPW = 32 / W, STEPS = KT / (4 * RPW);
            const uint32_t c = lane % W, r0 = (warp & 3) * RPW + lane / W;
            const auto copy_rows = [&](const void* base, uint64_t token, uint64_t head, uint32_t key0, unsigned char* tile_at) {
                const __half* src = static_cast<const __half*>(base) + (p.s.rq.token0 + key0 + r0) * token + p.hk * head + 8 * c;
                const uint32_t d = mma4::s_addr(tile_at) + (c >> 3) * C::PANEL;
#pragma unroll 4
                for (int i = 0; i < STEPS; ++i) {
                    const uint32_t rr = r0 + 4 * RPW * i;
                    const bool live = key0 + rr < p.s.rq.n;
                    const __half* from = live ? src + (uint64_t)(4 * RPW * i) * token : static_cast<const __half*>(base);
                    if (vec) {
                        copy16(d + swizzled(rr, c & 7), from, live);
                    } else {
                        __half h[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) h[e] = live ? from[e] : __ushort_as_half(0);
                        *reinterpret_cast<uint4*>(tile_at + (c >> 3) * C::PANEL + swizzled(rr, c & 7)) = *reinterpret_cast<const uint4*>(h);
                    }
                }
            };
            for (uint32_t tile = max(t0, p.s.past); tile < p.hi - p.u0; ++tile, ++done) {
                const uint32_t st = done % STAGES, use = done / STAGES, key0 = (tile - p.s.past) * KT;
                unsigned char* kd = smem + C::K + st * C::TILE;
                unsigned char* vd = smem + C::V + st * C::TILE;
                const bool all_see = key0 + KT - 1 <= p.tok0;   // every row sees every key
                if (use) wait<true>(&k_empty[st], (use - 1) & 1, err);
                __syncwarp();
                if (maps && all_see) {
                    fetch(&k_full[st], k_map, mma4::s_addr(kd), p.hk, p.s.rq.token0 + key0);
                    if (use) wait<true>(&v_empty[st], (use - 1) & 1, err);
                    __syncwarp();
                    fetch(&v_full[st], v_map, mma4::s_addr(vd), p.hk, p.s.rq.token0 + key0);
                    __syncwarp();
                    continue;
                }
                copy_rows(a.new_k, a.k_token, a.k_head, key0, kd);
                // A weight of zero does not keep an infinite or NaN value out of the rows that
                // are masked from it. Such a value row is taken as zeros, and its key as NaN,
                // which reaches the rows that see it and no other.
                if (use) wait<true>(&v_empty[st], (use - 1) & 1, err);
                copy_rows(a.new_v, a.v_token, a.v_head, key0, vd);
                asm volatile("cp.async.wait_all;" ::: "memory");
                __syncwarp();
#pragma unroll 4
                for (int i = 0; i < STEPS; ++i) {
                    const uint32_t off = (c >> 3) * C::PANEL + swizzled(r0 + 4 * RPW * i, c & 7);
                    const uint4 x = *reinterpret_cast<const uint4*>(vd + off);
                    const __half2* h = reinterpret_cast<const __half2*>(&x);
                    const __half2 top = __hmax2_nan(__hmax2_nan(__habs2(h[0]), __habs2(h[1])), __hmax2_nan(__habs2(h[2]), __habs2(h[3])));
                    const bool here = !(__low2float(top) <= 65504.0f && __high2float(top) <= 65504.0f);
                    const uint32_t who = __ballot_sync(0xffffffffu, here) >> (lane / W * W);
                    if (who & (uint32_t)((1ull << W) - 1)) {
                        *reinterpret_cast<uint4*>(vd + off) = make_uint4(0u, 0u, 0u, 0u);
                        *reinterpret_cast<uint4*>(kd + off) = make_uint4(0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu, 0x7FFF7FFFu);
                    }
                }
                filled(&k_full[st]);
                filled(&v_full[st]);
            }
        } while (p.next(a, before, least_new, end));
        // no copy of this CTA's is on its way when it leaves, whatever the waits did
        if (maps && warp == 8)
            for (uint32_t t = done > STAGES ? done - STAGES : 0; t < done; ++t) {
                const long long t0 = clock64();
                while ((!mbar_try_wait(&k_full[t % STAGES], (t / STAGES) & 1) || !mbar_try_wait(&v_full[t % STAGES], (t / STAGES) & 1)) &&
                       clock64() - t0 < WAIT_CYCLES) {}
            }
    } else {
        // --------------------------- the MMAs -----------------------------------------
        if (warp < 14) {
            // The whole warp walks the steps and one elected lane issues, so that the
            // operands' descriptors stay in uniform registers: under a condition on the
            // lane number each MMA took 190 cycles to issue against the 64 it runs.
            constexpr uint32_t ID_S = idesc(false, false, false, KS, ROWS);
            constexpr uint32_t ID_O = idesc(false, false, true, DH, ROWS);
            const int mt = warp - 12;
            const uint32_t base = mma4::s_addr(smem), q_at = base + C::Q + mt * C::TILE;
            const uint32_t s_at = tmem + C::S0 + 128 * mt, o_at = tmem + C::O0 + 128 * mt;
            uint32_t tiles = 0, parts = 0, steps = 0;              // done in front of this part
            do {
                const uint32_t n = (p.hi - p.lo) * (KT / KS), tile0 = tiles;
                tiles += p.hi - p.lo;
                if (mt == 1 && !p.second) {
                    // nothing to do in this part but to follow its tiles: a parity tells only
                    // neighbouring phases apart, and a tile is free once both warps say so
                    for (uint32_t kt = tile0; kt < tiles; ++kt) {
                        wait(&k_full[kt % STAGES], (kt / STAGES) & 1, err);
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&k_empty[kt % STAGES]);
                        wait(&v_full[kt % STAGES], (kt / STAGES) & 1, err);
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&v_empty[kt % STAGES]);
                    }
                    continue;
                }
                wait(&q_full[mt], parts & 1, err);
                ++parts;
                // scores of step q, two steps ahead of the combine of step q - 2 whose buffer
                // they take
                for (uint32_t q = 0; q < n + 2; ++q) {
                    const uint32_t kt = tile0 + q / 2, vt = kt - 1, half = q & 1, g = steps + q, buf = g & 1;
                    const uint32_t s_buf = s_at + KS * buf;
                    if (q < n && half == 0) wait(&k_full[kt % STAGES], (kt / STAGES) & 1, err);
                    if (q >= 2) {
                        if (half == 0) wait(&v_full[vt % STAGES], (vt / STAGES) & 1, err);
                        wait(&p_full[2 * mt + buf], ((g - 2) >> 1) & 1, err);
                    }
                    __syncwarp();
                    tc_fence_after();
                    if (elect_one()) {
                        if (q >= 2) {
                            const uint64_t v = desc128(base + C::V + (vt % STAGES) * C::TILE + half * (KS * 128), C::PANEL);
#pragma unroll
                            for (int k = 0; k < KS / 16; ++k) umma_ts(o_at, s_buf + 8 * k, v + k * (2048 >> 4), ID_O, q > 2 || k > 0);
                            if (q >= n) umma_commit(&o_done[mt]);          // the part's last two
                            if (half) umma_commit(&v_empty[vt % STAGES]);
                        }
                        if (q < n) {
                            const uint64_t qd = desc128(q_at, 16), kd = desc128(base + C::K + (kt % STAGES) * C::TILE + half * (KS * 128), 16);
#pragma unroll
                            for (int k = 0; k < DH / 16; ++k) {
                                const uint32_t off = ((k >> 2) * C::PANEL + (k & 3) * 32) >> 4;
                                umma(s_buf, qd + off, kd + off, ID_S, k > 0);
                            }
                            umma_commit(&s_full[2 * mt + buf]);
                            if (half) umma_commit(&k_empty[kt % STAGES]);
                        }
                    }
                    __syncwarp();
                }
                steps += n;
            } while (p.next(a, before, least_new, end));
            // nothing of this CTA's is in flight when its tensor memory goes
            if (elect_one()) umma_commit(&drained[mt]);
            for (const long long t0 = clock64(); !mbar_try_wait(&drained[mt], 0) && clock64() - t0 < WAIT_CYCLES;) {}
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 12) tmem_dealloc(tmem, 512);
    pdl_launch_dependents();
}

// x [tokens, heads, DH] with its strides as boxes of 64 dims x 1 head x 128 tokens
template <int DH>
bool map_of(const Attend& a, const void* x, uint64_t token, uint64_t head, CUtensorMap* map) {
    using Encode = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
    static const Encode encode = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult found;
        const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found);
        return e == cudaSuccess && found == cudaDriverEntryPointSuccess ? reinterpret_cast<Encode>(f) : nullptr;
    }();
    if (encode == nullptr) return false;
    const cuuint64_t dims[3] = {DH, a.n_kv_heads, a.tokens}, strides[2] = {2 * head, 2 * token};
    const cuuint32_t box[3] = {64, 1, KT}, steps[3] = {1, 1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<void*>(x), dims, strides, box, steps,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int DH, int GROUP>
cudaError_t launch_many(const Attend& a, uint32_t least_new, bool vec, uint32_t grid, void* ws, cudaStream_t stream) {
    using C = Cfg<DH>;
    auto kernel = many_kernel<DH, GROUP>;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_smem(kernel, 1024 + C::BEFORE + (MAX_ROWS + 1) * 4, done);
    if (e != cudaSuccess) return e;
    const size_t smem = 1024 + C::BEFORE + ((size_t)a.rows + 1) * 4;
    // whole tiles of own entries come by tensor copies, where their strides allow
    // (multiples of 16 bytes, and not 0)
    alignas(64) CUtensorMap k_map{}, v_map{};
    const bool maps = vec && a.k_token && a.k_head && a.v_token && a.v_head && map_of<DH>(a, a.new_k, a.k_token, a.k_head, &k_map) &&
                      map_of<DH>(a, a.new_v, a.v_token, a.v_head, &v_map);
    kernel<<<grid, THREADS, smem, stream>>>(a, least_new, vec, maps, static_cast<unsigned char*>(ws), k_map, v_map);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    return launch_join<__half, DH, COLS>(a, grid, static_cast<const unsigned char*>(ws), stream);
}

}  // namespace many
}  // namespace paged
}  // namespace kvq
