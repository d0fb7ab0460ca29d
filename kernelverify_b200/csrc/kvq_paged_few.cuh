// Paged attention for requests with few new tokens (a decode step, verified
// drafts): the cache is read once for up to 8 NT query columns, a column being
// one (token, query head) of a request, so the step is bound by the cache's
// bytes.
//
// A warp takes 32 cached positions at a time, as two blocks of 16: it streams
// them with 16-byte cp.async into its own ring (a page holds whole blocks; no
// warp waits for another), and keeps its own online softmax. The CTA's share is
// divided once more, into one run of tiles per warp: a unit inside one run is
// finished by its warp, and the parts of the others are joined when the CTA's
// warps are all done. With codes c, scales s, z = bias:
//
//   scores   S^T[pos, col] = sum_g ks[pos,g] (sum_{d in g} c[pos,d] q[col,d])
//                            + kz[pos,g] (sum_{d in g} q[col,d])
//   combine  O^T[d, col]   = sum_pos c[pos,d] (p[pos,col] vs[pos,g(d)])
//                            + sum_pos p[pos,col] vz[pos,g(d)]
//
// both as m16n8k16 fp16 MMAs with the codes as the A operand. For fp16 steps
// codes are never converted: the bits of c are the fp16 subnormal c * 2^-24
// (or, four bits higher, c * 2^-20), which the tensor cores multiply exactly,
// so a word of eight codes costs one shift and four ANDs; the integer pipe is
// what this kernel is short of next to memory. The factor 16 between the two
// is in the query fragments, and in the combine, where odd codes are rows of
// their own, in the result. ldmatrix.trans brings the V codes of two positions
// into one register. The tensor cores align a subnormal's products by its
// nominal exponent and so keep about 16 bits of their sums (measured 6e-6
// relative); fp32 steps convert their codes to c - 8. Which head dims (scores) and which positions (combine)
// a lane holds is free as long as both operands agree, and is chosen so that
// the packed words are used where they are loaded. The weights p vs reach the
// combine's B layout by one movmatrix per 8 x 8 block.
//
// Up to four columns (PAIR) leave half of an MMA's eight columns empty, and
// with them half of every lane's softmax. They are then held twice: columns 0
// to 3 stand for the tile's first block, 4 to 7 for its second. Scores are
// taken from the MMAs of the one block or the other, everything from there to
// the weights is done once for both, and the combine's MMAs of a block get the
// other half's weights as zeros. The two halves are two online softmaxes, joined
// at the end.
//
// Precision: products exact, sums fp32. Weights p vs of requests with up to SHORT
// cached positions go to the MMAs as two fp16 parts (2^-22 relative), those of longer
// ones as their fp16 rounding (2^-11 at most), and what that leaves times 7.5, the middle
// of the codes, joins the bias term: a weight's error meets c - 7.5 where it would meet
// c. (Root mean square error of an output against 64 bits, over that of its own
// rounding, 2.1e-4 of its magnitude; one part: 1.43 at 4 cached positions, 1.24 at 32, 1.07
// at 128, 1.04 at 256, 1.01 at 1024, 1.004 at 8192: fewer positions average less, as do
// more of them where the softmax rests on few; two parts: 1.000. They cost 12.5 us for
// 12.4 at 32 x 128, 37.4 for 36.2 at 256 x 256, and 70.7 for 66 at 32 x 8192.) fp32 steps carry
// three parts. Weights are held near the top of fp16's range: p is relative to a
// reference that the running maximum may pass by 2^14 before it moves (so
// accumulators are rarely rescaled), and vs is divided by a power of two above the
// largest |vs| met so far. Queries
// are scaled by a power of two per column (fp32 ones are three fp16 parts of
// that, and their MMAs start from zero and are added in fp32, since a long
// chain of additions in the tensor cores truncates).
//
// 32 requests of 8192 positions, 32 heads over 8 of 128: 66 us, 303 MB, 0.70 of the
// measured copy bandwidth; one of 131072: 42 us, 151 MB, 0.55. Neither memory nor a
// pipe is full: the schedulers issue in half of the cycles, from three warps each
// (168 registers a thread), and wait for the results of MMAs and shuffles and for
// the integer pipe, which is busy half of the time. What does not shrink with the
// cache is about 11 us (1 x 512): two launches, the running sums, one chain of loads
// (length, page, rows), the join.
#pragma once

#include <atomic>

#include "kvq_mma.cuh"
#include "kvq_paged_work.cuh"

namespace kvq {
namespace paged {
namespace few {

using mma4::ex2;
using mma4::mma_f16;

constexpr int BLK = 16, SUBS = 2;          // positions per block, blocks per tile
constexpr int TP = BLK * SUBS;
constexpr float RAISE = 14.0f, START = 5.0f;   // log2 room above the reference
constexpr uint32_t SHORT = 256;            // cached positions up to which fp16 weights have two parts (see above)

// A part of a unit that is not a warp's alone; cols = 0: none.
struct Info {
    uint32_t u0, u1, token0, hk, col0, cols;
};

template <typename T, int DH_, int GROUP_, int NT_, bool PAIR_>
struct Cfg {
    static constexpr bool PAIR = PAIR_;
    static_assert(!PAIR_ || NT_ == 1, "paired columns are one tile");
    static constexpr int DH = DH_, GROUP = GROUP_, NT = NT_;
    static constexpr bool HALF = sizeof(T) == 2;
    static constexpr int G = DH / GROUP;
    static constexpr int W = DH / 8;                // words per row
    static constexpr int SETS = DH / 32;            // runs of four words, one per lane of a quad
    static constexpr int MT = DH / 16;              // combine's 16-dim tiles
    static constexpr int QP = HALF ? 1 : 3;         // fp16 parts of a query
    static constexpr int COLS = PAIR ? 4 : 8 * NT;
    static constexpr int NB = PAIR ? 1 : SUBS;      // blocks whose weights a lane holds
    // One CTA per SM, its warps as many as registers and shared memory allow. (Two
    // CTAs of eight warps leave twice the parts to join, and the CTA that is
    // launched later runs behind the other: 1 x 131072 took 60 us so.)
    static constexpr int CW = HALF && NT == 1 ? 12 : 8, THREADS = 32 * CW;
    static constexpr int WB = BLK * W * 4, SB = BLK * G * (int)sizeof(T);
    static constexpr int VW = WB, KS = 2 * WB, KZ = KS + SB, VS = KZ + SB, VZ = VS + SB;
    static constexpr int BLOCK = VZ + SB;           // bytes of 16 positions
    static constexpr int STAGE = SUBS * BLOCK;
    static constexpr int NST = 2;                   // tiles per ring
    static constexpr int PART = COLS * DH;          // floats of a part's O
    static constexpr int HEADS = CW * STAGE * NST;  // fp32 [CW][COLS][DH]; the other parts lie in their warp's ring
    static constexpr int ML = HEADS + CW * PART * 4;            // fp32 [2][CW][2][COLS]: m and l, head and tail
    static constexpr int INFO = ML + 2 * CW * 2 * COLS * 4;     // Info [2][CW]
    static constexpr int BEFORE = (INFO + 2 * CW * (int)sizeof(Info) + 15) / 16 * 16;   // uint32 [rows + 1]
    static_assert(PART * 4 <= STAGE * NST, "a part fits a ring");
    static_assert(BEFORE + (MAX_ROWS + 1) * 4 <= 232448, "shared memory");
    static_assert(STAGE % 16 == 0 && HEADS % 16 == 0, "alignment");
};

__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(x));
    return d;
}
__device__ __forceinline__ uint32_t pack(float lo, float hi) {
    const __half2 h = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ float2 unpack(uint32_t x) { return __half22float2(*reinterpret_cast<const __half2*>(&x)); }
// (x, y) as N fp16 parts, each the rounding of what the ones before leave
template <int N>
__device__ __forceinline__ void parts_of(float x, float y, uint32_t (&h)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        h[i] = pack(x, y);
        const float2 f = unpack(h[i]);
        x -= f.x;
        y -= f.y;
    }
}
// Codes j and j + 4 of a word (or code j of two positions) as fp16x2, times 16
// for odd j: fp16 steps take c as a subnormal, in units of 2^-24; fp32 steps
// take c - 8 (1024 + c and 1024 + 16 c are exact, and so is the difference),
// since sums over codes of one sign would be far larger than what the bias then
// leaves of them.
template <bool HALF>
__device__ __forceinline__ uint32_t nib(uint32_t w, int j) {
    const uint32_t v = j & 2 ? w >> 8 : w, mask = j & 1 ? 0x00F000F0u : 0x000F000Fu;
    if constexpr (HALF) return v & mask;
    const uint32_t x = (v & mask) | 0x64006400u;
    const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(j & 1 ? 0x6480 : 0x6408)));
    return *reinterpret_cast<const uint32_t*>(&h);
}
// 2^e for a normal exponent
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }
// the G values of a position
template <int G>
__device__ __forceinline__ void scales_of(const __half* p, float (&x)[G]) {
    if constexpr (G == 1) {
        x[0] = __half2float(*p);
    } else {
#pragma unroll
        for (int i = 0; i < G; i += 2) {
            const float2 f = __half22float2(reinterpret_cast<const __half2*>(p)[i / 2]);
            x[i] = f.x;
            x[i + 1] = f.y;
        }
    }
}
template <int G>
__device__ __forceinline__ void scales_of(const float* p, float (&x)[G]) {
#pragma unroll
    for (int i = 0; i < G; ++i) x[i] = p[i];
}
__device__ __forceinline__ void store4(__half* p, float4 x) {
    *reinterpret_cast<uint2*>(p) = make_uint2(pack(x.x, x.y), pack(x.z, x.w));
}
__device__ __forceinline__ void store4(float* p, float4 x) { *reinterpret_cast<float4*>(p) = x; }
__device__ __forceinline__ void copy16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
// four 8 x 8 b16 tiles, transposed: lanes 8 i .. 8 i + 7 give tile i's rows;
// lane (g, t) receives rows 2t (low half) and 2t + 1 of column g in x[i]
__device__ __forceinline__ void ldsm_trans(uint32_t saddr, uint32_t (&x)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3])
                 : "r"(saddr));
}

// c (+)= a * b; fp32 steps add in fp32 registers (see the head of this file)
template <bool HALF>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (HALF) {
        mma_f16(c, a[0], a[1], a[2], a[3], b0, b1);
    } else {
        float d[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        mma_f16(d, a[0], a[1], a[2], a[3], b0, b1);
#pragma unroll
        for (int i = 0; i < 4; ++i) c[i] += d[i];
    }
}

// 8 consecutive elements as floats
template <typename T>
__device__ __forceinline__ void read8(const T* p, float (&x)[8]) {
    if ((reinterpret_cast<uintptr_t>(p) & 15) == 0) {
        uint4 raw[sizeof(T) / 2];
#pragma unroll
        for (int i = 0; i < (int)sizeof(T) / 2; ++i) raw[i] = reinterpret_cast<const uint4*>(p)[i];
        const T* v = reinterpret_cast<const T*>(raw);
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f32(v[i]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = to_f32(p[i]);
    }
}

template <typename T, int DH, int GROUP, int NT, bool PAIR>
__global__ void __launch_bounds__(Cfg<T, DH, GROUP, NT, PAIR>::THREADS, 1)
few_kernel(Attend a, uint32_t most_new, unsigned char* __restrict__ ws) {
    using C = Cfg<T, DH, GROUP, NT, PAIR>;
    constexpr int NB = C::NB;
    constexpr int G = C::G, COLS = C::COLS, QP = C::QP, CW = C::CW, THREADS = C::THREADS;
    constexpr bool HALF = C::HALF;
    constexpr float UNIT = HALF ? 16777216.0f : 1.0f;      // a code in an MMA is c / UNIT, or 16 c / UNIT
    // exponents of the power of two above |vs|: from below what the quantizer
    // stores (its smallest step is 1e-7) to fp16's largest; fp32 values are below 2^60
    // (own entries come in at the lowest one: 16 v 2^30 times weights of up to 2^14)
    constexpr int VEXP0 = HALF ? -14 : -30, VEXP1 = HALF ? 16 : 90;
    // the join's CTAs may come as soon as there is room: none before these CTAs,
    // which hold a whole SM's registers each, have left
    pdl_launch_dependents();
    extern __shared__ __align__(128) unsigned char smem[];
    uint32_t* before = reinterpret_cast<uint32_t*>(smem + C::BEFORE);
    Info* info = reinterpret_cast<Info*>(smem + C::INFO);
    const auto part_o = [&](int kind, int w) {      // kind 0: head (its unit began before the warp's run), 1: tail
        return reinterpret_cast<float*>(kind ? smem + w * C::STAGE * C::NST : smem + C::HEADS + w * C::PART * 4);
    };
    const auto part_ml = [&](int kind, int w) { return reinterpret_cast<float*>(smem + C::ML) + (kind * CW + w) * 2 * COLS; };
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    unsigned char* ring = smem + warp * C::STAGE * C::NST;
    if (tid == 0) reinterpret_cast<Split*>(ws)[blockIdx.x].parts = 0;
    const uint32_t H = a.n_kv_heads;
    const auto tiles_in = [](uint32_t ctx) { return max(1u, (ctx + TP - 1) / TP); };
    const auto col_tiles = [&](const Request& r) { return r.n > most_new ? 0u : (r.n * a.r + COLS - 1) / COLS; };
    const uint32_t total = sum_tiles<THREADS>(before, a.rows, [&](uint32_t b) {
        const Request r = request_of(a, b);
        return (uint64_t)col_tiles(r) * H * tiles_in(r.ctx);
    });
    const uint32_t run = (total + gridDim.x * CW - 1) / (gridDim.x * CW), share = run * CW;   // tiles per warp and CTA
    const uint64_t start64 = (uint64_t)blockIdx.x * share;
    if (start64 >= total) return;
    const uint32_t start = (uint32_t)start64, end = min(total, start + share);
    const uint32_t wstart = min(end, start + warp * run), wend = min(end, wstart + run), own = wend - wstart;
    if (lane < 2) info[lane * CW + warp].cols = 0;

    // ---- the warp's stream of tiles -----------------------------------------
    // lane i looks up the batch's i-th tile: the cache row of each block, and per
    // block whether it holds positions (bit) and its page id is in the pool (bad)
    uint32_t row_at[SUBS] = {0, 0}, held = 0, bad_id = 0;
    uint32_t bad = 0;                                  // stages with such a page
    const auto look = [&](uint32_t k0) {
        held = bad_id = 0;
        if (k0 + lane >= own) return;
        const uint32_t x = wstart + k0 + lane;
        const uint32_t b = row_of_tile(before, a.rows, x);
        const Request r = request_of(a, b);
        const uint32_t tiles = tiles_in(r.ctx), rem = x - before[b], unit = rem / tiles, hk = unit / col_tiles(r);
#pragma unroll
        for (int i = 0; i < SUBS; ++i) {
            const uint32_t pos = (rem - unit * tiles) * TP + i * BLK;
            if (pos >= r.ctx) break;
            uint32_t page = (uint32_t)a.block_tables[(size_t)b * a.width + (pos >> a.page_shift)];
            held |= 1u << i;
            if (page >= a.pages) {
                bad_id = 1;
                page = 0;
            }
            row_at[i] = ((page * H + hk) << a.page_shift) + (pos & ((1u << a.page_shift) - 1));
        }
    };
    // Every lane copies 16 bytes of each run. (A bulk copy per run takes its
    // operands from uniform registers, so six lanes that issue one each are walked
    // one after the other: 120 of 400 instructions per block.)
    constexpr int WCH = C::WB / 16, SCH = C::SB / 16, ALL = 4 * SCH;   // chunks of a run, of the four scale runs
    const unsigned char* kw0 = reinterpret_cast<const unsigned char*>(a.k.words) + lane * 16;
    const unsigned char* vw0 = reinterpret_cast<const unsigned char*>(a.v.words) + lane * 16;
    const unsigned char* sc0[(ALL + 31) / 32];
#pragma unroll
    for (int i = 0; i < (ALL + 31) / 32; ++i) {
        const int chunk = lane + 32 * i, run = chunk / SCH;
        const void* p = run == 0 ? a.k.scales : run == 1 ? a.k.biases : run == 2 ? a.v.scales : a.v.biases;
        sc0[i] = static_cast<const unsigned char*>(p) + (chunk % SCH) * 16;
    }
    const uint32_t ring_at = mma4::s_addr(ring) + lane * 16;
    const auto fill_tile = [&](uint32_t k) {
        if (k >= own) return;
        if ((k & 31) == 0) look(k);
        const uint32_t r0 = __shfl_sync(0xffffffffu, row_at[0], k & 31), r1 = __shfl_sync(0xffffffffu, row_at[1], k & 31);
        const uint32_t what = __shfl_sync(0xffffffffu, held | bad_id << SUBS, k & 31);
        const uint32_t s = k % C::NST;
        bad = what >> SUBS ? bad | (1u << s) : bad & ~(1u << s);
#pragma unroll
        for (int b = 0; b < SUBS; ++b) {
            if (!(what >> b & 1)) break;
            const uint64_t row = b ? r1 : r0;
            const uint32_t to = ring_at + s * C::STAGE + b * C::BLOCK;
#pragma unroll
            for (int i = 0; i < (WCH + 31) / 32; ++i)
                if (WCH >= 32 || lane < WCH) {
                    copy16(to + 512 * i, kw0 + row * (C::W * 4) + 512 * i);
                    copy16(to + C::VW + 512 * i, vw0 + row * (C::W * 4) + 512 * i);
                }
#pragma unroll
            for (int i = 0; i < (ALL + 31) / 32; ++i)
                if (lane + 32 * i < ALL) copy16(to + C::KS + 512 * i, sc0[i] + row * (G * sizeof(T)));
        }
    };
    // one group of copies per tile, empty ones among them, so that a tile's copies
    // are done when all but the last NST - 1 groups are
    const auto fill = [&](uint32_t k) {
        fill_tile(k);
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    for (int k = 0; k < C::NST; ++k) fill(k);

    const float scale2 = a.scale * 1.4426950408889634f;     // scores in log2 units
    // this lane's row address for ldsm_trans: tiles (positions 0..7, 8..15) x (16 bytes, the next 16)
    const uint32_t v_at = mma4::s_addr(ring) + C::VW + (lane & 15) * (C::W * 4) + (lane >> 4) * 16;
    uint32_t k = 0;                                          // the warp's next tile
    for (uint32_t at = wstart; at < wend;) {
        // ---- the unit this part of the run belongs to ----------------------------
        const uint32_t b = row_of_tile(before, a.rows, at);
        const Request rq = request_of(a, b);
        const uint32_t tiles = tiles_in(rq.ctx), nct = col_tiles(rq);
        const uint32_t unit = (at - before[b]) / tiles, hk = unit / nct, col0 = (unit - hk * nct) * COLS;
        const uint32_t u0 = before[b] + unit * tiles, u1 = u0 + tiles, seg_end = min(wend, u1);
        const uint32_t n_cols = rq.n * a.r;

        // query fragments: lane (g, t) holds column g's dims of its words
        uint32_t qf[QP][NT][C::SETS][4];
        float qs[NT][2][G], cs[NT][2];            // of columns 2t, 2t + 1
        const auto word_of = [&](int u) { return GROUP >= 64 ? 8 * (u >> 1) + 2 * t + (u & 1) : 4 * u + t; };
        constexpr auto group_of = [](int u) { return GROUP >= 64 ? (u >> 1) * 64 / GROUP : u; };
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const uint32_t c = col0 + nt * 8 + (PAIR ? g & 3 : g);
            float top = 0.0f, sum[G];
#pragma unroll
            for (int i = 0; i < G; ++i) sum[i] = 0.0f;
            const bool live = c < n_cols;
            const T* q = static_cast<const T*>(a.q) + (rq.token0 + c / a.r) * a.q_token + (hk * a.r + c % a.r) * a.q_head;
            float x[C::SETS][8];
#pragma unroll
            for (int u = 0; u < C::SETS; ++u) {
                if (live)
                    read8(q + 8 * word_of(u), x[u]);
                else
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[u][i] = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    sum[group_of(u)] += x[u][i];
                    top = fmaxf(top, fabsf(x[u][i]));
                }
            }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            // the column's largest |q| between 2^10 and 2^11 (zero and infinite ones as
            // they are), so that 16 q stays in range and small elements keep their bits
            const int e = top > 1e-30f && top < 1e30f ? (int)(__float_as_uint(top) >> 23) - 127 - 10 : 0;
            const float down = pow2(-e), up = pow2(e) * (scale2 * (UNIT / 16.0f));
#pragma unroll
            for (int u = 0; u < C::SETS; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t h[QP];
                    const float f = j & 1 ? down : 16.0f * down;       // the codes' other factor
                    parts_of<QP>(x[u][j] * f, x[u][j + 4] * f, h);
#pragma unroll
                    for (int i = 0; i < QP; ++i) qf[i][nt][u][j] = h[i];
                }
#pragma unroll
            for (int i = 0; i < G; ++i) {
                float v = sum[i] * scale2;
                v += __shfl_xor_sync(0xffffffffu, v, 1);
                v += __shfl_xor_sync(0xffffffffu, v, 2);
                qs[nt][0][i] = __shfl_sync(0xffffffffu, v, 8 * t);
                qs[nt][1][i] = __shfl_sync(0xffffffffu, v, 8 * t + 4);
            }
            cs[nt][0] = __shfl_sync(0xffffffffu, up, 8 * t);
            cs[nt][1] = __shfl_sync(0xffffffffu, up, 8 * t + 4);
        }

        // ref: what scores are relative to (0 until the column has one); room: how far
        // above it a score may go (-inf until then)
        float acc[C::MT][NT][4], ref[NT][2], room[NT][2], ob[NT][2][G], l[NT][2];
        int vexp = VEXP0;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                l[nt][c] = ref[nt][c] = 0.0f;
                room[nt][c] = -INFINITY;
#pragma unroll
                for (int i = 0; i < G; ++i) ob[nt][c][i] = 0.0f;
            }
#pragma unroll
            for (int m = 0; m < C::MT; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[m][nt][i] = 0.0f;
        }
        // top: a column's highest score, relative to ref. Moves the reference where it
        // is above the room, and returns by how much.
        const auto raise = [&](int nt, int c, float top) {
            if (!(top > room[nt][c])) return 0.0f;
            const float by = top - START, f = ex2(-by);
            ref[nt][c] += by;
            if (room[nt][c] == RAISE) {         // else there is nothing yet to rescale
                l[nt][c] *= f;
#pragma unroll
                for (int i = 0; i < G; ++i) ob[nt][c][i] *= f;
#pragma unroll
                for (int m = 0; m < C::MT; ++m) {
                    acc[m][nt][c] *= f;
                    acc[m][nt][2 + c] *= f;
                }
            }
            room[nt][c] = RAISE;
            return by;
        };
        // head dim of the combine's row g (hi = 0) or g + 8 of tile m: code 2 (m % 2) + hi
        // of the row's 16-bit unit; accumulators hold O UNIT / 2^vexp, times 16 for hi
        const auto dim_of = [&](int m, int hi) { return 32 * (m >> 1) + 4 * g + 2 * (m & 1) + hi; };

        // ---- the step's own entries, in the run where the unit begins --------------
        // Entry j against every column: the quad's lanes hold column g's q. One after the
        // other, in one warp: nothing for a few tokens, most of the time for fp32 chunks,
        // which take this kernel too (32 heads over 8 of 128: a first chunk of 1024 3.9 ms, of
        // 4096 54 ms; 1024 over 8192 6.0 ms, 24 TFLOP/s).
        const auto own_entries = [&]() {
            if (u0 < wstart) return;
            const uint32_t last = min(rq.n, (col0 + COLS - 1) / a.r + 1);
            const float unit = pow2(-vexp) / UNIT;
            for (uint32_t j = 0; j < last; ++j) {
                const T* nk = static_cast<const T*>(a.new_k) + (rq.token0 + j) * a.k_token + hk * a.k_head;
                const T* nv = static_cast<const T*>(a.new_v) + (rq.token0 + j) * a.v_token + hk * a.v_head;
                float dot[NT], dot16[NT];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) dot[nt] = dot16[nt] = 0.0f;
#pragma unroll
                for (int u = 0; u < C::SETS; ++u) {
                    float x[8];
                    read8(nk + 8 * word_of(u), x);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            float2 q = unpack(qf[QP - 1][nt][u][i]);
#pragma unroll
                            for (int p = QP - 2; p >= 0; --p) {
                                const float2 h = unpack(qf[p][nt][u][i]);
                                q.x += h.x;
                                q.y += h.y;
                            }
                            float& d = i & 1 ? dot[nt] : dot16[nt];
                            d += q.x * x[i];
                            d += q.y * x[i + 4];
                        }
                }
                float s[NT][2];
                bool sees[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    dot[nt] += dot16[nt] * 0.0625f;
                    dot[nt] += __shfl_xor_sync(0xffffffffu, dot[nt], 1);
                    dot[nt] += __shfl_xor_sync(0xffffffffu, dot[nt], 2);
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        s[nt][c] = __shfl_sync(0xffffffffu, dot[nt], 8 * t + 4 * c) * (cs[nt][c] * (16.0f / UNIT)) - ref[nt][c];
                        const uint32_t col = col0 + nt * 8 + 2 * t + c;
                        // columns past the last one are zero queries: any weight will do; a
                        // paired column counts its own entries once
                        sees[nt][c] = PAIR && t >= 2 ? false : col >= n_cols || j <= col / a.r;
                        if (!sees[nt][c]) s[nt][c] = -INFINITY;
                    }
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        s[nt][c] = ex2(s[nt][c] - raise(nt, c, s[nt][c]));
                        if (g == 0) l[nt][c] += s[nt][c];
                    }
                }
#pragma unroll
                for (int m = 0; m < C::MT; ++m)
#pragma unroll
                    for (int hi = 0; hi < 2; ++hi) {
                        const float v = to_f32(nv[dim_of(m, hi)]) * (hi ? 16.0f * unit : unit);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            // a weight of zero would not keep an infinity out
                            if (sees[nt][0]) acc[m][nt][2 * hi] += s[nt][0] * v;
                            if (sees[nt][1]) acc[m][nt][2 * hi + 1] += s[nt][1] * v;
                        }
                    }
            }
        };
        own_entries();

        // ---- the cached tiles ------------------------------------------------------
        float vlim = pow2(vexp), vinv = pow2(-vexp), vmid = 7.5f * vlim;
        // `weight_parts`: fp16 parts of a weight
        const auto cached_tiles = [&](auto weight_parts) {
            constexpr int PP = decltype(weight_parts)::value;
            for (; wstart + k < seg_end; ++k) {
                const uint32_t s = k % C::NST;
                asm volatile("cp.async.wait_group %0;" ::"n"(C::NST - 1) : "memory");
                __syncwarp();
                const unsigned char* stage = ring + s * C::STAGE;
                const uint32_t pos0 = (wstart + k - u0) * TP;
                const uint32_t valid = rq.ctx > pos0 ? rq.ctx - pos0 : 0;
                if (valid > 0) {
                    float p[NB][NT][4];                      // rows g (0, 1) and g + 8, columns 2t, 2t + 1
                    float vs[NB][2][G], vz[NB][2][G];
                    // scores: blocks and groups are independent chains of MMAs, taken in turn
                    float sacc[SUBS][NT][G][4];
#pragma unroll
                    for (int b = 0; b < SUBS; ++b)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int i = 0; i < G; ++i)
#pragma unroll
                                for (int c = 0; c < 4; ++c) sacc[b][nt][i][c] = 0.0f;
                    constexpr int PER = C::SETS / G;           // runs of words per group
#pragma unroll
                    for (int e = 0; e < PER; ++e)
#pragma unroll
                        for (int b = 0; b < SUBS; ++b)
#pragma unroll
                            for (int gi = 0; gi < G; ++gi) {
                                const int u = gi * PER + e;
                                static_assert(group_of(C::SETS - 1) == G - 1, "runs of a group are consecutive");
                                const uint32_t* kw = reinterpret_cast<const uint32_t*>(stage + b * C::BLOCK);
                                const uint32_t wa = kw[g * C::W + word_of(u)], wb = kw[(g + 8) * C::W + word_of(u)];
#pragma unroll
                                for (int i = 0; i < 2; ++i) {
                                    const uint32_t f[4] = {nib<HALF>(wa, 2 * i), nib<HALF>(wb, 2 * i), nib<HALF>(wa, 2 * i + 1),
                                                           nib<HALF>(wb, 2 * i + 1)};
#pragma unroll
                                    for (int x = 0; x < QP; ++x)
#pragma unroll
                                        for (int nt = 0; nt < NT; ++nt)
                                            mma<HALF>(sacc[b][nt][gi], f, qf[x][nt][u][2 * i], qf[x][nt][u][2 * i + 1]);
                                }
                            }
#pragma unroll
                    for (int b = 0; b < NB; ++b) {
                        const unsigned char* st = stage + (PAIR ? t >> 1 : b) * C::BLOCK;
                        if (PAIR) {
#pragma unroll
                            for (int i = 0; i < G; ++i)
#pragma unroll
                                for (int c = 0; c < 4; ++c) sacc[0][0][i][c] = t < 2 ? sacc[0][0][i][c] : sacc[1][0][i][c];
                        }
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const int at_pos = (g + 8 * h) * G;
                            float ks[G], kz[G];
                            scales_of(reinterpret_cast<const T*>(st + C::KS) + at_pos, ks);
                            scales_of(reinterpret_cast<const T*>(st + C::KZ) + at_pos, kz);
                            scales_of(reinterpret_cast<const T*>(st + C::VS) + at_pos, vs[b][h]);
                            scales_of(reinterpret_cast<const T*>(st + C::VZ) + at_pos, vz[b][h]);
                            if (!HALF) {                          // the codes' 8
#pragma unroll
                                for (int i = 0; i < G; ++i) {
                                    kz[i] = fmaf(8.0f, ks[i], kz[i]);
                                    vz[b][h][i] = fmaf(8.0f, vs[b][h][i], vz[b][h][i]);
                                }
                            }
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int c = 0; c < 2; ++c) {
                                    float x = sacc[b][nt][0][2 * h + c] * ks[0], z = -ref[nt][c];
#pragma unroll
                                    for (int i = 0; i < G; ++i) {
                                        if (i) x = fmaf(sacc[b][nt][i][2 * h + c], ks[i], x);
                                        z = fmaf(kz[i], qs[nt][c][i], z);
                                    }
                                    p[b][nt][2 * h + c] = fmaf(x, cs[nt][c], z);
                                }
                        }
                    }
                    if (valid < TP) {
                        // rows past the length may hold anything
#pragma unroll
                        for (int b = 0; b < NB; ++b)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                if ((uint32_t)((PAIR ? t >> 1 : b) * BLK + 8 * h + g) < valid) continue;
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) p[b][nt][2 * h] = p[b][nt][2 * h + 1] = -INFINITY;
#pragma unroll
                                for (int i = 0; i < G; ++i) vs[b][h][i] = vz[b][h][i] = 0.0f;
                            }
                    }
                    if (bad & (1u << s)) {
#pragma unroll
                        for (int b = 0; b < NB; ++b)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int c = 0; c < 4; ++c) p[b][nt][c] = NAN;
                    }
                    float top[NT][2], vtop = 0.0f;
                    bool over = false;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            top[nt][c] = fmaxf(p[0][nt][c], p[0][nt][2 + c]);
                            if (!PAIR) top[nt][c] = fmaxf(top[nt][c], fmaxf(p[NB - 1][nt][c], p[NB - 1][nt][2 + c]));
                            over |= top[nt][c] > room[nt][c];
                        }
                    if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int c = 0; c < 2; ++c) {
#pragma unroll
                                for (int o = 4; o < 32; o <<= 1) top[nt][c] = fmaxf(top[nt][c], __shfl_xor_sync(0xffffffffu, top[nt][c], o));
                                const float by = raise(nt, c, top[nt][c]);
#pragma unroll
                                for (int b = 0; b < NB; ++b) {
                                    p[b][nt][c] -= by;
                                    p[b][nt][2 + c] -= by;
                                }
                            }
                    }
#pragma unroll
                    for (int b = 0; b < NB; ++b)
#pragma unroll
                        for (int i = 0; i < G; ++i) vtop = fmaxf(vtop, fmaxf(fabsf(vs[b][0][i]), fabsf(vs[b][1][i])));
                    if (__any_sync(0xffffffffu, vtop >= vlim)) {
                        const int ve = min((int)(__reduce_max_sync(0xffffffffu, __float_as_uint(vtop)) >> 23) - 126, VEXP1);
                        if (ve > vexp) {               // |vs| < 2^ve
                            const float f = pow2(vexp - ve);
                            vexp = ve;
                            vlim = pow2(ve);
                            vinv = pow2(-ve);
                            vmid = 7.5f * vlim;
#pragma unroll
                            for (int m = 0; m < C::MT; ++m)
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                    for (int c = 0; c < 4; ++c) acc[m][nt][c] *= f;
                        }
                    }
                    uint32_t bf[G][NT][PP][2];
#pragma unroll
                    for (int b = 0; b < SUBS; ++b) {
                        if (!PAIR || b == 0) {
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int c = 0; c < 4; ++c) {
                                p[b][nt][c] = ex2(p[b][nt][c]);
                                l[nt][c & 1] += p[b][nt][c];
                            }
#pragma unroll
                        for (int i = 0; i < G; ++i)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const float sc = vs[b][h][i] * vinv;
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt) {
                                    uint32_t f[PP];
                                    const float w0 = p[b][nt][2 * h] * sc, w1 = p[b][nt][2 * h + 1] * sc;
                                    parts_of<PP>(w0, w1, f);
#pragma unroll
                                    for (int c = 0; c < 2; ++c) ob[nt][c][i] = fmaf(p[b][nt][2 * h + c], vz[b][h][i], ob[nt][c][i]);
                                    if constexpr (PP == 1) {
                                        const float2 r = unpack(f[0]);
                                        ob[nt][0][i] = fmaf(w0 - r.x, vmid, ob[nt][0][i]);
                                        ob[nt][1][i] = fmaf(w1 - r.y, vmid, ob[nt][1][i]);
                                    }
#pragma unroll
                                    for (int x = 0; x < PP; ++x) bf[i][nt][x][h] = movmatrix(f[x]);
                                }
                            }
                        }
                        uint32_t bm[G][NT][PP][2];              // the weights of this block
#pragma unroll
                        for (int i = 0; i < G; ++i)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int x = 0; x < PP; ++x)
#pragma unroll
                                    for (int h = 0; h < 2; ++h) bm[i][nt][x][h] = !PAIR || (g >> 2) == b ? bf[i][nt][x][h] : 0u;
                        const uint32_t va = v_at + s * C::STAGE + b * C::BLOCK;
#pragma unroll
                        for (int c2 = 0; c2 < DH / 64; ++c2) {
                            uint32_t w[4];              // 32 dims at positions 0..7 and 8..15, the next 32
                            ldsm_trans(va + 32 * c2, w);
                            uint32_t f[4][4];
#pragma unroll
                            for (int m = 0; m < 4; ++m) {
                                const int c = m >> 1, j = m & 1;
                                f[m][0] = nib<HALF>(w[2 * c], 2 * j);
                                f[m][1] = nib<HALF>(w[2 * c], 2 * j + 1);
                                f[m][2] = nib<HALF>(w[2 * c + 1], 2 * j);
                                f[m][3] = nib<HALF>(w[2 * c + 1], 2 * j + 1);
                            }
#pragma unroll
                            for (int x = 0; x < PP; ++x)
#pragma unroll
                                for (int m = 0; m < 4; ++m) {
                                    const int i = (2 * c2 + (m >> 1)) * 32 / GROUP;
#pragma unroll
                                    for (int nt = 0; nt < NT; ++nt)
                                        mma<HALF>(acc[4 * c2 + m][nt], f[m], bm[i][nt][x][0], bm[i][nt][x][1]);
                                }
                        }
                    }
                }
                __syncwarp();
                fill(k + C::NST);
            }
        };
        if constexpr (!HALF) cached_tiles(std::integral_constant<int, 3>{});
        else if (rq.ctx <= SHORT) cached_tiles(std::integral_constant<int, 2>{});
        else cached_tiles(std::integral_constant<int, 1>{});

        // ---- the part's result -------------------------------------------------------
        const float back = pow2(vexp) * UNIT;
        float own_m[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float bias[G];
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], o);
#pragma unroll
                for (int i = 0; i < G; ++i) {
                    bias[i] = ob[nt][c][i];
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) bias[i] += __shfl_xor_sync(0xffffffffu, bias[i], o);
                }
                own_m[nt][c] = room[nt][c] == RAISE ? ref[nt][c] : -INFINITY;
#pragma unroll
                for (int m = 0; m < C::MT; ++m)
#pragma unroll
                    for (int hi = 0; hi < 2; ++hi)
                        acc[m][nt][2 * hi + c] = acc[m][nt][2 * hi + c] * (hi ? back / 16.0f : back) + bias[(m >> 1) * 32 / GROUP];
            }
        if (PAIR) {
            // the second block's columns are two lanes on in the quad
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const float m2 = __shfl_xor_sync(0xffffffffu, own_m[0][c], 2), m = fmaxf(own_m[0][c], m2);
                const float l2 = __shfl_xor_sync(0xffffffffu, l[0][c], 2);
                const float f = own_m[0][c] == m ? 1.0f : ex2(own_m[0][c] - m), f2 = m2 == m ? 1.0f : ex2(m2 - m);
                own_m[0][c] = m;
                l[0][c] = l[0][c] * f + l2 * f2;
#pragma unroll
                for (int k2 = 0; k2 < C::MT; ++k2)
#pragma unroll
                    for (int hi = 0; hi < 2; ++hi) {
                        float& x = acc[k2][0][2 * hi + c];
                        const float y = __shfl_xor_sync(0xffffffffu, x, 2);
                        x = x * f + y * f2;
                    }
            }
        }
        const bool writes = !PAIR || t < 2, head = u0 < wstart;
        if (!head && u1 <= wend) {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const uint32_t cc = col0 + nt * 8 + 2 * t + c;
                    if (!writes || cc >= n_cols) continue;
                    const float inv = 1.0f / l[nt][c];
                    T* out = static_cast<T*>(a.out) + ((size_t)(rq.token0 + cc / a.r) * a.n_heads + hk * a.r + cc % a.r) * DH;
#pragma unroll
                    for (int m = 0; m < C::MT; m += 2)
                        store4(out + dim_of(m, 0), make_float4(acc[m][nt][c] * inv, acc[m][nt][2 + c] * inv,
                                                               acc[m + 1][nt][c] * inv, acc[m + 1][nt][2 + c] * inv));
                }
        } else {
            __syncwarp();                           // a tail lies in the ring, which is done with
            float* o = part_o(!head, warp);
            float* ml = part_ml(!head, warp);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int col = nt * 8 + 2 * t + c;
                    if (!writes) continue;
                    if (g == 0) {
                        ml[col] = own_m[nt][c];
                        ml[COLS + col] = l[nt][c];
                    }
#pragma unroll
                    for (int m = 0; m < C::MT; m += 2)
                        *reinterpret_cast<float4*>(&o[col * DH + dim_of(m, 0)]) =
                            make_float4(acc[m][nt][c], acc[m][nt][2 + c], acc[m + 1][nt][c], acc[m + 1][nt][2 + c]);
                }
            if (lane == 0)
                info[(head ? 0 : CW) + warp] = {u0, u1, rq.token0, hk, col0, min((uint32_t)COLS, n_cols - col0)};
        }
        at = seg_end;
    }

    // ---- the parts of units that several warps shared, joined in their order ----------
    __syncthreads();
    float* slots = reinterpret_cast<float*>(ws + split_bytes(gridDim.x)) + 2 * (size_t)blockIdx.x * slot_floats(COLS, DH);
    for (int first = -1; first < CW; ++first) {
        // a unit's first part here: warp 0's head (the unit began before the share) or a tail
        const Info u = info[first < 0 ? 0 : CW + first];
        if (u.cols == 0) continue;
        const int w0 = max(first, 0), w1 = (int)((min(u.u1, end) - 1 - start) / run);
        const bool whole = u.u0 >= start && u.u1 <= end;
        float* slot = slots + (u.u0 >= start ? slot_floats(COLS, DH) : 0);
        for (int i = tid; i < (int)u.cols * (DH / 4); i += THREADS) {
            const int col = i / (DH / 4), d = i % (DH / 4) * 4;
            float m = part_ml(first >= 0, w0)[col];
            for (int w = w0 + 1; w <= w1; ++w) m = fmaxf(m, part_ml(0, w)[col]);
            float sum = 0.0f;
            float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (int w = w0; w <= w1; ++w) {
                const int kind = w == w0 && first >= 0;
                const float f = ex2(part_ml(kind, w)[col] - m);
                const float4 x = *reinterpret_cast<const float4*>(&part_o(kind, w)[col * DH + d]);
                sum += f * part_ml(kind, w)[COLS + col];
                o.x += f * x.x;
                o.y += f * x.y;
                o.z += f * x.z;
                o.w += f * x.w;
            }
            if (whole) {
                const uint32_t c = u.col0 + col, tok = u.token0 + c / a.r, hd = u.hk * a.r + c % a.r;
                store4(static_cast<T*>(a.out) + ((size_t)tok * a.n_heads + hd) * DH + d,
                       make_float4(o.x / sum, o.y / sum, o.z / sum, o.w / sum));
            } else {
                *reinterpret_cast<float4*>(&slot[2 * COLS + col * DH + d]) = o;
                if (d == 0) {
                    slot[col] = m;
                    slot[COLS + col] = sum;
                }
            }
        }
        if (tid == 0 && u.u0 >= start && u.u1 > end)
            reinterpret_cast<Split*>(ws)[blockIdx.x] = {(u.u1 - 1) / share - blockIdx.x + 1, u.token0, u.hk, u.col0, u.cols};
    }
}

template <typename T, int DH, int GROUP, int NT, bool PAIR>
cudaError_t launch_few(const Attend& a, uint32_t most_new, uint32_t grid, void* ws, cudaStream_t stream) {
    using C = Cfg<T, DH, GROUP, NT, PAIR>;
    const size_t smem = C::BEFORE + ((size_t)a.rows + 1) * 4;
    auto kernel = few_kernel<T, DH, GROUP, NT, PAIR>;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_smem(kernel, C::BEFORE + (MAX_ROWS + 1) * 4, done);
    if (e != cudaSuccess) return e;
    kernel<<<grid, C::THREADS, smem, stream>>>(a, most_new, static_cast<unsigned char*>(ws));
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    return launch_join<T, DH, C::COLS>(a, grid, static_cast<const unsigned char*>(ws), stream);
}

}  // namespace few
}  // namespace paged
}  // namespace kvq
