// Paged attention for requests with few new tokens (a decode step, verified
// drafts): the cache is read once for up to 8 NT query columns, a column being
// one (token, query head) of a request, so the step is bound by the cache's
// bytes.
//
// A warp takes 32 cached positions at a time, as two blocks of 16: it streams
// them with 16-byte cp.async into its own ring (a page holds whole blocks; no
// warp waits for another), and keeps its own online softmax; the CTA's warps are
// joined when a unit ends. With codes c, scales s, z = bias:
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
// Precision: products exact, sums fp32. The weights are carried as PP fp16
// parts (2: 2^-22 relative, for fp16 steps; 3 for fp32 steps), held near the
// top of fp16's range: p is relative to a reference that the running maximum
// may pass by 2^14 before it moves (so accumulators are rarely rescaled), and
// vs is divided by a power of two above the largest |vs| met so far. Queries
// are scaled by a power of two per column (fp32 ones are three fp16 parts of
// that, and their MMAs start from zero and are added in fp32, since a long
// chain of additions in the tensor cores truncates).
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

template <typename T, int DH_, int GROUP_, int NT_>
struct Cfg {
    static constexpr int DH = DH_, GROUP = GROUP_, NT = NT_;
    static constexpr bool HALF = sizeof(T) == 2;
    static constexpr int G = DH / GROUP;
    static constexpr int W = DH / 8;                // words per row
    static constexpr int SETS = DH / 32;            // runs of four words, one per lane of a quad
    static constexpr int MT = DH / 16;              // combine's 16-dim tiles
    static constexpr int QP = HALF ? 1 : 3, PP = HALF ? 2 : 3;
    static constexpr int COLS = 8 * NT;
    // One CTA per SM: sixteen warps where 128 registers do, else eight. (Two CTAs
    // of eight leave twice the parts to join, and the CTA that is launched later
    // runs behind the other: 1 x 131072 took 60 us so.)
    static constexpr int CW = HALF && NT == 1 ? 16 : 8, THREADS = 32 * CW;
    static constexpr int HW = 8;                    // warps joined at once
    static constexpr int WB = BLK * W * 4, SB = BLK * G * (int)sizeof(T);
    static constexpr int VW = WB, KS = 2 * WB, KZ = KS + SB, VS = KZ + SB, VZ = VS + SB;
    static constexpr int BLOCK = VZ + SB;           // bytes of 16 positions
    static constexpr int STAGE = SUBS * BLOCK;
    static constexpr int NST = 2;                   // tiles per ring
    static constexpr int LD = DH + 4;               // floats per combined row (no bank conflicts)
    static constexpr int COMB = CW * STAGE * NST;   // fp32 [HW][COLS][LD], then m and l [CW][COLS]
    static constexpr int ML = COMB + HW * COLS * LD * 4;
    static constexpr int BEFORE = ML + 2 * CW * COLS * 4;      // uint32 [rows + 1]
    static_assert(STAGE % 16 == 0 && COMB % 16 == 0 && BEFORE % 16 == 0, "alignment");
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

template <typename T, int DH, int GROUP, int NT>
__global__ void __launch_bounds__(Cfg<T, DH, GROUP, NT>::THREADS, 1)
few_kernel(Attend a, uint32_t most_new, unsigned char* __restrict__ ws) {
    using C = Cfg<T, DH, GROUP, NT>;
    constexpr int G = C::G, COLS = C::COLS, QP = C::QP, PP = C::PP, CW = C::CW, HW = C::HW, THREADS = C::THREADS;
    constexpr bool HALF = C::HALF;
    constexpr float UNIT = HALF ? 16777216.0f : 1.0f;      // a code in an MMA is c / UNIT, or 16 c / UNIT
    // exponents of the power of two above |vs|: from below what the quantizer
    // stores (its smallest step is 1e-7) to the type's largest
    constexpr int VEXP0 = HALF ? -14 : -30, VEXP1 = HALF ? 16 : 90;
    // the join's CTAs may come as soon as there is room: none before these CTAs,
    // which hold a whole SM's registers each, have left
    pdl_launch_dependents();
    extern __shared__ __align__(128) unsigned char smem[];
    uint32_t* before = reinterpret_cast<uint32_t*>(smem + C::BEFORE);
    float* comb = reinterpret_cast<float*>(smem + C::COMB);
    float* comb_m = reinterpret_cast<float*>(smem + C::ML);
    float* comb_l = comb_m + CW * COLS;
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
    // a whole round of the warps is the least a CTA takes
    const uint32_t share = ((total + gridDim.x - 1) / gridDim.x + CW - 1) / CW * CW;
    const uint64_t start64 = (uint64_t)blockIdx.x * share;
    if (start64 >= total) return;
    const uint32_t start = (uint32_t)start64, end = min(total, start + share);

    // ---- the warp's stream of tiles -----------------------------------------
    // lane i looks up the batch's i-th tile: the cache row of each block, and per
    // block whether it holds positions (bit) and its page id is in the pool (bad)
    uint32_t row_at[SUBS] = {0, 0}, held = 0, bad_id = 0;
    uint32_t bad = 0;                                  // stages with such a page
    const auto look = [&](uint32_t k0) {
        const uint64_t x64 = (uint64_t)start + warp + (uint64_t)CW * (k0 + lane);
        held = bad_id = 0;
        if (x64 >= end) return;
        const uint32_t x = (uint32_t)x64;
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
    const uint32_t own = end - start > (uint32_t)warp ? (end - start - warp + CW - 1) / CW : 0;   // the warp's tiles
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
    for (uint32_t at = start; at < end;) {
        // ---- the unit this part of the share belongs to --------------------------
        const uint32_t b = row_of_tile(before, a.rows, at);
        const Request rq = request_of(a, b);
        const uint32_t tiles = tiles_in(rq.ctx), nct = col_tiles(rq);
        const uint32_t unit = (at - before[b]) / tiles, hk = unit / nct, col0 = (unit - hk * nct) * COLS;
        const uint32_t u0 = before[b] + unit * tiles, u1 = u0 + tiles, seg_end = min(end, u1);
        const uint32_t n_cols = rq.n * a.r;

        // query fragments: lane (g, t) holds column g's dims of its words
        uint32_t qf[QP][NT][C::SETS][4];
        float qs[NT][2][G], cs[NT][2];            // of columns 2t, 2t + 1
        const auto word_of = [&](int u) { return GROUP >= 64 ? 8 * (u >> 1) + 2 * t + (u & 1) : 4 * u + t; };
        constexpr auto group_of = [](int u) { return GROUP >= 64 ? (u >> 1) * 64 / GROUP : u; };
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const uint32_t c = col0 + nt * 8 + g;
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

        // ---- the step's own entries, in the share where the unit begins -----------
        // Entry j against every column: the quad's lanes hold column g's q.
        const auto own_entries = [&]() {
            if (u0 < start) return;
            const uint32_t last = min(rq.n, (col0 + COLS - 1) / a.r + 1);
            const float unit = pow2(-vexp) / UNIT;
            for (uint32_t j = warp; j < last; j += CW) {
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
                        // columns past the last one are zero queries: any weight will do
                        sees[nt][c] = col >= n_cols || j <= col / a.r;
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
        float vlim = pow2(vexp), vinv = pow2(-vexp);
        for (; k < own && start + warp + k * CW < seg_end; ++k) {
            const uint32_t s = k % C::NST;
            asm volatile("cp.async.wait_group %0;" ::"n"(C::NST - 1) : "memory");
            __syncwarp();
            const unsigned char* stage = ring + s * C::STAGE;
            const uint32_t pos0 = (start + warp + k * CW - u0) * TP;
            const uint32_t valid = rq.ctx > pos0 ? rq.ctx - pos0 : 0;
            if (valid > 0) {
                float p[SUBS][NT][4];                      // rows g (0, 1) and g + 8, columns 2t, 2t + 1
                float vs[SUBS][2][G], vz[SUBS][2][G];
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
                for (int b = 0; b < SUBS; ++b) {
                    const unsigned char* st = stage + b * C::BLOCK;
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
                    for (int b = 0; b < SUBS; ++b)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            if ((uint32_t)(b * BLK + 8 * h + g) < valid) continue;
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) p[b][nt][2 * h] = p[b][nt][2 * h + 1] = -INFINITY;
#pragma unroll
                            for (int i = 0; i < G; ++i) vs[b][h][i] = vz[b][h][i] = 0.0f;
                        }
                }
                if (bad & (1u << s)) {
#pragma unroll
                    for (int b = 0; b < SUBS; ++b)
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
                        top[nt][c] = fmaxf(fmaxf(p[0][nt][c], p[0][nt][2 + c]), fmaxf(p[1][nt][c], p[1][nt][2 + c]));
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
                            for (int b = 0; b < SUBS; ++b) {
                                p[b][nt][c] -= by;
                                p[b][nt][2 + c] -= by;
                            }
                        }
                }
#pragma unroll
                for (int b = 0; b < SUBS; ++b)
#pragma unroll
                    for (int i = 0; i < G; ++i) vtop = fmaxf(vtop, fmaxf(fabsf(vs[b][0][i]), fabsf(vs[b][1][i])));
                if (__any_sync(0xffffffffu, vtop >= vlim)) {
                    const int ve = min((int)(__reduce_max_sync(0xffffffffu, __float_as_uint(vtop)) >> 23) - 126, VEXP1);
                    if (ve > vexp) {               // |vs| < 2^ve
                        const float f = pow2(vexp - ve);
                        vexp = ve;
                        vlim = pow2(ve);
                        vinv = pow2(-ve);
#pragma unroll
                        for (int m = 0; m < C::MT; ++m)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int c = 0; c < 4; ++c) acc[m][nt][c] *= f;
                    }
                }
#pragma unroll
                for (int b = 0; b < SUBS; ++b) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int c = 0; c < 4; ++c) {
                            p[b][nt][c] = ex2(p[b][nt][c]);
                            l[nt][c & 1] += p[b][nt][c];
                        }
                    uint32_t bf[G][NT][PP][2];
#pragma unroll
                    for (int i = 0; i < G; ++i)
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float sc = vs[b][h][i] * vinv;
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt) {
                                uint32_t f[PP];
                                parts_of<PP>(p[b][nt][2 * h] * sc, p[b][nt][2 * h + 1] * sc, f);
#pragma unroll
                                for (int c = 0; c < 2; ++c) ob[nt][c][i] = fmaf(p[b][nt][2 * h + c], vz[b][h][i], ob[nt][c][i]);
#pragma unroll
                                for (int x = 0; x < PP; ++x) bf[i][nt][x][h] = movmatrix(f[x]);
                            }
                        }
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
                                    mma<HALF>(acc[4 * c2 + m][nt], f[m], bf[i][nt][x][0], bf[i][nt][x][1]);
                            }
                    }
                }
            }
            __syncwarp();
            fill(k + C::NST);
        }

        // ---- the warps' results of this part, joined ---------------------------------
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
        const auto leave = [&]() {
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    const int col = nt * 8 + 2 * t + c;
                    if (g == 0) {
                        comb_m[warp * COLS + col] = own_m[nt][c];
                        comb_l[warp * COLS + col] = l[nt][c];
                    }
#pragma unroll
                    for (int m = 0; m < C::MT; ++m)
#pragma unroll
                        for (int hi = 0; hi < 2; ++hi)
                            comb[((warp % HW) * COLS + col) * C::LD + dim_of(m, hi)] = acc[m][nt][2 * hi + c];
                }
        };
        if constexpr (CW > HW) {
            // the upper half's results go to the lower half's warps first
            if (warp >= HW) leave();
            __syncthreads();
            if (warp < HW) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        const int col = nt * 8 + 2 * t + c;
                        const float m2 = comb_m[(warp + HW) * COLS + col], m = fmaxf(own_m[nt][c], m2);
                        const float f = own_m[nt][c] == m ? 1.0f : ex2(own_m[nt][c] - m), f2 = m2 == m ? 1.0f : ex2(m2 - m);
                        own_m[nt][c] = m;
                        l[nt][c] = l[nt][c] * f + comb_l[(warp + HW) * COLS + col] * f2;
#pragma unroll
                        for (int k2 = 0; k2 < C::MT; ++k2)
#pragma unroll
                            for (int hi = 0; hi < 2; ++hi) {
                                float& x = acc[k2][nt][2 * hi + c];
                                x = x * f + comb[(warp * COLS + col) * C::LD + dim_of(k2, hi)] * f2;
                            }
                    }
            }
        }
        if (warp < HW) leave();
        __syncthreads();
        const bool whole = u0 >= start && u1 <= end;
        float* slot = reinterpret_cast<float*>(ws + split_bytes(gridDim.x)) +
                      (2 * (size_t)blockIdx.x + (u0 >= start ? 1 : 0)) * slot_floats(COLS, DH);
        for (int i = tid; i < COLS * DH / 4; i += THREADS) {
            const int col = i / (DH / 4), d = i % (DH / 4) * 4;
            const uint32_t c = col0 + col;
            if (c >= n_cols) continue;
            float m = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < HW; ++w) m = fmaxf(m, comb_m[w * COLS + col]);
            float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < HW; ++w) {
                const float f = ex2(comb_m[w * COLS + col] - m);
                const float4 x = *reinterpret_cast<const float4*>(&comb[(w * COLS + col) * C::LD + d]);
                sum += f * comb_l[w * COLS + col];
                o.x += f * x.x;
                o.y += f * x.y;
                o.z += f * x.z;
                o.w += f * x.w;
            }
            if (whole) {
                const uint32_t tok = rq.token0 + c / a.r, head = hk * a.r + c % a.r;
                alignas(16) T v[4] = {from_f32<T>(o.x / sum), from_f32<T>(o.y / sum), from_f32<T>(o.z / sum),
                                      from_f32<T>(o.w / sum)};
                T* dst = static_cast<T*>(a.out) + ((size_t)tok * a.n_heads + head) * DH + d;
                if constexpr (HALF) *reinterpret_cast<uint2*>(dst) = *reinterpret_cast<const uint2*>(v);
                else *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(v);
            } else {
                *reinterpret_cast<float4*>(&slot[2 * COLS + col * DH + d]) = o;
                if (d == 0) {
                    slot[col] = m;
                    slot[COLS + col] = sum;
                }
            }
        }
        if (tid == 0 && u0 >= start && u1 > end)
            reinterpret_cast<Split*>(ws)[blockIdx.x] = {(u1 - 1) / share - blockIdx.x + 1, rq.token0, hk, col0,
                                                        min((uint32_t)COLS, n_cols - col0)};
        __syncthreads();
        at = seg_end;
    }
}

template <typename T, int DH, int GROUP, int NT>
cudaError_t launch_few(const Attend& a, uint32_t most_new, uint32_t grid, void* ws, cudaStream_t stream) {
    using C = Cfg<T, DH, GROUP, NT>;
    const size_t smem = C::BEFORE + ((size_t)a.rows + 1) * 4;
    auto kernel = few_kernel<T, DH, GROUP, NT>;
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
