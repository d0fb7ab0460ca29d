// Paged attention for requests with few new tokens (a decode step, verified
// drafts): the cache is read once for up to 8 NT query columns, a column being
// one (token, query head) of a request, so the step is bound by the cache's
// bytes.
//
// A warp takes 16 cached positions at a time: it streams them with
// cp.async.bulk into its own ring (a page holds whole tiles; no warp waits for
// another), and keeps its own online softmax; the CTA's eight warps are joined
// when a unit ends. With codes c, scales s, z = bias:
//
//   scores   S^T[pos, col] = sum_g ks[pos,g] (sum_{d in g} c[pos,d] q[col,d])
//                            + kz[pos,g] (sum_{d in g} q[col,d])
//   combine  O^T[d, col]   = sum_pos c[pos,d] (p[pos,col] vs[pos,g(d)])
//                            + sum_pos p[pos,col] vz[pos,g(d)]
//
// both as m16n8k16 fp16 MMAs with the codes as the A operand. Codes are never
// converted: the bits of c are the fp16 subnormal c * 2^-24, which the tensor
// cores multiply exactly, so two codes cost one shift and one AND, and the 2^24
// goes into the scale. Which head dims (scores) and which positions (combine)
// a lane holds is free as long as both operands agree, and is chosen so that
// the packed words are used where they are loaded. The weights p vs reach the
// combine's B layout by one movmatrix per 8 x 8 block.
//
// Precision: products exact, sums fp32. The weights are carried as PP fp16
// parts (2: 2^-22 relative, for fp16 steps; 3 for fp32 steps), held near the
// top of fp16's range: p is relative to a reference that the running maximum
// may pass by 2^14 before it moves (so accumulators are rarely rescaled), and
// vs is divided by a power of two above the largest |vs| met so far. fp32
// queries are three fp16 parts of q divided by a power of two per column, and
// their MMAs start from zero and are added in fp32, since a long chain of
// additions in the tensor cores truncates.
#pragma once

#include <atomic>

#include "kvq_mma.cuh"
#include "kvq_paged_work.cuh"

namespace kvq {
namespace paged {
namespace few {

using mma4::bulk_g2s;
using mma4::ex2;
using mma4::mbar_arrive;
using mma4::mbar_expect_tx;
using mma4::mbar_init;
using mma4::mbar_wait;
using mma4::mma_f16;

constexpr int CW = 8;                     // warps
constexpr int THREADS = 32 * CW;
constexpr int TP = 16;                    // positions per tile
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
    static constexpr int WB = TP * W * 4, SB = TP * G * (int)sizeof(T);
    static constexpr int VW = WB, KS = 2 * WB, KZ = KS + SB, VS = KZ + SB, VZ = VS + SB;
    static constexpr int STAGE = VZ + SB;
    static constexpr int NST = 4;                   // tiles in flight per warp
    static constexpr int LD = DH + 4;               // floats per combined row (no bank conflicts)
    static constexpr int COMB = CW * STAGE * NST;   // fp32 [CW][COLS][LD], then m and l [CW][COLS]
    static constexpr int ML = COMB + CW * COLS * LD * 4;
    static constexpr int BAR = ML + 2 * CW * COLS * 4;
    static constexpr int BEFORE = BAR + CW * NST * 8 + 16;     // uint32 [rows + 1]
    static constexpr int MIN_CTAS = NT == 1 && HALF ? 2 : 1;
    static_assert(STAGE % 16 == 0 && COMB % 16 == 0 && BAR % 8 == 0 && BEFORE % 16 == 0, "alignment");
};

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
    uint32_t d;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(sel));
    return d;
}
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
// codes j and j + 4 of a word (or of two words' halves) as subnormal fp16x2:
// c, or c - 8 (exact) for fp32 steps, whose sums over codes of one sign would
// be far larger than what the bias then leaves of them
template <bool HALF>
__device__ __forceinline__ uint32_t nib(uint32_t w, int j) {
    uint32_t x = (w >> (4 * j)) & 0x000F000Fu;
    if constexpr (!HALF) {
        const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&x), __half2half2(__ushort_as_half(8)));
        x = *reinterpret_cast<const uint32_t*>(&h);
    }
    return x;
}
__device__ __forceinline__ float pow2(int e) { return ldexpf(1.0f, e); }

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
__global__ void __launch_bounds__(THREADS, (Cfg<T, DH, GROUP, NT>::MIN_CTAS))
few_kernel(Attend a, uint32_t most_new, unsigned char* __restrict__ ws) {
    using C = Cfg<T, DH, GROUP, NT>;
    constexpr int G = C::G, COLS = C::COLS, QP = C::QP, PP = C::PP;
    constexpr bool HALF = C::HALF;
    // exponents of the power of two above |vs|: from below what the quantizer
    // stores (its smallest step is 1e-7) to the type's largest
    constexpr int VEXP0 = HALF ? -14 : -30, VEXP1 = HALF ? 16 : 100;
    extern __shared__ __align__(128) unsigned char smem[];
    uint32_t* before = reinterpret_cast<uint32_t*>(smem + C::BEFORE);
    float* comb = reinterpret_cast<float*>(smem + C::COMB);
    float* comb_m = reinterpret_cast<float*>(smem + C::ML);
    float* comb_l = comb_m + CW * COLS;
    int* err = reinterpret_cast<int*>(smem + C::BEFORE - 16);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, g = lane >> 2, t = lane & 3;
    unsigned char* ring = smem + warp * C::STAGE * C::NST;
    uint64_t* bar = reinterpret_cast<uint64_t*>(smem + C::BAR) + warp * C::NST;

    if (lane == 0) {
        for (int s = 0; s < C::NST; ++s) mbar_init(&bar[s], 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (tid == 0) {
        *err = 0;
        reinterpret_cast<Split*>(ws)[blockIdx.x].parts = 0;
    }
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
    uint64_t row_at = 0;          // lane i: first cache row of the batch's i-th tile
    uint32_t kind = 0;            // 0 no positions, 1 a page, 2 a page id outside the pool
    uint32_t bad = 0;             // stages that hold such a page
    const auto look = [&](uint32_t k0) {
        const uint64_t x64 = (uint64_t)start + warp + (uint64_t)CW * (k0 + lane);
        kind = 0;
        if (x64 >= end) return;
        const uint32_t x = (uint32_t)x64;
        const uint32_t b = row_of_tile(before, a.rows, x);
        const Request r = request_of(a, b);
        const uint32_t tiles = tiles_in(r.ctx), rem = x - before[b], unit = rem / tiles;
        const uint32_t pos = (rem - unit * tiles) * TP, hk = unit / col_tiles(r);
        if (pos >= r.ctx) return;
        uint32_t page = (uint32_t)a.block_tables[(size_t)b * a.width + (pos >> a.page_shift)];
        kind = 1;
        if (page >= a.pages) {
            kind = 2;
            page = 0;
        }
        row_at = (((uint64_t)page * H + hk) << a.page_shift) + (pos & ((1u << a.page_shift) - 1));
    };
    const uint32_t own = end - start > (uint32_t)warp ? (end - start - warp + CW - 1) / CW : 0;   // the warp's tiles
    const auto fill = [&](uint32_t k) {
        if (k >= own) return;
        if ((k & 31) == 0) look(k);
        const uint64_t row = __shfl_sync(0xffffffffu, row_at, k & 31);
        const uint32_t what = __shfl_sync(0xffffffffu, kind, k & 31);
        const uint32_t s = k % C::NST;
        bad = what == 2 ? bad | (1u << s) : bad & ~(1u << s);
        if (what == 0) {
            if (lane == 0) mbar_arrive(&bar[s]);
            return;
        }
        if (lane == 0) mbar_expect_tx(&bar[s], C::STAGE);
        __syncwarp();
        if (lane < 6) {
            const int half = lane >= 3, part = lane - 3 * half;
            const Pool& p = half ? a.v : a.k;
            const unsigned char* src = part == 0 ? reinterpret_cast<const unsigned char*>(p.words) + row * (C::W * 4)
                                       : static_cast<const unsigned char*>(part == 1 ? p.scales : p.biases) + row * (G * sizeof(T));
            const int off = part == 0 ? half * C::WB : C::KS + (2 * half + part - 1) * C::SB;
            bulk_g2s(ring + s * C::STAGE + off, src, part == 0 ? C::WB : C::SB, &bar[s], mma4::evict_first_policy());
        }
    };
    for (int k = 0; k < C::NST; ++k) fill(k);

    const float scale2 = a.scale * 1.4426950408889634f;     // scores in log2 units
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
        float qs[NT][2][G], cs[NT][2];
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
            float down = 1.0f, up = 1.0f;
            if constexpr (!HALF) {
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                // the column's largest |q| at 2^12 (zero, huge and infinite ones as they are)
                const int e = top > 1e-30f && top < 1e30f ? (int)(__float_as_uint(top) >> 23) - 127 - 12 : 0;
                down = pow2(-e);
                up = pow2(e);
            }
#pragma unroll
            for (int u = 0; u < C::SETS; ++u)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    uint32_t h[QP];
                    parts_of<QP>(x[u][j] * down, x[u][j + 4] * down, h);
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
            cs[nt][0] = __shfl_sync(0xffffffffu, up, 8 * t) * scale2 * 16777216.0f;
            cs[nt][1] = __shfl_sync(0xffffffffu, up, 8 * t + 4) * scale2 * 16777216.0f;
        }

        float acc[C::MT][NT][4], ob[NT][2][G], l[NT][2], ref[NT][2];
        int vexp = VEXP0;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                l[nt][c] = 0.0f;
                ref[nt][c] = -INFINITY;
#pragma unroll
                for (int i = 0; i < G; ++i) ob[nt][c][i] = 0.0f;
            }
#pragma unroll
            for (int m = 0; m < C::MT; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[m][nt][i] = 0.0f;
        }
        // moves a column's reference where a score passed it by more than RAISE
        const auto raise = [&](int nt, float top0, float top1) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const float top = c ? top1 : top0;
                if (!(top - ref[nt][c] > RAISE)) continue;
                const float to = top - START, f = ex2(ref[nt][c] - to);
                ref[nt][c] = to;
                l[nt][c] *= f;
#pragma unroll
                for (int i = 0; i < G; ++i) ob[nt][c][i] *= f;
#pragma unroll
                for (int m = 0; m < C::MT; ++m) {
                    acc[m][nt][c] *= f;
                    acc[m][nt][2 + c] *= f;
                }
            }
        };
        // head dim of the combine's row g (hi = 0) or g + 8 of tile m
        const auto dim_of = [&](int m, int hi) {
            if (GROUP >= 64) return 8 * (8 * (m >> 2) + g) + (m & 3) + 4 * hi;
            return 8 * (8 * (m >> 2) + 4 * ((m >> 1) & 1) + (g & 3)) + 4 * (g >> 2) + 2 * (m & 1) + hi;
        };

        // ---- the step's own entries, in the share where the unit begins -----------
        // Entry j against every column: the quad's lanes hold column g's q.
        const auto own_entries = [&]() {
            if (u0 < start) return;
            const uint32_t last = min(rq.n, (col0 + COLS - 1) / a.r + 1);
            const float unit_v = pow2(-vexp) * 5.9604644775390625e-8f;     // accumulators hold O / 2^(24 + vexp)
            for (uint32_t j = warp; j < last; j += CW) {
                const T* nk = static_cast<const T*>(a.new_k) + (rq.token0 + j) * a.k_token + hk * a.k_head;
                const T* nv = static_cast<const T*>(a.new_v) + (rq.token0 + j) * a.v_token + hk * a.v_head;
                float dot[NT];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) dot[nt] = 0.0f;
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
                            dot[nt] += q.x * x[i];
                            dot[nt] += q.y * x[i + 4];
                        }
                }
                float s[NT][2];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    dot[nt] += __shfl_xor_sync(0xffffffffu, dot[nt], 1);
                    dot[nt] += __shfl_xor_sync(0xffffffffu, dot[nt], 2);
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        s[nt][c] = __shfl_sync(0xffffffffu, dot[nt], 8 * t + 4 * c) * cs[nt][c] * 5.9604644775390625e-8f;
                        const uint32_t col = col0 + nt * 8 + 2 * t + c;
                        // columns past the last one are zero queries: any weight will do
                        if (col < n_cols && j > col / a.r) s[nt][c] = -INFINITY;
                    }
                    raise(nt, s[nt][0], s[nt][1]);
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        s[nt][c] = s[nt][c] == -INFINITY ? 0.0f : ex2(s[nt][c] - ref[nt][c]);
                        if (g == 0) l[nt][c] += s[nt][c];
                        s[nt][c] *= unit_v;
                    }
                }
#pragma unroll
                for (int m = 0; m < C::MT; ++m)
#pragma unroll
                    for (int hi = 0; hi < 2; ++hi) {
                        const float v = to_f32(nv[dim_of(m, hi)]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            acc[m][nt][2 * hi] += s[nt][0] * v;
                            acc[m][nt][2 * hi + 1] += s[nt][1] * v;
                        }
                    }
            }
        };
        own_entries();

        // ---- the cached tiles ------------------------------------------------------
        // fragment row r (and k index r of the combine) is the tile's position
        // r / 2 + 4 (r % 2) in each half of eight: the lanes of a quad then read
        // consecutive rows
        const int pa = (g >> 1) + 4 * (g & 1), pb = pa + 8;
        for (; k < own && start + warp + k * CW < seg_end; ++k) {
            const uint32_t s = k % C::NST;
            if (!mbar_wait(&bar[s], (k / C::NST) & 1)) *err = 1;
            const unsigned char* st = ring + s * C::STAGE;
            const uint32_t pos0 = (start + warp + k * CW - u0) * TP;
            const uint32_t valid = rq.ctx > pos0 ? rq.ctx - pos0 : 0;
            if (valid > 0) {
                float sacc[NT][G][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int i = 0; i < G; ++i)
#pragma unroll
                        for (int c = 0; c < 4; ++c) sacc[nt][i][c] = 0.0f;
                const uint32_t* kw = reinterpret_cast<const uint32_t*>(st);
#pragma unroll
                for (int u = 0; u < C::SETS; ++u) {
                    const uint32_t wa = kw[pa * C::W + word_of(u)], wb = kw[pb * C::W + word_of(u)];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        const uint32_t f[4] = {nib<HALF>(wa, 2 * i), nib<HALF>(wb, 2 * i), nib<HALF>(wa, 2 * i + 1), nib<HALF>(wb, 2 * i + 1)};
#pragma unroll
                        for (int p = 0; p < QP; ++p)
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
                                mma<HALF>(sacc[nt][group_of(u)], f, qf[p][nt][u][2 * i], qf[p][nt][u][2 * i + 1]);
                    }
                }
                const T* ks = reinterpret_cast<const T*>(st + C::KS);
                const T* kz = reinterpret_cast<const T*>(st + C::KZ);
                const T* vs = reinterpret_cast<const T*>(st + C::VS);
                const T* vz = reinterpret_cast<const T*>(st + C::VZ);
                float p[NT][4];
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 4; ++c) p[nt][c] = 0.0f;
                float vsa[G], vsb[G], vza[G], vzb[G];
                float vtop = 0.0f;
#pragma unroll
                for (int i = 0; i < G; ++i) {
                    const float sa = to_f32(ks[pa * G + i]), sb = to_f32(ks[pb * G + i]);
                    float za = to_f32(kz[pa * G + i]), zb = to_f32(kz[pb * G + i]);
                    if (!HALF) {
                        za = fmaf(8.0f, sa, za);
                        zb = fmaf(8.0f, sb, zb);
                    }
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            p[nt][c] += sacc[nt][i][c] * sa * cs[nt][c] + za * qs[nt][c][i];
                            p[nt][2 + c] += sacc[nt][i][2 + c] * sb * cs[nt][c] + zb * qs[nt][c][i];
                        }
                    vsa[i] = to_f32(vs[pa * G + i]);
                    vsb[i] = to_f32(vs[pb * G + i]);
                    vza[i] = to_f32(vz[pa * G + i]);
                    vzb[i] = to_f32(vz[pb * G + i]);
                    if (!HALF) {                    // the codes' 8
                        vza[i] = fmaf(8.0f, vsa[i], vza[i]);
                        vzb[i] = fmaf(8.0f, vsb[i], vzb[i]);
                    }
                }
                if (valid < TP) {
                    // rows past the length may hold anything
                    const bool oa = (uint32_t)pa >= valid, obb = (uint32_t)pb >= valid;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            if (oa) p[nt][c] = -INFINITY;
                            if (obb) p[nt][2 + c] = -INFINITY;
                        }
#pragma unroll
                    for (int i = 0; i < G; ++i) {
                        if (oa) vsa[i] = vza[i] = 0.0f;
                        if (obb) vsb[i] = vzb[i] = 0.0f;
                    }
                }
                if (bad & (1u << s)) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int c = 0; c < 4; ++c) p[nt][c] = NAN;
                }
                bool over = false;
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 2; ++c) over |= fmaxf(p[nt][c], p[nt][2 + c]) - ref[nt][c] > RAISE;
                if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        float top[2];
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            top[c] = fmaxf(p[nt][c], p[nt][2 + c]);
#pragma unroll
                            for (int o = 4; o < 32; o <<= 1) top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], o));
                        }
                        raise(nt, top[0], top[1]);
                    }
                }
#pragma unroll
                for (int i = 0; i < G; ++i) vtop = fmaxf(vtop, fmaxf(fabsf(vsa[i]), fabsf(vsb[i])));
                const int ve = min((int)(__reduce_max_sync(0xffffffffu, __float_as_uint(vtop)) >> 23) - 126, VEXP1);
                if (ve > vexp) {                   // |vs| < 2^ve
                    const float f = pow2(vexp - ve);
                    vexp = ve;
#pragma unroll
                    for (int m = 0; m < C::MT; ++m)
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                            for (int c = 0; c < 4; ++c) acc[m][nt][c] *= f;
                }
                const float vinv = pow2(-vexp);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        p[nt][c] = ex2(p[nt][c] - ref[nt][c]);
                        p[nt][2 + c] = ex2(p[nt][2 + c] - ref[nt][c]);
                        l[nt][c] += p[nt][c] + p[nt][2 + c];
                    }
                uint32_t bf[G][NT][PP][2];
#pragma unroll
                for (int i = 0; i < G; ++i) {
                    const float sa = vsa[i] * vinv, sb = vsb[i] * vinv;
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                        for (int c = 0; c < 2; ++c) ob[nt][c][i] += p[nt][c] * vza[i] + p[nt][2 + c] * vzb[i];
                        uint32_t ha[PP], hb[PP];
                        parts_of<PP>(p[nt][0] * sa, p[nt][1] * sa, ha);
                        parts_of<PP>(p[nt][2] * sb, p[nt][3] * sb, hb);
#pragma unroll
                        for (int x = 0; x < PP; ++x) {
                            bf[i][nt][x][0] = movmatrix(ha[x]);
                            bf[i][nt][x][1] = movmatrix(hb[x]);
                        }
                    }
                }
                const uint32_t* vw = reinterpret_cast<const uint32_t*>(st + C::VW);
#pragma unroll
                for (int m4 = 0; m4 < C::MT / 4; ++m4) {
                    if constexpr (GROUP >= 64) {
                        uint32_t w[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) w[i] = vw[(t + 4 * i) * C::W + 8 * m4 + g];
                        const uint32_t lo01 = prmt(w[0], w[1], 0x5410), hi01 = prmt(w[0], w[1], 0x7632);
                        const uint32_t lo23 = prmt(w[2], w[3], 0x5410), hi23 = prmt(w[2], w[3], 0x7632);
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint32_t f[4] = {nib<HALF>(lo01, j), nib<HALF>(hi01, j), nib<HALF>(lo23, j), nib<HALF>(hi23, j)};
#pragma unroll
                            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                for (int x = 0; x < PP; ++x)
                                    mma<HALF>(acc[4 * m4 + j][nt], f, bf[m4 * 64 / GROUP][nt][x][0], bf[m4 * 64 / GROUP][nt][x][1]);
                        }
                    } else {
                        const uint32_t sel = g < 4 ? 0x5410 : 0x7632;
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            uint32_t w[4];
#pragma unroll
                            for (int i = 0; i < 4; ++i) w[i] = vw[(t + 4 * i) * C::W + 8 * m4 + 4 * q + (g & 3)];
                            const uint32_t w01 = prmt(w[0], w[1], sel), w23 = prmt(w[2], w[3], sel);
#pragma unroll
                            for (int j = 0; j < 2; ++j) {
                                const uint32_t f[4] = {nib<HALF>(w01, 2 * j), nib<HALF>(w01, 2 * j + 1), nib<HALF>(w23, 2 * j), nib<HALF>(w23, 2 * j + 1)};
#pragma unroll
                                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                                    for (int x = 0; x < PP; ++x)
                                        mma<HALF>(acc[4 * m4 + 2 * q + j][nt], f, bf[2 * m4 + q][nt][x][0], bf[2 * m4 + q][nt][x][1]);
                            }
                        }
                    }
                }
            }
            __syncwarp();
            fill(k + C::NST);
        }

        // ---- the warps' results of this part, joined ---------------------------------
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                const int col = nt * 8 + 2 * t + c;
                float bias[G], sum = l[nt][c];
#pragma unroll
                for (int o = 4; o < 32; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
#pragma unroll
                for (int i = 0; i < G; ++i) {
                    bias[i] = ob[nt][c][i];
#pragma unroll
                    for (int o = 4; o < 32; o <<= 1) bias[i] += __shfl_xor_sync(0xffffffffu, bias[i], o);
                }
                if (g == 0) {
                    comb_m[warp * COLS + col] = ref[nt][c];
                    comb_l[warp * COLS + col] = sum;
                }
#pragma unroll
                for (int m = 0; m < C::MT; ++m)
#pragma unroll
                    for (int hi = 0; hi < 2; ++hi) {
                        constexpr auto group_of_tile = [](int mm) { return GROUP >= 64 ? (mm >> 2) * 64 / GROUP : mm >> 1; };
                        comb[(warp * COLS + col) * C::LD + dim_of(m, hi)] =
                            acc[m][nt][2 * hi + c] * 16777216.0f * pow2(vexp) + bias[group_of_tile(m)];
                    }
            }
        __syncthreads();
        const bool whole = u0 >= start && u1 <= end;
        float* slot = reinterpret_cast<float*>(ws + split_bytes(gridDim.x)) +
                      (2 * (size_t)blockIdx.x + (u0 >= start ? 1 : 0)) * slot_floats(COLS, DH);
        const bool failed = *reinterpret_cast<volatile int*>(err) != 0;
        for (int i = tid; i < COLS * DH / 4; i += THREADS) {
            const int col = i / (DH / 4), d = i % (DH / 4) * 4;
            const uint32_t c = col0 + col;
            if (c >= n_cols) continue;
            float m = -INFINITY, sum = 0.0f;
#pragma unroll
            for (int w = 0; w < CW; ++w) m = fmaxf(m, comb_m[w * COLS + col]);
            float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int w = 0; w < CW; ++w) {
                const float f = ex2(comb_m[w * COLS + col] - m);
                const float4 x = *reinterpret_cast<const float4*>(&comb[(w * COLS + col) * C::LD + d]);
                sum += f * comb_l[w * COLS + col];
                o.x += f * x.x;
                o.y += f * x.y;
                o.z += f * x.z;
                o.w += f * x.w;
            }
            if (failed) o.x = o.y = o.z = o.w = NAN;
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
    pdl_launch_dependents();
}

template <typename T, int DH, int GROUP, int NT>
cudaError_t launch_few(const Attend& a, uint32_t most_new, uint32_t grid, void* ws, cudaStream_t stream) {
    using C = Cfg<T, DH, GROUP, NT>;
    const size_t smem = C::BEFORE + ((size_t)a.rows + 1) * 4;
    auto kernel = few_kernel<T, DH, GROUP, NT>;
    static std::atomic<uint64_t> done{0};
    cudaError_t e = allow_smem(kernel, C::BEFORE + (MAX_ROWS + 1) * 4, done);
    if (e != cudaSuccess) return e;
    kernel<<<grid, THREADS, smem, stream>>>(a, most_new, static_cast<unsigned char*>(ws));
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    return launch_join<T, DH, C::COLS>(a, grid, static_cast<const unsigned char*>(ws), stream);
}

}  // namespace few
}  // namespace paged
}  // namespace kvq
