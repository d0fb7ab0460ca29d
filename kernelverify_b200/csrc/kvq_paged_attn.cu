// Which kernel serves a step's requests, on how many CTAs, and the workspace
// they need. Decided from the sizes the host knows (types, heads and the bounds
// on lengths), never from lengths on the device, so a captured step keeps its
// launches.
#include "kvq_launch.h"
#include "kvq_paged_attn.h"
#include "kvq_paged_work.cuh"

namespace kvq {
namespace paged {

namespace {

struct Choice {
    uint32_t few_most;       // new tokens of a request up to which the few kernel takes it (0: none)
    uint32_t cols;           // its query columns per pass
    uint32_t few_grid, many_grid;
    bool vec;
    bool fits;               // the tiles can be counted in 31 bits
};

uint32_t grid_for(uint64_t tiles, uint64_t least, uint64_t most) {
    const uint64_t n = (tiles + least - 1) / least;
    return (uint32_t)(n < 1 ? 1 : (n > most ? most : n));
}

Choice choose(const Attend& a) {
    Choice c{};
    c.fits = true;
    const uint64_t cols = (uint64_t)a.max_new * a.r, sms = (uint64_t)sm_count();
    const uint64_t rows = a.rows < a.tokens ? a.rows : a.tokens;
    c.few_most = 0xFFFFFFFFu;
    c.cols = a.dtype == KVQ_F32 ? 8 : cols <= 4 ? 4 : cols <= 8 ? 8 : 16;
    if (a.dtype == KVQ_F16 && a.r <= 128 && cols > 16) {
        // one request: the many kernel alone, whatever it brings
        c.cols = a.r <= 4 ? 4 : 8;
        c.few_most = a.rows == 1 ? 0 : (a.r >= c.cols ? 1 : c.cols / a.r);
        // units have at most 256 query rows
        const uint64_t tu = 2 * (128 / a.r), units = (uint64_t)a.n_kv_heads * (a.tokens / tu + rows);
        const uint64_t tiles = units * (((uint64_t)a.max_ctx + a.max_new) / MANY_KEYS + 2);
        c.fits = tiles < TOO_MANY;
        c.many_grid = grid_for(tiles, 4, sms);
        const size_t es = 2;
        c.vec = true;
        for (const void* p : {a.q, a.new_k, a.new_v}) c.vec = c.vec && reinterpret_cast<uintptr_t>(p) % 16 == 0;
        for (uint64_t st : {a.q_token, a.q_head, a.k_token, a.k_head, a.v_token, a.v_head}) c.vec = c.vec && st * es % 16 == 0;
    }
    if (c.few_most) {
        // no CTA for less than a tile per warp
        const uint64_t few = c.few_most < a.max_new ? c.few_most : a.max_new, w = c.cols;
        const uint64_t tiles = rows * a.n_kv_heads * ((few * a.r + w - 1) / w) * ((uint64_t)a.max_ctx / 32 + 1);
        c.fits = c.fits && tiles < TOO_MANY;
        c.few_grid = grid_for(tiles, a.dtype == KVQ_F16 && c.cols <= 8 ? 12 : 8, sms);
    }
    return c;
}

size_t few_bytes(const Attend& a, const Choice& c) {
    if (!c.few_most) return 0;
    return (split_bytes(c.few_grid) + 2 * (size_t)c.few_grid * slot_floats(c.cols, a.head_dim) * sizeof(float) + 255) / 256 * 256;
}
size_t many_bytes(const Attend& a, const Choice& c) {
    if (!c.many_grid) return 0;
    return split_bytes(c.many_grid) + 2 * (size_t)c.many_grid * slot_floats(MANY_COLS, a.head_dim) * sizeof(float);
}

}  // namespace

bool attend_fits(const Attend& a) { return a.tokens == 0 || a.max_new == 0 || choose(a).fits; }

size_t attend_workspace(const Attend& a) {
    if (a.tokens == 0 || a.max_new == 0) return 0;
    const Choice c = choose(a);
    return few_bytes(a, c) + many_bytes(a, c);
}

cudaError_t launch_attend(const Attend& a, void* ws, cudaStream_t s) {
    const Choice c = choose(a);
    if (c.many_grid) {
        const cudaError_t e = launch_many_f16(a, c.few_most + 1, c.vec, c.many_grid,
                                              static_cast<unsigned char*>(ws) + few_bytes(a, c), s);
        if (e != cudaSuccess) return e;
    }
    if (!c.few_most) return cudaSuccess;
    if (a.dtype == KVQ_F16) return launch_few_f16(a, c.cols, c.few_most, c.few_grid, ws, s);
    return launch_few_f32(a, c.few_most, c.few_grid, ws, s);
}

}  // namespace paged
}  // namespace kvq
