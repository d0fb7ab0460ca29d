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

// us on a B200 below: 8 cache heads of 128, groups of 64, a captured call.
//
// A request is the few kernel's while its columns (new tokens x shared heads) fit
// two passes of 16, where the two are even. 32 requests of 8192 cached positions,
// R = 4, n new tokens each, few / many: n = 1 66 / 219, n = 4 116 / 221, n = 6
// 188 / 222, n = 8 216 / 224, n = 9 with a third pass 301 / 224; 32 of 1024, n = 8:
// 56 / 58, n = 9 63 / 58; one of 131072, n = 8: 119 / 117, n = 9 152 / 118. 31 of 8192
// with two tokens each beside a chunk of 512 over 8192: 173 / 353 with all of them units
// of the many kernel.
constexpr uint32_t FEW_COLS = 32;

// Columns per pass. Up to four are held once per block of a tile (4 columns: 66
// against 69 with 8, 32 x 8192). Two tiles of eight save a pass but leave room for
// 8 warps instead of 12: 16 columns 116 against 126 (32 x 8192, n = 4), 66 against 68
// (1 x 131072, R = 8, n = 2), 43 either way (32 x 8192 of 2 cache heads, R = 16), but 41
// against 38 (32 x 1024) and 20 against 15 (1 x 32768 of one cache head, R = 16), where a
// warp has few tiles. 24 columns are three passes of eight (188) or two of sixteen (208).
uint32_t columns(uint64_t cols, uint64_t row_tiles, uint64_t sms) {
    if (cols <= 4) return 4;
    const uint64_t p8 = (cols + 7) / 8, p16 = (cols + 15) / 16;
    return p8 == 2 * p16 && row_tiles * p8 > 20 * 12 * sms ? 16 : 8;
}

Choice choose(const Attend& a) {
    Choice c{};
    c.fits = true;
    const uint64_t cols = (uint64_t)a.max_new * a.r, sms = (uint64_t)sm_count();
    const uint64_t rows = a.rows < a.tokens ? a.rows : a.tokens;
    const uint64_t row_tiles = rows * a.n_kv_heads * ((uint64_t)a.max_ctx / 32 + 1);
    c.few_most = 0xFFFFFFFFu;
    if (a.dtype == KVQ_F32) {
        c.cols = 8;
    } else if (a.r > 128 || cols <= FEW_COLS) {
        c.cols = columns(cols, row_tiles, sms);
    } else {
        // one request: the many kernel alone (its bound is what it brings, but for a
        // padded batch), so that no second pair of launches finds nothing to do
        c.few_most = rows == 1 ? 0 : FEW_COLS / a.r;
        // (8 for R <= 8: against 4 they cost 31 single tokens of 8192 2 us of 169 and save as
        // many pairs 46 of 218, beside a chunk of 512 over 8192)
        c.cols = columns(a.r > 8 ? a.r : 8, row_tiles, sms);
        // units have at most 256 query rows; no CTA for less than two tiles (64 tokens
        // over 512: 21 us, as with one; with four 22, with eight 27)
        const uint64_t tu = 2 * (128 / a.r), units = (uint64_t)a.n_kv_heads * (a.tokens / tu + rows);
        const uint64_t tiles = units * (((uint64_t)a.max_ctx + a.max_new) / MANY_KEYS + 2 + MANY_UNIT);
        c.fits = tiles < TOO_MANY;
        c.many_grid = grid_for(tiles, 2, sms);
        const size_t es = 2;
        c.vec = true;
        for (const void* p : {a.q, a.new_k, a.new_v}) c.vec = c.vec && reinterpret_cast<uintptr_t>(p) % 16 == 0;
        for (uint64_t st : {a.q_token, a.q_head, a.k_token, a.k_head, a.v_token, a.v_head}) c.vec = c.vec && st * es % 16 == 0;
    }
    if (c.few_most) {
        // passes of a request, of all of them at most one each more than their tokens fill
        const uint64_t few = c.few_most < a.max_new ? c.few_most : a.max_new, w = c.cols;
        const uint64_t each = rows * ((few * a.r + w - 1) / w), all = (uint64_t)a.tokens * a.r / w + rows;
        const uint64_t tiles = (each < all ? each : all) * a.n_kv_heads * ((uint64_t)a.max_ctx / 32 + 1);
        c.fits = c.fits && tiles < TOO_MANY;
        // no CTA for less than a tile per warp (1 x 512: 11.7 us, with two per warp 13.3)
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
