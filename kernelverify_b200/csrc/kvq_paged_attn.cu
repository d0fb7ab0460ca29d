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
    int nt;              // few: column tiles of 8
    uint32_t cols, grid;
};

Choice choose(const Attend& a) {
    Choice c{};
    const uint64_t cols = (uint64_t)a.max_new * a.r;
    c.nt = a.dtype == KVQ_F16 && cols > 8 ? 2 : 1;
    c.cols = 8u * c.nt;
    const uint64_t per_sm = a.dtype == KVQ_F16 && c.nt == 1 ? 2 : 1;
    // tiles the step can have at most: no CTA for less than a round of eight
    const uint64_t tokens = a.tokens, ct = (cols + c.cols - 1) / c.cols;
    const uint64_t units = (uint64_t)(a.rows < tokens ? a.rows : tokens) * a.n_kv_heads * ct;
    const uint64_t tiles = units * ((uint64_t)a.max_ctx / 16 + 1);
    uint64_t grid = per_sm * (uint64_t)sm_count();
    if (grid > (tiles + 7) / 8) grid = (tiles + 7) / 8;
    c.grid = (uint32_t)(grid < 1 ? 1 : grid);
    return c;
}

}  // namespace

size_t attend_workspace(const Attend& a) {
    if (a.tokens == 0 || a.max_new == 0) return 0;
    const Choice c = choose(a);
    return split_bytes(c.grid) + 2 * (size_t)c.grid * slot_floats(c.cols, a.head_dim) * sizeof(float);
}

cudaError_t launch_attend(const Attend& a, void* ws, cudaStream_t s) {
    const Choice c = choose(a);
    if (a.dtype == KVQ_F16) return launch_few_f16(a, c.nt, 0xFFFFFFFFu, c.grid, ws, s);
    return launch_few_f32(a, 0xFFFFFFFFu, c.grid, ws, s);
}

}  // namespace paged
}  // namespace kvq
