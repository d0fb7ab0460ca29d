// Launchers of the paged attention's kernels, one translation unit per element
// type; kvq_paged_attn.cu chooses among them.
#pragma once

#include "kvq_paged.h"

namespace kvq {
namespace paged {

// Requests with at most most_new new tokens, `cols` (4, 8 or 16; 8 for fp32)
// query columns per pass over the cache, on `grid` CTAs.
cudaError_t launch_few_f16(const Attend& a, uint32_t cols, uint32_t most_new, uint32_t grid, void* ws, cudaStream_t s);
cudaError_t launch_few_f32(const Attend& a, uint32_t most_new, uint32_t grid, void* ws, cudaStream_t s);

// Requests with at least least_new new tokens (at most 128 query heads per
// cache head); vec: every row of q, new_k and new_v is 16-byte aligned.
// MANY_UNIT: what a unit of its work counts besides its key tiles.
constexpr uint32_t MANY_COLS = 256, MANY_KEYS = 128, MANY_UNIT = 3;
cudaError_t launch_many_f16(const Attend& a, uint32_t least_new, bool vec, uint32_t grid, void* ws, cudaStream_t s);

}  // namespace paged
}  // namespace kvq
