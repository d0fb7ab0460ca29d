// The few-token paged attention for float16 steps.
#include "kvq_paged_attn.h"
#include "kvq_paged_few.cuh"

namespace kvq {
namespace paged {

template <int DH, int GROUP>
static cudaError_t go(const Attend& a, uint32_t cols, uint32_t most_new, uint32_t grid, void* ws, cudaStream_t s) {
    if (cols == 4) return few::launch_few<__half, DH, GROUP, 1, true>(a, most_new, grid, ws, s);
    if (cols == 8) return few::launch_few<__half, DH, GROUP, 1, false>(a, most_new, grid, ws, s);
    return few::launch_few<__half, DH, GROUP, 2, false>(a, most_new, grid, ws, s);
}

cudaError_t launch_few_f16(const Attend& a, uint32_t cols, uint32_t most_new, uint32_t grid, void* ws, cudaStream_t s) {
    switch (a.head_dim * 1000 + a.group) {
        case 64032: return go<64, 32>(a, cols, most_new, grid, ws, s);
        case 64064: return go<64, 64>(a, cols, most_new, grid, ws, s);
        case 128032: return go<128, 32>(a, cols, most_new, grid, ws, s);
        case 128064: return go<128, 64>(a, cols, most_new, grid, ws, s);
        case 128128: return go<128, 128>(a, cols, most_new, grid, ws, s);
    }
    return cudaErrorInvalidValue;
}

}  // namespace paged
}  // namespace kvq
