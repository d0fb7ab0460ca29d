// The few-token paged attention for float32 steps.
#include "kvq_paged_attn.h"
#include "kvq_paged_few.cuh"

namespace kvq {
namespace paged {

cudaError_t launch_few_f32(const Attend& a, uint32_t most_new, uint32_t grid, void* ws, cudaStream_t s) {
    switch (a.head_dim * 1000 + a.group) {
        case 64032: return few::launch_few<float, 64, 32, 1, false>(a, most_new, grid, ws, s);
        case 64064: return few::launch_few<float, 64, 64, 1, false>(a, most_new, grid, ws, s);
        case 128032: return few::launch_few<float, 128, 32, 1, false>(a, most_new, grid, ws, s);
        case 128064: return few::launch_few<float, 128, 64, 1, false>(a, most_new, grid, ws, s);
        case 128128: return few::launch_few<float, 128, 128, 1, false>(a, most_new, grid, ws, s);
    }
    return cudaErrorInvalidValue;
}

}  // namespace paged
}  // namespace kvq
