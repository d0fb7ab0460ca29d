// The many-token paged attention (float16 steps).
#include "kvq_paged_attn.h"
#include "kvq_paged_many.cuh"

namespace kvq {
namespace paged {

cudaError_t launch_many_f16(const Attend& a, uint32_t least_new, bool vec, uint32_t grid, void* ws, cudaStream_t s) {
    switch (a.head_dim * 1000 + a.group) {
        case 64032: return many::launch_many<64, 32>(a, least_new, vec, grid, ws, s);
        case 64064: return many::launch_many<64, 64>(a, least_new, vec, grid, ws, s);
        case 128032: return many::launch_many<128, 32>(a, least_new, vec, grid, ws, s);
        case 128064: return many::launch_many<128, 64>(a, least_new, vec, grid, ws, s);
        case 128128: return many::launch_many<128, 128>(a, least_new, vec, grid, ws, s);
    }
    return cudaErrorInvalidValue;
}

}  // namespace paged
}  // namespace kvq
