// Internal launchers of the paged 4-bit cache (block tables, append, gather,
// attention); the C entry points in kvq_paged_abi.cu validate and dispatch to
// them. And the error and device checks they share with kvq_abi.cu.
#pragma once

#include <cuda_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "kvq_b200.h"

namespace kvq {

// The calling thread's last error, set from a printf format; returns `code`.
int api_fail(int code, const char* fmt, ...);
// KVQ_OK when the current device is an sm_100.
int api_device_ok();

namespace paged {

// Rows of a batch: each CTA of the tables and attention kernels scans the
// whole batch's lengths into shared memory (4 bytes a row, twice).
constexpr uint32_t MAX_ROWS = 4096;

// One packed half of the cache: words [pages, HKV, page, DH/8], scales and
// biases [pages, HKV, page, DH/GROUP].
struct Pool {
    uint32_t* words;
    void* scales;
    void* biases;
};

struct Tables {
    const int32_t* lens;
    const int32_t* step;       // new tokens (build) or the length to keep (truncate)
    int32_t* block_tables;     // [rows, width]
    int32_t* free_pages;       // [pool]
    const int32_t* n_free;
    uint32_t rows, width, pool, page_shift, max_tokens;
    int32_t* cu_new;
    int64_t* slots;
    int32_t* positions;
    int32_t* lens_out;
    int32_t* n_free_out;
    int32_t* status;
};
cudaError_t launch_build_tables(const Tables& t, cudaStream_t stream);
cudaError_t launch_truncate(const Tables& t, cudaStream_t stream);

// Rows by slot: keys / values [tokens, HKV, DH] on one side, the pools on the
// other. Strides in elements; the pool has `slots_end` slots.
struct Rows {
    const void* src[2];        // append: keys, values
    uint64_t token_stride[2], head_stride[2];
    Pool pool[2];
    void* dst[2];              // gather: keys, values (contiguous)
    const int64_t* slots;
    uint64_t slots_end;
    uint32_t tokens, heads, head_dim, group, page_shift;
    int dtype, out_dtype;
    bool vec;                  // source rows are 16-byte aligned
};
cudaError_t launch_append(const Rows& r, cudaStream_t stream);
cudaError_t launch_gather(const Rows& r, cudaStream_t stream);

// One attention step over the pages (kvq_paged_args, checked).
struct Attend {
    const void* q;
    const void* new_k;
    const void* new_v;
    void* out;
    Pool k, v;
    const int32_t* block_tables;
    const int32_t* ctx_lens;
    const int32_t* cu_new;
    uint64_t q_token, q_head, k_token, k_head, v_token, v_head;   // element strides
    uint32_t rows, tokens, n_heads, n_kv_heads, r, head_dim, group;
    uint32_t page_shift, pages, width, max_ctx, max_new;
    int dtype;
    float scale;
};

}  // namespace paged
}  // namespace kvq
