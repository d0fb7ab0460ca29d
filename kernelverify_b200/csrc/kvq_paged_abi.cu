// C entry points of the paged 4-bit cache: every argument is checked here,
// before a kernel can index with it.
#include <math.h>

#include "kvq_paged.h"

namespace kvq {
namespace paged {
bool attend_fits(const Attend& a);
size_t attend_workspace(const Attend& a);
cudaError_t launch_attend(const Attend& a, void* workspace, cudaStream_t stream);
}  // namespace paged
}  // namespace kvq

namespace {

using kvq::api_device_ok;
using kvq::api_fail;
using namespace kvq::paged;

bool aligned(const void* p, size_t n) { return (reinterpret_cast<uintptr_t>(p) % n) == 0; }

int launched(cudaError_t e, const char* what) {
    if (e == cudaSuccess) return KVQ_OK;
    return api_fail(KVQ_ERR_LAUNCH, "%s: %s (%s)", what, cudaGetErrorName(e), cudaGetErrorString(e));
}

int page_shift_of(uint32_t page) {
    switch (page) {
        case 16: return 4;
        case 32: return 5;
        case 64: return 6;
        case 128: return 7;
    }
    return -1;
}

int check_page(uint32_t page) {
    if (page_shift_of(page) < 0) return api_fail(KVQ_ERR_INVALID, "page_size %u is not supported (16, 32, 64 or 128)", page);
    return KVQ_OK;
}

int check_cache(uint32_t head_dim, uint32_t group, uint32_t dtype, uint32_t pages, uint32_t page, uint32_t heads) {
    if (head_dim != 64 && head_dim != 128)
        return api_fail(KVQ_ERR_INVALID, "head_dim %u is not supported (64 or 128)", head_dim);
    if (group != 32 && group != 64 && group != 128)
        return api_fail(KVQ_ERR_INVALID, "group_size %u is not supported (32, 64 or 128)", group);
    if (head_dim % group) return api_fail(KVQ_ERR_INVALID, "group_size %u does not divide head_dim %u", group, head_dim);
    if (dtype != KVQ_F16 && dtype != KVQ_F32) return api_fail(KVQ_ERR_INVALID, "dtype %u is not KVQ_F16 or KVQ_F32", dtype);
    if (int rc = check_page(page)) return rc;
    if (pages == 0 || pages > 0x7FFFFFFFu) return api_fail(KVQ_ERR_INVALID, "a pool of %u pages: 1 to 2^31 - 1", pages);
    if (heads == 0 || heads > 32767) return api_fail(KVQ_ERR_INVALID, "%u cache heads: 1 to 32767", heads);
    if ((uint64_t)pages * heads * page > 0xFFFFFFFFull)
        return api_fail(KVQ_ERR_INVALID, "a pool of %u pages x %u heads x %u rows: at most 2^32 - 1 rows", pages, heads, page);
    return KVQ_OK;
}

int check_pool(const kvq_packed& p) {
    if (!p.words || !p.scales || !p.biases) return api_fail(KVQ_ERR_INVALID, "a pool pointer is NULL");
    if (!aligned(p.words, 16) || !aligned(p.scales, 16) || !aligned(p.biases, 16))
        return api_fail(KVQ_ERR_INVALID, "the pools must be 16-byte aligned");
    return KVQ_OK;
}

bool overlap(const void* a, size_t na, const void* b, size_t nb) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + nb && y < x + na;
}

int check_tables(const kvq_tables* a, bool build) {
    if (!a) return api_fail(KVQ_ERR_INVALID, "args is NULL");
    if (!a->lens || !a->step || !a->block_tables || !a->free_pages || !a->n_free || !a->lens_out || !a->n_free_out)
        return api_fail(KVQ_ERR_INVALID, "a required pointer is NULL");
    if (int rc = check_page(a->page_size)) return rc;
    if (a->rows == 0 || a->rows > MAX_ROWS) return api_fail(KVQ_ERR_INVALID, "%u rows: 1 to %u", a->rows, MAX_ROWS);
    if (a->pool == 0 || a->pool > 0x7FFFFFFFu) return api_fail(KVQ_ERR_INVALID, "a stack of %u pages: 1 to 2^31 - 1", a->pool);
    if (a->width == 0 || (uint64_t)a->width * a->page_size > 0x7FFFFFFFull || (uint64_t)a->width * a->rows > 0x7FFFFFFFull)
        return api_fail(KVQ_ERR_INVALID, "block tables of %u columns: positions and entries must stay below 2^31", a->width);
    const void* in4[] = {a->lens, a->step, a->block_tables, a->free_pages, a->n_free, a->lens_out, a->n_free_out,
                         a->cu_new, a->positions, a->status};
    for (const void* p : in4)
        if (p && !aligned(p, 4)) return api_fail(KVQ_ERR_INVALID, "a pointer is not 4-byte aligned");
    if (build) {
        if (!a->cu_new || !a->status || (a->max_tokens && (!a->slots || !a->positions)))
            return api_fail(KVQ_ERR_INVALID, "a required pointer is NULL");
        if (!aligned(a->slots, 8)) return api_fail(KVQ_ERR_INVALID, "slots must be 8-byte aligned");
        if (a->max_tokens > 0x7FFFFFFFu) return api_fail(KVQ_ERR_INVALID, "max_tokens %u above 2^31 - 1", a->max_tokens);
    }
    // Every CTA reads the lengths, the tables and the stack, and again for each token,
    // while others write: nothing that is written may lie over anything else.
    const size_t rb = 4ull * a->rows, tokens = build ? a->max_tokens : 0;
    const struct { const void* p; size_t n; bool written; } spans[] = {
        {a->lens, rb, false}, {a->step, rb, false}, {a->n_free, 4, false},
        {a->block_tables, rb * a->width, build}, {a->free_pages, 4ull * a->pool, !build},
        {a->lens_out, rb, true}, {a->n_free_out, 4, true}, {a->cu_new, build ? rb + 4 : 0, true},
        {a->status, build ? 4u : 0u, true}, {a->slots, 8 * tokens, true}, {a->positions, 4 * tokens, true}};
    constexpr int N = sizeof spans / sizeof *spans;
    for (int i = 0; i < N; ++i)
        for (int j = 0; j < i; ++j)
            if ((spans[i].written || spans[j].written) && spans[i].n && spans[j].n &&
                overlap(spans[i].p, spans[i].n, spans[j].p, spans[j].n))
                return api_fail(KVQ_ERR_INVALID, "an output overlaps an input or another output");
    return KVQ_OK;
}

Tables tables_of(const kvq_tables* a) {
    Tables t{};
    t.lens = a->lens;
    t.step = a->step;
    t.block_tables = a->block_tables;
    t.free_pages = a->free_pages;
    t.n_free = a->n_free;
    t.rows = a->rows;
    t.width = a->width;
    t.pool = a->pool;
    t.page_shift = (uint32_t)page_shift_of(a->page_size);
    t.max_tokens = a->max_tokens;
    t.cu_new = a->cu_new;
    t.slots = a->slots;
    t.positions = a->positions;
    t.lens_out = a->lens_out;
    t.n_free_out = a->n_free_out;
    t.status = a->status;
    return t;
}

int rows_of(const kvq_paged_rows* a, bool append, Rows* r) {
    if (!a) return api_fail(KVQ_ERR_INVALID, "args is NULL");
    if (int rc = check_cache(a->head_dim, a->group_size, a->dtype, a->pages, a->page_size, a->n_kv_heads)) return rc;
    if (int rc = check_pool(a->k)) return rc;
    if (int rc = check_pool(a->v)) return rc;
    if (a->tokens > 0x7FFFFFFFu) return api_fail(KVQ_ERR_INVALID, "%u tokens: at most 2^31 - 1", a->tokens);
    if (a->tokens && (!a->keys || !a->values || !a->slots)) return api_fail(KVQ_ERR_INVALID, "a required pointer is NULL");
    if (!aligned(a->slots, 8)) return api_fail(KVQ_ERR_INVALID, "slots must be 8-byte aligned");
    const size_t esz = a->dtype == KVQ_F16 ? 2 : 4;
    r->pool[0] = {const_cast<uint32_t*>(a->k.words), const_cast<void*>(a->k.scales), const_cast<void*>(a->k.biases)};
    r->pool[1] = {const_cast<uint32_t*>(a->v.words), const_cast<void*>(a->v.scales), const_cast<void*>(a->v.biases)};
    r->slots = a->slots;
    r->slots_end = (uint64_t)a->pages * a->page_size;
    r->tokens = a->tokens;
    r->heads = a->n_kv_heads;
    r->head_dim = a->head_dim;
    r->group = a->group_size;
    r->page_shift = (uint32_t)page_shift_of(a->page_size);
    r->dtype = (int)a->dtype;
    r->out_dtype = (int)a->out_dtype;
    if (append) {
        if (!aligned(a->keys, esz) || !aligned(a->values, esz))
            return api_fail(KVQ_ERR_INVALID, "keys and values must be %zu-byte aligned", esz);
        r->src[0] = a->keys;
        r->src[1] = a->values;
        const uint64_t st[4] = {a->k_token_stride, a->k_head_stride, a->v_token_stride, a->v_head_stride};
        r->vec = aligned(a->keys, 16) && aligned(a->values, 16);
        for (uint64_t s : st) r->vec = r->vec && s * esz % 16 == 0;
        r->token_stride[0] = st[0];
        r->head_stride[0] = st[1];
        r->token_stride[1] = st[2];
        r->head_stride[1] = st[3];
    } else {
        if (a->out_dtype != a->dtype && a->out_dtype != KVQ_F32)
            return api_fail(KVQ_ERR_INVALID, "out_dtype %u: the cache's dtype or KVQ_F32", a->out_dtype);
        if (!aligned(a->keys, 16) || !aligned(a->values, 16))
            return api_fail(KVQ_ERR_INVALID, "keys and values must be 16-byte aligned");
        r->dst[0] = const_cast<void*>(a->keys);
        r->dst[1] = const_cast<void*>(a->values);
    }
    return KVQ_OK;
}

// What the call writes may lie over nothing else of it: a row would hold a mixture of
// two, or be read after it was written.
int check_rows_apart(const kvq_paged_rows* a, bool append) {
    const size_t es = a->dtype == KVQ_F16 ? 2 : 4, oes = a->out_dtype == KVQ_F16 ? 2 : 4;
    const size_t held = (size_t)a->pages * a->n_kv_heads * a->page_size, words = held * a->head_dim / 2,
                 scales = held * (a->head_dim / a->group_size) * es;
    const auto rows = [&](uint64_t token, uint64_t head) -> size_t {
        if (!append) return (size_t)a->tokens * a->n_kv_heads * a->head_dim * oes;
        return ((a->tokens - 1) * token + (a->n_kv_heads - 1) * head + a->head_dim) * es;
    };
    const struct { const void* p; size_t n; bool written; } spans[] = {
        {a->k.words, words, append}, {a->k.scales, scales, append}, {a->k.biases, scales, append},
        {a->v.words, words, append}, {a->v.scales, scales, append}, {a->v.biases, scales, append},
        {a->keys, rows(a->k_token_stride, a->k_head_stride), !append},
        {a->values, rows(a->v_token_stride, a->v_head_stride), !append}, {a->slots, 8ull * a->tokens, false}};
    constexpr int N = sizeof spans / sizeof *spans;
    for (int i = 0; i < N; ++i)
        for (int j = 0; j < i; ++j)
            if ((spans[i].written || spans[j].written) && overlap(spans[i].p, spans[i].n, spans[j].p, spans[j].n))
                return api_fail(KVQ_ERR_INVALID, "an array that is written overlaps another one of the call");
    return KVQ_OK;
}

int attend_of(const kvq_paged_args* a, Attend* p) {
    if (!a) return api_fail(KVQ_ERR_INVALID, "args is NULL");
    if (int rc = check_cache(a->head_dim, a->group_size, a->dtype, a->pages, a->page_size, a->n_kv_heads)) return rc;
    if (int rc = check_pool(a->k)) return rc;
    if (int rc = check_pool(a->v)) return rc;
    if (!a->block_tables || !a->ctx_lens || !a->cu_new) return api_fail(KVQ_ERR_INVALID, "a required pointer is NULL");
    if (a->tokens && (!a->q || !a->new_k || !a->new_v)) return api_fail(KVQ_ERR_INVALID, "a required pointer is NULL");
    if (a->rows == 0 || a->rows > MAX_ROWS) return api_fail(KVQ_ERR_INVALID, "%u rows: 1 to %u", a->rows, MAX_ROWS);
    if (a->n_heads == 0 || a->n_heads % a->n_kv_heads)
        return api_fail(KVQ_ERR_INVALID, "n_heads %u is not a multiple of n_kv_heads %u", a->n_heads, a->n_kv_heads);
    if (a->n_heads > 65535) return api_fail(KVQ_ERR_INVALID, "%u query heads: at most 65535", a->n_heads);
    if (a->tokens > 0x7FFFFFFFu || a->max_new > 0x7FFFFFFFu || (uint64_t)a->tokens * a->n_heads > 0x7FFFFFFFull)
        return api_fail(KVQ_ERR_INVALID, "too many tokens: tokens * n_heads must stay below 2^31");
    if (a->max_ctx > (uint64_t)a->width * a->page_size)
        return api_fail(KVQ_ERR_INVALID, "max_ctx %u exceeds the block tables' %u pages of %u", a->max_ctx, a->width, a->page_size);
    if (a->max_ctx > 0x7FFFFFFFu - a->max_new) return api_fail(KVQ_ERR_INVALID, "positions must stay below 2^31");
    const size_t esz = a->dtype == KVQ_F16 ? 2 : 4;
    for (const void* x : {a->q, a->new_k, a->new_v})
        if (!aligned(x, esz)) return api_fail(KVQ_ERR_INVALID, "a tensor pointer is not %zu-byte aligned", esz);
    for (const void* x : {(const void*)a->block_tables, (const void*)a->ctx_lens, (const void*)a->cu_new})
        if (!aligned(x, 4)) return api_fail(KVQ_ERR_INVALID, "block_tables, ctx_lens and cu_new must be 4-byte aligned");
    p->q = a->q;
    p->new_k = a->new_k;
    p->new_v = a->new_v;
    p->k = {const_cast<uint32_t*>(a->k.words), const_cast<void*>(a->k.scales), const_cast<void*>(a->k.biases)};
    p->v = {const_cast<uint32_t*>(a->v.words), const_cast<void*>(a->v.scales), const_cast<void*>(a->v.biases)};
    p->block_tables = a->block_tables;
    p->ctx_lens = a->ctx_lens;
    p->cu_new = a->cu_new;
    p->q_token = a->q_token_stride;
    p->q_head = a->q_head_stride;
    p->k_token = a->k_token_stride;
    p->k_head = a->k_head_stride;
    p->v_token = a->v_token_stride;
    p->v_head = a->v_head_stride;
    p->rows = a->rows;
    p->tokens = a->tokens;
    p->n_heads = a->n_heads;
    p->n_kv_heads = a->n_kv_heads;
    p->r = a->n_heads / a->n_kv_heads;
    p->head_dim = a->head_dim;
    p->group = a->group_size;
    p->page_shift = (uint32_t)page_shift_of(a->page_size);
    p->pages = a->pages;
    p->width = a->width;
    p->max_ctx = a->max_ctx;
    p->max_new = a->max_new < a->tokens ? a->max_new : a->tokens;
    p->dtype = (int)a->dtype;
    p->scale = 1.0f / sqrtf((float)a->head_dim);
    if (!attend_fits(*p)) return api_fail(KVQ_ERR_INVALID, "max_ctx and max_new allow too many tiles for one step: lower them or split the batch");
    return KVQ_OK;
}

}  // namespace

extern "C" {

int kvq_paged_tables(const kvq_tables* a, void* stream) {
    if (int rc = check_tables(a, true)) return rc;
    if (int rc = api_device_ok()) return rc;
    return launched(launch_build_tables(tables_of(a), static_cast<cudaStream_t>(stream)), "block tables");
}

int kvq_paged_truncate(const kvq_tables* a, void* stream) {
    if (int rc = check_tables(a, false)) return rc;
    if (int rc = api_device_ok()) return rc;
    return launched(launch_truncate(tables_of(a), static_cast<cudaStream_t>(stream)), "truncate");
}

int kvq_paged_append(const kvq_paged_rows* a, void* stream) {
    Rows r{};
    if (int rc = rows_of(a, true, &r)) return rc;
    if (int rc = api_device_ok()) return rc;
    if (r.tokens == 0) return KVQ_OK;
    if (int rc = check_rows_apart(a, true)) return rc;
    return launched(launch_append(r, static_cast<cudaStream_t>(stream)), "paged append");
}

int kvq_paged_gather(const kvq_paged_rows* a, void* stream) {
    Rows r{};
    if (int rc = rows_of(a, false, &r)) return rc;
    if (int rc = api_device_ok()) return rc;
    if (r.tokens == 0) return KVQ_OK;
    if (int rc = check_rows_apart(a, false)) return rc;
    return launched(launch_gather(r, static_cast<cudaStream_t>(stream)), "paged gather");
}

size_t kvq_paged_workspace_bytes(const kvq_paged_args* a) {
    Attend p{};
    return attend_of(a, &p) ? 0 : attend_workspace(p);
}

int kvq_paged_attend(const kvq_paged_args* a, void* out, void* workspace, size_t workspace_bytes, void* stream) {
    Attend p{};
    if (int rc = attend_of(a, &p)) return rc;
    if (p.tokens && !out) return api_fail(KVQ_ERR_INVALID, "out is NULL");
    if (!aligned(out, 16)) return api_fail(KVQ_ERR_INVALID, "out must be 16-byte aligned");
    p.out = out;
    const size_t need = attend_workspace(p);
    if (need && (workspace == nullptr || workspace_bytes < need))
        return api_fail(KVQ_ERR_INVALID, "workspace of %zu bytes is smaller than the %zu this call needs", workspace_bytes, need);
    if (need && !aligned(workspace, 256)) return api_fail(KVQ_ERR_INVALID, "workspace is not 256-byte aligned");
    if (p.tokens) {
        // rows and parts are written while others are still read, the lengths and offsets
        // that the reads follow among them
        const size_t es = p.dtype == KVQ_F16 ? 2 : 4, n = (size_t)p.tokens * p.n_heads * p.head_dim * es;
        const auto span = [&](uint64_t token, uint64_t heads, uint64_t head) {
            return ((p.tokens - 1) * token + (heads - 1) * head + p.head_dim) * es;
        };
        const size_t held = ((size_t)p.pages * p.n_kv_heads << p.page_shift), words = held * p.head_dim / 2,
                     scales = held * (p.head_dim / p.group) * es;
        const struct { const void* p; size_t n; } ins[] = {
            {p.q, span(p.q_token, p.n_heads, p.q_head)}, {p.new_k, span(p.k_token, p.n_kv_heads, p.k_head)},
            {p.new_v, span(p.v_token, p.n_kv_heads, p.v_head)}, {p.k.words, words}, {p.k.scales, scales},
            {p.k.biases, scales}, {p.v.words, words}, {p.v.scales, scales}, {p.v.biases, scales},
            {p.block_tables, 4ull * p.rows * p.width}, {p.ctx_lens, 4ull * p.rows}, {p.cu_new, 4ull * p.rows + 4}};
        for (const auto& i : ins) {
            if (overlap(out, n, i.p, i.n)) return api_fail(KVQ_ERR_INVALID, "out overlaps an input");
            if (need && overlap(workspace, need, i.p, i.n)) return api_fail(KVQ_ERR_INVALID, "the workspace overlaps an input");
        }
        if (need && overlap(workspace, need, out, n)) return api_fail(KVQ_ERR_INVALID, "the workspace overlaps out");
    }
    if (int rc = api_device_ok()) return rc;
    if (p.tokens == 0 || p.max_new == 0) return KVQ_OK;
    return launched(launch_attend(p, workspace, static_cast<cudaStream_t>(stream)), "paged attention");
}

}  // extern "C"
