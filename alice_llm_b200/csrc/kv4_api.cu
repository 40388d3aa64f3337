// The alice_kv4_* entry points: handles, checks of arguments, what a step works on (csrc/kv4.cuh).
#include <algorithm>
#include <cmath>
#include <new>
#include <vector>

#include "abi_internal.cuh"
#include "kv4.cuh"
#include "kv4_plan.cuh"
#include "rows.cuh"

using namespace alice;

struct alice_kv4 {
    alice_engine* e;
    Kv4Shape shape;
    uint8_t* pool;
};

struct alice_kv4_batch {
    alice_engine* e;
    Kv4Shape shape;               // of the caches it serves; pages: of the one it was made for
    uint32_t group, max_seqs, max_tokens, max_pages, max_jobs;
    uint8_t* blob = nullptr;      // the arrays of `plan`
    float* part = nullptr;
    unsigned int* tickets = nullptr;
    Kv4Plan plan{};
    Kv4Head now{};                // what `set` gave last
};

#define CU(call)                                                        \
    do {                                                                \
        cudaError_t err__ = (call);                                     \
        if (err__ != cudaSuccess) return alice_cuda_fail(err__, #call); \
    } while (0)

namespace {

int check_rows(const char* who, const char* name, const alice_engine* e, const alice_buf* x, uint32_t tokens, size_t& ld, size_t dim) {
    if (!x) return alice_fail(ALICE_E_INVALID, "%s: %s is null", who, name);
    if (x->e != e) return alice_fail(ALICE_E_INVALID, "%s: %s belongs to another engine", who, name);
    if (ld == 0) ld = dim;
    if (ld < dim || ld % 4 || ld > ((size_t)1 << 40)) return alice_fail(ALICE_E_SHAPE, "%s: rows of %s are %zu floats apart; a multiple of 4 of at least %zu is wanted", who, name, ld, dim);
    if (!rows_fit(x->len, tokens, ld, dim)) return alice_fail(ALICE_E_SHAPE, "%s: %s holds %zu floats, less than %u rows of %zu that are %zu apart", who, name, x->len, tokens, dim, ld);
    return ALICE_OK;
}

// tokens that a buffer has rows for
uint32_t room(const alice_buf* x, size_t ld, size_t dim) { return x->len < dim ? 0 : (uint32_t)std::min<size_t>((x->len - dim) / ld + 1, 0xffffffffu); }

int check_rope(const char* who, const alice_engine* e, const alice_buf* table, uint32_t dims, uint32_t neox, uint32_t dim, uint32_t rows, Kv4Rope& out) {
    out = Kv4Rope{};
    if (!table) return dims ? alice_fail(ALICE_E_INVALID, "%s: %u rotated dims without a table", who, dims) : (int)ALICE_OK;
    if (table->e != e) return alice_fail(ALICE_E_INVALID, "%s: the rotation table belongs to another engine", who);
    if (dims == 0 || dims % 16 || dims > dim) return alice_fail(ALICE_E_SHAPE, "%s: %u rotated dims; a multiple of 16 up to %u is wanted", who, dims, dim);
    if (neox > 1) return alice_fail(ALICE_E_INVALID, "%s: neox is 0 or 1", who);
    if (table->len < (size_t)rows * dims) return alice_fail(ALICE_E_SHAPE, "%s: the rotation table has %zu rows, positions reach %u", who, table->len / dims, rows);
    out.table = table->p; out.dims = dims; out.neox = neox;
    out.rows = (uint32_t)std::min<size_t>(table->len / dims, 0xffffffffu);
    return ALICE_OK;
}

int check_pair(const char* who, const alice_engine* e, const alice_kv4* c, const alice_kv4_batch* b) {
    if (!e || !c || !b) return alice_fail(ALICE_E_INVALID, "%s: null argument", who);
    if (c->e != e || b->e != e) return alice_fail(ALICE_E_INVALID, "%s: cache or batch belongs to another engine", who);
    if (c->shape.page_tokens != b->shape.page_tokens || c->shape.kv_heads != b->shape.kv_heads || c->shape.dim != b->shape.dim)
        return alice_fail(ALICE_E_SHAPE, "%s: the batch was made for a cache of another shape", who);
    if (b->now.seqs && b->now.top_page >= c->shape.pages) return alice_fail(ALICE_E_SHAPE, "%s: the batch names page %u of %u", who, b->now.top_page, c->shape.pages);
    return ALICE_OK;
}

}  // namespace

extern "C" {

int32_t alice_kv4_create(alice_engine* e, uint32_t pages, uint32_t page_tokens, uint32_t kv_heads, uint32_t head_dim, alice_kv4** out) {
    const char* who = "alice_kv4_create";
    if (!e || !out) return alice_fail(ALICE_E_INVALID, "%s: null argument", who);
    *out = nullptr;
    const int rc = kv4_check_shape(who, pages, page_tokens, kv_heads, head_dim);
    if (rc) return rc;
    const Kv4Shape s{pages, page_tokens, kv_heads, head_dim};
    CU(cudaSetDevice(e->device));
    void* p = nullptr;
    CU(cudaMalloc(&p, s.bytes()));
    const cudaError_t err = cudaMemsetAsync(p, 0, s.bytes(), e->stream);
    auto* c = err == cudaSuccess ? new (std::nothrow) alice_kv4{e, s, static_cast<uint8_t*>(p)} : nullptr;
    if (!c) {
        cudaFree(p);
        return err != cudaSuccess ? alice_cuda_fail(err, who) : alice_fail(ALICE_E_NOMEM, "%s: host allocation failed", who);
    }
    alice_engine_retain(e);
    *out = c;
    return ALICE_OK;
}

int32_t alice_kv4_free(alice_kv4* c) {
    if (!c) return ALICE_OK;
    alice_quiesce(c->e);
    cudaFree(c->pool);
    alice_engine_release(c->e);
    delete c;
    return ALICE_OK;
}

int32_t alice_kv4_batch_create(alice_engine* e, const alice_kv4* cache, uint32_t heads, uint32_t max_seqs, uint32_t max_tokens, uint32_t max_pages,
                               alice_kv4_batch** out) {
    const char* who = "alice_kv4_batch_create";
    if (!e || !cache || !out) return alice_fail(ALICE_E_INVALID, "%s: null argument", who);
    *out = nullptr;
    if (cache->e != e) return alice_fail(ALICE_E_INVALID, "%s: the cache belongs to another engine", who);
    const Kv4Shape& s = cache->shape;
    const int rc = kv4_check_limits(who, s.kv_heads, s.dim, heads, max_seqs, max_tokens, max_pages);
    if (rc) return rc;
    auto* b = new (std::nothrow) alice_kv4_batch{};
    if (!b) return alice_fail(ALICE_E_NOMEM, "%s: host allocation failed", who);
    b->e = e; b->shape = s; b->group = heads / s.kv_heads;
    b->max_seqs = max_seqs; b->max_tokens = max_tokens; b->max_pages = max_pages;
    b->max_jobs = kv4_max_jobs(max_seqs, max_tokens, b->group, s.dim);
    alice_engine_retain(e);
    size_t at = 0;
    auto take = [&](size_t words) { const size_t o = at; at += (words * 4 + 15) & ~size_t(15); return o; };
    const size_t o_job = take((size_t)b->max_jobs * (sizeof(Kv4Job) / 4)), o_head = take(sizeof(Kv4Head) / 4), o_jtile = take(b->max_jobs), o_token = take((size_t)max_tokens * 4),
                 o_table = take((size_t)max_seqs * max_pages);
    cudaError_t err = cudaSetDevice(e->device);
    if (err == cudaSuccess) err = cudaMalloc(reinterpret_cast<void**>(&b->blob), at);
    if (err == cudaSuccess) err = cudaMalloc(reinterpret_cast<void**>(&b->part), kv4_part_floats(s.dim, e->num_sms) * sizeof(float));
    if (err == cudaSuccess) err = cudaMalloc(reinterpret_cast<void**>(&b->tickets), (size_t)e->num_sms * sizeof(unsigned int));
    if (err == cudaSuccess) err = cudaMemsetAsync(b->blob, 0, at, e->stream);
    if (err == cudaSuccess) err = cudaMemsetAsync(b->tickets, 0, (size_t)e->num_sms * sizeof(unsigned int), e->stream);
    if (err != cudaSuccess) { alice_kv4_batch_free(b); return alice_cuda_fail(err, who); }
    auto u32 = [&](size_t o) { return reinterpret_cast<const uint32_t*>(b->blob + o); };
    b->plan.head = reinterpret_cast<const Kv4Head*>(b->blob + o_head);
    b->plan.token = reinterpret_cast<const Kv4Token*>(b->blob + o_token);
    b->plan.job = reinterpret_cast<const Kv4Job*>(b->blob + o_job); b->plan.job_tile = u32(o_jtile);
    b->plan.table = u32(o_table); b->plan.table_ld = max_pages;
    *out = b;
    return ALICE_OK;
}

int32_t alice_kv4_batch_free(alice_kv4_batch* b) {
    if (!b) return ALICE_OK;
    alice_quiesce(b->e);
    cudaFree(b->blob);
    cudaFree(b->part);
    cudaFree(b->tickets);
    alice_engine_release(b->e);
    delete b;
    return ALICE_OK;
}

int32_t alice_kv4_batch_check(uint32_t pages, uint32_t page_tokens, uint32_t max_seqs, uint32_t max_tokens, uint32_t max_pages, uint32_t seqs, const uint32_t* past,
                              const uint32_t* tokens, const uint32_t* tables, uint32_t table_ld) {
    try {
        return kv4_check_batch("alice_kv4_batch_check", pages, page_tokens, max_seqs, max_tokens, max_pages, seqs, past, tokens, tables, table_ld);
    } catch (const std::exception&) {
        return alice_fail(ALICE_E_NOMEM, "alice_kv4_batch_check: host allocation failed");
    }
}

int32_t alice_kv4_batch_set(alice_kv4_batch* b, uint32_t seqs, const uint32_t* past, const uint32_t* tokens, const uint32_t* tables, uint32_t table_ld) {
    const char* who = "alice_kv4_batch_set";
    if (!b) return alice_fail(ALICE_E_INVALID, "%s: null batch", who);
    try {
        const int rc = kv4_check_batch(who, b->shape.pages, b->shape.page_tokens, b->max_seqs, b->max_tokens, b->max_pages, seqs, past, tokens, tables, table_ld);
        if (rc) return rc;
        if (b->e->dead) return alice_fail(ALICE_E_INVALID, "%s: the engine is gone", who);
        CU(cudaSetDevice(b->e->device));
        cudaStream_t st = b->e->stream;
        cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
        CU(cudaStreamIsCapturing(st, &capturing));
        if (capturing != cudaStreamCaptureStatusNone) return alice_cuda_fail(cudaErrorStreamCaptureUnsupported, "alice_kv4_batch_set: lengths and pages of a captured stream");
        Kv4HostPlan h;
        const bool fits = kv4_make_plan(h, b->shape.dim, b->shape.kv_heads, b->shape.page_tokens, b->group, seqs, past, tokens, tables, table_ld, b->max_pages);
        if (!fits || (uint64_t)h.head.tiles * b->shape.kv_heads > 0x7fffffffull)     // tiles of all heads are numbered in 32 bits
            return alice_fail(ALICE_E_SHAPE, "%s: too many tokens over too many positions for one step", who);
        // copies from pageable memory: the vectors have been read when a call returns
        auto up = [&](const auto* dst, const auto& src) -> cudaError_t {
            return src.empty() ? cudaSuccess : cudaMemcpyAsync(const_cast<void*>(static_cast<const void*>(dst)), src.data(), src.size() * sizeof(src[0]), cudaMemcpyHostToDevice, st);
        };
        CU(up(b->plan.job, h.job)); CU(up(b->plan.job_tile, h.job_tile));
        CU(up(b->plan.token, h.token)); CU(up(b->plan.table, h.table));
        CU(cudaMemcpyAsync(const_cast<Kv4Head*>(b->plan.head), &h.head, sizeof(Kv4Head), cudaMemcpyHostToDevice, st));
        b->now = h.head;
    } catch (const std::exception&) {
        return alice_fail(ALICE_E_NOMEM, "%s: host allocation failed", who);
    }
    return ALICE_OK;
}

static int rows_call(const char* who, alice_engine* e, const alice_kv4* c, const alice_kv4_batch* b, const alice_buf* k, size_t k_ld, const alice_buf* v, size_t v_ld,
                     Kv4RowsArgs& a) {
    int rc = check_pair(who, e, c, b);
    if (rc) return rc;
    const size_t dim = (size_t)c->shape.kv_heads * c->shape.dim;
    if ((rc = check_rows(who, "k", e, k, b->now.tokens, k_ld, dim))) return rc;
    if ((rc = check_rows(who, "v", e, v, b->now.tokens, v_ld, dim))) return rc;
    a.plan = b->plan; a.shape = c->shape; a.pool = c->pool; a.k = k->p; a.v = v->p; a.k_ld = k_ld; a.v_ld = v_ld;
    a.most_tokens = std::min(room(k, k_ld, dim), room(v, v_ld, dim)); a.status = e->status;
    CU(cudaSetDevice(e->device));
    return ALICE_OK;
}

int32_t alice_kv4_append(alice_engine* e, alice_kv4* c, const alice_kv4_batch* b, const alice_buf* k, size_t k_stride, const alice_buf* v, size_t v_stride,
                         const alice_buf* rope, uint32_t rot_dims, uint32_t neox) {
    const char* who = "alice_kv4_append";
    Kv4RowsArgs a{};
    int rc = rows_call(who, e, c, b, k, k_stride, v, v_stride, a);
    if (!rc) rc = check_rope(who, e, rope, rot_dims, neox, c->shape.dim, b->now.end, a.rope);
    if (rc) return rc;
    CU(launch_kv4_append(a, b->now.tokens, e->num_sms, e->stream, e->pdl));
    return ALICE_OK;
}

int32_t alice_kv4_read(alice_engine* e, const alice_kv4* c, const alice_kv4_batch* b, alice_buf* k, size_t k_stride, alice_buf* v, size_t v_stride) {
    const char* who = "alice_kv4_read";
    Kv4RowsArgs a{};
    const int rc = rows_call(who, e, c, b, k, k_stride, v, v_stride, a);
    if (rc) return rc;
    const size_t dim = (size_t)c->shape.kv_heads * c->shape.dim;
    // side by side in one buffer is fine; the same floats for both are not, nor at a replay with more tokens
    a.most_tokens = (uint32_t)rows_apart(a.k, a.k_ld, dim, a.v, a.v_ld, dim, a.most_tokens);
    if (k->p == v->p || a.most_tokens < b->now.tokens) return alice_fail(ALICE_E_INVALID, "%s: k and v share memory", who);
    CU(launch_kv4_read(a, b->now.tokens, e->num_sms, e->stream, e->pdl));
    return ALICE_OK;
}

int32_t alice_kv4_attention(alice_engine* e, const alice_kv4* c, const alice_kv4_batch* b, const alice_buf* q, size_t q_stride, alice_buf* out, size_t out_stride,
                            const alice_buf* rope, uint32_t rot_dims, uint32_t neox, float scale) {
    const char* who = "alice_kv4_attention";
    int rc = check_pair(who, e, c, b);
    if (rc) return rc;
    Kv4AttnArgs a{};
    const size_t dim = (size_t)c->shape.kv_heads * b->group * c->shape.dim;
    if ((rc = check_rows(who, "q", e, q, b->now.tokens, q_stride, dim))) return rc;
    if ((rc = check_rows(who, "out", e, out, b->now.tokens, out_stride, dim))) return rc;
    if ((rc = check_rope(who, e, rope, rot_dims, neox, c->shape.dim, b->now.end, a.rope))) return rc;
    if (!std::isfinite(scale)) return alice_fail(ALICE_E_INVALID, "%s: scale is not finite", who);
    // a query is read by several CTAs, at any time before the last of its output is there; a replay may have more tokens
    a.most_tokens = (uint32_t)rows_apart(q->p, q_stride, dim, out->p, out_stride, dim, std::min(room(q, q_stride, dim), room(out, out_stride, dim)));
    if (q->p == out->p || a.most_tokens < b->now.tokens) return alice_fail(ALICE_E_INVALID, "%s: q and out share memory", who);
    CU(cudaSetDevice(e->device));
    a.plan = b->plan; a.shape = c->shape; a.pool = c->pool; a.q = q->p; a.out = out->p; a.q_ld = q_stride; a.out_ld = out_stride;
    a.group = b->group; a.scale = scale; a.part = b->part; a.tickets = b->tickets; a.status = e->status;
    a.rows = b->now.prompt_jobs && !b->now.jobs ? 0 : std::max(b->now.rows, 4u);      // a capture of an empty batch is one of single tokens
    a.prompt_jobs = b->now.prompt_jobs; a.end = b->now.end;
    if (a.prompt_jobs) {      // a captured call meets longer sequences
        cudaStreamCaptureStatus capturing = cudaStreamCaptureStatusNone;
        CU(cudaStreamIsCapturing(e->stream, &capturing));
        if (capturing != cudaStreamCaptureStatusNone) a.end = (uint32_t)std::min<uint64_t>((uint64_t)b->max_pages * b->shape.page_tokens, 0x7fffffffu);
    }
    CU(launch_kv4_attention(a, e->num_sms, e->stream, e->pdl));
    return ALICE_OK;
}

}  // extern "C"
