// Entry points of the paged KV-cache operators (include/gfd_b200.h): argument checks,
// device-memory checks and launches.

#include <cstring>
#include <new>

#include "internal.h"
#include "kv.h"

using namespace gfdb;

namespace {

struct Region {
    const void* p;
    uint64_t bytes;
    const char* what;
};

// Every region lies in device memory of the context's GPU (regions of no bytes pass).  The driver
// is asked once per allocation and call: arrays of one allocation follow one another often.
int check_regions(gfd_ctx* ctx, const char* call, const Region* r, int n) {
    uint64_t lo[16], hi[16];
    int known = 0;
    for (int i = 0; i < n; ++i) {
        const uint64_t a = reinterpret_cast<uint64_t>(r[i].p), b = a + r[i].bytes;
        if (r[i].p == nullptr || r[i].bytes == 0) continue;
        bool in = false;
        for (int k = 0; k < known && !in; ++k) in = a >= lo[k] && b <= hi[k] && b > a;
        if (in) continue;
        if (!check_dev(ctx, a, r[i].bytes))
            return set_error(ctx, GFD_ERR_INVALID, "%s: %s is not inside one device allocation of GPU %d", call, r[i].what, ctx->device);
        const Range* range = ctx->dev_ranges.find(a, r[i].bytes);
        if (range != nullptr && known < 16) {
            lo[known] = range->lo;
            hi[known++] = range->hi;
        }
    }
    return GFD_OK;
}

KvCacheView view(const gfd_kv_cache& c) {
    KvCacheView v;
    v.k = static_cast<const char*>(c.k);
    v.v = static_cast<const char*>(c.v);
    v.block_stride = c.blocks > 1 ? 2 * c.block_stride : 0;
    v.token_stride = 2 * c.token_stride;
    v.head_stride = c.heads > 1 ? 2 * c.head_stride : 0;
    v.blocks = static_cast<int32_t>(c.blocks);
    v.block_tokens = c.block_tokens;
    v.heads = c.heads;
    return v;
}

KvBatchView view(const gfd_kv_batch& b, const gfd_kv_cache& c) {
    KvBatchView v;
    v.row_start = b.row_start;
    v.kv_len = b.kv_len;
    v.table = b.table;
    v.table_stride = b.table_stride;
    v.capacity = static_cast<int64_t>(b.table_width) * c.block_tokens;
    v.rows = static_cast<int32_t>(b.rows);
    v.seqs = b.seqs;
    v.table_width = b.table_width;
    return v;
}

KvRowsView view(const gfd_kv_rows& r, int64_t rows, int64_t heads, int elt) {
    return KvRowsView{static_cast<char*>(r.data), rows > 1 ? r.row_stride * elt : 0, heads > 1 ? r.head_stride * elt : 0};
}

KvPlan plan_attend(const gfd_ctx* ctx, const gfd_kv_cache& c, const gfd_kv_batch& b, const gfd_kv_attend_args& a, int64_t shared_len) {
    return kv_plan(c, b, a, shared_len, kv_decode_workers(ctx->num_sms, c.head_dim), kv_prompt_ctas(ctx->num_sms));
}

int append(gfd_ctx* ctx, const gfd_kv_cache* c, const gfd_kv_batch* b, const gfd_kv_append_args* a, void* stream) {
    if (c == nullptr || b == nullptr || a == nullptr) return set_error(ctx, GFD_ERR_INVALID, "kv_append: NULL argument");
    uint64_t cache_bytes = 0, kb = 0, vb = 0, qb = 0, qob = 0;
    const char* why = kv_check_cache(*c, true, &cache_bytes);
    if (!why) why = kv_check_batch(*b, *c, 0);
    if (!why) why = kv_check_append(*a, *c);
    const bool empty = b->rows == 0 || b->seqs == 0;
    if (!why && !empty) why = kv_check_rows(a->k, b->rows, c->heads, c->head_dim, c->dtype, false, &kb);
    if (!why && !empty) why = kv_check_rows(a->v, b->rows, c->heads, c->head_dim, c->dtype, false, &vb);
    if (!why && !empty && a->q_heads > 0) {
        why = kv_check_rows(a->q, b->rows, a->q_heads, c->head_dim, c->dtype, false, &qb);
        if (!why) why = kv_check_rows(a->q_out, b->rows, a->q_heads, c->head_dim, c->dtype, true, &qob);
    }
    if (why) return set_error(ctx, GFD_ERR_INVALID, "kv_append: %s", why);
    if (empty) return GFD_OK;
    const Region regions[] = {{c->k, cache_bytes, "the cache's K"},
                              {c->v, cache_bytes, "the cache's V"},
                              {a->k.data, kb, "k"},
                              {a->v.data, vb, "v"},
                              {a->q.data, qb, "q"},
                              {a->q_out.data, qob, "q_out"},
                              {b->row_start, (static_cast<uint64_t>(b->seqs) + 1) * 4, "row_start"},
                              {b->kv_len, static_cast<uint64_t>(b->seqs) * 4, "kv_len"},
                              {b->table, kv_table_bytes(*b), "table"},
                              {a->inv_freq, static_cast<uint64_t>(a->rot_dim) * 2, "inv_freq"},
                              {a->positions, static_cast<uint64_t>(b->rows) * 4, "positions"},
                              {a->status, 4, "status"}};
    const int rc = check_regions(ctx, "kv_append", regions, static_cast<int>(sizeof(regions) / sizeof(regions[0])));
    if (rc != GFD_OK) return rc;
    KvAppendParams p;
    std::memset(&p, 0, sizeof(p));
    p.cache = view(*c);
    p.batch = view(*b, *c);
    p.k = view(a->k, b->rows, c->heads, 2);
    p.v = view(a->v, b->rows, c->heads, 2);
    if (a->q_heads > 0) {
        p.q = view(a->q, b->rows, a->q_heads, 2);
        p.q_out = view(a->q_out, b->rows, a->q_heads, 2);
    }
    p.inv_freq = a->inv_freq;
    p.positions = a->positions;
    p.status = a->status;
    p.q_heads = a->q_heads;
    p.rot_dim = a->rot_dim;
    p.interleaved = a->interleaved != 0;
    cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
    const cudaError_t e = launch_kv_append(p, c->head_dim, c->dtype, ctx->num_sms, st);
    return e == cudaSuccess ? GFD_OK : cuda_error(ctx, e, "kv_append: kernel launch");
}

int attend(gfd_ctx* ctx, const char* call, const gfd_kv_cache* c, const gfd_kv_batch* b, const int32_t* shared_table,
           int64_t shared_len, const gfd_kv_attend_args* a, void* stream) {
    if (c == nullptr || b == nullptr || a == nullptr) return set_error(ctx, GFD_ERR_INVALID, "%s: NULL argument", call);
    uint64_t cache_bytes = 0, qb = 0, ob = 0;
    const char* why = kv_check_cache(*c, false, &cache_bytes);
    if (!why) why = kv_check_batch(*b, *c, shared_len);
    if (!why) why = kv_check_attend(*a, *c);
    if (!why && shared_len > 0 && (shared_table == nullptr || !kv_aligned(shared_table, 4))) why = "shared_table is NULL or not 4-byte aligned";
    const bool empty = b->rows == 0 || b->seqs == 0;
    if (!why && !empty) why = kv_check_rows(a->q, b->rows, a->q_heads, c->head_dim, c->dtype, false, &qb);
    if (!why && !empty) why = kv_check_rows(a->out, b->rows, a->q_heads, c->head_dim, a->out_dtype, true, &ob);
    if (why) return set_error(ctx, GFD_ERR_INVALID, "%s: %s", call, why);
    if (empty) return GFD_OK;
    const KvPlan plan = plan_attend(ctx, *c, *b, *a, shared_len);  // (divides by the heads: after the checks)
    const size_t need = plan.bytes;
    if (need > 0 && (a->workspace == nullptr || !kv_aligned(a->workspace, 256))) why = "workspace is NULL or not 256-byte aligned";
    else if (a->workspace_bytes < need) why = "workspace is smaller than gfd_kv_attend_workspace says";
    if (why) return set_error(ctx, GFD_ERR_INVALID, "%s: %s", call, why);
    const uint64_t shared_blocks = (static_cast<uint64_t>(shared_len) + c->block_tokens - 1) / c->block_tokens;
    const Region regions[] = {{c->k, cache_bytes, "the cache's K"},
                              {c->v, cache_bytes, "the cache's V"},
                              {a->q.data, qb, "q"},
                              {a->out.data, ob, "out"},
                              {b->row_start, (static_cast<uint64_t>(b->seqs) + 1) * 4, "row_start"},
                              {b->kv_len, static_cast<uint64_t>(b->seqs) * 4, "kv_len"},
                              {b->table, kv_table_bytes(*b), "table"},
                              {shared_table, shared_blocks * 4, "shared_table"},
                              {a->lse, static_cast<uint64_t>(b->rows) * a->q_heads * 4, "lse"},
                              {a->alibi, static_cast<uint64_t>(a->q_heads) * 4, "alibi"},
                              {a->prefix_len, static_cast<uint64_t>(b->seqs) * 4, "prefix_len"},
                              {a->workspace, need, "workspace"},
                              {a->status, 4, "status"}};
    const int rc = check_regions(ctx, call, regions, static_cast<int>(sizeof(regions) / sizeof(regions[0])));
    if (rc != GFD_OK) return rc;
    KvAttendParams p;
    std::memset(&p, 0, sizeof(p));
    p.cache = view(*c);
    p.batch = view(*b, *c);
    p.q = view(a->q, b->rows, a->q_heads, 2);
    p.out = view(a->out, b->rows, a->q_heads, kv_elt(a->out_dtype));
    p.lse = a->lse;
    p.alibi = a->alibi;
    p.prefix_len = a->prefix_len;
    p.shared_table = shared_len > 0 ? shared_table : nullptr;
    p.status = a->status;
    p.shared_len = static_cast<int32_t>(shared_len);
    p.q_heads = a->q_heads;
    p.group = a->q_heads / c->heads;
    p.group_magic = ((1ull << 44) + p.group - 1) / p.group;
    const uint32_t pages = c->block_tokens / kKvPage;
    p.page_magic = ((1ull << 32) + pages - 1) / pages;
    p.max_q_len = a->max_q_len;
    p.causal = a->causal != 0;
    p.window = a->window;
    p.scale = a->scale;
    p.softcap = a->softcap;
    p.scale2 = a->scale * 1.4426950408889634f;
    p.cap_x = a->softcap > 0.0f ? a->scale / a->softcap : 0.0f;
    p.cap2 = a->softcap * 1.4426950408889634f;
    // scores of 10 and more would show the rounding of these factors in lse
    const double factor = a->softcap > 0.0f ? static_cast<double>(p.cap_x) * p.cap2 : static_cast<double>(p.scale2);
    p.to_ln = static_cast<float>(a->alibi != nullptr || factor == 0.0 ? 0.6931471805599453 : a->scale / factor);
    p.out_f32 = a->out_dtype == GFD_FP32;
    p.few_rows = plan.few ? kKvFewRows : 0;
    cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
    char* ws = static_cast<char*>(a->workspace);
    const KvEncodeFn encode = driver().tensor_map;
    KvMaps maps;
    if (plan.many || shared_len > 0) {
        if (encode == nullptr) return set_error(ctx, GFD_ERR_UNSUPPORTED, "%s: the driver has no cuTensorMapEncodeTiled", call);
        if (!kv_make_maps(&maps, p, c->head_dim, c->dtype, encode))
            return set_error(ctx, GFD_ERR_INVALID, "%s: the cache's shape does not fit a tensor map", call);
        p.q_mapped = maps.q_mapped;
    }
    KvAttendParams own = p;
    if (shared_len > 0) {
        // the results over the own keys go to the workspace in 32 bits, the pass over the prefix finishes
        own.out = KvRowsView{ws + plan.own_out, static_cast<int64_t>(a->q_heads) * c->head_dim * 4, static_cast<int64_t>(c->head_dim) * 4};
        own.lse = reinterpret_cast<float*>(ws + plan.own_lse);
        own.skipped_lse = own.lse;
        own.out_f32 = 1;
    }
    cudaError_t e = cudaSuccess;
    bool chained = false;  // launches of this call overlap
    if (e == cudaSuccess && plan.few) {
        own.line = kv_line_at(ws + plan.few_line, kv_decode_workers(ctx->num_sms, c->head_dim));
        e = launch_kv_decode(own, c->head_dim, c->dtype, ctx->num_sms, chained, st);
        chained = true;
    }
    if (e == cudaSuccess && plan.many) {
        own.line = kv_line_at(ws + plan.many_line, kv_prompt_ctas(ctx->num_sms));
        e = launch_kv_prompt(own, c->head_dim, c->dtype, ctx->num_sms, maps, chained, st);
        chained = true;
    }
    if (e == cudaSuccess && shared_len > 0) {
        KvAttendParams pre = p;
        pre.shared_pass = 1;
        pre.own_out = reinterpret_cast<const float*>(ws + plan.own_out);
        pre.own_lse = own.lse;
        pre.line = kv_line_at(ws + plan.prefix_line, kv_prompt_ctas(ctx->num_sms));
        e = launch_kv_prompt(pre, c->head_dim, c->dtype, ctx->num_sms, maps, chained, st);
    }
    return e == cudaSuccess ? GFD_OK : cuda_error(ctx, e, "kv_attend: kernel launch");
}

int merge(gfd_ctx* ctx, const gfd_kv_merge_args* a, void* stream) {
    if (a == nullptr) return set_error(ctx, GFD_ERR_INVALID, "kv_merge: NULL argument");
    uint64_t pb = 0, ob = 0;
    const char* why = kv_check_merge(*a);
    if (!why && a->rows > 0) why = kv_check_rows(a->parts, a->rows, a->heads, a->head_dim, a->part_dtype, false, &pb);
    if (!why && a->rows > 0) why = kv_check_rows(a->out, a->rows, a->heads, a->head_dim, a->out_dtype, true, &ob);
    if (why) return set_error(ctx, GFD_ERR_INVALID, "kv_merge: %s", why);
    if (a->rows == 0) return GFD_OK;
    pb += static_cast<uint64_t>(a->part_count - 1) * a->part_stride * kv_elt(a->part_dtype);
    const uint64_t n = static_cast<uint64_t>(a->rows) * a->heads;
    const Region regions[] = {{a->parts.data, pb, "parts"},
                              {a->part_lse, n * a->part_count * 4, "part_lse"},
                              {a->out.data, ob, "out"},
                              {a->lse, n * 4, "lse"}};
    const int rc = check_regions(ctx, "kv_merge", regions, 4);
    if (rc != GFD_OK) return rc;
    KvMergeParams p;
    std::memset(&p, 0, sizeof(p));
    p.parts = view(a->parts, a->rows, a->heads, kv_elt(a->part_dtype));
    p.part_stride = a->part_count > 1 ? a->part_stride * kv_elt(a->part_dtype) : 0;
    p.part_lse = a->part_lse;
    p.out = view(a->out, a->rows, a->heads, kv_elt(a->out_dtype));
    p.lse = a->lse;
    p.rows = static_cast<int32_t>(a->rows);
    p.heads = a->heads;
    p.part_count = a->part_count;
    cudaStream_t st = stream ? static_cast<cudaStream_t>(stream) : ctx->stream;
    const cudaError_t e = launch_kv_merge(p, a->head_dim, a->part_dtype, a->out_dtype, ctx->num_sms, st);
    return e == cudaSuccess ? GFD_OK : cuda_error(ctx, e, "kv_merge: kernel launch");
}

// No C++ exception leaves a C entry point (the range registry allocates).
template <typename F>
int guarded(gfd_ctx* ctx, F f) {
    if (ctx == nullptr) return GFD_ERR_INVALID;
    try {
        std::lock_guard<std::mutex> lk(ctx->mu);
        CtxScope scope(ctx->cu_ctx);
        return f();
    } catch (const std::bad_alloc&) {
        return GFD_ERR_NOMEM;
    } catch (...) {
        return GFD_ERR_STATE;
    }
}

}  // namespace

extern "C" {

int gfd_kv_append(gfd_ctx* ctx, const gfd_kv_cache* cache, const gfd_kv_batch* batch, const gfd_kv_append_args* args,
                  void* stream) {
    return guarded(ctx, [&] { return append(ctx, cache, batch, args, stream); });
}

int gfd_kv_attend(gfd_ctx* ctx, const gfd_kv_cache* cache, const gfd_kv_batch* batch, const gfd_kv_attend_args* args,
                  void* stream) {
    return guarded(ctx, [&] { return attend(ctx, "kv_attend", cache, batch, nullptr, 0, args, stream); });
}

int gfd_kv_attend_shared(gfd_ctx* ctx, const gfd_kv_cache* cache, const gfd_kv_batch* batch, const int32_t* shared_table,
                         int64_t shared_len, const gfd_kv_attend_args* args, void* stream) {
    return guarded(ctx, [&] { return attend(ctx, "kv_attend_shared", cache, batch, shared_table, shared_len, args, stream); });
}

int gfd_kv_attend_workspace(gfd_ctx* ctx, const gfd_kv_cache* cache, const gfd_kv_batch* batch,
                            const gfd_kv_attend_args* args, int64_t shared_len, size_t* bytes) {
    return guarded(ctx, [&] {
        if (bytes == nullptr || cache == nullptr || batch == nullptr || args == nullptr)
            return set_error(ctx, GFD_ERR_INVALID, "kv_attend_workspace: NULL argument");
        uint64_t unused = 0;
        const char* why = kv_check_cache(*cache, false, &unused);
        if (!why) why = kv_check_workspace(*cache, *batch, *args, shared_len);
        if (why) return set_error(ctx, GFD_ERR_INVALID, "kv_attend_workspace: %s", why);
        *bytes = plan_attend(ctx, *cache, *batch, *args, shared_len).bytes;
        return static_cast<int>(GFD_OK);
    });
}

int gfd_kv_merge(gfd_ctx* ctx, const gfd_kv_merge_args* args, void* stream) {
    return guarded(ctx, [&] { return merge(ctx, args, stream); });
}

}  // extern "C"
