// C exports of the paged KV-cache checks and sequence arithmetic (gfd_b200/csrc/kv_check.h)
// for the CPU tests.
#include <cstddef>

#include "kv_check.h"

using namespace gfdb;

extern "C" {

const char* gfdt_kv_cache(const gfd_kv_cache* c, int write, uint64_t* bytes) { return kv_check_cache(*c, write != 0, bytes); }
const char* gfdt_kv_batch(const gfd_kv_batch* b, const gfd_kv_cache* c, int64_t shared) { return kv_check_batch(*b, *c, shared); }
// workspace of a call on a GPU of `sms`; kernels: bit 0 kv_decode, bit 1 kv_prompt
uint64_t gfdt_kv_workspace(const gfd_kv_cache* c, int64_t rows, int32_t seqs, int32_t q_heads, int32_t max_q_len, int64_t shared, int sms,
                           int* kernels) {
    gfd_kv_batch b{};
    gfd_kv_attend_args a{};
    b.rows = rows, b.seqs = seqs, a.q_heads = q_heads, a.max_q_len = max_q_len;
    const KvPlan p = kv_plan(*c, b, a, shared, sms * 4 * (c->head_dim == 64 ? 3 : 2), sms);
    *kernels = (p.few ? 1 : 0) + (p.many ? 2 : 0);
    return p.bytes;
}
uint64_t gfdt_kv_table_bytes(const gfd_kv_batch* b) { return kv_table_bytes(*b); }
const char* gfdt_kv_append(const gfd_kv_append_args* a, const gfd_kv_cache* c) { return kv_check_append(*a, *c); }
const char* gfdt_kv_attend(const gfd_kv_attend_args* a, const gfd_kv_cache* c) { return kv_check_attend(*a, *c); }
const char* gfdt_kv_check_workspace(const gfd_kv_cache* c, const gfd_kv_batch* b, const gfd_kv_attend_args* a, int64_t shared) {
    return kv_check_workspace(*c, *b, *a, shared);
}
const char* gfdt_kv_merge(const gfd_kv_merge_args* a) { return kv_check_merge(*a); }
const char* gfdt_kv_rows(const gfd_kv_rows* r, int64_t rows, int64_t heads, int64_t dim, int32_t dtype, int out, uint64_t* bytes) {
    return kv_check_rows(*r, rows, heads, dim, dtype, out != 0, bytes);
}
void gfdt_kv_span(int32_t p, int32_t n, int32_t prefix, int32_t window, int causal, int32_t* out) {
    const KvSpan s = kv_span(p, n, prefix, window, causal != 0);
    out[0] = s.pre, out[1] = s.lo, out[2] = s.hi;
}
int gfdt_kv_seq(int32_t start, int32_t end, int32_t len, int64_t capacity, int32_t max_q, int32_t* out) {
    const KvSeq q = kv_seq(start, end, len, capacity, max_q);
    out[0] = q.row0, out[1] = q.rows, out[2] = q.keys;
    return q.ok;
}
void gfdt_kv_tiles(const int32_t* span, int32_t base, int32_t len, int32_t size, int32_t* out) {
    const KvTiles t = kv_tiles(kv_clip(KvSpan{span[0], span[1], span[2]}, base, len), size);
    out[0] = t.npre, out[1] = t.first, out[2] = t.count;
}
// at(0) .. at(n), n returned
int gfdt_kv_cuts(int64_t total, uint32_t most, int64_t* at) {
    const KvCuts c(total, most);
    for (int i = 0; i <= c.n() && c.n() > 0; ++i) at[i] = c.at(i);
    return c.n();
}
uint32_t gfdt_kv_last_before(int64_t total, uint32_t most, uint32_t c, int64_t end) { return KvCuts(total, most).last_before(c, end); }
int64_t gfdt_kv_div(int64_t a, int64_t b) { return kv_div(a, b); }
// sizes and last offsets of the argument structures
void gfdt_kv_layout(uint64_t* out) {
    const uint64_t v[] = {sizeof(gfd_kv_cache),       offsetof(gfd_kv_cache, dtype),
                          sizeof(gfd_kv_batch),       offsetof(gfd_kv_batch, table_width),
                          sizeof(gfd_kv_rows),        offsetof(gfd_kv_rows, head_stride),
                          sizeof(gfd_kv_append_args), offsetof(gfd_kv_append_args, interleaved),
                          sizeof(gfd_kv_attend_args), offsetof(gfd_kv_attend_args, softcap),
                          sizeof(gfd_kv_merge_args),  offsetof(gfd_kv_merge_args, out_dtype)};
    for (unsigned i = 0; i < sizeof(v) / sizeof(v[0]); ++i) out[i] = v[i];
}
}
