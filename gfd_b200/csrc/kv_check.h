#pragma once
// Argument checks of the paged KV-cache entry points and the sequence arithmetic that
// their kernels share with the host.  Nothing here touches CUDA state, so the CPU tests
// compile it with a plain C++ compiler.

#include <cmath>
#include <cstddef>
#include <cstdint>
#include <initializer_list>

#include "gfd_b200.h"

#if defined(__CUDACC__)
#define GFD_HD __host__ __device__ __forceinline__
#else
#define GFD_HD inline
#endif

namespace gfdb {

constexpr int kKvPage = 16;           // tokens one load takes: block_tokens is a multiple
constexpr int kKvMaxHeads = 1024;
constexpr int kKvMaxBlockTokens = 1024;
constexpr int kKvMaxParts = 1024;
constexpr int64_t kKvMaxTokens = 1ll << 30;  // positions of a sequence, so that they fit 32 bits with room

// ---------------------------------------------------------------------------
// Sequences
// ---------------------------------------------------------------------------
// Rows [row0, row0 + rows) of sequence s and its keys; ok == false: skipped (BAD_LENGTH).
struct KvSeq {
    int32_t row0;
    int32_t rows;
    int32_t keys;  // kv_len
    bool ok;
};

GFD_HD KvSeq kv_seq(int32_t start, int32_t end, int32_t kv_len, int64_t capacity, int32_t max_q_len) {
    KvSeq q{start, end - start, kv_len, true};
    if (q.rows > 0 && (kv_len < q.rows || kv_len > capacity || (max_q_len > 0 && q.rows > max_q_len))) q.ok = false;
    if (q.rows <= 0) q.rows = q.keys = 0;  // nothing to do, whatever kv_len says
    return q;
}

// What the row at position p sees of n keys: [0, pre) and [lo, hi).  lo >= pre and
// hi >= lo, so the two never overlap.
struct KvSpan {
    int32_t pre, lo, hi;
};

GFD_HD KvSpan kv_span(int32_t p, int32_t n, int32_t prefix, int32_t window, bool causal) {
    KvSpan s;
    s.pre = prefix < 0 ? 0 : (prefix > n ? n : prefix);
    s.hi = causal ? (p + 1 < n ? p + 1 : n) : n;
    s.lo = window > 0 && p + 1 > window ? p + 1 - window : 0;
    if (s.lo < s.pre) s.lo = s.pre;
    if (s.hi < s.lo) s.hi = s.lo;
    return s;
}

// The span within the keys [base, base + len), in their own count.
GFD_HD KvSpan kv_clip(KvSpan s, int32_t base, int32_t len) {
    auto c = [&](int32_t x) { return x < base ? 0 : (x - base > len ? len : x - base); };
    return KvSpan{c(s.pre), c(s.lo), c(s.hi)};
}

// Tiles of `size` keys that hold a visible key of some row: tiles [0, npre), then
// [first, first + count - npre).  The span's lo and hi are the least and the greatest of the rows'.
struct KvTiles {
    int32_t npre, first, count;
    GFD_HD int32_t at(int32_t i) const { return i < npre ? i : i - npre + first; }
};

GFD_HD KvTiles kv_tiles(KvSpan s, int32_t size) {
    KvTiles t;
    t.npre = (s.pre + size - 1) / size;
    t.first = s.lo / size;
    if (t.first < t.npre) t.first = t.npre;
    const int32_t end = s.hi > s.lo ? (s.hi + size - 1) / size : 0;
    t.count = t.npre + (end > t.first ? end - t.first : 0);
    return t;
}

// a / b for a >= 0, b > 0; the 64-bit division costs several times the 32-bit one.
GFD_HD int64_t kv_div(int64_t a, int64_t b) {
    return ((a | b) >> 32) == 0 ? static_cast<int64_t>(static_cast<uint32_t>(a) / static_cast<uint32_t>(b)) : a / b;
}

// All tiles of a launch form one line, unit after unit; stretch c is [at(c), at(c + 1)), at least one
// tile each, n() of them.  A unit inside one stretch is finished there.  One that is cut leaves
// partial results, one in each stretch it touches, in slot 1 of the one where it begins and slot 0
// of the others; they are joined at the first cut inside the unit.
struct KvCuts {
    int64_t each;
    uint32_t more, ctas;
    GFD_HD KvCuts(int64_t total, uint32_t most) {
        ctas = total < static_cast<int64_t>(most) ? static_cast<uint32_t>(total) : most;
        each = ctas > 0 ? kv_div(total, ctas) : 0;
        more = ctas > 0 ? static_cast<uint32_t>(total - each * ctas) : 0;
    }
    GFD_HD int n() const { return static_cast<int>(ctas); }
    GFD_HD int64_t at(uint32_t c) const { return each * c + more * c / ctas; }  // more * c < 2^32: ctas <= 2^16
    // The last cut before position `end` of the line, c being one.
    GFD_HD uint32_t last_before(uint32_t c, int64_t end) const {
        uint32_t hi = ctas - 1;
        while (c < hi) {
            const uint32_t mid = c + (hi - c + 1) / 2;
            if (at(mid) < end) c = mid;
            else hi = mid - 1;
        }
        return c;
    }
};

// What the joining kernel finds for a stretch: the rows of the unit that the stretch's cut is the first
// to divide, left in parts: slot 1 of the stretch before it, slot 0 of this one and the next ones.
struct KvCut {
    int32_t parts;  // 0: nothing to join
    int32_t row0, packed0, packed, h;
};

// ---------------------------------------------------------------------------
// An attention call's kernels and workspace
// ---------------------------------------------------------------------------
constexpr int kKvManyRows = 256;  // packed rows of a unit of kv_prompt
constexpr int kKvFewRows = 16;  // packed rows (rows x group) up to which kv_decode takes a sequence

// Bytes of a line's cuts and slots.
inline size_t kv_line_bytes(int ctas, int slot_rows, int head_dim) {
    return (sizeof(KvCut) * ctas + 255) / 256 * 256 +
           (static_cast<size_t>(ctas) * 2 * (static_cast<size_t>(slot_rows) * head_dim + 2 * slot_rows) * sizeof(float) + 255) / 256 * 256;
}

// Which kernels a call runs, and where each keeps its intermediate results in the workspace.
struct KvPlan {
    bool few, many;       // kv_decode takes the sequences of few rows, kv_prompt the others
    size_t few_line, many_line, prefix_line;  // offsets of the kernels' lines
    size_t own_out, own_lse;                  // behind a shared prefix: results over the own keys
    size_t bytes;
};

// few_workers, many_ctas: the stretches of the two kernels on this GPU.  The cache has been checked.  A batch
// of no more rows, sequences, rows a sequence and shared tokens never needs more bytes than one of more: the
// kernels that run depend on how the rows can be spread over the sequences, the room does not.
inline KvPlan kv_plan(const gfd_kv_cache& c, const gfd_kv_batch& b, const gfd_kv_attend_args& a, int64_t shared_len, int few_workers,
                      int many_ctas) {
    KvPlan r{};
    if (b.rows <= 0 || b.seqs <= 0 || a.q_heads <= 0) return r;
    const int64_t group = a.q_heads / c.heads > 0 ? a.q_heads / c.heads : 1;
    const int64_t most = a.max_q_len > 0 && a.max_q_len < b.rows ? a.max_q_len : b.rows;  // rows of a sequence
    r.many = most * group > kKvFewRows;
    // Where every sequence has many rows (no row left over: one has at least what the others cannot
    // have), kv_prompt takes them all, whatever they turn out to be: two launches less, 10 us.
    const int64_t least = b.rows - (b.seqs - 1) * most;
    r.few = group <= kKvFewRows && (!r.many || least * group <= kKvFewRows);
    size_t at = 0;
    auto take = [&](size_t n) {
        const size_t here = at;
        at += (n + 255) / 256 * 256;
        return here;
    };
    const size_t many_bytes = kv_line_bytes(many_ctas, kKvManyRows, c.head_dim);
    if (group <= kKvFewRows) r.few_line = take(kv_line_bytes(few_workers, kKvFewRows, c.head_dim));
    if (r.many) r.many_line = take(many_bytes);
    if (shared_len > 0) {
        r.prefix_line = take(many_bytes);
        r.own_out = take(static_cast<size_t>(b.rows) * a.q_heads * c.head_dim * sizeof(float));
        r.own_lse = take(static_cast<size_t>(b.rows) * a.q_heads * sizeof(float));
    }
    r.bytes = at;
    return r;
}

// ---------------------------------------------------------------------------
// Checks: each returns nullptr, or what is wrong
// ---------------------------------------------------------------------------
inline int kv_elt(int32_t dtype) { return dtype == GFD_FP32 ? 4 : 2; }

inline bool kv_aligned(const void* p, uint64_t n) { return (reinterpret_cast<uint64_t>(p) & (n - 1)) == 0; }

// Bytes from the first to behind the last element of [n0][n1][...][inner], or 0 when that
// does not fit 2^62.
inline uint64_t kv_extent(const int64_t* n, const int64_t* stride, int dims, int64_t inner, int elt) {
    unsigned __int128 e = static_cast<unsigned __int128>(inner);
    for (int i = 0; i < dims; ++i) {
        if (n[i] <= 0 || stride[i] < 0) return 0;
        e += static_cast<unsigned __int128>(n[i] - 1) * static_cast<unsigned __int128>(stride[i]);
    }
    e *= static_cast<unsigned>(elt);
    return (e >> 62) != 0 ? 0 : static_cast<uint64_t>(e);
}

// True when no two index tuples of [n0][n1].. share an element (strides nest in some order).
inline bool kv_distinct(const int64_t* n, const int64_t* stride, int dims, int64_t inner) {
    bool used[4] = {};
    unsigned __int128 span = static_cast<unsigned __int128>(inner);
    for (int k = 0; k < dims; ++k) {
        int best = -1;
        for (int i = 0; i < dims; ++i)
            if (!used[i] && n[i] > 1 && (best < 0 || stride[i] < stride[best])) best = i;
        if (best < 0) break;
        used[best] = true;
        if (stride[best] < 0 || static_cast<unsigned __int128>(stride[best]) < span) return false;
        span += static_cast<unsigned __int128>(n[best] - 1) * static_cast<unsigned __int128>(stride[best]);
    }
    return true;
}

// A row array; `out`: written, so its elements must be distinct.  *bytes: its extent.
inline const char* kv_check_rows(const gfd_kv_rows& r, int64_t rows, int64_t heads, int64_t dim, int32_t dtype, bool out,
                                 uint64_t* bytes) {
    const int64_t n[2] = {rows, heads};
    const int64_t st[2] = {rows > 1 ? r.row_stride : 0, heads > 1 ? r.head_stride : 0};
    if (r.data == nullptr) return "a row array is NULL";
    if (!kv_aligned(r.data, 16)) return "a row array is not 16-byte aligned";
    if (st[0] < 0 || st[1] < 0 || st[0] % 8 != 0 || st[1] % 8 != 0) return "row and head strides must be multiples of 8, not negative";
    *bytes = kv_extent(n, st, 2, dim, kv_elt(dtype));
    if (*bytes == 0) return "a row array is too large";
    if (out && !kv_distinct(n, st, 2, dim)) return "elements of an output row array overlap";
    return nullptr;
}

inline const char* kv_check_cache(const gfd_kv_cache& c, bool write, uint64_t* bytes) {
    if (c.dtype != GFD_BF16 && c.dtype != GFD_FP16) return "the cache is neither bf16 nor fp16";
    if (c.head_dim != 64 && c.head_dim != 128) return "head_dim must be 64 or 128";
    if (c.heads < 1 || c.heads > kKvMaxHeads) return "bad number of KV heads";
    if (c.block_tokens < kKvPage || c.block_tokens > kKvMaxBlockTokens || c.block_tokens % kKvPage != 0)
        return "block_tokens must be a multiple of 16, at most 1024";
    if (c.blocks < 1 || c.blocks > 0x7fffffffll) return "bad number of blocks";
    if (c.k == nullptr || c.v == nullptr) return "K or V of the cache is NULL";
    if (!kv_aligned(c.k, 16) || !kv_aligned(c.v, 16)) return "the cache is not 16-byte aligned";
    const int64_t n[3] = {c.blocks, c.block_tokens, c.heads};
    const int64_t st[3] = {c.blocks > 1 ? c.block_stride : 0, c.token_stride, c.heads > 1 ? c.head_stride : 0};
    for (int64_t s : st)
        if (s < 0 || s % 8 != 0 || s >= (1ll << 38)) return "cache strides must be multiples of 8, not negative and below 2^38";
    if (!kv_distinct(n, st, 3, c.head_dim)) return "elements of the cache overlap";
    *bytes = kv_extent(n, st, 3, c.head_dim, 2);
    if (*bytes == 0) return "the cache is too large";
    if (write && c.k == c.v) return "K and V are the same array";
    return nullptr;
}

// Bytes of the block table of a batch that was checked.
inline uint64_t kv_table_bytes(const gfd_kv_batch& b) {
    const int64_t n[1] = {b.seqs}, st[1] = {b.seqs > 1 ? b.table_stride : 0};
    return b.table_width == 0 ? 0 : kv_extent(n, st, 1, b.table_width, sizeof(int32_t));
}

inline const char* kv_check_batch(const gfd_kv_batch& b, const gfd_kv_cache& c, int64_t shared_len) {
    if (b.rows < 0 || b.rows > 0x3fffffffll) return "bad number of rows";
    if (b.seqs < 0 || b.seqs > GFD_KV_MAX_SEQS) return "bad number of sequences";
    if (b.rows == 0 || b.seqs == 0) return nullptr;
    if (b.table_width < 0 || b.table_stride < 0 || (b.seqs > 1 && b.table_stride < b.table_width)) return "bad block table shape";
    if (b.table_width > 0 && kv_table_bytes(b) == 0) return "the block table is too large";
    if (shared_len < 0 || shared_len + static_cast<int64_t>(b.table_width) * c.block_tokens > kKvMaxTokens)
        return "more than 2^30 tokens in a sequence's table";
    if (b.row_start == nullptr || b.kv_len == nullptr || (b.table == nullptr && b.table_width > 0))
        return "row_start, kv_len or table is NULL";
    if (!kv_aligned(b.row_start, 4) || !kv_aligned(b.kv_len, 4) || !kv_aligned(b.table, 4))
        return "row_start, kv_len or table is not 4-byte aligned";
    return nullptr;
}

inline const char* kv_check_append(const gfd_kv_append_args& a, const gfd_kv_cache& c) {
    if (a.q_heads < 0 || a.q_heads > 8 * kKvMaxHeads) return "bad number of query heads";
    if (a.rot_dim < 0 || a.rot_dim > c.head_dim || a.rot_dim % 16 != 0) return "rot_dim must be a multiple of 16, at most head_dim";
    if (a.rot_dim > 0 && (a.inv_freq == nullptr || !kv_aligned(a.inv_freq, 4))) return "inv_freq is NULL or not 4-byte aligned";
    if (!kv_aligned(a.positions, 4) || !kv_aligned(a.status, 4)) return "positions or status is not 4-byte aligned";
    if (a.q_heads > 0 && a.q.data == a.q_out.data && (a.q.row_stride != a.q_out.row_stride || a.q.head_stride != a.q_out.head_stride))
        return "q_out is q with other strides";
    return nullptr;
}

inline const char* kv_check_attend(const gfd_kv_attend_args& a, const gfd_kv_cache& c) {
    if (a.q_heads < 1 || a.q_heads > 8 * kKvMaxHeads || a.q_heads % c.heads != 0)
        return "query heads must be a multiple of the cache's heads";
    if (a.out_dtype != c.dtype && a.out_dtype != GFD_FP32) return "out must be of the cache's type or fp32";
    if (a.max_q_len < 0) return "max_q_len is negative";
    if (a.window < 0 || a.window > kKvMaxTokens) return "bad window";
    if (!std::isfinite(a.scale)) return "scale is not finite";
    if (!std::isfinite(a.softcap) || a.softcap < 0.0f) return "softcap must be finite and not negative";
    if (a.softcap > 0.0f && (!std::isfinite(a.scale / a.softcap) || a.softcap > 1e30f)) return "softcap is out of range";
    if (a.q.data == a.out.data && a.q.data != nullptr) return "out must not be q";  // (no rows, no pointers)
    if (!kv_aligned(a.lse, 4) || !kv_aligned(a.alibi, 4) || !kv_aligned(a.prefix_len, 4) || !kv_aligned(a.status, 4))
        return "lse, alibi, prefix_len or status is not 4-byte aligned";
    return nullptr;
}

// What gfd_kv_attend_workspace reads, within the limits of the calls themselves (so that nothing wraps).
inline const char* kv_check_workspace(const gfd_kv_cache& c, const gfd_kv_batch& b, const gfd_kv_attend_args& a, int64_t shared_len) {
    if (b.rows < 0 || b.rows > 0x3fffffffll) return "bad number of rows";
    if (b.seqs < 0 || b.seqs > GFD_KV_MAX_SEQS) return "bad number of sequences";
    if (a.q_heads < 1 || a.q_heads > 8 * kKvMaxHeads || a.q_heads % c.heads != 0)
        return "query heads must be a multiple of the cache's heads";
    if (a.max_q_len < 0) return "max_q_len is negative";
    if (shared_len < 0 || shared_len > kKvMaxTokens) return "bad shared_len";
    return nullptr;
}

inline const char* kv_check_merge(const gfd_kv_merge_args& a) {
    if (a.rows < 0 || a.rows > 0x3fffffffll) return "bad number of rows";
    if (a.part_count < 1 || a.part_count > kKvMaxParts) return "bad number of parts";
    if (a.heads < 1 || a.heads > 8 * kKvMaxHeads) return "bad number of heads";
    if (a.head_dim != 64 && a.head_dim != 128) return "head_dim must be 64 or 128";
    for (int32_t t : {a.part_dtype, a.out_dtype})
        if (t != GFD_BF16 && t != GFD_FP16 && t != GFD_FP32) return "unknown type";
    if (a.part_stride < 0 || a.part_stride % 8 != 0) return "part_stride must be a multiple of 8, not negative";
    if (a.part_count > 1 && a.part_stride > (1ll << 40)) return "part_stride is too large";
    if ((a.rows > 0 && a.part_lse == nullptr) || !kv_aligned(a.part_lse, 4) || !kv_aligned(a.lse, 4)) return "part_lse is NULL, or part_lse or lse not 4-byte aligned";
    if (a.rows > 0)
        for (int i = 0; i < a.part_count; ++i)
            if (static_cast<const char*>(a.parts.data) + static_cast<int64_t>(i) * a.part_stride * kv_elt(a.part_dtype) == a.out.data)
                return "out must not be a part";
    return nullptr;
}

}  // namespace gfdb
