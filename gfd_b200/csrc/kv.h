#pragma once
// Kernel parameters and launchers of the paged KV-cache operators (kv*.cu, kv_api.cpp).

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "gfd_b200.h"
#include "kv_check.h"

namespace gfdb {

struct KvCacheView {
    const char* k;
    const char* v;
    int64_t block_stride, token_stride, head_stride;  // bytes
    int32_t blocks, block_tokens, heads;
};

struct KvBatchView {
    const int32_t* row_start;
    const int32_t* kv_len;
    const int32_t* table;
    int64_t table_stride;
    int64_t capacity;  // tokens a table row can name
    int32_t rows, seqs, table_width;
};

struct KvRowsView {
    char* data;
    int64_t row_stride, head_stride;  // bytes
};

struct KvAppendParams {
    KvCacheView cache;
    KvBatchView batch;
    KvRowsView k, v, q, q_out;
    const float* inv_freq;
    const int32_t* positions;
    uint32_t* status;
    int32_t q_heads, rot_dim, interleaved;
};

// Where a stretch of the line of tiles begins (KvCuts).
struct KvPlace {
    int64_t begin;            // the unit's first tile on the line
    int32_t t, count;         // tile t of the unit's `count`
    int32_t row0;             // first row of its sequence
    int32_t packed0, packed;  // packed rows [packed0, packed0 + packed) of the sequence
    int32_t h, s;             // KV head, sequence
};

// A launch's cuts and partial results, one and two slots per stretch: the sums of kRows packed rows
// ([rows][D] of kv_decode, [D / 4][rows][4] of kv_prompt, so that its threads of neighbouring rows
// write side by side), then the rows' base and weight sum.
struct KvLine {
    KvCut* cuts;
    float* slots;
};

constexpr uint32_t kKvSkipped = 0xffffffffu;  // a NaN that no sum leaves

struct KvAttendParams {
    KvCacheView cache;
    KvBatchView batch;
    KvRowsView q, out;
    float* lse;
    const float* alibi;
    const int32_t* prefix_len;
    const int32_t* shared_table;
    uint32_t* status;
    int32_t shared_len;
    int32_t q_heads, group;
    uint64_t group_magic;  // ceil(2^44 / group), see kv_div_group
    uint64_t page_magic;   // ceil(2^32 / pages of a block), see kv_div_pages
    int32_t max_q_len, causal, window;
    float scale, softcap;
    float scale2;    // scale in base 2
    float cap_x;     // scale / softcap
    float cap2;      // softcap in base 2
    float to_ln;     // from the kernels' base-2 scores to natural ones: ln 2, and what rounded off scale2 or cap_x and cap2
    int32_t out_f32;
    int32_t few_rows;  // sequences of at most so many packed rows are kv_decode's
    int32_t q_mapped;      // kv_prompt: Q comes by its tensor map
    int32_t shared_pass;   // kv_prompt: all rows against the shared prefix, joined with
    const float* own_out;  // what was found over the own keys, [rows][q_heads][D]
    const float* own_lse;  // and its lse; kKvSkipped for rows of skipped sequences
    float* skipped_lse;    // where the passes over the own keys leave those marks; null: nowhere
    KvLine line;
};

struct KvMergeParams {
    KvRowsView parts;
    int64_t part_stride;  // bytes
    const float* part_lse;
    KvRowsView out;
    float* lse;
    int32_t rows, heads, part_count;
};

// dtype: GFD_* of the cache.  chained: the launch may start before the one before it on the stream has
// ended (it was made by the same call and touches nothing of this one's, or waits for it).
cudaError_t launch_kv_append(const KvAppendParams& p, int head_dim, int dtype, int num_sms, cudaStream_t st);
cudaError_t launch_kv_join_few(const KvAttendParams& p, int head_dim, int dtype, int stretches, cudaStream_t st);
cudaError_t launch_kv_join_many(const KvAttendParams& p, int head_dim, int dtype, int stretches, cudaStream_t st);
int kv_decode_workers(int num_sms, int head_dim);  // each with a stretch of the line
int kv_prompt_ctas(int num_sms);
// cuTensorMapEncodeTiled, resolved through the runtime (libcuda is not linked)
using KvEncodeFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
struct KvMaps {
    CUtensorMap k, v;  // the cache as kv_prompt reads it
    CUtensorMap q;     // and the rows, where `q_mapped`
    bool q_mapped;
};
bool kv_make_maps(KvMaps* maps, const KvAttendParams& p, int head_dim, int dtype, KvEncodeFn encode);
cudaError_t launch_kv_prompt(const KvAttendParams& p, int head_dim, int dtype, int num_sms, const KvMaps& maps, bool chained, cudaStream_t st);
cudaError_t launch_kv_decode(const KvAttendParams& p, int head_dim, int dtype, int num_sms, bool chained, cudaStream_t st);

// A line laid out in the kv_line_bytes at p.
inline KvLine kv_line_at(void* p, int ctas) {
    return KvLine{static_cast<KvCut*>(p), reinterpret_cast<float*>(static_cast<char*>(p) + (sizeof(KvCut) * ctas + 255) / 256 * 256)};
}
cudaError_t launch_kv_merge(const KvMergeParams& p, int head_dim, int part_dtype, int out_dtype, int num_sms, cudaStream_t st);

}  // namespace gfdb
