#pragma once
// Kernel parameters and launchers of the paged KV-cache operators (kv*.cu, kv_api.cpp).

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
    int32_t max_q_len, causal, window;
    float scale, softcap;
    float scale2;    // scale in base 2
    float cap_rate;  // 2 log2(e) / softcap
    int32_t out_f32;
    int32_t skip_few;  // the plain kernel leaves sequences of at most kKvFewRows packed rows out
    float* partial;    // kv_decode's partial results
};

constexpr int kKvFewRows = 16;  // packed rows (rows x group) up to which kv_decode takes a sequence

struct KvMergeParams {
    KvRowsView parts;
    int64_t part_stride;  // bytes
    const float* part_lse;
    KvRowsView out;
    float* lse;
    int32_t rows, heads, part_count;
};

// dtype: GFD_* of the cache; out: of the output rows
cudaError_t launch_kv_append(const KvAppendParams& p, int head_dim, int dtype, int num_sms, cudaStream_t st);
cudaError_t launch_kv_attend(const KvAttendParams& p, int head_dim, int dtype, int out_dtype, int num_sms, cudaStream_t st);
cudaError_t launch_kv_decode(const KvAttendParams& p, int head_dim, int dtype, int num_sms, cudaStream_t st);
size_t kv_decode_workspace(int num_sms, int head_dim);
cudaError_t launch_kv_merge(const KvMergeParams& p, int head_dim, int part_dtype, int out_dtype, int num_sms,
                            cudaStream_t st);

}  // namespace gfdb
