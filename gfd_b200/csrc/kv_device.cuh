#pragma once
// Device helpers shared by the paged KV-cache kernels.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "kv.h"

namespace gfdb {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// 2^x by the hardware instruction: within 2^-22 of the value, results below 2^-126 are 0
__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <typename T>
struct Pack;  // 8 elements of T <-> 8 floats, and rounding to nearest even
template <>
struct Pack<__nv_bfloat16> {
    static __device__ __forceinline__ void load(const char* p, float (&f)[8]) {
        const uint4 q = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(w[i] << 16);
            f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ uint32_t pair(float a, float b) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ void store(char* p, const float (&f)[8]) {
        *reinterpret_cast<uint4*>(p) = make_uint4(pair(f[0], f[1]), pair(f[2], f[3]), pair(f[4], f[5]), pair(f[6], f[7]));
    }
};
template <>
struct Pack<__half> {
    static __device__ __forceinline__ void load(const char* p, float (&f)[8]) {
        const uint4 q = *reinterpret_cast<const uint4*>(p);
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            f[2 * i] = v.x;
            f[2 * i + 1] = v.y;
        }
    }
    static __device__ __forceinline__ uint32_t pair(float a, float b) {
        const __half2 h = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    static __device__ __forceinline__ void store(char* p, const float (&f)[8]) {
        *reinterpret_cast<uint4*>(p) = make_uint4(pair(f[0], f[1]), pair(f[2], f[3]), pair(f[4], f[5]), pair(f[6], f[7]));
    }
};
template <>
struct Pack<float> {
    static __device__ __forceinline__ void load(const char* p, float (&f)[8]) {
        *reinterpret_cast<float4*>(&f[0]) = reinterpret_cast<const float4*>(p)[0];
        *reinterpret_cast<float4*>(&f[4]) = reinterpret_cast<const float4*>(p)[1];
    }
    static __device__ __forceinline__ void store(char* p, const float (&f)[8]) {
        reinterpret_cast<float4*>(p)[0] = *reinterpret_cast<const float4*>(&f[0]);
        reinterpret_cast<float4*>(p)[1] = *reinterpret_cast<const float4*>(&f[4]);
    }
};

// row_start rises from >= 0 to <= rows (every thread of the CTA calls; same answer for all).
__device__ __forceinline__ bool kv_starts_ok(const KvBatchView& b) {
    bool bad = false;
    for (int i = threadIdx.x; i < b.seqs; i += blockDim.x) {
        const int32_t a = b.row_start[i], e = b.row_start[i + 1];
        bad |= a < 0 || a > e || e > b.rows;
    }
    return __syncthreads_or(bad) == 0;
}

__device__ __forceinline__ void kv_report(uint32_t* status, uint32_t bits) {
    if (status != nullptr && bits != 0) atomicOr(status, bits);
}

// Address of token j of a sequence (its own table and the shared prefix in front of it);
// null: the block id is outside the cache.
__device__ __forceinline__ int32_t kv_block(const KvBatchView& b, int s, int32_t j, int32_t bt, const int32_t* shared_table,
                                            int32_t shared_len, int32_t* place) {
    const int32_t* t = shared_table;
    if (j >= shared_len) {
        t = b.table + s * b.table_stride;
        j -= shared_len;
    }
    *place = j % bt;
    return t[j / bt];
}

}  // namespace gfdb
