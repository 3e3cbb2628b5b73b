#pragma once
// Device helpers shared by the paged KV-cache kernels.

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <type_traits>

#include "kv.h"

namespace gfdb {

constexpr float kLog2e = 1.4426950408889634f;

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
    static __device__ __forceinline__ void unpair(uint32_t w, float& a, float& b) {
        a = __uint_as_float(w << 16);
        b = __uint_as_float(w & 0xffff0000u);
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
    static __device__ __forceinline__ void unpair(uint32_t w, float& a, float& b) {
        const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w));
        a = v.x;
        b = v.y;
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

// Launches of one call overlap (programmatic dependent launch): each lets the next one start at
// once and, before it reads what an earlier one wrote or ends, waits for that one to complete.  As
// every CTA waits before it ends, the completion of a launch implies that of all before it.
__device__ __forceinline__ void kv_let_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void kv_wait_last() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// n / group for 0 <= n < 2^31: the rounded-up reciprocal errs by less than group <= 2^13 in 2^44, so
// n times it stays below the next whole quotient.
__device__ __forceinline__ int32_t kv_div_group(const KvAttendParams& p, int32_t n) {
    return static_cast<int32_t>(__umul64hi(static_cast<uint64_t>(n) << 20, p.group_magic));
}

// n / (pages of a block) for 0 <= n < 2^26 and up to 64 pages: n times pages stays below 2^32.
__device__ __forceinline__ int32_t kv_div_pages(const KvAttendParams& p, int32_t n) {
    return static_cast<int32_t>(static_cast<uint64_t>(n) * p.page_magic >> 32);
}

__device__ __forceinline__ void kv_report(uint32_t* status, uint32_t bits) {
    if (status != nullptr && bits != 0) atomicOr(status, bits);
}

// What CTA c's cut leaves to join, for the CTA whose stretch begins at `at`.
__device__ __forceinline__ KvCut kv_cut(const KvCuts& cuts, uint32_t c, const KvPlace& at) {
    KvCut k{0, at.row0, at.packed0, at.packed, at.h};
    if (c > 0 && at.t > 0 && cuts.at(c - 1) <= at.begin) k.parts = static_cast<int32_t>(cuts.last_before(c, at.begin + at.count) - c) + 2;
    return k;
}

// Marks the rows of a sequence that is skipped, for the pass over the shared prefix (one thread calls).
__device__ __forceinline__ void kv_mark_skipped(const KvAttendParams& p, int s) {
    if (p.skipped_lse == nullptr) return;
    const int64_t from = static_cast<int64_t>(p.batch.row_start[s]) * p.q_heads, to = static_cast<int64_t>(p.batch.row_start[s + 1]) * p.q_heads;
    for (int64_t i = from; i < to; ++i) reinterpret_cast<uint32_t*>(p.skipped_lse)[i] = kKvSkipped;
}

__device__ __forceinline__ float kv_lse(const KvAttendParams& p, float base, float sum) {
    return sum == 0.0f ? -INFINITY : fmaf(base, p.to_ln, logf(sum));
}

// What becomes of a row's sums (relative to 2^base, weights adding up to sum): multiplied by `scale`
// they are the result; behind a shared prefix the result over the own keys, times `own`, is
// added.  base and sum: of both together.
struct KvFinish {
    float scale, own, base, sum;
};
template <bool kShared>
__device__ __forceinline__ KvFinish kv_finish(const KvAttendParams& p, float base, float sum, float own_lse) {
    KvFinish f{0.0f, 0.0f, base, sum};
    const float own = kShared ? own_lse / p.to_ln : -INFINITY;
    if (own == -INFINITY) {
        if (sum != 0.0f) f.scale = 1.0f / sum;
        return f;
    }
    f.base = fmaxf(base, own);
    const float a = base == -INFINITY ? (sum == 0.0f ? 0.0f : 1.0f) : fast_exp2(base - f.base), b = fast_exp2(own - f.base);
    f.sum = (sum == 0.0f ? 0.0f : sum * a) + b;
    f.scale = a / f.sum;
    f.own = b / f.sum;
    return f;
}

// Pairs of 32-bit numbers, one instruction for both.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t r, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}

// cap * tanh(x) in base 2 for any x: tanh x = 1 - 2 / (1 + e^2x), to about 2^-21
__device__ __forceinline__ float kv_tanh2(const KvAttendParams& p, float x) {
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + fast_exp2(x * (2.0f * kLog2e))));
    return fmaf(-2.0f * p.cap2, r, p.cap2);
}

// cap * tanh in base 2 of both products, |cap_x times them| up to 3/4: tanh x is x P(x^2) on the FMA units, P = 1 + ...
// of degree 5 by least largest relative error (2^-24.9; 2^-22.9 with the roundings).
__device__ __forceinline__ uint64_t kv_tanh2_small(const KvAttendParams& p, uint64_t z) {
    const uint64_t x = mul2(z, pack2(p.cap_x, p.cap_x)), y = mul2(x, x);
    uint64_t q = fma2(y, pack2(-0.004769490100443363f, -0.004769490100443363f), pack2(0.019664913415908813f, 0.019664913415908813f));
    q = fma2(q, y, pack2(-0.0533902570605278f, -0.0533902570605278f));
    q = fma2(q, y, pack2(0.13326521217823029f, 0.13326521217823029f));
    q = fma2(q, y, pack2(-0.3333306908607483f, -0.3333306908607483f));
    q = fma2(q, y, pack2(1.0f, 1.0f));
    return mul2(mul2(q, x), pack2(p.cap2, p.cap2));
}

// N products of queries and keys to scores in base 2: scaled, capped where the call has a cap.
// Where a thread's products all lie within three quarters of the cap tanh is a polynomial; usually those of the
// whole warp do, and the special-function unit, which the exponentials need, is left out.  The choice, and
// with it a result's last bits, goes by what the row sees and not by its neighbours: otherwise the largest
// product is looked for among the keys that `sees` (of 32 keys a word, asked where `masked`).
template <int N, typename F>
__device__ __forceinline__ void kv_cap(const KvAttendParams& p, uint32_t* z, bool masked, F sees) {
    if (p.softcap > 0.0f) {
        float m = 0.0f;
#pragma unroll
        for (int e = 0; e < N; ++e) m = fmaxf(m, fabsf(__uint_as_float(z[e])));
        if (__all_sync(0xffffffffu, m * fabsf(p.cap_x) <= 0.75f)) {
#pragma unroll
            for (int e = 0; e < N; e += 2) {
                float a, b;
                unpack2(kv_tanh2_small(p, pack2(__uint_as_float(z[e]), __uint_as_float(z[e + 1]))), a, b);
                z[e] = __float_as_uint(a);
                z[e + 1] = __float_as_uint(b);
            }
        } else {
            if (masked) {
                m = 0.0f;
#pragma unroll
                for (int k = 0; k < N; k += 32) {
                    const uint32_t some = sees(k);
#pragma unroll
                    for (int e = k; e < k + 32 && e < N; ++e)
                        if (some >> (e - k) & 1u) m = fmaxf(m, fabsf(__uint_as_float(z[e])));
                }
            }
            const bool small = m * fabsf(p.cap_x) <= 0.75f;
#pragma unroll
            for (int e = 0; e < N; e += 2) {
                const float x = __uint_as_float(z[e]), y = __uint_as_float(z[e + 1]);
                float a, b;
                unpack2(kv_tanh2_small(p, pack2(x, y)), a, b);
                z[e] = __float_as_uint(small ? a : kv_tanh2(p, x * p.cap_x));
                z[e + 1] = __float_as_uint(small ? b : kv_tanh2(p, y * p.cap_x));
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) z[e] = __float_as_uint(__uint_as_float(z[e]) * p.scale2);
    }
}

template <typename... P, typename... A>
cudaError_t kv_launch(void (*kernel)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, bool chained, A... args) {
    if (smem > 32 * 1024) {  // with the static part more than 48 KB
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
        if (e != cudaSuccess) return e;
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = chained ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

}  // namespace gfdb
