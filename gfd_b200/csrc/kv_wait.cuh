#pragma once
// Barriers in shared memory whose waits are bounded: what kv_prompt's warps hand work to one another with.

#include <cuda_runtime.h>

#include <cstdint>

namespace gfdb {

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

__device__ __forceinline__ void bar_init(uint32_t bar, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n.reg .pred q;\nmbarrier.try_wait.parity.shared::cta.b64 q, [%1], %2;\nselp.u32 %0, 1, 0, q;\n}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ uint64_t clock_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}

// What a block's waits go by.  One warp watches: its waits run out when the block has got nowhere for the limit.
// `steps` counts what the block does (a tile takes microseconds, a unit of a long context may take seconds), and
// while `held` it waits for launches before it, which takes as long as they take.  The other warps' waits end
// when the watching one's did, which costs them no clock.
struct KvWaits {
    int gave_up;
    int held;
    uint32_t steps;
};
constexpr uint64_t kWaitLimitNs = 10000000000ull;

// false: the waits ran out
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int* gave_up) {
    for (uint32_t i = 1; !bar_try(bar, parity); ++i)
        if ((i & 255u) == 0 && *gave_up != 0) return false;
    return true;
}

// The same, of the warp that watches.
__device__ __forceinline__ bool bar_watch(uint32_t bar, uint32_t parity, volatile KvWaits* w, uint64_t limit_ns = kWaitLimitNs) {
    uint64_t t0 = 0;
    uint32_t steps = 0;
    for (uint32_t i = 1; !bar_try(bar, parity); ++i) {
        if ((i & 63u) != 0) continue;
        if (w->gave_up != 0) return false;
        const uint64_t now = clock_ns();
        if (t0 == 0 || w->steps != steps || w->held != 0) {
            t0 = now;
            steps = w->steps;
        } else if (now - t0 > limit_ns) {
            w->gave_up = 1;
            return false;
        }
    }
    return true;
}

// For copies and products in flight before a block ends, whether waits ran out or not: they land by themselves.
__device__ __forceinline__ void bar_drain(uint32_t bar, uint32_t parity, uint64_t limit_ns = kWaitLimitNs) {
    const uint64_t t0 = clock_ns();
    while (!bar_try(bar, parity) && clock_ns() - t0 < limit_ns) {
    }
}

}  // namespace gfdb
