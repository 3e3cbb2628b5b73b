// The bounded waits of the paged attention for many rows (gfd_b200/csrc/kv_wait.cuh), run out on barriers that
// nothing arrives at: one warp watches with a short limit, another waits without a clock.  Steps of the block
// and launches before it keep them waiting; the next work runs as ever.
#include "../../gfd_b200/csrc/kv_wait.cuh"

#include <chrono>

#include "common.h"

using namespace gfdb;
using clk = std::chrono::steady_clock;

constexpr uint64_t kLimitNs = 100ull * 1000 * 1000;  // 100 ms

__device__ void pass_ns(uint64_t ns) {
    const uint64_t t0 = clock_ns();
    while (clock_ns() - t0 < ns) __nanosleep(1000);
}

// out: what the watching and the waiting warp got, and whether the block gave up.
__global__ void wait_kernel(int step_ms, int held_ms, bool arrive, int* out) {
    __shared__ uint64_t bar;
    __shared__ KvWaits waits;
    const int warp = threadIdx.x / 32;
    if (threadIdx.x == 0) {
        waits = KvWaits{0, held_ms > 0, 0};
        bar_init(smem_addr(&bar), 1);
    }
    __syncthreads();
    volatile KvWaits* w = &waits;
    if (warp == 0) {
        const bool ok = bar_watch(smem_addr(&bar), 0, w, kLimitNs);
        if (threadIdx.x == 0) out[0] = ok;
    } else if (warp == 1) {
        const bool ok = bar_wait(smem_addr(&bar), 0, &w->gave_up);
        if (threadIdx.x == 32) out[1] = ok;
    } else if (threadIdx.x == 64) {
        for (int ms = 0; ms < step_ms; ms += 5) {
            pass_ns(5000000);
            w->steps = w->steps + 1;
        }
        pass_ns(held_ms * 1000000ull);
        w->held = 0;
        if (arrive) bar_arrive(smem_addr(&bar));
    }
    __syncthreads();
    if (threadIdx.x == 0) out[2] = w->gave_up;
}

__global__ void drain_kernel() {
    __shared__ uint64_t bar;
    if (threadIdx.x == 0) bar_init(smem_addr(&bar), 1);
    __syncthreads();
    bar_drain(smem_addr(&bar), 0, kLimitNs);
    bar_drain(smem_addr(&bar), 1, kLimitNs);  // the phase before the first counts as done: no wait
}

static void run(const char* name, int step_ms, int held_ms, bool arrive, bool ok, double least_ms) {
    int* out = nullptr;
    CK(cudaHostAlloc(&out, 3 * sizeof(int), cudaHostAllocMapped));
    out[0] = out[1] = out[2] = -1;
    const auto t0 = clk::now();
    wait_kernel<<<1, 96>>>(step_ms, held_ms, arrive, out);
    const cudaError_t e = cudaDeviceSynchronize();
    const double ms = std::chrono::duration<double, std::milli>(clk::now() - t0).count();
    char detail[160];
    snprintf(detail, sizeof(detail), "watch=%d wait=%d gave_up=%d after %.0f ms", out[0], out[1], out[2], ms);
    report(name, e == cudaSuccess && out[0] == ok && out[1] == ok && out[2] == !ok && ms >= least_ms && ms < 5000, detail);
    cudaFreeHost(out);
}

int main() {
    CK(cudaSetDevice(0));
    run("kv_wait_arrives", 0, 0, true, true, 0);
    run("kv_wait_runs_out", 0, 0, false, false, 90);
    run("kv_wait_steps_keep_it", 400, 0, true, true, 390);
    run("kv_wait_runs_out_after_the_last_step", 300, 0, false, false, 390);
    run("kv_wait_held_by_launches_before", 0, 400, true, true, 390);
    run("kv_wait_runs_out_once_not_held", 0, 300, false, false, 390);
    const auto t0 = clk::now();
    drain_kernel<<<1, 32>>>();
    const cudaError_t e = cudaDeviceSynchronize();
    const double ms = std::chrono::duration<double, std::milli>(clk::now() - t0).count();
    report("kv_drain_ends", e == cudaSuccess && ms >= 90 && ms < 1000);
    run("kv_wait_next_launch", 0, 0, true, true, 0);
    return g_failures ? 1 : 0;
}
