// Attention for sequences with many rows (prompts, chunks, drafts of wide groups) on the
// 5th-generation tensor cores.
//
// A unit is 256 packed rows ((row, query head of the KV head's group) pairs, rows outermost) of one
// sequence against the keys they see, 128 at a time; two halves A and B of 128 rows share
// the keys.  Per half and tile: S = Q K^T (tcgen05.mma, 128 x 128 x D, both operands in shared
// memory), a softmax thread per row takes its row of S out of tensor memory, writes the weights
// back over it in the 16-bit type, and O += P V (P from tensor memory, V from shared memory,
// O in tensor memory).  While one half is in softmax the other one's products run.
//
// The running maximum moves only when a row's scores grow by more than 2^8 over it: until then
// the weights are at most 2^8 and the sums stay in tensor memory untouched, so the rescaling
// of O is rare.  Sums and maxima are 32-bit; the weights' rounding to the 16-bit type for the
// second product is the only one before the result's.
//
// Roles: warps 0-3 softmax of half A, 4-7 of half B, warp 8 issues the products, warp 9 loads K
// and V (TMA boxes of 16 tokens x 64 elements, so that every page is found by its id).
// Units lie on one line of tiles that the CTAs (one per SM) share evenly; a cut unit leaves
// partial sums for kv_join_kernel, as in kv_decode.cu.

#include <cuda.h>

#include <type_traits>

#include "kv_device.cuh"

namespace gfdb {
namespace {

constexpr int kRows = kKvManyRows;  // packed rows of a unit
constexpr int kHalf = 128;          // rows of a half: one tensor-core tile
constexpr int kTile = 128;          // keys of a step
constexpr int kPages = kTile / kKvPage;
constexpr int kThreads = 320;
constexpr int kBadRing = 8;         // tiles whose bad pages are remembered

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }

// ---- barriers: every wait is bounded ----
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
constexpr uint64_t kWaitLimitNs = 2000000000ull;
__device__ __forceinline__ uint64_t clock_ns() {
    uint64_t t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
// false: the wait ran out, or another warp's did
__device__ __noinline__ bool bar_wait_slow(uint32_t bar, uint32_t parity, volatile int* gave_up) {
    const uint64_t t0 = clock_ns();
    for (;;) {
        for (int i = 0; i < 64; ++i)
            if (bar_try(bar, parity)) return true;
        if (*gave_up != 0) return false;
        if (clock_ns() - t0 > kWaitLimitNs) {
            *gave_up = 1;
            return false;
        }
    }
}
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, volatile int* gave_up) {
    for (int i = 0; i < 16; ++i)
        if (bar_try(bar, parity)) return true;
    return bar_wait_slow(bar, parity, gave_up);
}

// ---- tensor memory and products ----
__device__ __forceinline__ void tm_ld32(uint32_t addr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, "
        "%19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void tm_st32(uint32_t addr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, "
        "%18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]),
        "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31]),
        "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tm_st16(uint32_t addr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
        : "memory");
}
// waits for the loads issued so far; r, loaded by one of them, is not read before
__device__ __forceinline__ void tm_wait32(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), "+r"(r[8]),
                   "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]), "+r"(r[16]),
                   "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]),
                   "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
}
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// Shared-memory operand in 128-byte swizzle: rows of 128 bytes in groups of 8 (1024 bytes).
// group: bytes from one group of 8 rows to the next; block: bytes between 64-element blocks of a
// row-major second operand's columns (not used by the K-major ones).
__device__ __forceinline__ uint64_t operand(uint32_t addr, uint32_t block, uint32_t group) {
    return static_cast<uint64_t>((addr & 0x3ffffu) >> 4) | static_cast<uint64_t>(block >> 4) << 16 |
           static_cast<uint64_t>(group >> 4) << 32 | 1ull << 46 | 2ull << 61;
}
// 32-bit sums of 16-bit products; second operand's columns contiguous (trans) or not
template <typename T>
__device__ __forceinline__ constexpr uint32_t product(int m, int n, bool trans) {
    const uint32_t fmt = std::is_same<T, __half>::value ? 0u : 1u;
    return 1u << 4 | fmt << 7 | fmt << 10 | (trans ? 1u << 16 : 0u) | static_cast<uint32_t>(n >> 3) << 17 |
           static_cast<uint32_t>(m >> 4) << 24;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a),
                 "l"(b), "r"(idesc), "r"(add ? 1u : 0u)
                 : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool add) {
    asm volatile("{\n.reg .pred p;\nsetp.ne.u32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d), "r"(a),
                 "l"(b), "r"(idesc), "r"(add ? 1u : 0u)
                 : "memory");
}
__device__ __forceinline__ void tma_page(uint32_t dst, const CUtensorMap* map, int x, int head, int place, int block, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(map), "r"(x), "r"(head), "r"(place), "r"(block), "r"(bar)
        : "memory");
}

// ---------------------------------------------------------------------------
// Units
// ---------------------------------------------------------------------------
// What the launch walks over: the sequences with many rows, or (shared pass) all rows of the
// batch as one sequence against the shared prefix.
struct Many {
    KvSeq q;       // rows and keys (keys in the count of this pass)
    int32_t tiles; // row tiles
    bool bad;
};

__device__ __forceinline__ Many many_seq(const KvAttendParams& p, int s) {
    const KvBatchView& b = p.batch;
    Many r;
    if (p.shared_pass) {
        r.q = KvSeq{b.row_start[0], b.row_start[b.seqs] - b.row_start[0], p.shared_len, true};
        r.bad = false;
    } else {
        r.q = kv_seq(b.row_start[s], b.row_start[s + 1], b.kv_len[s], b.capacity, p.max_q_len);
        r.bad = !r.q.ok;
        if (r.bad || r.q.rows * p.group <= kKvFewRows) r.q.rows = r.q.keys = 0;
    }
    r.tiles = static_cast<int32_t>((static_cast<int64_t>(r.q.rows) * p.group + kRows - 1) / kRows);
    return r;
}

struct Unit {
    KvSpan all;  // pre, least lo, greatest hi of its rows
    KvTiles tiles;
    int32_t packed0, packed;
};

__device__ __forceinline__ Unit many_unit(const KvAttendParams& p, int s, const KvSeq& q, int rt) {
    Unit u;
    const int64_t packed = static_cast<int64_t>(q.rows) * p.group;
    u.packed0 = rt * kRows;
    u.packed = static_cast<int32_t>(min(static_cast<int64_t>(kRows), packed - u.packed0));
    if (p.shared_pass) {
        // every row stands behind the prefix; with a window the rows nearest to it see most
        u.all = KvSpan{0, 0, p.shared_len};
        if (p.window > 0 && p.prefix_len == nullptr) u.all.lo = min(p.shared_len, max(0, p.shared_len + 1 - p.window));
        if (p.window > 0 && u.all.lo >= p.shared_len) u.all.hi = u.all.lo = p.shared_len;
    } else {
        const int32_t n = p.shared_len + q.keys, pos0 = n - q.rows;
        const int32_t prefix = p.prefix_len != nullptr ? p.prefix_len[s] : 0;
        const KvSpan first = kv_clip(kv_span(pos0 + u.packed0 / p.group, n, prefix, p.window, p.causal != 0), p.shared_len, q.keys);
        const KvSpan last =
            kv_clip(kv_span(pos0 + (u.packed0 + u.packed - 1) / p.group, n, prefix, p.window, p.causal != 0), p.shared_len, q.keys);
        u.all = KvSpan{first.pre, first.lo, last.hi};
    }
    u.tiles = kv_tiles(u.all, kTile);
    if (u.tiles.count == 0) u.tiles = KvTiles{1, 0, 1};  // rows that see nothing are written all the same
    return u;
}

struct Cursor {
    Many m;
    Unit u;
    int32_t s, h, rt, t, end;
    int64_t left;
    bool done;

    __device__ __forceinline__ void enter(const KvAttendParams& p, const KvPlace& at, int64_t len) {
        s = at.s;
        h = at.h;
        rt = at.packed0 / kRows;
        t = at.t;
        m = many_seq(p, s);
        u = many_unit(p, s, m.q, rt);
        clamp(len);
    }
    __device__ __forceinline__ void clamp(int64_t l) {
        done = l <= 0;
        end = static_cast<int32_t>(min(static_cast<int64_t>(u.tiles.count), t + l));
        left = l - (end - t);
    }
    // The line runs over KV heads, within a head over sequences, within a sequence over row tiles.
    __device__ __forceinline__ void next(const KvAttendParams& p) {
        if (left <= 0) {
            done = true;
            return;
        }
        t = 0;
        if (++rt >= m.tiles) {
            rt = 0;
            do {
                if (++s >= (p.shared_pass ? 1 : p.batch.seqs)) {
                    s = 0;
                    ++h;
                }
                m = many_seq(p, s);
            } while (m.tiles == 0);
        }
        u = many_unit(p, s, m.q, rt);
        clamp(left);
    }
};

// Inclusive sum over the CTA's threads.
__device__ __forceinline__ int64_t cta_scan(int64_t v, int64_t* warps, int64_t* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += y;
    }
    __syncthreads();
    if (lane == 31) warps[warp] = v;
    __syncthreads();
    int64_t before = 0, all = 0;
    for (int w = 0; w < kThreads / 32; ++w) {
        if (w < warp) before += warps[w];
        all += warps[w];
    }
    *total = all;
    return v + before;
}

// ---------------------------------------------------------------------------
// Shared memory
// ---------------------------------------------------------------------------
template <int D>
struct Shape {
    static constexpr int kBlocks = D / 64;                // 64-element blocks of a row
    static constexpr int kOperand = kHalf * D * 2;        // bytes of Q of a half, K or V of a tile
    static constexpr int kBlock = kHalf * 128;            // bytes of a 64-element block of one
    static constexpr int kSlots = 4;                      // K and V tiles in flight
    static constexpr int kSmem = 2 * kOperand + kSlots * kOperand + 1024;
    static constexpr uint32_t kColumns = 512;             // S, S, O, O
    static constexpr uint32_t kO = 256;                   // O of half A
};

struct Bars {
    uint64_t full[8], empty[8];
    uint64_t q[2], s[2], p[2], o[2];
};

template <typename T>
struct Shift {  // weights reach 2^(shift + 8): fp16 keeps them clear of its small values' coarse steps
    static constexpr float value = std::is_same<T, __half>::value ? 6.0f : 0.0f;
};
constexpr float kGrow = 8.0f;

template <typename T, int D, bool kPlain>
__global__ void __launch_bounds__(kThreads, 1)
    kv_prompt_kernel(const KvAttendParams p, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v) {
    using S = Shape<D>;
    extern __shared__ char smem_raw[];
    __shared__ Bars bars;
    __shared__ KvPlace s_place;
    __shared__ int64_t s_warps[kThreads / 32];
    __shared__ uint32_t s_tmem;
    __shared__ int s_gave_up;
    __shared__ uint32_t s_bad[kBadRing];
    char* smem = reinterpret_cast<char*>((reinterpret_cast<uint64_t>(smem_raw) + 1023) & ~1023ull);
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const KvBatchView& b = p.batch;

    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (t == 0) {
        s_place = KvPlace{};
        s_gave_up = 0;
        for (int i = 0; i < S::kSlots; ++i) {
            bar_init(smem_addr(&bars.full[i]), 1);
            bar_init(smem_addr(&bars.empty[i]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            bar_init(smem_addr(&bars.q[i]), kHalf);
            bar_init(smem_addr(&bars.s[i]), 1);
            bar_init(smem_addr(&bars.p[i]), kHalf);
            bar_init(smem_addr(&bars.o[i]), 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }

    // ---- this CTA's stretch of the line ----
    int64_t len = 0;
    {
        const bool ok = kv_starts_ok(b);  // syncs
        if (!ok && blockIdx.x == 0 && t == 0) kv_report(p.status, GFD_KV_BAD_LENGTH);
        const int seqs = !ok ? 0 : (p.shared_pass ? 1 : b.seqs);
        // first row tile of every sequence, kept where the operands will lie
        int32_t* first = reinterpret_cast<int32_t*>(smem);
        const int per = (seqs + kThreads - 1) / kThreads;
        int64_t mine = 0, row_tiles = 0;
        for (int s = t * per; s < min((t + 1) * per, seqs); ++s) {
            const Many m = many_seq(p, s);
            if (m.bad && blockIdx.x == 0) kv_report(p.status, GFD_KV_BAD_LENGTH);
            mine += m.tiles;
        }
        int64_t run = cta_scan(mine, s_warps, &row_tiles) - mine;
        for (int s = t * per; s < min((t + 1) * per, seqs); ++s) {
            first[s] = static_cast<int32_t>(run);
            run += many_seq(p, s).tiles;
        }
        __syncthreads();
        // tiles of this thread's row tiles, then where the stretch begins
        const int64_t each = (row_tiles + kThreads - 1) / kThreads;
        const int64_t u0 = min(t * each, row_tiles), u1 = min(u0 + each, row_tiles);
        int s0 = 0;
        if (u0 < u1) {
            int lo = 0, hi = seqs - 1;
            while (lo < hi) {
                const int mid = (lo + hi + 1) / 2;
                if (first[mid] <= u0) lo = mid;
                else hi = mid - 1;
            }
            s0 = lo;
        }
        int64_t per_head = 0, total = 0, at = 0;
        bool none = false;
        for (int pass = 0; pass < 2; ++pass) {
            int s = s0;
            Many m{};
            if (u0 < u1) m = many_seq(p, s);
            int64_t sum = 0;
            for (int64_t u = u0; u < u1; ++u) {
                while (u - first[s] >= m.tiles) m = many_seq(p, ++s);
                const int rt = static_cast<int>(u - first[s]);
                const Unit x = many_unit(p, s, m.q, rt);
                if (pass == 1 && !none) {
                    const int64_t want = at % per_head, here = mine + sum;
                    if (want >= here && want < here + x.tiles.count) {
                        s_place.s = s;
                        s_place.h = static_cast<int32_t>(at / per_head);
                        s_place.t = static_cast<int32_t>(want - here);
                        s_place.count = x.tiles.count;
                        s_place.begin = at - (want - here);
                        s_place.row0 = m.q.row0;
                        s_place.packed0 = x.packed0;
                        s_place.packed = x.packed;
                    }
                }
                sum += x.tiles.count;
            }
            if (pass == 0) {
                mine = cta_scan(sum, s_warps, &per_head) - sum;
                total = per_head * p.cache.heads;
                const KvCuts cuts(total, gridDim.x);
                none = static_cast<int>(blockIdx.x) >= cuts.n();
                if (!none) {
                    at = cuts.at(blockIdx.x);
                    len = cuts.at(blockIdx.x + 1) - at;
                }
            }
        }
        __syncthreads();
        if (t == 0) {
            s_place.total = total;
            p.line.places[blockIdx.x] = s_place;
        }
    }
    if (len <= 0) return;

    if (warp == 8) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)), "r"(S::kColumns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tm_before();
    __syncthreads();
    tm_after();
    const uint32_t tmem = s_tmem;
    const uint32_t sq = smem_addr(smem), ring = sq + 2 * S::kOperand;
    volatile int* gave_up = &s_gave_up;
    const KvPlace place = s_place;

    if (warp == 9) {
        // ---- K and V ----
        Cursor c;
        c.enter(p, place, len);
        int slot = 0, seen = 0;  // seen: tiles so far
        uint32_t phase = 0;      // bit i: parity that slot i's `empty` has to reach
        bool good = true;
        const int pages = p.cache.block_tokens / kKvPage;
        while (good && !c.done) {
            const int32_t* table = p.shared_pass ? p.shared_table : b.table + c.s * b.table_stride;
            const int32_t n = c.m.q.keys;
            for (; good && c.t < c.end; ++c.t, ++seen) {
                const int32_t j0 = c.u.tiles.at(c.t) * kTile;
                // lane i: page i % 8 of the tile
                const int32_t j = j0 + (lane % kPages) * kKvPage;
                int32_t id = p.cache.blocks;  // a block outside the map: loads as zeros
                bool bad = false;
                if ((j < c.u.all.pre || (j + kKvPage > c.u.all.lo && j < c.u.all.hi)) && j < n) {
                    id = table[j / kKvPage / pages];
                    if (id < 0 || id >= p.cache.blocks) {
                        bad = true;
                        id = p.cache.blocks;
                        kv_report(p.status, GFD_KV_BAD_PAGE);
                    }
                }
                const int32_t in_block = (j / kKvPage % pages) * kKvPage;
                const uint32_t bad_pages = __ballot_sync(0xffffffffu, bad) & 0xffu;
                // a page that the sequence ends in: V's tokens behind the end are kept out by hand,
                // whatever lies there would meet weights of zero
                const int32_t rest = n - j0;
                const int cut_page = rest > 0 && rest < kTile && rest % kKvPage != 0 ? rest / kKvPage : -1;
                for (int which = 0; good && which < 2; ++which) {  // K, V
                    const uint32_t full = smem_addr(&bars.full[slot]);
                    good = bar_wait(smem_addr(&bars.empty[slot]), ((phase >> slot) & 1u) ^ 1u, gave_up);
                    if (!good) break;
                    const uint32_t dst = ring + slot * S::kOperand;
                    const bool by_hand = which == 1 && cut_page >= 0;
                    if (which == 0 && lane == 0) s_bad[seen % kBadRing] = bad_pages;
                    if (by_hand) {
                        const int32_t hid = __shfl_sync(0xffffffffu, id, cut_page), hpl = __shfl_sync(0xffffffffu, in_block, cut_page);
                        const char* src = p.cache.v + (hid < p.cache.blocks ? hid : 0) * p.cache.block_stride + hpl * p.cache.token_stride +
                                          c.h * p.cache.head_stride;
                        for (int i = lane; i < kKvPage * D / 8; i += 32) {
                            const int r = i / (D / 8), ch = i % (D / 8);
                            uint4 v = make_uint4(0, 0, 0, 0);
                            if (hid < p.cache.blocks && r < rest % kKvPage)
                                v = *reinterpret_cast<const uint4*>(src + r * p.cache.token_stride + 16 * ch);
                            const uint32_t o = dst + (ch / 8) * S::kBlock + (cut_page * kKvPage + r) * 128 + (((ch % 8) ^ (r & 7)) << 4);
                            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(o), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    }
                    __syncwarp();
                    if (lane == 0) bar_expect(full, S::kOperand - (by_hand ? kKvPage * D * 2 : 0));
                    __syncwarp();
                    const int page = lane % kPages, block = lane / kPages;
                    if (block < S::kBlocks && !(by_hand && page == cut_page))
                        tma_page(dst + block * S::kBlock + page * kKvPage * 128, which == 0 ? &map_k : &map_v, block * 64, c.h, in_block, id,
                                 full);
                    phase ^= 1u << slot;
                    slot = slot + 1 == S::kSlots ? 0 : slot + 1;
                }
            }
            if (good) c.next(p);
        }
        if (!good) {
            // the copies in flight land before the block ends: `full` flips once more for each slot
            // that was filled and not yet waited for
            for (int i = 0; i < S::kSlots; ++i) {
                const uint64_t t0 = clock_ns();
                while (!bar_try(smem_addr(&bars.full[i]), ((phase >> i) & 1u) ^ 1u) && clock_ns() - t0 < kWaitLimitNs) {
                }
            }
        }
    } else if (warp == 8) {
        // ---- products ----
        if (lane == 0) {
            Cursor c;
            c.enter(p, place, len);
            int slot = 0;
            uint32_t full_phase = 0, q_phase = 0, p_phase = 0;
            bool good = true;
            constexpr uint32_t kQk = product<T>(kHalf, kTile, false);
            constexpr uint32_t kPv = product<T>(kHalf, D, true);
            auto scores = [&](int x, int k) {
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    const uint32_t o = (i / 4) * S::kBlock + (i % 4) * 32;
                    mma_ss(tmem + x * kTile, operand(sq + x * S::kOperand + o, 16, 1024), operand(ring + k * S::kOperand + o, 16, 1024), kQk,
                           i > 0);
                }
            };
            while (good && !c.done) {
                const int halves = c.u.packed > kHalf ? 2 : 1;
                const int nt = c.end - c.t;
                for (int x = 0; good && x < halves; ++x) {
                    good = bar_wait(smem_addr(&bars.q[x]), (q_phase >> x) & 1u, gave_up);
                    q_phase ^= 1u << x;
                }
                if (good) good = bar_wait(smem_addr(&bars.full[slot]), (full_phase >> slot) & 1u, gave_up);
                if (!good) break;
                tm_after();
                for (int x = 0; x < halves; ++x) {
                    scores(x, slot);
                    tm_commit(smem_addr(&bars.s[x]));
                }
                tm_commit(smem_addr(&bars.empty[slot]));
                full_phase ^= 1u << slot;
                slot = slot + 1 == S::kSlots ? 0 : slot + 1;
                for (int i = 0; good && i < nt; ++i) {
                    const int v = slot, k = slot + 1 == S::kSlots ? 0 : slot + 1;
                    good = bar_wait(smem_addr(&bars.full[v]), (full_phase >> v) & 1u, gave_up);
                    full_phase ^= 1u << v;
                    for (int x = 0; good && x < halves; ++x) {
                        good = bar_wait(smem_addr(&bars.p[x]), (p_phase >> x) & 1u, gave_up);
                        p_phase ^= 1u << x;
                        if (!good) break;
                        tm_after();
#pragma unroll
                        for (int j = 0; j < kTile / 16; ++j)
                            mma_ts(tmem + S::kO + x * D, tmem + x * kTile + j * 8, operand(ring + v * S::kOperand + j * 2048, S::kBlock, 1024),
                                   kPv, i > 0 || j > 0);
                        if (x == halves - 1) tm_commit(smem_addr(&bars.empty[v]));
                        if (i + 1 < nt) {
                            if (x == 0) {
                                good = bar_wait(smem_addr(&bars.full[k]), (full_phase >> k) & 1u, gave_up);
                                full_phase ^= 1u << k;
                                if (!good) break;
                                tm_after();
                            }
                            scores(x, k);
                            tm_commit(smem_addr(&bars.s[x]));
                            if (x == halves - 1) tm_commit(smem_addr(&bars.empty[k]));
                        } else {
                            tm_commit(smem_addr(&bars.o[x]));
                        }
                    }
                    slot = k;
                    if (i + 1 < nt) slot = k + 1 == S::kSlots ? 0 : k + 1;
                }
                if (good) c.next(p);
            }
        }
        __syncwarp();
    } else {
        // ---- softmax: one thread per packed row ----
        const int x = warp >> 2;
        const int rr = t & (kHalf - 1);                                        // row of the half
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;  // this warp's lanes of tensor memory
        const uint32_t ts = tmem + lanes + x * kTile, to = tmem + lanes + S::kO + x * D;
        Cursor c;
        c.enter(p, place, len);
        uint32_t s_phase = 0, o_phase = 0;
        int seen = 0;
        bool good = true;
        while (good && !c.done) {
            const int32_t t0 = c.t, nt = c.end - c.t;
            if (x * kHalf >= c.u.packed) {  // this half has no rows
                seen += nt;
                c.next(p);
                continue;
            }
            const int r = x * kHalf + rr;  // row of the unit
            const bool valid = r < c.u.packed;
            const int32_t packed = c.u.packed0 + (valid ? r : 0);
            const int64_t row = c.m.q.row0 + packed / p.group;
            const int32_t head = c.h * p.group + packed % p.group;
            // position and span; rows that do not exist see everything, of a zero query
            int32_t pos = p.shared_len + c.m.q.keys - c.m.q.rows + packed / p.group;
            const int32_t base_key = p.shared_pass ? 0 : p.shared_len;
            KvSpan sp{0x7fffffff, 0, 0};
            if (valid) {
                int s = c.s;
                int32_t n = p.shared_len + c.m.q.keys;
                if (p.shared_pass) {
                    pos = 0x3fffffff;
                    n = p.shared_len;
                    if (p.window > 0 || p.prefix_len != nullptr || !kPlain) {
                        int lo = 0, hi = b.seqs - 1;
                        while (lo < hi) {
                            const int mid = (lo + hi + 1) / 2;
                            if (b.row_start[mid] <= row) lo = mid;
                            else hi = mid - 1;
                        }
                        s = lo;
                        n = p.shared_len + b.kv_len[s];
                        pos = n - (b.row_start[s + 1] - static_cast<int32_t>(row));
                    }
                }
                sp = kv_clip(kv_span(pos, n, p.prefix_len != nullptr ? p.prefix_len[s] : 0, p.window, p.causal != 0), base_key, c.m.q.keys);
            }
            const float slope = !kPlain && p.alibi != nullptr ? p.alibi[head] : 0.0f;
            // this row of Q; the sign of the scale goes into it
            {
                const char* src = p.q.data + row * p.q.row_stride + head * p.q.head_stride;
                const uint32_t flip = kPlain && p.scale2 < 0.0f ? 0x80008000u : 0u;
                const uint32_t dst = sq + x * S::kOperand + rr * 128;
#pragma unroll
                for (int i = 0; i < D / 8; ++i) {
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (valid) v = *reinterpret_cast<const uint4*>(src + 16 * i);
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + (i / 8) * S::kBlock + (((i % 8) ^ (rr & 7)) << 4)),
                                 "r"(v.x ^ flip), "r"(v.y ^ flip), "r"(v.z ^ flip), "r"(v.w ^ flip)
                                 : "memory");
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                bar_arrive(smem_addr(&bars.q[x]));
            }
            const float scale = kPlain ? fabsf(p.scale2) : 1.0f;
            float base = -INFINITY, l = 0.0f;  // the weights' base (2^base), -inf before the first key; their sum
            for (int i = 0; i < nt; ++i, ++seen) {
                good = bar_wait(smem_addr(&bars.s[x]), s_phase & 1u, gave_up);
                s_phase ^= 1u;
                if (!good) break;
                tm_after();
                const int32_t j0 = c.u.tiles.at(t0 + i) * kTile;
                const uint32_t bad = *reinterpret_cast<volatile uint32_t*>(&s_bad[seen % kBadRing]);
                const bool inside = (j0 >= sp.lo && j0 + kTile <= sp.hi) || sp.pre >= j0 + kTile;
                const bool masked = __any_sync(0xffffffffu, !inside) || bad != 0;
                uint32_t buf[2][32];
                // the scores' maximum; what cap, bias and masks make of them goes back in place
                float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
                tm_ld32(ts, buf[0]);
#pragma unroll
                for (int k = 0; k < kTile / 32; ++k) {
                    uint32_t* z = buf[k & 1];
                    tm_wait32(z);
                    if (k + 1 < kTile / 32) tm_ld32(ts + 32 * (k + 1), buf[(k + 1) & 1]);
                    if (!kPlain)
#pragma unroll
                        for (int e = 0; e < 32; ++e)
                            z[e] = __float_as_uint(kv_score2<false>(p, __uint_as_float(z[e]), slope, base_key + j0 + 32 * k + e - pos));
                    if (masked)
#pragma unroll
                        for (int e = 0; e < 32; ++e) {
                            const int32_t j = j0 + 32 * k + e;
                            const bool sees = (j < sp.pre || (j >= sp.lo && j < sp.hi)) && !((bad >> ((32 * k + e) / kKvPage)) & 1u);
                            z[e] = sees ? z[e] : 0xff800000u;
                        }
#pragma unroll
                    for (int e = 0; e < 32; ++e) m4[e & 3] = fmaxf(m4[e & 3], __uint_as_float(z[e]));
                    if (!kPlain || masked) tm_st32(ts + 32 * k, z);
                }
                if (!kPlain || masked) tm_wait_st();
                const float top = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3])) * scale - Shift<T>::value;
                const bool grew = top > base + kGrow || (base == -INFINITY && top > -INFINITY);
                if (__any_sync(0xffffffffu, grew)) {
                    const float to_base = fmaxf(base, top);
                    const float keep = to_base == -INFINITY ? 1.0f : fast_exp2(base - to_base);
                    base = to_base;
                    l *= keep;
                    if (i > 0) {
                        for (int k = 0; k < D / 32; ++k) {
                            uint32_t* o = buf[1];
                            tm_ld32(to + 32 * k, o);
                            tm_wait32(o);
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                            tm_st32(to + 32 * k, o);
                        }
                    }
                }
                tm_ld32(ts, buf[0]);
                const float less = base == -INFINITY ? 0.0f : base;
                float l4[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int k = 0; k < kTile / 32; ++k) {
                    const uint32_t* z = buf[k & 1];
                    tm_wait32(buf[k & 1]);
                    // the weights of columns 32 k .. 32 k + 31 take columns 16 k .. 16 k + 15, read before
                    if (k + 1 < kTile / 32) tm_ld32(ts + 32 * (k + 1), buf[(k + 1) & 1]);
                    uint32_t w[16];
#pragma unroll
                    for (int e = 0; e < 32; e += 2) {
                        const float a = fast_exp2(fmaf(__uint_as_float(z[e]), scale, -less));
                        const float d = fast_exp2(fmaf(__uint_as_float(z[e + 1]), scale, -less));
                        l4[(e / 2) & 3] += a + d;
                        w[e / 2] = Pack<T>::pair(a, d);
                    }
                    tm_st16(ts + 16 * k, w);
                }
                l += (l4[0] + l4[1]) + (l4[2] + l4[3]);
                tm_wait_st();
                tm_before();
                bar_arrive(smem_addr(&bars.p[x]));
            }
            if (!good) break;
            good = bar_wait(smem_addr(&bars.o[x]), o_phase & 1u, gave_up);
            o_phase ^= 1u;
            if (!good) break;
            tm_after();

            // ---- the unit's rows ----
            const bool whole = t0 == 0 && c.end == c.u.tiles.count;
            float* slot = p.line.slots + (2 * static_cast<int64_t>(blockIdx.x) + (t0 == 0 ? 1 : 0)) * (static_cast<int64_t>(kRows) * (D + 2));
            const float inv = !whole ? 1.0f : (l == 0.0f ? 0.0f : 1.0f / l);
            bool odd = false;
            for (int k = 0; k < D / 32; ++k) {
                uint32_t o[32];
                tm_ld32(to + 32 * k, o);
                tm_wait32(o);
                float f[32];
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                    f[e] = __uint_as_float(o[e]);
                    odd |= !(fabsf(f[e]) < INFINITY);
                    f[e] = l == 0.0f ? 0.0f : f[e] * inv;
                }
                if (valid) {
                    if (whole) {
                        kv_store_out<T>(p, row, head, 32 * k, f, 32);
                    } else {
                        for (int e = 0; e < 32; e += 4)
                            *reinterpret_cast<float4*>(slot + static_cast<int64_t>(r) * D + 32 * k + e) = *reinterpret_cast<const float4*>(f + e);
                    }
                }
            }
            if (valid) {
                if (whole) {
                    if (p.lse != nullptr) p.lse[row * p.q_heads + head] = l == 0.0f ? -INFINITY : base * kLn2 + logf(l);
                } else {
                    slot[static_cast<int64_t>(kRows) * D + r] = base;
                    slot[static_cast<int64_t>(kRows) * D + kRows + r] = l;
                }
            }
            for (uint32_t redo = __ballot_sync(0xffffffffu, odd && valid && l != 0.0f); redo != 0; redo &= redo - 1) {
                const int src = __ffs(redo) - 1;
                KvExact y;
                y.table = p.shared_pass ? p.shared_table : b.table + c.s * b.table_stride;
                y.tiles = c.u.tiles;
                y.seen = KvSpan{__shfl_sync(0xffffffffu, sp.pre, src), __shfl_sync(0xffffffffu, sp.lo, src), __shfl_sync(0xffffffffu, sp.hi, src)};
                y.base = base_key;
                y.pos = __shfl_sync(0xffffffffu, pos, src);
                y.t0 = t0;
                y.t1 = c.end;
                y.size = kTile;
                y.row = __shfl_sync(0xffffffffu, row, src);
                y.head = __shfl_sync(0xffffffffu, head, src);
                y.kvh = c.h;
                const float rb = __shfl_sync(0xffffffffu, base, src), ri = __shfl_sync(0xffffffffu, inv, src);
                const int rrow = __shfl_sync(0xffffffffu, r, src);
                constexpr int kEach = D / 32;
                float part[4];
                kv_exact_row<T, D, kPlain>(p, y, rb, part);
                for (int e = 0; e < kEach; ++e) {
                    part[e] *= ri;
                    if (!whole) {
                        slot[static_cast<int64_t>(rrow) * D + lane * kEach + e] = part[e];
                    } else {
                        char* at = p.out.data + y.row * p.out.row_stride + y.head * p.out.head_stride;
                        if (p.out_f32) reinterpret_cast<float*>(at)[lane * kEach + e] = part[e];
                        else reinterpret_cast<T*>(at)[lane * kEach + e] = static_cast<T>(part[e]);
                    }
                }
            }
            tm_before();
            c.next(p);
        }
    }

    // ---- end ----
    tm_before();
    __syncthreads();
    tm_after();
    if (t == 0 && s_gave_up != 0) kv_report(p.status, GFD_KV_GAVE_UP);
    if (warp == 8) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::kColumns) : "memory");
}

// The cache's K or V as [blocks][tokens][heads][D], read in boxes of 16 tokens x 64 elements.
bool make_map(CUtensorMap* map, const KvAttendParams& p, const char* base, int head_dim, int dtype, KvEncodeFn encode) {
    const cuuint64_t row = static_cast<cuuint64_t>(head_dim) * 2;
    cuuint64_t dims[4] = {static_cast<cuuint64_t>(head_dim), static_cast<cuuint64_t>(p.cache.heads),
                          static_cast<cuuint64_t>(p.cache.block_tokens), static_cast<cuuint64_t>(p.cache.blocks)};
    // the stride of a dimension of one is not used, but has to be one that the map takes
    cuuint64_t strides[3] = {p.cache.heads > 1 ? static_cast<cuuint64_t>(p.cache.head_stride) : row,
                             static_cast<cuuint64_t>(p.cache.token_stride),
                             p.cache.blocks > 1 ? static_cast<cuuint64_t>(p.cache.block_stride) : row};
    cuuint32_t box[4] = {64, 1, kKvPage, 1}, ones[4] = {1, 1, 1, 1};
    return encode(map, dtype == GFD_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<char*>(base),
                  dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D>
cudaError_t launch(const KvAttendParams& p, const CUtensorMap& k, const CUtensorMap& v, int ctas, cudaStream_t st) {
    const bool plain = p.softcap == 0.0f && p.alibi == nullptr && p.scale2 != 0.0f;
    auto* f = plain ? kv_prompt_kernel<T, D, true> : kv_prompt_kernel<T, D, false>;
    cudaError_t e = cudaFuncSetAttribute(f, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<D>::kSmem);
    if (e != cudaSuccess) return e;
    f<<<ctas, kThreads, Shape<D>::kSmem, st>>>(p, k, v);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    return launch_kv_join(p, D, std::is_same<T, __half>::value ? GFD_FP16 : GFD_BF16, ctas, kRows, st);
}

}  // namespace

int kv_prompt_ctas(int num_sms) { return num_sms; }

cudaError_t launch_kv_prompt(const KvAttendParams& p, int head_dim, int dtype, int num_sms, KvEncodeFn encode, cudaStream_t st) {
    CUtensorMap k, v;
    if (!make_map(&k, p, p.cache.k, head_dim, dtype, encode) || !make_map(&v, p, p.cache.v, head_dim, dtype, encode))
        return cudaErrorInvalidValue;
    const int ctas = kv_prompt_ctas(num_sms);
    if (dtype == GFD_BF16) return head_dim == 64 ? launch<__nv_bfloat16, 64>(p, k, v, ctas, st) : launch<__nv_bfloat16, 128>(p, k, v, ctas, st);
    return head_dim == 64 ? launch<__half, 64>(p, k, v, ctas, st) : launch<__half, 128>(p, k, v, ctas, st);
}

}  // namespace gfdb
