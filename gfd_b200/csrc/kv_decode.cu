// Attention for sequences with few rows (decode steps, short drafts): at most 16 packed rows
// per KV head, where a packed row is one (row, query head) pair of the head's group.
//
// The work is reading the cache once: 4 D bytes per key and KV head against 4 D * 16 operations,
// so memory bounds it.  All (sequence, KV head) units are laid out as one line of 16-key tiles (one
// page or part of one) and every warp takes an equal stretch (KvCuts): a batch of mixed lengths,
// one long context and a hundred short ones keep every SM equally busy, with nothing known on
// the host.  A unit that a cut divides leaves partial sums in the workspace, joined by
// kv_join_few_kernel.
//
// The warps run alone: each has its own ring of stages filled with 16-byte cp.async (8 KB a stage,
// 192 KB in flight on an SM; block ids fetched 32 stages at a time), its own running maximum and
// sum, scores and sums by mma.m16n8k16 from ldmatrix fragments (KvRows16), and writes its rows from
// registers.  After the stretches are found there is no barrier.
//
// Measured: 64 sequences of up to 8192 tokens, 8 heads of 128, in 171 us with their join, 6.0 TB/s; two of
// 131 thousand, 24 query heads of 64 behind a cap, in 100 us, 5.1 TB/s (there 12 rows' scores and the cap's
// polynomial fill half of the issue slots).  128 elements a head take 213-217 registers, two CTAs an SM; 64
// take 158-160, and the third CTA is worth 123 -> 102 us.

#include <type_traits>

#include "kv_rows.cuh"
#include "kv_wait.cuh"

namespace gfdb {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;
template <int D>
constexpr int kPerSm = D == 64 ? 3 : 2;  // CTAs of an SM
constexpr int kLeast = 2;       // tiles of a stretch, where there are enough: a part costs its joining about as much
constexpr int kRows = kKvFewRows;

// 16 bytes into shared memory, zeros where !take
__device__ __forceinline__ void copy16(uint32_t dst, const char* src, bool take) {
    asm volatile("cp.async.cg.shared.global.L2::128B [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(take ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// One sequence as this kernel sees it: its rows and, in the count of its own keys (behind the
// shared prefix), what its rows see together.
struct Seq {
    KvSeq q;
    KvSpan all;  // pre, least lo, greatest hi
    KvTiles tiles;
    bool bad;
};

__device__ __forceinline__ Seq few_seq(const KvAttendParams& p, int s) {
    const KvBatchView& b = p.batch;
    Seq r;
    r.q = kv_seq(b.row_start[s], b.row_start[s + 1], b.kv_len[s], b.capacity, p.max_q_len);
    r.bad = !r.q.ok;
    if (r.bad || static_cast<int64_t>(r.q.rows) * p.group > kRows) r.q.rows = r.q.keys = 0;
    r.all = KvSpan{0, 0, 0};
    r.tiles = KvTiles{0, 0, 0};
    if (r.q.rows > 0) {
        const int32_t n = p.shared_len + r.q.keys;
        const int32_t prefix = p.prefix_len != nullptr ? p.prefix_len[s] : 0;
        const KvSpan first = kv_clip(kv_span(n - r.q.rows, n, prefix, p.window, p.causal != 0), p.shared_len, r.q.keys);
        const KvSpan last = kv_clip(kv_span(n - 1, n, prefix, p.window, p.causal != 0), p.shared_len, r.q.keys);
        r.all = KvSpan{first.pre, first.lo, last.hi};
        r.tiles = kv_tiles(r.all, kKvPage);
        // a sequence that sees none of its own keys still has rows to write
        if (r.tiles.count == 0) r.tiles = KvTiles{1, 0, 1};
    }
    return r;
}

// Where the stretches of this CTA's warps begin on the line, found together.  *cuts: the line's cuts;
// false: the row starts do not rise.
__device__ __forceinline__ bool find_places(const KvAttendParams& p, KvCuts* cuts, KvPlace* places) {
    __shared__ int64_t s_warp[kWarps];
    const KvBatchView& b = p.batch;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const int per = (b.seqs + kThreads - 1) / kThreads, s_lo = min(t * per, b.seqs), s_hi = min(s_lo + per, b.seqs);
    int64_t sum = 0;
    bool bad = false;
    Seq q;
    for (int s = s_lo; s < s_hi; ++s) {
        const int32_t from = b.row_start[s], to = b.row_start[s + 1];
        bad |= from < 0 || from > to || to > b.rows;
        q = few_seq(p, s);
        if (q.bad && blockIdx.x == 0) {
            kv_report(p.status, GFD_KV_BAD_LENGTH);
            if (from >= 0 && to <= b.rows) kv_mark_skipped(p, s);
        }
        sum += static_cast<int64_t>(q.tiles.count) * p.cache.heads;
    }
    int64_t incl = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    if (lane == 31) s_warp[warp] = incl;
    if (__syncthreads_or(bad) != 0) {
        if (blockIdx.x == 0 && t == 0) kv_report(p.status, GFD_KV_BAD_LENGTH);
        return false;
    }
    int64_t run = incl - sum, total = 0;
    for (int w = 0; w < kWarps; ++w) {
        if (w < warp) run += s_warp[w];
        total += s_warp[w];
    }
    const int64_t most = (total + kLeast - 1) / kLeast;
    *cuts = KvCuts(total, static_cast<uint32_t>(min(static_cast<int64_t>(kWarps) * gridDim.x, most)));
    for (int s = s_lo; s < s_hi; ++s) {
        if (per > 1) q = few_seq(p, s);
        const int32_t n = q.tiles.count;
        const int64_t here = static_cast<int64_t>(n) * p.cache.heads;
        if (n > 0)
            for (int w = 0; w < kWarps; ++w) {
                const int worker = w * gridDim.x + blockIdx.x;
                if (worker >= cuts->n()) break;
                const int64_t at = cuts->at(worker) - run;
                if (at < 0 || at >= here) continue;
                KvPlace& x = places[w];
                x.s = s;
                x.h = static_cast<int32_t>(kv_div(at, n));
                x.t = static_cast<int32_t>(at - static_cast<int64_t>(x.h) * n);
                x.count = n;
                x.begin = run + static_cast<int64_t>(x.h) * n;
                x.row0 = q.q.row0;
                x.packed0 = 0;
                x.packed = q.q.rows * p.group;
            }
        run += here;
    }
    __syncthreads();
    return true;
}

// Walks the units of a stretch.
struct Cursor {
    Seq q;
    int32_t s, h, t, end;  // tiles [t, end) of the unit lie in the stretch
    int64_t left;          // tiles of the stretch behind `end`
    bool done;

    __device__ __forceinline__ void enter(const KvAttendParams& p, int32_t s_, int32_t h_, int32_t t_, int64_t left_) {
        s = s_;
        h = h_;
        t = t_;
        q = few_seq(p, s);
        clamp(left_);
    }
    __device__ __forceinline__ void clamp(int64_t l) {
        done = l <= 0;
        end = static_cast<int32_t>(min(static_cast<int64_t>(q.tiles.count), t + l));
        left = l - (end - t);
    }
    __device__ __forceinline__ void next_unit(const KvAttendParams& p) {
        if (left <= 0) {
            done = true;
            return;
        }
        t = 0;
        if (++h == p.cache.heads) {
            h = 0;
            do {
                q = few_seq(p, ++s);
            } while (q.tiles.count == 0);
        }
        clamp(left);
    }
};

template <int D>
struct Shape {
    static constexpr int kStages = 3;
    static constexpr int kRow = 2 * D;                   // bytes of a key
    static constexpr int kStage = 2 * kKvPage * kRow;  // K and V of 16 keys
    static constexpr int kRing = kStages * kStage;
    static constexpr int kSmem = kWarps * kRing;
};

template <typename T, int D, bool kPlain>
__global__ void __launch_bounds__(kThreads, kPerSm<D>) kv_decode_kernel(const KvAttendParams p) {
    using S = Shape<D>;
    constexpr int kSteps = D / 16;
    constexpr int kChunks = D / 8;   // 16-byte pieces of a key
    constexpr int kTile = kKvPage;   // keys of a tile
    extern __shared__ __align__(128) char smem[];
    __shared__ KvPlace s_place[kWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // neighbouring stretches lie on different SMs, so that a short line is spread over all of them
    const int worker = warp * gridDim.x + blockIdx.x;
    const KvBatchView& b = p.batch;

    kv_let_next();
    KvCuts cuts(0, 0);
    if (!find_places(p, &cuts, s_place) || worker >= cuts.n()) {
        if (lane == 0) p.line.cuts[worker].parts = 0;
        kv_wait_last();
        return;
    }
    Cursor load, use;
    load.enter(p, s_place[warp].s, s_place[warp].h, s_place[warp].t, cuts.at(worker + 1) - cuts.at(worker));
    use = load;

    // ---- stages ----
    const uint32_t ring = smem_addr(smem) + warp * S::kRing;
    const int pages = p.cache.block_tokens / kKvPage;
    int32_t ids = -1;       // lane i: block id of tile ids_from + i
    int32_t ids_from = 0;
    bool ids_ok = false;
    uint32_t live = 0;      // bit i: the stage issued i stages ago holds keys
    int put = 0;
    // lane i of a step copies piece i % kChunks of key i / kChunks, kStep keys a step
    constexpr int kStep = 32 / kChunks;
    const int64_t lane_off = lane / kChunks * p.cache.token_stride + 16 * (lane % kChunks);
    const int64_t step_off = kStep * p.cache.token_stride;
    const uint32_t lane_to = ring + lane / kChunks * S::kRow + ((lane % kChunks ^ lane / kChunks) << 4);
    auto issue = [&]() {
        live <<= 1;
        if (!load.done) {
            const KvSpan& a = load.q.all;
            if (!ids_ok || load.t >= ids_from + 32) {
                if (!ids_ok && lane < 2 * kRows) {
                    // a new unit: its rows of Q set out as well
                    const int r = lane / 2, of = kv_div_group(p, r);
                    if (r < load.q.q.rows * p.group && (D == 128 || lane % 2 == 0))
                        asm volatile("prefetch.global.L1 [%0];" ::"l"(p.q.data + (load.q.q.row0 + of) * p.q.row_stride +
                                                                      (load.h * p.group + r - of * p.group) * p.q.head_stride + 128 * (lane % 2)));
                }
                ids_from = load.t;
                ids_ok = true;
                const int32_t i = ids_from + lane;
                ids = -1;
                if (i < load.end) {
                    const int32_t j = load.q.tiles.at(i) * kTile;
                    if (j < a.pre || (j + kTile > a.lo && j < a.hi)) {
                        ids = b.table[load.s * b.table_stride + kv_div_pages(p, j / kTile)];
                        if (ids < 0 || ids >= p.cache.blocks) {
                            kv_report(p.status, GFD_KV_BAD_PAGE);
                            ids = -1;
                        }
                    }
                }
            }
            const int32_t id = __shfl_sync(0xffffffffu, ids, load.t - ids_from);
            if (id >= 0) {
                live |= 1u;
                const int32_t page = load.q.tiles.at(load.t), j = page * kTile;
                const int32_t place = (page - kv_div_pages(p, page) * pages) * kKvPage;
                const int64_t off = id * p.cache.block_stride + place * p.cache.token_stride + load.h * p.cache.head_stride + lane_off;
                const char* k = p.cache.k + off;
                const char* v = p.cache.v + off;
                const uint32_t to = lane_to + put * S::kStage;
                if ((j >= a.lo && j + kTile <= a.hi) || j + kTile <= a.pre) {
#pragma unroll
                    for (int i = 0; i < kKvPage / kStep; ++i) {
                        const uint32_t at = (to ^ (((i * kStep) & 7) << 4)) + i * kStep * S::kRow;
                        copy16(at, k, true);
                        copy16(at + kTile * S::kRow, v, true);
                        k += step_off;
                        v += step_off;
                    }
                } else {
                    // keys no row sees stay zero, so that what lies there cannot reach a sum
#pragma unroll 1
                    for (int i = 0; i < kKvPage / kStep; ++i) {
                        const int32_t key = j + i * kStep + lane / kChunks;
                        const bool take = key < a.pre || (key >= a.lo && key < a.hi);
                        const uint32_t at = (to ^ (((i * kStep) & 7) << 4)) + i * kStep * S::kRow;
                        copy16(at, k, take);
                        copy16(at + kTile * S::kRow, v, take);
                        k += step_off;
                        v += step_off;
                    }
                }
            }
            if (++load.t == load.end) {
                load.next_unit(p);
                ids_ok = false;
            }
        }
        copy_commit();
        put = put + 1 == S::kStages ? 0 : put + 1;
    };
#pragma unroll
    for (int i = 0; i < S::kStages - 1; ++i) issue();
    if (lane == 0) p.line.cuts[worker] = kv_cut(cuts, worker, s_place[warp]);  // while the first keys are on their way

    // ---- units ----
    int get = 0;
    const int row_a = lane >> 2;  // this thread's rows: row_a and row_a + 8
    while (!use.done) {
        const int32_t rows = use.q.q.rows * p.group;
        const int32_t n = p.shared_len + use.q.q.keys;
        KvRows16<T, D, kPlain> w;
        w.begin(rows);
        const int prefix = p.prefix_len != nullptr ? p.prefix_len[use.s] : 0;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int r = row_a + 8 * x;
            const int i = kv_div_group(p, r), head = use.h * p.group + r - i * p.group;
            w.pos[x] = n - use.q.q.rows + i;
            w.sp[x] = KvSpan{0, 0, 0};
            if (r < rows) {
                w.sp[x] = kv_clip(kv_span(w.pos[x], n, prefix, p.window, p.causal != 0), p.shared_len, use.q.q.keys);
                if (!kPlain && p.alibi != nullptr) w.slope[x] = p.alibi[head] * kLog2e;
            }
            w.load_q(x, p.q.data + (use.q.q.row0 + i) * p.q.row_stride + head * p.q.head_stride, r < rows);
        }
        const int32_t t0 = use.t;

        for (; use.t < use.end; ++use.t) {
            issue();
            copy_wait<S::kStages - 1>();
            __syncwarp();
            if ((live >> (S::kStages - 1)) & 1u) {
                const uint32_t kb = ring + get * S::kStage, vb = kb + kTile * S::kRow;
                const int32_t j0 = use.q.tiles.at(use.t) * kTile;
                // (the rows of one token see the same keys, and the others are zeros)
                const uint32_t odd = use.q.q.rows > 1 && w.cut(j0) ? w.odd_keys(vb) : 0u;
                w.tile(p, kb, vb, j0, p.shared_len, odd, vb);
            }
            __syncwarp();
            get = get + 1 == S::kStages ? 0 : get + 1;
        }

        // ---- the unit's rows ----
        const bool whole = t0 == 0 && use.end == use.q.tiles.count;
        float* slot = p.line.slots + (2 * static_cast<int64_t>(worker) + (t0 == 0 ? 1 : 0)) * (kRows * D + 2 * kRows);
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            if (8 * x >= rows) break;
            float l = w.l[x];
            l += __shfl_xor_sync(0xffffffffu, l, 1);
            l += __shfl_xor_sync(0xffffffffu, l, 2);
            const int r = row_a + 8 * x, i = kv_div_group(p, r), head = use.h * p.group + r - i * p.group;
            const int64_t row = use.q.q.row0 + i;
            if (r >= rows) continue;
            const float inv = !whole ? 1.0f : (l == 0.0f ? 0.0f : 1.0f / l);
            char* dst = whole ? p.out.data + row * p.out.row_stride + head * p.out.head_stride : reinterpret_cast<char*>(slot + r * D);
            const bool wide = !whole || p.out_f32;
#pragma unroll
            for (int y = 0; y < 2 * kSteps; ++y) {
                const float v0 = w.acc[y][2 * x] * inv, v1 = w.acc[y][2 * x + 1] * inv;
                if (wide) reinterpret_cast<float2*>(dst)[4 * y + (lane & 3)] = make_float2(v0, v1);
                else reinterpret_cast<uint32_t*>(dst)[4 * y + (lane & 3)] = Pack<T>::pair(v0, v1);
            }
            if ((lane & 3) == 0) {
                if (!whole) {
                    slot[kRows * D + r] = w.m[x];
                    slot[kRows * D + kRows + r] = l;
                } else if (p.lse != nullptr) {
                    p.lse[row * p.q_heads + head] = kv_lse(p, w.m[x], l);
                }
            }
        }
        __syncwarp();
        use.next_unit(p);
    }
    copy_wait<0>();
    kv_wait_last();
}

template <typename T, int D>
cudaError_t launch(const KvAttendParams& p, int num_sms, bool chained, cudaStream_t st) {
    const int ctas = num_sms * kPerSm<D>;
    const bool plain = p.softcap == 0.0f && p.alibi == nullptr;
    const cudaError_t e = kv_launch(plain ? kv_decode_kernel<T, D, true> : kv_decode_kernel<T, D, false>, dim3(ctas), kThreads,
                                    Shape<D>::kSmem, st, chained, p);
    if (e != cudaSuccess) return e;
    return launch_kv_join_few(p, D, std::is_same<T, __half>::value ? GFD_FP16 : GFD_BF16, kWarps * ctas, st);
}

}  // namespace

int kv_decode_workers(int num_sms, int head_dim) { return num_sms * kWarps * (head_dim == 64 ? kPerSm<64> : kPerSm<128>); }

cudaError_t launch_kv_decode(const KvAttendParams& p, int head_dim, int dtype, int num_sms, bool chained, cudaStream_t st) {
    if (dtype == GFD_BF16)
        return head_dim == 64 ? launch<__nv_bfloat16, 64>(p, num_sms, chained, st) : launch<__nv_bfloat16, 128>(p, num_sms, chained, st);
    return head_dim == 64 ? launch<__half, 64>(p, num_sms, chained, st) : launch<__half, 128>(p, num_sms, chained, st);
}

}  // namespace gfdb
