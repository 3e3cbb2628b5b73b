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
// No pipe is full: with 128 elements a head the tensor pipe is active 58 % of the time and the special function
// unit, which takes the exponentials, 59 %; with 64 it is 35 and 65 %, the issue slots 37 and 43 %.  What bounds a tile
// is the chain of scores, maximum, exponentials and sums of a half, with two softmax warps a scheduler to hide
// it.  8192 rows on 8192 keys and 32 heads take 866 us, 1270 TFLOP/s, 467 us causal; with 64 elements 721 us,
// 762 TFLOP/s, 392 us causal; 752 and 687 us causal behind a cap (calls with pauses between them; back to back the
// power cap takes a sixth).  Short units wait for O to be written before the next one's sums begin: 16 prompts of
// 512 rows take 93 us, 737 TFLOP/s.
//
// Roles: warps 0-3 softmax of half A, 4-7 of half B; 8-11 write finished rows while the softmax
// is in the next unit; 12 issues the products, 13 loads K and V (TMA boxes of 16 tokens x 64
// elements, so that every page is found by its id), 14 loads Q (a box of the group's heads x rows where
// the heads divide 128), 15 walks the units and watches over the others' waits.  Units whose values held a NaN
// or an infinity are summed once more at the end (sum_again).  Units lie
// on one line of tiles that the CTAs (one per SM) share evenly; a cut unit leaves partial sums
// for kv_join_many_kernel, as in kv_decode.cu.

#include <cuda.h>

#include <type_traits>

#include "kv_rows.cuh"
#include "kv_wait.cuh"

namespace gfdb {
namespace {

constexpr int kRows = kKvManyRows;  // packed rows of a unit
constexpr int kHalf = 128;          // rows of a half: one tensor-core tile
constexpr int kTile = 128;          // keys of a step
constexpr int kPages = kTile / kKvPage;
constexpr int kThreads = 512;
constexpr int kAux = 80, kMain = 176;  // registers of the helpers' and the softmax warps: 256 x (80 + 176) = 64 K
// On the line every unit is as much longer than its tiles: what beginning and finishing one costs
// (1 to 3 come out alike within 2 %, 5 and 8 slower).
constexpr int kUnitCost = 2;
constexpr int kBadRing = 8;         // tiles whose bad pages are remembered
constexpr int kOddUnits = 1024;     // units of a CTA that are marked one by one; the last mark is the others'

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
__device__ __forceinline__ void tm_st16(uint32_t addr, const uint32_t* r) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(r[0]),
        "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
        "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(addr)
        : "memory");
}
__device__ __forceinline__ void tm_ld16(uint32_t addr, uint32_t* r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
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
__device__ __forceinline__ void tm_wait16(uint32_t* r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]), 
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ bool elect_one() {
    uint32_t ok;
    asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(ok));
    return ok != 0;
}
__device__ __forceinline__ void tm_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// Shared-memory operand in 128-byte swizzle: rows of 128 bytes in groups of 8 (1024 bytes, the
// stride in bits 32-45), descriptor version 1.  The low word holds the address, and for a row-major
// second operand the bytes from one 64-element block of its columns to the next.
constexpr uint32_t kOperandHigh = (1024u >> 4) | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t operand(uint32_t addr, uint32_t block) { return (addr >> 4) | (block >> 4) << 16; }
// 32-bit sums of 16-bit products; second operand's columns contiguous (trans) or not
template <typename T>
__device__ __forceinline__ constexpr uint32_t product(int m, int n, bool trans) {
    const uint32_t fmt = std::is_same<T, __half>::value ? 0u : 1u;
    return 1u << 4 | fmt << 7 | fmt << 10 | (trans ? 1u << 16 : 0u) | static_cast<uint32_t>(n >> 3) << 17 |
           static_cast<uint32_t>(m >> 4) << 24;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n.reg .pred p;\n.reg .b64 x, y;\nmov.b64 x, {%1, %5};\nmov.b64 y, {%2, %5};\nsetp.ne.u32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(add ? 1u : 0u), "n"(kOperandHigh)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
    asm volatile(
        "{\n.reg .pred p;\n.reg .b64 y;\nmov.b64 y, {%2, %5};\nsetp.ne.u32 p, %4, 0;\n"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n}" ::"r"(d),
        "r"(a), "r"(b), "r"(idesc), "r"(add ? 1u : 0u), "n"(kOperandHigh)
        : "memory");
}
__device__ __forceinline__ void tma_page(uint32_t dst, const CUtensorMap* map, int x, int head, int place, int block, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
        "l"(map), "r"(x), "r"(head), "r"(place), "r"(block), "r"(bar)
        : "memory");
}
// 32 bytes; `wide`: both ends of them on 32
__device__ __forceinline__ void store8(uint64_t to, const uint32_t* r, bool wide) {
    if (wide) {
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]),
                     "r"(r[5]), "r"(r[6]), "r"(r[7])
                     : "memory");
    } else {
        *reinterpret_cast<uint4*>(to) = make_uint4(r[0], r[1], r[2], r[3]);
        *reinterpret_cast<uint4*>(to + 16) = make_uint4(r[4], r[5], r[6], r[7]);
    }
}
__device__ __forceinline__ void tma_rows(uint32_t dst, const CUtensorMap* map, int x, int head, int row, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
        "l"(map), "r"(x), "r"(head), "r"(row), "r"(bar)
        : "memory");
}
__device__ __forceinline__ void tma_rows_ahead(const CUtensorMap* map, int x, int head, int row) {  // into L2
    asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global [%0, {%1, %2, %3}];" ::"l"(map), "r"(x), "r"(head), "r"(row) : "memory");
}

// ---------------------------------------------------------------------------
// Units
// ---------------------------------------------------------------------------
// What the rows of sequence s see of the shared prefix together: the first of them sees furthest back.  All of it
// behind the prefix or in a skipped or empty sequence: nothing.
__device__ __forceinline__ KvSpan seen_of_prefix(const KvAttendParams& p, int s) {
    const KvBatchView& b = p.batch;
    const KvSeq q = kv_seq(b.row_start[s], b.row_start[s + 1], b.kv_len[s], b.capacity, p.max_q_len);
    if (!q.ok || q.rows == 0) return KvSpan{0, p.shared_len, p.shared_len};
    const int32_t n = p.shared_len + q.keys, prefix = p.prefix_len != nullptr ? p.prefix_len[s] : 0;
    return kv_clip(kv_span(n - q.rows, n, prefix, p.window, p.causal != 0), 0, p.shared_len);
}

// What the launch walks over: the sequences with many rows, or (shared pass) all rows of the
// batch as one sequence against the shared prefix.
struct Many {
    KvSeq q;       // rows and keys (keys in the count of this pass)
    int32_t tiles; // row tiles
    bool bad;
};

template <bool kShared>
__device__ __forceinline__ Many many_seq(const KvAttendParams& p, int s) {
    const KvBatchView& b = p.batch;
    Many r;
    if (kShared) {
        r.q = KvSeq{b.row_start[0], b.row_start[b.seqs] - b.row_start[0], p.shared_len, true};
        r.bad = false;
    } else {
        r.q = kv_seq(b.row_start[s], b.row_start[s + 1], b.kv_len[s], b.capacity, p.max_q_len);
        r.bad = !r.q.ok;
        if (r.bad || static_cast<int64_t>(r.q.rows) * p.group <= p.few_rows) r.q.rows = r.q.keys = 0;
    }
    r.tiles = static_cast<int32_t>((static_cast<int64_t>(r.q.rows) * p.group + kRows - 1) / kRows);
    return r;
}

struct Unit {
    KvSpan all;  // pre, least lo, greatest hi of its rows
    KvTiles tiles;
    int32_t packed0, packed;
};

// seen: what the batch's rows see together of the shared prefix (shared pass)
template <bool kShared>
__device__ __forceinline__ Unit many_unit(const KvAttendParams& p, int s, const KvSeq& q, int rt, const KvSpan& seen) {
    Unit u;
    const int64_t packed = static_cast<int64_t>(q.rows) * p.group;
    u.packed0 = rt * kRows;
    u.packed = static_cast<int32_t>(min(static_cast<int64_t>(kRows), packed - u.packed0));
    if (kShared) {
        u.all = seen;
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

template <bool kShared>
struct Cursor {
    Many m;
    Unit u;
    int32_t s, h, rt, t, end;  // tiles [t, end) of the unit lie in the stretch
    int64_t begin, to;         // of the unit's first tile, and of the stretch's end, on the line
    bool done;

    __device__ __forceinline__ void enter(const KvAttendParams& p, const KvPlace& at, int64_t to_, const KvSpan& seen) {
        s = at.s;
        h = at.h;
        rt = at.packed0 / kRows;
        t = at.t;
        begin = at.begin;
        to = to_;
        m = many_seq<kShared>(p, s);
        u = many_unit<kShared>(p, s, m.q, rt, seen);
        clamp();
    }
    __device__ __forceinline__ void clamp() {
        end = static_cast<int32_t>(min(static_cast<int64_t>(u.tiles.count), max(to - begin, static_cast<int64_t>(0))));
        done = t >= end;
    }
    // The line runs over KV heads, within a head over sequences, within a sequence over row tiles.
    __device__ __forceinline__ void next(const KvAttendParams& p, const KvSpan& seen) {
        begin += u.tiles.count + kUnitCost;
        if (begin >= to) {
            done = true;
            return;
        }
        t = 0;
        if (++rt >= m.tiles) {
            rt = 0;
            do {
                if (++s >= (kShared ? 1 : p.batch.seqs)) {
                    s = 0;
                    ++h;
                }
                m = many_seq<kShared>(p, s);
            } while (m.tiles == 0);
        }
        u = many_unit<kShared>(p, s, m.q, rt, seen);
        clamp();
    }
};

// A unit as the walking warp hands it to the others.
struct Desc {
    int32_t s, h;
    int32_t t0, nt;              // its tiles in this CTA
    int32_t count;               // all its tiles
    int32_t npre, first;         // KvTiles
    int32_t pre, lo, hi;         // what its rows see together
    int32_t packed0, packed;
    int32_t row0, rows, keys;    // of its sequence
    int32_t prefix;
    __device__ __forceinline__ int32_t key(int i) const {  // first key of tile t0 + i
        const int32_t t = t0 + i;
        return (t < npre ? t : t - npre + first) * kTile;
    }
};

// Tiles [t0, t1) of a unit; none when t1 <= t0.
template <bool kShared>
__device__ __forceinline__ Desc describe(const KvAttendParams& p, int s, int h, int t0, int t1, const KvSeq& q, const Unit& u) {
    Desc d;
    d.s = s;
    d.h = h;
    d.t0 = t0;
    d.nt = max(t1 - t0, 0);
    d.count = u.tiles.count;
    d.npre = u.tiles.npre;
    d.first = u.tiles.first;
    d.pre = u.all.pre;
    d.lo = u.all.lo;
    d.hi = u.all.hi;
    d.packed0 = u.packed0;
    d.packed = u.packed;
    d.row0 = q.row0;
    d.rows = q.rows;
    d.keys = q.keys;
    d.prefix = !kShared && p.prefix_len != nullptr ? p.prefix_len[s] : 0;
    return d;
}

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

constexpr int kUnitRing = 4;
constexpr int kUnitReaders = 4 + 4 + 4 + 3;  // warps

struct Bars {
    uint64_t full[4], empty[4];                       // K and V slots
    uint64_t unit[kUnitRing], unit_read[kUnitRing];
    uint64_t q[2], q_read[2], s[2], p[2], p2[2];      // Q there / products with it done, scores, weights in two parts
    uint64_t o[2], o_read[2], ml[2], ml_read[2];      // sums done / taken, their base and weight sum
    uint64_t last, done;                              // all products done, all rows written
};

template <typename T>
struct Shift {  // weights reach 2^(shift + 8): fp16 keeps them clear of its small values' coarse steps
    static constexpr float value = std::is_same<T, __half>::value ? 6.0f : 0.0f;
};
constexpr float kGrow = 8.0f;

// Position of row r of the unit and what it sees of this pass's keys; rows that do not exist see
// everything.  `exact`: the position itself is needed, not only the span.
template <bool kShared>
__device__ __forceinline__ KvSpan row_span(const KvAttendParams& p, const Desc& u, int r, int32_t* pos, bool exact) {
    *pos = 0;
    if (r >= u.packed) return KvSpan{0x7fffffff, 0, 0};
    const int32_t of = kv_div_group(p, u.packed0 + r);
    int32_t n = p.shared_len + u.keys, prefix = u.prefix;
    *pos = n - u.rows + of;
    if (kShared) {
        // all rows of the batch: the position is that of the row's own sequence, and without a
        // window, a prefix mask or a bias it does not matter
        const KvBatchView& b = p.batch;
        n = p.shared_len;
        *pos = 0x3fffffff;
        if (exact || p.window > 0 || p.prefix_len != nullptr) {
            const int32_t row = u.row0 + of;
            int lo = 0, hi = b.seqs - 1;
            while (lo < hi) {
                const int mid = (lo + hi + 1) / 2;
                if (b.row_start[mid] <= row) lo = mid;
                else hi = mid - 1;
            }
            n = p.shared_len + min(max(b.kv_len[lo], 0), static_cast<int32_t>(b.capacity));
            *pos = n - (b.row_start[lo + 1] - row);
            prefix = p.prefix_len != nullptr ? p.prefix_len[lo] : 0;
        }
    }
    return kv_clip(kv_span(*pos, n, prefix, p.window, p.causal != 0), kShared ? 0 : p.shared_len, u.keys);
}

// the n lowest bits, n clamped to 0 .. 32
__device__ __forceinline__ uint32_t below(int32_t n) { return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u); }

// 2^x of both, without the special function unit: 2^n from the exponent's bits, n the nearest whole
// number, times a polynomial of degree 5 in x - n (least relative error on [-1/2, 1/2], 1 at 0; off by
// at most 2^-22.5 in 32-bit arithmetic).  Below -126 it falls to 0, and from -127 on, -infinity
// too, it is 0.  x < 127; a NaN gives 0.
__device__ __forceinline__ uint64_t poly_exp2(uint64_t x) {
    float a, b;
    unpack2(x, a, b);
    x = pack2(fmaxf(a, -127.0f), fmaxf(b, -127.0f));
    const uint64_t n = add2(x, pack2(12582912.0f, 12582912.0f));  // 3 * 2^22: the sum's low bits are n
    const uint64_t r = add2(x, fma2(n, pack2(-1.0f, -1.0f), pack2(12582912.0f, 12582912.0f)));
    uint64_t y = fma2(r, pack2(0.001326472731307149f, 0.001326472731307149f), pack2(0.009671512991189957f, 0.009671512991189957f));
    y = fma2(y, r, pack2(0.05550733581185341f, 0.05550733581185341f));
    y = fma2(y, r, pack2(0.24022242426872253f, 0.24022242426872253f));
    y = fma2(y, r, pack2(0.6931470036506653f, 0.6931470036506653f));
    y = fma2(y, r, pack2(1.0f, 1.0f));
    float na, nb;
    unpack2(y, a, b);
    unpack2(n, na, nb);
    return pack2(__uint_as_float(__float_as_uint(a) + (__float_as_uint(na) << 23)),
                 __uint_as_float(__float_as_uint(b) + (__float_as_uint(nb) << 23)));
}

// Pairs out of 16 that take poly_exp2.  With 64 elements a head the special function unit is the busiest pipe
// and one pair is worth 2 % (non-causal, 8192 rows on 8192 keys, 32 heads: 763 us with none, 747 with 1, 744 with 2);
// with 128 it is no busier than the tensor pipe and a pair costs 2 % (causal: 489 us, 500 with 1).
template <int D>
struct ByPoly {
    static constexpr int value = D == 64 ? 1 : 0;
};

// largest of three; NaN if one is
__device__ __forceinline__ float max3(float a, float b, float c) {
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}

// ---------------------------------------------------------------------------
// Units whose sums met a NaN or an infinity
// ---------------------------------------------------------------------------
// A value that a row's mask hides reaches its sum as 0 * NaN, so units with sums that are not finite are summed
// once more, by the softmax warps when the stretch is done and nothing waits: 128 rows at a time, 16 a warp, such
// values taken out of the tile on its way into shared memory and added to the sums of the rows that see them
// (KvRows16).  A result that is to be NaN or infinite comes out as that.  8192 causal rows of 32 heads of 128 take
// 1.8 ms when the last key alone holds a NaN and 5.3 ms when every unit meets one, 0.50 ms otherwise.
constexpr int kAgainThreads = 256;
__device__ __forceinline__ void again_sync() { asm volatile("bar.sync 2, %0;" ::"n"(kAgainThreads) : "memory"); }

template <typename T, int D, bool kPlain, bool kShared>
__device__ __forceinline__ void sum_again(const KvAttendParams& p, const KvPlace& from, int64_t to, uint32_t smem, uint32_t* flags,
                                          const uint8_t* marks, const KvSpan& seen) {
    using Rows = KvRows16<T, D, kPlain>;
    constexpr int kRow = 2 * D, kChunks = D / 8, kSub = kTile / kKvPage;
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const uint32_t sk = smem, sv = sk + kTile * kRow, raw = sv + kTile * kRow;  // K, V without such values, V
    const int pages = p.cache.block_tokens / kKvPage;
    const int32_t base_key = kShared ? 0 : p.shared_len;
    if (t < 2 * kSub) flags[t] = 0;
    again_sync();
    Cursor<kShared> c;
    c.enter(p, from, to, seen);
    int turn = 0;
    for (int i = 0; !c.done; ++i, c.next(p, seen)) {
        if (marks[min(i, kOddUnits - 1)] == 0) continue;
        const Desc u = describe<kShared>(p, c.s, c.h, c.t, c.end, c.m.q, c.u);
        const int32_t* table = kShared ? p.shared_table : p.batch.table + u.s * p.batch.table_stride;
        const bool whole = u.nt == u.count;
        for (int half = 0; half < u.packed; half += kHalf) {
            const int first = half + warp * 16;
            Rows w;
            w.begin(max(0, min(16, u.packed - first)));
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int r = first + lane / 4 + 8 * x;
                const int32_t packed = u.packed0 + (r < u.packed ? r : 0), of = kv_div_group(p, packed);
                const int32_t head = u.h * p.group + packed - of * p.group;
                w.sp[x] = row_span<kShared>(p, u, r, &w.pos[x], true);
                if (!kPlain && p.alibi != nullptr) w.slope[x] = p.alibi[head] * kLog2e;
                w.load_q(x, p.q.data + static_cast<int64_t>(u.row0 + of) * p.q.row_stride + head * p.q.head_stride, r < u.packed);
            }
            for (int k = 0; k < u.nt; ++k, turn ^= 1) {
                const int32_t j0 = u.key(k);
                uint32_t* flag = flags + turn * kSub;  // per 16 keys: bit 31 some are there, bit i key i's values are not all finite
                for (int e = t; e < kTile * kChunks; e += kAgainThreads) {
                    const int key = e / kChunks, piece = e % kChunks;
                    const int32_t j = j0 + key, page = j / kKvPage;
                    uint4 a = make_uint4(0, 0, 0, 0), v = a;
                    if (j < u.pre || (j >= u.lo && j < u.hi)) {
                        const int32_t in = kv_div_pages(p, page), id = table[in];
                        if (id >= 0 && id < p.cache.blocks) {
                            const int64_t at = id * p.cache.block_stride + ((page - in * pages) * kKvPage + j % kKvPage) * p.cache.token_stride +
                                               u.h * p.cache.head_stride + 16 * piece;
                            a = *reinterpret_cast<const uint4*>(p.cache.k + at);
                            v = *reinterpret_cast<const uint4*>(p.cache.v + at);
                            if (piece == 0) atomicOr(flag + key / kKvPage, 1u << 31);
                            if ((kv_odd<T>(v.x) | kv_odd<T>(v.y) | kv_odd<T>(v.z) | kv_odd<T>(v.w)) != 0)
                                atomicOr(flag + key / kKvPage, 1u << (key % kKvPage));
                        }
                    }
                    const uint32_t to_piece = key * kRow + ((piece ^ (key & 7)) << 4);
                    Rows::sts16(sk + to_piece, a.x, a.y, a.z, a.w);
                    Rows::sts16(sv + to_piece, kv_finite<T>(v.x), kv_finite<T>(v.y), kv_finite<T>(v.z), kv_finite<T>(v.w));
                    Rows::sts16(raw + to_piece, v.x, v.y, v.z, v.w);
                }
                again_sync();
                if (t < kSub) flags[(turn ^ 1) * kSub + t] = 0;
                if (w.rows > 0)
                    for (int y = 0; y < kSub; ++y) {
                        const uint32_t f = flag[y];
                        if (f >> 31 == 0) continue;
                        const uint32_t at = y * kKvPage * kRow;
                        w.tile(p, sk + at, sv + at, j0 + y * kKvPage, base_key, f & 0xffffu, raw + at);
                    }
                again_sync();
            }
            float* slot = p.line.slots + (2 * static_cast<int64_t>(blockIdx.x) + (u.t0 == 0 ? 1 : 0)) * (static_cast<int64_t>(kRows) * (D + 2));
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                float l = w.l[x];
                l += __shfl_xor_sync(0xffffffffu, l, 1);
                l += __shfl_xor_sync(0xffffffffu, l, 2);
                const int r = first + lane / 4 + 8 * x, d0 = 2 * (lane & 3);
                if (r >= u.packed) continue;
                if (!whole) {
#pragma unroll
                    for (int y = 0; y < D / 8; ++y) {
                        const int d = 8 * y + d0;
                        *reinterpret_cast<float2*>(slot + (static_cast<int64_t>(d / 4) * kRows + r) * 4 + d % 4) = make_float2(w.acc[y][2 * x], w.acc[y][2 * x + 1]);
                    }
                    if (d0 == 0) {
                        slot[static_cast<int64_t>(kRows) * D + r] = w.m[x];
                        slot[static_cast<int64_t>(kRows) * D + kRows + r] = l;
                    }
                    continue;
                }
                const int32_t packed = u.packed0 + r, of = kv_div_group(p, packed);
                const int64_t row = u.row0 + of, place = row * p.q_heads + u.h * p.group + packed - of * p.group;
                const int32_t head = u.h * p.group + packed - of * p.group;
                const float own_lse = kShared ? p.own_lse[place] : -INFINITY;
                if (kShared && __float_as_uint(own_lse) == kKvSkipped) continue;
                const KvFinish f = kv_finish<kShared>(p, w.m[x], l, own_lse);
                char* dst = p.out.data + row * p.out.row_stride + head * p.out.head_stride;
#pragma unroll
                for (int y = 0; y < D / 8; ++y) {
                    const int d = 8 * y + d0;
                    float a = w.acc[y][2 * x] * f.scale, b = w.acc[y][2 * x + 1] * f.scale;
                    if (kShared && f.own != 0.0f) {
                        const float2 o = *reinterpret_cast<const float2*>(p.own_out + place * D + d);
                        a = fmaf(o.x, f.own, a);
                        b = fmaf(o.y, f.own, b);
                    }
                    if (p.out_f32) *reinterpret_cast<float2*>(dst + 4 * d) = make_float2(a, b);
                    else *reinterpret_cast<uint32_t*>(dst + 2 * d) = Pack<T>::pair(a, b);
                }
                if (p.lse != nullptr && d0 == 0) p.lse[place] = kv_lse(p, f.base, f.sum);
            }
        }
    }
}

// kShared: the pass over a shared prefix
template <typename T, int D, bool kPlain, bool kShared>
__global__ void __launch_bounds__(kThreads, 1)
    kv_prompt_kernel(const KvAttendParams p, const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v,
                     const __grid_constant__ CUtensorMap map_q) {
    using S = Shape<D>;
    extern __shared__ char smem_raw[];
    __shared__ Bars bars;
    __shared__ KvPlace s_place;
    __shared__ KvSpan s_seen;                         // of the shared prefix, by the batch's rows together
    __shared__ int32_t s_reach[kThreads / 32][2];
    __shared__ int64_t s_warps[kThreads / 32];
    __shared__ uint32_t s_tmem;
    __shared__ KvWaits s_waits;
    __shared__ uint32_t s_bad[kBadRing];
    __shared__ uint8_t s_marks[kOddUnits];            // units to be summed again
    __shared__ uint32_t s_flags[2 * kTile / kKvPage];  // of sum_again
    __shared__ Desc s_unit[kUnitRing];
    __shared__ float s_base[2][kHalf], s_sum[2][kHalf];
    __shared__ const char* s_rows[kRows];
    char* smem = reinterpret_cast<char*>((reinterpret_cast<uint64_t>(smem_raw) + 1023) & ~1023ull);
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    const KvBatchView& b = p.batch;

    kv_let_next();
    if (t == 0) {
        s_waits.gave_up = 0;
        s_waits.held = kShared;  // until the warps that write have waited for the passes over the own keys
        s_waits.steps = 0;
        for (int i = 0; i < S::kSlots; ++i) {
            bar_init(smem_addr(&bars.full[i]), 1);
            bar_init(smem_addr(&bars.empty[i]), 1);
        }
        for (int i = 0; i < kUnitRing; ++i) {
            bar_init(smem_addr(&bars.unit[i]), 1);
            bar_init(smem_addr(&bars.unit_read[i]), kUnitReaders);
        }
        for (int i = 0; i < 2; ++i) {
            bar_init(smem_addr(&bars.q[i]), 1);
            bar_init(smem_addr(&bars.q_read[i]), 1);
            bar_init(smem_addr(&bars.s[i]), 1);
            bar_init(smem_addr(&bars.p[i]), 4);
            bar_init(smem_addr(&bars.p2[i]), 4);
            bar_init(smem_addr(&bars.o[i]), 1);
            bar_init(smem_addr(&bars.o_read[i]), 4);
            bar_init(smem_addr(&bars.ml[i]), 4);
            bar_init(smem_addr(&bars.ml_read[i]), 4);
        }
        bar_init(smem_addr(&bars.last), 1);
        bar_init(smem_addr(&bars.done), 4);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }

    for (int i = t; i < kOddUnits; i += kThreads) s_marks[i] = 0;
    if (warp == 12) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(&s_tmem)), "r"(S::kColumns)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (t == 13 * 32) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_k) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&map_v) : "memory");
        if (p.q_mapped) asm volatile("prefetch.tensormap [%0];" ::"l"(&map_q) : "memory");
    }

    // ---- this CTA's stretch of the line, its first unit for all roles ----
    int64_t stretch_end = 0;
    {
        // the sequences' row tiles; each sequence's first one is kept where the operands will lie
        int32_t* first = reinterpret_cast<int32_t*>(smem);
        const int per = (b.seqs + kThreads - 1) / kThreads, s_lo = min(t * per, b.seqs), s_hi = min(s_lo + per, b.seqs);
        int64_t mine = 0, row_tiles = 0;
        bool bad_starts = false;
        int32_t pre = 0, lo = p.shared_len;
        for (int s = s_lo; s < s_hi; ++s) {
            const int32_t from = b.row_start[s], to = b.row_start[s + 1];
            bad_starts |= from < 0 || from > to || to > b.rows;
            if (kShared) {
                if (p.window > 0) {
                    const KvSpan x = seen_of_prefix(p, s);
                    pre = max(pre, x.pre);
                    lo = min(lo, x.lo);
                }
                continue;
            }
            const Many m = many_seq<kShared>(p, s);
            if (m.bad && blockIdx.x == 0) {
                kv_report(p.status, GFD_KV_BAD_LENGTH);
                if (from >= 0 && to <= b.rows) kv_mark_skipped(p, s);
            }
            mine += m.tiles;
        }
        if (kShared) {
            pre = __reduce_max_sync(0xffffffffu, pre);
            lo = __reduce_min_sync(0xffffffffu, lo);
            if (lane == 0) {
                s_reach[warp][0] = pre;
                s_reach[warp][1] = lo;
            }
        }
        const bool ok = __syncthreads_or(bad_starts) == 0;
        if (!ok && blockIdx.x == 0 && t == 0) kv_report(p.status, GFD_KV_BAD_LENGTH);
        const int seqs = !ok ? 0 : (kShared ? 1 : b.seqs);
        if (kShared) {
            for (int w = 0; w < kThreads / 32; ++w) {
                pre = max(pre, s_reach[w][0]);
                lo = min(lo, s_reach[w][1]);
            }
            // (without a window every row sees all of it)
            if (p.window == 0) lo = 0;
            if (t == 0) s_seen = lo < p.shared_len ? KvSpan{pre, max(lo, pre), p.shared_len} : KvSpan{pre, pre, pre};
            first[0] = 0;
            row_tiles = ok ? many_seq<kShared>(p, 0).tiles : 0;
        } else {
            int64_t run = cta_scan(mine, s_warps, &row_tiles) - mine;
            if (!ok) row_tiles = 0;
            for (int s = s_lo; s < s_hi; ++s) {
                first[s] = static_cast<int32_t>(run);
                if (per > 1) run += many_seq<kShared>(p, s).tiles;
            }
        }
        __syncthreads();
        // tiles of this thread's row tiles, then where the stretch begins
        const int64_t each = (row_tiles + kThreads - 1) / kThreads;
        const int64_t u0 = min(t * each, row_tiles), u1 = min(u0 + each, row_tiles);
        int s0 = 0;
        Many m0{};
        if (u0 < u1) {
            int lo = 0, hi = seqs - 1;
            while (lo < hi) {
                const int mid = (lo + hi + 1) / 2;
                if (first[mid] <= u0) lo = mid;
                else hi = mid - 1;
            }
            s0 = lo;
            m0 = many_seq<kShared>(p, s0);
        }
        int64_t per_head = 0, total = 0, want = -1, head = 0;
        for (int pass = 0; pass < 2; ++pass) {
            int s = s0;
            Many m = m0;
            int64_t here = pass == 0 ? 0 : mine;
            for (int64_t u = u0; u < u1; ++u) {
                while (u - first[s] >= m.tiles) m = many_seq<kShared>(p, ++s);
                const int rt = static_cast<int>(u - first[s]);
                const Unit x = many_unit<kShared>(p, s, m.q, rt, s_seen);
                if (want >= here && want < here + x.tiles.count + kUnitCost) {
                    const int64_t begin = head * per_head + here + kUnitCost;
                    const int32_t t0 = static_cast<int32_t>(max(want - here - kUnitCost, static_cast<int64_t>(0)));
                    s_place.s = s;
                    s_place.h = static_cast<int32_t>(head);
                    s_place.t = t0;
                    s_place.count = x.tiles.count;
                    s_place.begin = begin;
                    s_place.row0 = m.q.row0;
                    s_place.packed0 = x.packed0;
                    s_place.packed = x.packed;
                    const int64_t t1 = min(static_cast<int64_t>(x.tiles.count), max(stretch_end - begin, static_cast<int64_t>(0)));
                    s_unit[0] = describe<kShared>(p, s, static_cast<int32_t>(head), t0, static_cast<int32_t>(t1), m.q, x);
                }
                here += x.tiles.count + kUnitCost;
            }
            if (pass == 0) {
                mine = cta_scan(here, s_warps, &per_head) - here;
                total = per_head * p.cache.heads;
                const KvCuts cuts(total, gridDim.x);
                if (static_cast<int>(blockIdx.x) < cuts.n()) {
                    const int64_t at = cuts.at(blockIdx.x);
                    stretch_end = cuts.at(blockIdx.x + 1);
                    head = kv_div(at, per_head);
                    want = at - head * per_head;
                }
            }
        }
        // (threads of CTAs without a stretch have found no place)
        __syncthreads();
        if (t == kThreads - 1)
            p.line.cuts[blockIdx.x] = stretch_end > 0 ? kv_cut(KvCuts(total, gridDim.x), blockIdx.x, s_place) : KvCut{};
    }
    tm_before();
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // `first` lay where Q goes
    __syncthreads();
    tm_after();
    const uint32_t tmem = s_tmem;
    if (stretch_end == 0) {
        if (warp == 12) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::kColumns) : "memory");
        kv_wait_last();
        return;
    }
    const uint32_t sq = smem_addr(smem), ring = sq + 2 * S::kOperand;
    volatile KvWaits* waits = &s_waits;
    volatile int* gave_up = &s_waits.gave_up;
    // The next unit, read by a whole warp (every role takes every unit, in order).
    int unit = 0;
    auto take = [&](Desc* d) -> bool {
        const int i = unit % kUnitRing;
        if (!bar_wait(smem_addr(&bars.unit[i]), (unit / kUnitRing) & 1, gave_up)) return false;
        *d = s_unit[i];
        __syncwarp();
        if (lane == 0) bar_arrive(smem_addr(&bars.unit_read[i]));
        ++unit;
        return d->nt > 0;
    };

    if (warp < 8) {
        // ---- softmax: one thread per packed row ----
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kMain));
        const int x = warp >> 2;
        const int rr = t & (kHalf - 1);                                        // row of the half
        const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;  // this warp's lanes of tensor memory
        const uint32_t ts = tmem + lanes + x * kTile, to = tmem + lanes + S::kO + x * D;
        const int32_t base_key = kShared ? 0 : p.shared_len;
        uint32_t s_phase = 0, ml_phase = 0;
        int seen = 0;
        Desc u;
        while (take(&u)) {
            if (x * kHalf >= u.packed) {  // this half has no rows
                seen += u.nt;
                continue;
            }
            int32_t pos;
            const KvSpan sp = row_span<kShared>(p, u, x * kHalf + rr, &pos, !kPlain);
            float slope = 0.0f;
            if (!kPlain && p.alibi != nullptr) slope = p.alibi[u.h * p.group + (u.packed0 + x * kHalf + rr) % p.group] * kLog2e;
            const float scale = kPlain ? p.scale2 : 1.0f;
            float base = -INFINITY, l = 0.0f;  // the weights' base (2^base), -inf before the first key; their sum
            bool good = true;
            for (int i = 0; i < u.nt; ++i, ++seen) {
                good = bar_wait(smem_addr(&bars.s[x]), s_phase, gave_up);
                s_phase ^= 1u;
                if (!good) break;
                tm_after();
                const int32_t j0 = u.key(i);
                const uint32_t bad = *reinterpret_cast<volatile uint32_t*>(&s_bad[seen % kBadRing]);
                const bool inside = (j0 >= sp.lo && j0 + kTile <= sp.hi) || sp.pre >= j0 + kTile;
                const bool masked = __any_sync(0xffffffffu, !inside) || bad != 0;
                uint32_t z[kTile];
#pragma unroll
                for (int k = 0; k < kTile; k += 32) tm_ld32(ts + k, z + k);
#pragma unroll
                for (int k = 0; k < kTile; k += 32) tm_wait32(z + k);
                // keys [j0 + k, j0 + k + 32) that the row sees, a bit each
                auto sees = [&](int k) {
                    const int32_t j = j0 + k;
                    const uint32_t out = (((bad >> (k / kKvPage)) & 1u) ? 0x0000ffffu : 0u) | (((bad >> (k / kKvPage)) & 2u) ? 0xffff0000u : 0u);
                    return (below(sp.pre - j) | (below(sp.hi - j) & ~below(sp.lo - j))) & ~out;
                };
                if (!kPlain) {
                    kv_cap<kTile>(p, z, masked, sees);
                    if (p.alibi != nullptr) {
                        const float d0 = static_cast<float>(base_key + j0 - pos);
                        const uint64_t from = pack2(d0, d0), by = pack2(slope, slope);
#pragma unroll
                        for (int e = 0; e < kTile; e += 2) {
                            float a, c;
                            unpack2(fma2(add2(from, pack2(static_cast<float>(e), static_cast<float>(e + 1))), by,
                                         pack2(__uint_as_float(z[e]), __uint_as_float(z[e + 1]))), a, c);
                            z[e] = __float_as_uint(a);
                            z[e + 1] = __float_as_uint(c);
                        }
                    }
                }
                if (masked)
#pragma unroll
                    for (int k = 0; k < kTile; k += 32) {
                        const uint32_t some = sees(k);
#pragma unroll
                        for (int e = 0; e < 32; ++e) z[k + e] = (some & (1u << e)) != 0 ? z[k + e] : 0xff800000u;
                    }
                float m8[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) m8[e] = __uint_as_float(z[e]);
#pragma unroll
                for (int e = 8; e < 120; e += 16)
#pragma unroll
                    for (int y = 0; y < 8; ++y) m8[y] = max3(m8[y], __uint_as_float(z[e + 2 * y]), __uint_as_float(z[e + 2 * y + 1]));
#pragma unroll
                for (int y = 0; y < 4; ++y) m8[y] = max3(m8[y], __uint_as_float(z[120 + 2 * y]), __uint_as_float(z[121 + 2 * y]));
                const float most = max3(max3(m8[0], m8[1], m8[2]), max3(m8[3], m8[4], m8[5]), max3(m8[6], m8[7], m8[7]));
                if (!(most < INFINITY)) l = __int_as_float(0x7fffffff);  // a NaN or an infinity among the scores
                const float top = most * scale - Shift<T>::value;
                const bool grew = top > base + kGrow || (base == -INFINITY && top > -INFINITY);
                if (__any_sync(0xffffffffu, grew)) {
                    // (a row's base moves by its own scores alone, so that its roundings do not go by its neighbours)
                    const float keep = grew ? fast_exp2(base - top) : 1.0f;
                    base = grew ? top : base;
                    l *= keep;
                    if (i > 0) {
#pragma unroll 1
                        for (int k = 0; k < D; k += 16) {
                            uint32_t o[16];
                            tm_ld16(to + k, o);
                            tm_wait16(o);
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * keep);
                            tm_st16(to + k, o);
                        }
                    }
                }
                const float less = base == -INFINITY ? 0.0f : -base;
                const uint64_t scale_2 = pack2(scale, scale), less_2 = pack2(less, less);
                uint64_t sum0 = 0, sum1 = 0;  // pairs of 0.0f
#pragma unroll
                for (int k = 0; k < kTile; k += 32) {
                    uint32_t w[16];
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        float a, c;
                        unpack2(fma2(pack2(__uint_as_float(z[k + 2 * e]), __uint_as_float(z[k + 2 * e + 1])), scale_2, less_2), a, c);
                        if (kPlain && e >= 16 - ByPoly<D>::value) {
                            unpack2(poly_exp2(pack2(a, c)), a, c);
                        } else {
                            a = fast_exp2(a);
                            c = fast_exp2(c);
                        }
                        if (e & 1) sum1 = add2(sum1, pack2(a, c));
                        else sum0 = add2(sum0, pack2(a, c));
                        w[e] = Pack<T>::pair(a, c);
                    }
                    tm_st16(ts + k / 2, w);
                    if (k == 32 || k == 96) {
                        tm_wait_st();
                        tm_before();
                        __syncwarp();
                        if (lane == 0) bar_arrive(smem_addr(k == 32 ? &bars.p[x] : &bars.p2[x]));
                    }
                }
                {
                    float a, c;
                    unpack2(add2(sum0, sum1), a, c);
                    l += a + c;
                }
            }
            if (!good) break;
            // base and sum go to the warps that write the rows
            if (!bar_wait(smem_addr(&bars.ml_read[x]), ml_phase ^ 1u, gave_up)) break;
            ml_phase ^= 1u;
            s_base[x][rr] = base;
            s_sum[x][rr] = l;
            __syncwarp();
            if (lane == 0) bar_arrive(smem_addr(&bars.ml[x]));
        }
        // the warps that write are done, and with them all copies and products
        __syncwarp();
        asm volatile("bar.sync 1, 384;" ::: "memory");
        uint32_t some = 0;
        for (int i = lane; i < kOddUnits; i += 32) some |= s_marks[i];
        if (__any_sync(0xffffffffu, some != 0) && *gave_up == 0) {
            if (kShared) kv_wait_last();
            sum_again<T, D, kPlain, kShared>(p, s_place, stretch_end, sq, s_flags, s_marks, s_seen);
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kAux));
        if (warp < 12) {
            // ---- finished rows ----
            const uint32_t lanes = static_cast<uint32_t>((warp & 3) * 32) << 16;
            // rows that begin on 32 bytes are written 32 bytes at a time
            const bool wide = ((reinterpret_cast<uint64_t>(p.out.data) | p.out.row_stride | p.out.head_stride) & 31) == 0;
            uint32_t o_phase = 0;  // bit x
            bool good = true;
            if (kShared) {
                kv_wait_last();  // the results over the own keys, which finish here
                if (t == 8 * 32) waits->held = 0;
            }
            // The unit is read where it lies, and given back when its rows are written: with a copy of it
            // in registers this loop's spilled, and with 2/3 of the SM's memory taken by
            // operands, what is spilled comes back from L2.
            for (; good; ++unit) {
                const Desc& u = s_unit[unit % kUnitRing];
                if (!bar_wait(smem_addr(&bars.unit[unit % kUnitRing]), (unit / kUnitRing) & 1, gave_up) || u.nt <= 0) break;
                const bool whole = u.nt == u.count;
                float* slot = p.line.slots + (2 * static_cast<int64_t>(blockIdx.x) + (u.t0 == 0 ? 1 : 0)) * (static_cast<int64_t>(kRows) * (D + 2));
                for (int x = 0; x * kHalf < u.packed; ++x) {
                    const int rr = (warp & 3) * 32 + lane, r = x * kHalf + rr;
                    const int32_t packed = u.packed0 + (r < u.packed ? r : 0);
                    const int32_t of = kv_div_group(p, packed);
                    const int64_t row = u.row0 + of;
                    const int32_t head = u.h * p.group + packed - of * p.group;
                    const float own_lse = kShared ? p.own_lse[row * p.q_heads + head] : -INFINITY;
                    const bool valid = r < u.packed && (!whole || !kShared || __float_as_uint(own_lse) != kKvSkipped);
                    uint64_t dst = 0;
                    if (valid && whole) dst = reinterpret_cast<uint64_t>(p.out.data + row * p.out.row_stride + head * p.out.head_stride);
                    const uint32_t phase = (o_phase >> x) & 1u;
                    o_phase ^= 1u << x;
                    good = bar_wait(smem_addr(&bars.ml[x]), phase, gave_up) && bar_wait(smem_addr(&bars.o[x]), phase, gave_up);
                    if (!good) break;
                    tm_after();
                    const float base = s_base[x][rr], l = s_sum[x][rr];
                    __syncwarp();
                    if (lane == 0) bar_arrive(smem_addr(&bars.ml_read[x]));
                    uint64_t odd0 = 0, odd1 = 0;      // pairs of 0.0f, NaN once a sum is not finite
                    KvFinish f{1.0f, 0.0f, base, l};  // what becomes of the sums
                    const float* own = nullptr;
                    if (whole) {
                        f = kv_finish<kShared>(p, base, l, own_lse);
                        if (kShared && valid && f.own != 0.0f) own = p.own_out + (row * p.q_heads + head) * D;
                    }
#pragma unroll 1
                    for (int k = 0; k < D; k += 32) {
                        uint32_t o[32];
                        tm_ld32(tmem + lanes + S::kO + x * D + k, o);
                        tm_wait32(o);
                        if (k + 32 == D) {
                            tm_before();
                            __syncwarp();
                            if (lane == 0) bar_arrive(smem_addr(&bars.o_read[x]));
                        }
                        const uint64_t by = pack2(f.scale, f.scale);
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            const uint64_t v = pack2(__uint_as_float(o[e]), __uint_as_float(o[e + 1]));
                            uint64_t& odd = e & 2 ? odd1 : odd0;
                            odd = fma2(v, 0, odd);
                            float a, c;
                            unpack2(mul2(v, by), a, c);
                            o[e] = __float_as_uint(a);
                            o[e + 1] = __float_as_uint(c);
                        }
                        if (!whole) {
                            // partial sums: 4 elements of 32 rows side by side
                            if (valid)
#pragma unroll
                                for (int e = 0; e < 32; e += 4)
                                    *reinterpret_cast<uint4*>(slot + (static_cast<int64_t>((k + e) / 4) * kRows + r) * 4) =
                                        make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                            continue;
                        }
                        if (kShared && own != nullptr)
#pragma unroll
                            for (int e = 0; e < 32; e += 4) {
                                const float4 y = *reinterpret_cast<const float4*>(own + k + e);
                                o[e] = __float_as_uint(fmaf(y.x, f.own, __uint_as_float(o[e])));
                                o[e + 1] = __float_as_uint(fmaf(y.y, f.own, __uint_as_float(o[e + 1])));
                                o[e + 2] = __float_as_uint(fmaf(y.z, f.own, __uint_as_float(o[e + 2])));
                                o[e + 3] = __float_as_uint(fmaf(y.w, f.own, __uint_as_float(o[e + 3])));
                            }
                        if (dst == 0) continue;
                        if (p.out_f32) {
#pragma unroll
                            for (int e = 0; e < 32; e += 8) store8(dst + 4 * (k + e), o + e, wide);
                        } else {
#pragma unroll
                            for (int e = 0; e < 16; ++e) o[e] = Pack<T>::pair(__uint_as_float(o[2 * e]), __uint_as_float(o[2 * e + 1]));
                            store8(dst + 2 * k, o, wide);
                            store8(dst + 2 * k + 32, o + 8, wide);
                        }
                    }
                    if (valid) {
                        if (whole) {
                            if (p.lse != nullptr) p.lse[row * p.q_heads + head] = kv_lse(p, f.base, f.sum);
                        } else {
                            slot[static_cast<int64_t>(kRows) * D + r] = base;
                            slot[static_cast<int64_t>(kRows) * D + kRows + r] = l;
                        }
                    }
                    float odd, odd_c;
                    unpack2(add2(odd0, odd1), odd, odd_c);
                    odd += odd_c;
                    // (a weight sum that is not finite makes the row NaN as it is)
                    const uint32_t again = __ballot_sync(0xffffffffu, valid && odd != 0.0f && l < INFINITY);
                    if (again != 0 && lane == 0) *const_cast<volatile uint8_t*>(&s_marks[min(unit, kOddUnits - 1)]) = 1;
                }
                __syncwarp();
                if (lane == 0) bar_arrive(smem_addr(&bars.unit_read[unit % kUnitRing]));
            }
            __syncwarp();
            if (lane == 0) bar_arrive(smem_addr(&bars.done));
            asm volatile("bar.arrive 1, 384;" ::: "memory");
        } else if (warp == 12) {
            // ---- products: the whole warp walks, one thread issues ----
            int slot = 0;
            uint32_t full_phase = 0, q_phase = 0, p_phase = 0, or_phase = 0;
            constexpr uint32_t kQk = product<T>(kHalf, kTile, false);
            constexpr uint32_t kPv = product<T>(kHalf, D, true);
            const uint32_t q_low = operand(sq, 16), k_low = operand(ring, 16), v_low = operand(ring, S::kBlock);
            auto scores = [&](int x, int k) {
                const uint32_t a = q_low + x * (S::kOperand >> 4), c = k_low + k * (S::kOperand >> 4);
#pragma unroll
                for (int i = 0; i < D / 16; ++i) {
                    constexpr int kStep = S::kBlock >> 4;
                    mma_ss(tmem + x * kTile, a + (i / 4) * kStep + (i % 4) * 2, c + (i / 4) * kStep + (i % 4) * 2, kQk, i > 0);
                }
            };
            auto sums = [&](int x, int v, int j0, int j1, bool add) {
                const uint32_t c = v_low + v * (S::kOperand >> 4);
#pragma unroll
                for (int j = j0; j < j1; ++j) mma_ts(tmem + S::kO + x * D, tmem + x * kTile + j * 8, c + j * (2048 >> 4), kPv, add || j > 0);
            };
            uint32_t steps = 0;
            Desc u;
            bool good = true;
            while (good && take(&u)) {
                const int halves = u.packed > kHalf ? 2 : 1, nt = u.nt;
                good = bar_wait(smem_addr(&bars.full[slot]), (full_phase >> slot) & 1u, gave_up);
                for (int x = 0; good && x < halves; ++x) {
                    good = bar_wait(smem_addr(&bars.q[x]), (q_phase >> x) & 1u, gave_up);
                    q_phase ^= 1u << x;
                    if (!good) break;
                    tm_after();
                    if (elect_one()) {
                        scores(x, slot);
                        tm_commit(smem_addr(&bars.s[x]));
                        if (nt == 1) tm_commit(smem_addr(&bars.q_read[x]));
                        if (x == halves - 1) tm_commit(smem_addr(&bars.empty[slot]));
                    }
                    __syncwarp();
                }
                full_phase ^= 1u << slot;
                slot = slot + 1 == S::kSlots ? 0 : slot + 1;
                for (int i = 0; good && i < nt; ++i) {
                    const int v = slot, k = slot + 1 == S::kSlots ? 0 : slot + 1;
                    const bool more = i + 1 < nt;
                    good = bar_wait(smem_addr(&bars.full[v]), (full_phase >> v) & 1u, gave_up);
                    full_phase ^= 1u << v;
                    for (int x = 0; good && x < halves; ++x) {
                        if (i == 0) {  // the last unit's sums have been taken
                            good = bar_wait(smem_addr(&bars.o_read[x]), ((or_phase >> x) & 1u) ^ 1u, gave_up);
                            or_phase ^= 1u << x;
                            if (!good) break;
                        }
                        // the weights come in two parts of 64 keys
                        good = bar_wait(smem_addr(&bars.p[x]), (p_phase >> x) & 1u, gave_up);
                        if (!good) break;
                        tm_after();
                        if (elect_one()) sums(x, v, 0, kTile / 32, i > 0);
                        __syncwarp();
                        good = bar_wait(smem_addr(&bars.p2[x]), (p_phase >> x) & 1u, gave_up);
                        p_phase ^= 1u << x;
                        if (!good) break;
                        if (more && x == 0) {
                            good = bar_wait(smem_addr(&bars.full[k]), (full_phase >> k) & 1u, gave_up);
                            full_phase ^= 1u << k;
                            if (!good) break;
                        }
                        tm_after();
                        if (elect_one()) {
                            sums(x, v, kTile / 32, kTile / 16, true);
                            if (x == halves - 1) tm_commit(smem_addr(&bars.empty[v]));
                            if (more) {
                                scores(x, k);
                                tm_commit(smem_addr(&bars.s[x]));
                                if (i + 2 == nt) tm_commit(smem_addr(&bars.q_read[x]));
                                if (x == halves - 1) tm_commit(smem_addr(&bars.empty[k]));
                            } else {
                                tm_commit(smem_addr(&bars.o[x]));
                            }
                        }
                        __syncwarp();
                    }
                    slot = k;
                    if (more) slot = k + 1 == S::kSlots ? 0 : k + 1;
                    if (lane == 0) waits->steps = ++steps;
                }
            }
            // tensor memory and the operands stay until the last product is done
            if (elect_one()) tm_commit(smem_addr(&bars.last));
            __syncwarp();
            bar_drain(smem_addr(&bars.last), 0);
        } else if (warp == 13) {
            // ---- K and V ----
            int slot = 0, seen = 0;  // seen: tiles so far
            uint32_t phase = 0;      // bit i: parity that slot i's `empty` has to reach
            const int pages = p.cache.block_tokens / kKvPage;
            Desc u;
            bool good = true;
            while (good && take(&u)) {
                const int32_t* table = kShared ? p.shared_table : b.table + u.s * b.table_stride;
                const int32_t n = u.keys;
                for (int i = 0; good && i < u.nt; ++i, ++seen) {
                    const int32_t j0 = u.key(i);
                    // lane i: page i % 8 of the tile
                    const int32_t j = j0 + (lane % kPages) * kKvPage;
                    int32_t id = p.cache.blocks;  // a block outside the map: loads as zeros
                    bool bad = false;
                    if ((j < u.pre || (j + kKvPage > u.lo && j < u.hi)) && j < n) {
                        id = table[kv_div_pages(p, j / kKvPage)];
                        if (id < 0 || id >= p.cache.blocks) {
                            bad = true;
                            id = p.cache.blocks;
                            kv_report(p.status, GFD_KV_BAD_PAGE);
                        }
                    }
                    const int32_t in_block = (j / kKvPage - kv_div_pages(p, j / kKvPage) * pages) * kKvPage;
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
                            const char* src = p.cache.v + (hid < p.cache.blocks ? hid : 0) * p.cache.block_stride +
                                              hpl * p.cache.token_stride + u.h * p.cache.head_stride;
                            for (int y = lane; y < kKvPage * D / 8; y += 32) {
                                const int r = y / (D / 8), ch = y % (D / 8);
                                uint4 v = make_uint4(0, 0, 0, 0);
                                if (hid < p.cache.blocks && r < rest % kKvPage)
                                    v = *reinterpret_cast<const uint4*>(src + r * p.cache.token_stride + 16 * ch);
                                const uint32_t o = dst + (ch / 8) * S::kBlock + (cut_page * kKvPage + r) * 128 + (((ch % 8) ^ (r & 7)) << 4);
                                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(o), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w)
                                             : "memory");
                            }
                            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        }
                        __syncwarp();
                        if (lane == 0) bar_expect(full, S::kOperand - (by_hand ? kKvPage * D * 2 : 0));
                        __syncwarp();
                        const int page = lane % kPages, block = lane / kPages;
                        if (block < S::kBlocks && !(by_hand && page == cut_page))
                            tma_page(dst + block * S::kBlock + page * kKvPage * 128, which == 0 ? &map_k : &map_v, block * 64, u.h, in_block,
                                     id, full);
                        phase ^= 1u << slot;
                        slot = slot + 1 == S::kSlots ? 0 : slot + 1;
                    }
                }
            }
            // the copies in flight land before the block ends: `full` flips once more for each slot that was filled
            for (int i = 0; i < S::kSlots; ++i) bar_drain(smem_addr(&bars.full[i]), ((phase >> i) & 1u) ^ 1u);
        } else if (warp == 14) {
            // ---- Q ----
            uint32_t phase = 0;  // bit x
            if (p.q_mapped) {
                // a box of [64 elements][heads of the group][rows]: packed rows in order.  Rows behind
                // the sequence's last one bring whatever follows it into rows that nothing is written for.
                Desc u;
                bool good = true;
                while (good && take(&u)) {
                    const int head = u.h * p.group, row = u.row0 + kv_div_group(p, u.packed0), by = kHalf / p.group;
                    if (lane < 2 * S::kBlocks && lane / S::kBlocks * kHalf < u.packed)
                        tma_rows_ahead(&map_q, lane % S::kBlocks * 64, head, row + lane / S::kBlocks * by);
                    for (int x = 0; good && x * kHalf < u.packed; ++x) {
                        good = bar_wait(smem_addr(&bars.q_read[x]), ((phase >> x) & 1u) ^ 1u, gave_up);
                        if (!good) break;
                        phase ^= 1u << x;
                        const uint32_t there = smem_addr(&bars.q[x]);
                        if (lane == 0) bar_expect(there, S::kOperand);
                        __syncwarp();
                        if (lane < S::kBlocks)
                            tma_rows(sq + x * S::kOperand + lane * S::kBlock, &map_q, lane * 64, head, row + x * by, there);
                    }
                }
                for (int x = 0; x < 2; ++x) bar_drain(smem_addr(&bars.q[x]), ((phase >> x) & 1u) ^ 1u);  // likewise
            }
            // groups and strides that no box has: every row by neighbouring lanes, zeros for rows that do not exist
            constexpr int kLanes = D / 8, kPer = 32 / kLanes;  // lanes of a row, rows a step
            const int ch = lane % kLanes, sub = lane / kLanes;
            const uint32_t to = sq + (ch / 8) * S::kBlock + sub * 128;
            Desc u;
            bool good = !p.q_mapped;
            while (good && take(&u)) {
                // where the unit's rows lie, and a start on bringing them into L2
                __syncwarp();
                for (int r = lane; r < u.packed; r += 32) {
                    const int32_t packed = u.packed0 + r, of = kv_div_group(p, packed);
                    const char* at = p.q.data + static_cast<int64_t>(u.row0 + of) * p.q.row_stride +
                                     (u.h * p.group + packed - of * p.group) * p.q.head_stride;
                    s_rows[r] = at;
                    asm volatile("prefetch.global.L2 [%0];" ::"l"(at));
                    if (D == 128) asm volatile("prefetch.global.L2 [%0];" ::"l"(at + 128));
                }
                __syncwarp();
                for (int x = 0; good && x * kHalf < u.packed; ++x) {
                    good = bar_wait(smem_addr(&bars.q_read[x]), ((phase >> x) & 1u) ^ 1u, gave_up);
                    phase ^= 1u << x;
                    if (!good) break;
                    const int n = min(kHalf, u.packed - x * kHalf);
#pragma unroll 8
                    for (int y = 0; y < kHalf; y += kPer) {
                        const char* at = p.q.data;
                        const bool live = y + sub < n;
                        if (live) at = s_rows[x * kHalf + y + sub] + 16 * ch;
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to + x * S::kOperand + y * 128 +
                                                                                           (((ch % 8) ^ ((y + sub) & 7)) << 4)),
                                     "l"(at), "r"(live ? 16 : 0)
                                     : "memory");
                    }
                    asm volatile("cp.async.wait_all;" ::: "memory");
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) bar_arrive(smem_addr(&bars.q[x]));
                }
            }
        } else {
            // ---- the units of the stretch; the first one is there.  This warp watches over the others' waits ----
            if (lane == 0) bar_arrive(smem_addr(&bars.unit[0]));
            Cursor<kShared> c;
            c.enter(p, s_place, stretch_end, s_seen);
            for (int i = 1; !c.done; ++i) {
                c.next(p, s_seen);
                const int k = i % kUnitRing;
                if (!bar_watch(smem_addr(&bars.unit_read[k]), ((i / kUnitRing) & 1) ^ 1, waits)) break;
                if (lane == 0) {
                    s_unit[k] = describe<kShared>(p, c.s, c.h, c.t, c.done ? c.t : c.end, c.m.q, c.u);
                    bar_arrive(smem_addr(&bars.unit[k]));
                }
                __syncwarp();
            }
            bar_watch(smem_addr(&bars.done), 0, waits);
        }
    }

    // ---- end ----
    tm_before();
    __syncthreads();
    tm_after();
    if (t == 0 && s_waits.gave_up != 0) kv_report(p.status, GFD_KV_GAVE_UP);
    if (warp == 12) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(S::kColumns) : "memory");
    kv_wait_last();
}

// The cache's K or V as [blocks][tokens][heads][D], read in boxes of 16 tokens x 64 elements.
bool make_map(CUtensorMap* map, const KvCacheView& c, const char* base, int head_dim, int dtype, KvEncodeFn encode) {
    const cuuint64_t row = static_cast<cuuint64_t>(head_dim) * 2;
    const cuuint64_t dims[4] = {static_cast<cuuint64_t>(head_dim), static_cast<cuuint64_t>(c.heads), static_cast<cuuint64_t>(c.block_tokens),
                                static_cast<cuuint64_t>(c.blocks)};
    // the stride of a dimension of one is not used, but has to be one that the map takes
    const cuuint64_t strides[3] = {c.heads > 1 ? static_cast<cuuint64_t>(c.head_stride) : row, static_cast<cuuint64_t>(c.token_stride),
                                   c.blocks > 1 ? static_cast<cuuint64_t>(c.block_stride) : row};
    const cuuint32_t box[4] = {64, 1, kKvPage, 1}, ones[4] = {1, 1, 1, 1};
    return encode(map, dtype == GFD_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<char*>(base),
                  dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Q as [rows][heads][D], read in boxes of 128 packed rows x 64 elements.  Not where a group's heads do
// not divide 128, nor with strides that no map takes (rows or heads that are one and the same, say).
bool make_rows_map(CUtensorMap* map, const KvAttendParams& p, int head_dim, int dtype, KvEncodeFn encode) {
    const cuuint64_t row = static_cast<cuuint64_t>(head_dim) * 2;
    if (p.group > kHalf || kHalf % p.group != 0 || (p.q_heads > 1 && p.q.head_stride == 0) || (p.batch.rows > 1 && p.q.row_stride == 0))
        return false;
    const cuuint64_t dims[3] = {static_cast<cuuint64_t>(head_dim), static_cast<cuuint64_t>(p.q_heads), static_cast<cuuint64_t>(p.batch.rows)};
    const cuuint64_t strides[2] = {p.q_heads > 1 ? static_cast<cuuint64_t>(p.q.head_stride) : row,
                                   p.batch.rows > 1 ? static_cast<cuuint64_t>(p.q.row_stride) : row};
    const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(p.group), static_cast<cuuint32_t>(kHalf / p.group)}, ones[3] = {1, 1, 1};
    return encode(map, dtype == GFD_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, p.q.data, dims, strides, box,
                  ones, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <typename T, int D>
cudaError_t launch(const KvAttendParams& p, const KvMaps& maps, int ctas, bool chained, cudaStream_t st) {
    const bool plain = p.softcap == 0.0f && p.alibi == nullptr && p.scale2 > 0.0f;
    auto* f = p.shared_pass ? (plain ? kv_prompt_kernel<T, D, true, true> : kv_prompt_kernel<T, D, false, true>)
                            : (plain ? kv_prompt_kernel<T, D, true, false> : kv_prompt_kernel<T, D, false, false>);
    const cudaError_t e = kv_launch(f, dim3(ctas), kThreads, Shape<D>::kSmem, st, chained, p, maps.k, maps.v, maps.q);
    if (e != cudaSuccess) return e;
    return launch_kv_join_many(p, D, std::is_same<T, __half>::value ? GFD_FP16 : GFD_BF16, ctas, st);
}

}  // namespace

int kv_prompt_ctas(int num_sms) { return num_sms; }

bool kv_make_maps(KvMaps* maps, const KvAttendParams& p, int head_dim, int dtype, KvEncodeFn encode) {
    *maps = KvMaps{};
    maps->q_mapped = make_rows_map(&maps->q, p, head_dim, dtype, encode);
    return make_map(&maps->k, p.cache, p.cache.k, head_dim, dtype, encode) && make_map(&maps->v, p.cache, p.cache.v, head_dim, dtype, encode);
}

cudaError_t launch_kv_prompt(const KvAttendParams& p, int head_dim, int dtype, int num_sms, const KvMaps& maps, bool chained, cudaStream_t st) {
    const int ctas = kv_prompt_ctas(num_sms);
    if (dtype == GFD_BF16) return head_dim == 64 ? launch<__nv_bfloat16, 64>(p, maps, ctas, chained, st) : launch<__nv_bfloat16, 128>(p, maps, ctas, chained, st);
    return head_dim == 64 ? launch<__half, 64>(p, maps, ctas, chained, st) : launch<__half, 128>(p, maps, ctas, chained, st);
}

}  // namespace gfdb
