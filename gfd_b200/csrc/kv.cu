// Paged KV-cache operators: append with rotation, merge of partial results, and the join of an
// attention launch's own partial results.

#include "kv_device.cuh"

namespace gfdb {
namespace {

// ---------------------------------------------------------------------------
// Append
// ---------------------------------------------------------------------------
// A head is cut into items of 16 elements that one thread moves: item i < rot_dim / 16
// holds the 8 pairs that rotate together (two 16-byte pieces rot_dim / 2 apart, or 16
// neighbours when interleaved), the items above copy.  A CTA takes kRows rows: their
// places and the sines and cosines of their rot_dim / 2 angles are formed once in shared
// memory and serve all K and Q heads.  Angles: p * inv_freq is exact in 64 bits up to
// p = 2^29, and a turn is taken off in 64 bits before the 32-bit sine, so a position of a
// million is as accurate as a small one.
constexpr int kAppendThreads = 256;

template <typename T, int D>
__global__ void __launch_bounds__(kAppendThreads) kv_append_kernel(const KvAppendParams p, int rows_per_cta) {
    constexpr int kMaxRows = 4;
    __shared__ float s_cos[kMaxRows][D / 2], s_sin[kMaxRows][D / 2];
    __shared__ int32_t s_seq[kMaxRows], s_block[kMaxRows], s_place[kMaxRows], s_pos[kMaxRows];
    const KvBatchView& b = p.batch;
    const int t = threadIdx.x;
    const int32_t row0 = blockIdx.x * rows_per_cta;
    const int nrows = min(rows_per_cta, b.rows - row0);
    if (t < kMaxRows) s_seq[t] = -1;
    if (!kv_starts_ok(b)) {  // syncs
        if (blockIdx.x == 0 && t == 0) kv_report(p.status, GFD_KV_BAD_LENGTH);
        return;
    }
    for (int s = t; s < b.seqs; s += kAppendThreads) {
        const int32_t a = b.row_start[s], e = b.row_start[s + 1];
        if (a >= row0 + nrows || e <= row0 || a == e) continue;
        const KvSeq q = kv_seq(a, e, b.kv_len[s], b.capacity, 0);
        if (!q.ok) {
            kv_report(p.status, GFD_KV_BAD_LENGTH);
            continue;
        }
        for (int i = max(a - row0, 0); i < min(e - row0, nrows); ++i) {
            const int32_t pos = q.keys - q.rows + (row0 + i - a);
            int32_t place;
            const int32_t block = kv_block(b, s, pos, p.cache.block_tokens, nullptr, 0, &place);
            s_seq[i] = s;
            s_place[i] = place;
            s_block[i] = block >= 0 && block < p.cache.blocks ? block : -1;
            if (s_block[i] < 0) kv_report(p.status, GFD_KV_BAD_PAGE);
            s_pos[i] = p.positions != nullptr ? p.positions[row0 + i] : pos;
        }
    }
    __syncthreads();
    const int half = p.rot_dim / 2;
    for (int i = t; i < nrows * half; i += kAppendThreads) {
        const int r = i / half, f = i % half;
        if (s_seq[r] < 0) continue;
        constexpr double kPerTurn = 0.15915494309189535;  // 1 / (2 pi)
        double turns = static_cast<double>(s_pos[r]) * static_cast<double>(p.inv_freq[f]) * kPerTurn;
        turns -= rint(turns);
        float sn, cs;
        sincospif(static_cast<float>(2.0 * turns), &sn, &cs);
        s_cos[r][f] = cs;
        s_sin[r][f] = sn;
    }
    __syncthreads();

    constexpr int kItems = D / 16;
    const int kvh = p.cache.heads;
    const int per_row = (p.q_heads + 2 * kvh) * kItems;
    for (int i = t; i < nrows * per_row; i += kAppendThreads) {
        const int r = i / per_row, rest = i % per_row;
        if (s_seq[r] < 0) continue;
        int h = rest / kItems;
        const int it = rest % kItems;
        const int64_t row = row0 + r;
        const char* src;
        char* dst;
        bool turn = it < p.rot_dim / 16;
        if (h < p.q_heads) {
            src = p.q.data + row * p.q.row_stride + h * p.q.head_stride;
            dst = p.q_out.data + row * p.q_out.row_stride + h * p.q_out.head_stride;
        } else {
            h -= p.q_heads;
            const bool is_v = h >= kvh;
            if (is_v) h -= kvh;
            const KvRowsView& x = is_v ? p.v : p.k;
            if (s_block[r] < 0) continue;
            src = x.data + row * x.row_stride + h * x.head_stride;
            dst = const_cast<char*>(is_v ? p.cache.v : p.cache.k) + s_block[r] * p.cache.block_stride +
                  s_place[r] * p.cache.token_stride + h * p.cache.head_stride;
            turn = turn && !is_v;
        }
        if (!turn) {
            const int e = it * 16;
            // the pairs of the split form lie rot_dim / 2 apart; what is copied is contiguous
            const uint4 x0 = *reinterpret_cast<const uint4*>(src + 2 * e), x1 = *reinterpret_cast<const uint4*>(src + 2 * e + 16);
            *reinterpret_cast<uint4*>(dst + 2 * e) = x0;
            *reinterpret_cast<uint4*>(dst + 2 * e + 16) = x1;
            continue;
        }
        const int e0 = p.interleaved ? it * 16 : it * 8;
        const int e1 = p.interleaved ? e0 + 8 : e0 + half;
        float a[8], c[8];
        Pack<T>::load(src + 2 * e0, a);
        Pack<T>::load(src + 2 * e1, c);
        const float* cs = &s_cos[r][it * 8];
        const float* sn = &s_sin[r][it * 8];
        if (p.interleaved) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float x = a[2 * j], y = a[2 * j + 1];
                a[2 * j] = x * cs[j] - y * sn[j];
                a[2 * j + 1] = x * sn[j] + y * cs[j];
                const float u = c[2 * j], w = c[2 * j + 1];
                c[2 * j] = u * cs[4 + j] - w * sn[4 + j];
                c[2 * j + 1] = u * sn[4 + j] + w * cs[4 + j];
            }
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float x = a[j], y = c[j];
                a[j] = x * cs[j] - y * sn[j];
                c[j] = x * sn[j] + y * cs[j];
            }
        }
        Pack<T>::store(dst + 2 * e0, a);
        Pack<T>::store(dst + 2 * e1, c);
    }
}

// ---------------------------------------------------------------------------
// Merge: one group of D / 8 threads per (row, head), 8 elements a thread
// ---------------------------------------------------------------------------
constexpr int kMergeThreads = 256;

template <typename T, typename O, int D>
__global__ void __launch_bounds__(kMergeThreads) kv_merge_kernel(const KvMergeParams p) {
    constexpr int kLanes = D / 8;
    kv_wait_last();
    const int64_t n = static_cast<int64_t>(p.rows) * p.heads;
    const int lane = threadIdx.x % kLanes;
    const int64_t step = static_cast<int64_t>(gridDim.x) * (kMergeThreads / kLanes);
    for (int64_t u = blockIdx.x * static_cast<int64_t>(kMergeThreads / kLanes) + threadIdx.x / kLanes; u < n; u += step) {
        const int64_t row = u / p.heads, h = u % p.heads;
        if (p.last_marks && __float_as_uint(p.part_lse[(p.part_count - 1) * n + u]) == kKvUnwritten) continue;
        float m = -INFINITY;
        for (int i = 0; i < p.part_count; ++i) m = fmaxf(m, p.part_lse[i * n + u]);
        const float base = m == -INFINITY ? 0.0f : m;
        float acc[8] = {}, total = 0.0f;
        const char* src = p.parts.data + row * p.parts.row_stride + h * p.parts.head_stride + lane * 8 * sizeof(T);
        for (int i = 0; i < p.part_count; ++i) {
            const float l = p.part_lse[i * n + u];
            if (l == -INFINITY) continue;
            const float w = expf(l - base);
            total += w;
            float f[8];
            Pack<T>::load(src + i * p.part_stride, f);
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] = fmaf(w, f[e], acc[e]);
        }
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] = total == 0.0f ? 0.0f : acc[e] * inv;
        Pack<O>::store(p.out.data + row * p.out.row_stride + h * p.out.head_stride + lane * 8 * sizeof(O), acc);
        if (lane == 0 && p.lse != nullptr) p.lse[u] = total == 0.0f ? -INFINITY : base + logf(total);
    }
}

// ---------------------------------------------------------------------------
// Join of an attention launch's partial results.
//
// Every CTA reads the launch's places, lists the units that a cut divides and takes its share of
// their rows, a warp per row: lane i first weighs part i (32 at a time), then every lane sums D / 32
// elements over the parts, in their order.  Three rounds of loads, each of them wide.
// ---------------------------------------------------------------------------
constexpr int kJoinThreads = 256;
constexpr int kJoinCtas = 512;  // most CTAs of the launch to join

template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) kv_join_kernel(const KvAttendParams p, int ctas, int slot_rows) {
    __shared__ int32_t s_cut[kJoinCtas], s_row[kJoinCtas + 1];
    __shared__ int32_t s_count[kJoinThreads / 32][2];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5;
    constexpr int kEach = D / 32;
    kv_let_next();
    kv_wait_last();
    const KvCuts cuts(p.line.places[0].total, ctas);
    // cuts that are the first inside their unit: the list of units, and where their rows begin
    int units = 0, rows = 0;
    for (int c0 = 1; c0 < cuts.n(); c0 += kJoinThreads) {
        const int c = c0 + t;
        int mine = 0;
        if (c < cuts.n()) {
            const KvPlace& u = p.line.places[c];
            if (u.t > 0 && cuts.at(c - 1) <= u.begin) mine = u.packed;
        }
        const unsigned ball = __ballot_sync(0xffffffffu, mine > 0);
        int incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += y;
        }
        if (lane == 31) {
            s_count[warp][0] = __popc(ball);
            s_count[warp][1] = incl;
        }
        __syncthreads();
        int k = units + __popc(ball & ((1u << lane) - 1u)), r = rows + incl - mine;
        for (int w = 0; w < kJoinThreads / 32; ++w) {
            if (w < warp) {
                k += s_count[w][0];
                r += s_count[w][1];
            }
            units += s_count[w][0];
            rows += s_count[w][1];
        }
        if (mine > 0) {
            s_cut[k] = c;
            s_row[k] = r;
        }
        __syncthreads();
    }
    const int64_t size = static_cast<int64_t>(slot_rows) * (D + 2);
    for (int i = blockIdx.x * (kJoinThreads / 32) + warp; i < rows; i += gridDim.x * (kJoinThreads / 32)) {
        int lo = 0, hi = units - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) / 2;
            if (s_row[mid] <= i) lo = mid;
            else hi = mid - 1;
        }
        const int c = s_cut[lo], r = i - s_row[lo];
        const KvPlace& u = p.line.places[c];
        const int64_t end = u.begin + u.count;
        const int32_t packed = u.packed0 + r, h = u.h, row0 = u.row0;
        // part 0 is CTA c - 1 (slot 1), part x >= 1 CTA c - 1 + x (slot 0), to the last cut inside the unit
        const float* base = p.line.slots + (2 * static_cast<int64_t>(c - 1)) * size;
        float m = -INFINITY, l = 0.0f, sum[kEach] = {};
        for (int x0 = 0;; x0 += 32) {
            const int x = x0 + lane;
            const bool live = x == 0 || (c - 1 + x < cuts.n() && cuts.at(c - 1 + x) < end);
            const float* slot = base + (x == 0 ? size : 2 * x * size);
            float pm = -INFINITY, pl = 0.0f;
            if (live) {
                pm = slot[slot_rows * D + r];
                pl = slot[slot_rows * D + slot_rows + r];
            }
            float top = pm;
#pragma unroll
            for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            top = fmaxf(top, m);
            const float keep = m == -INFINITY ? 0.0f : fast_exp2(m - top);
            const float w = pm == -INFINITY ? 0.0f : fast_exp2(pm - top);
            float part = pm == -INFINITY ? pl : pl * w;  // -inf: 0, or NaN from scores that are NaN
#pragma unroll
            for (int o = 16; o; o >>= 1) part += __shfl_xor_sync(0xffffffffu, part, o);
            l = (m == -INFINITY ? l : l * keep) + part;
            m = top;
#pragma unroll
            for (int e = 0; e < kEach; ++e) sum[e] *= keep;
            const int n = __popc(__ballot_sync(0xffffffffu, live));
#pragma unroll 8
            for (int y = 0; y < n; ++y) {
                const float wy = __shfl_sync(0xffffffffu, w, y);
                const float* v = base + (x0 + y == 0 ? size : 2 * (x0 + y) * size) + r * D + lane * kEach;
                float f[kEach];
                if constexpr (kEach == 4) *reinterpret_cast<float4*>(f) = *reinterpret_cast<const float4*>(v);
                else *reinterpret_cast<float2*>(f) = *reinterpret_cast<const float2*>(v);
                if (wy != 0.0f)
#pragma unroll
                    for (int e = 0; e < kEach; ++e) sum[e] = fmaf(f[e], wy, sum[e]);
            }
            if (n < 32) break;
        }
        const int32_t of = kv_div_group(p, packed);
        const int64_t row = row0 + of;
        const int head = h * p.group + packed - of * p.group;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
        char* at = p.out.data + row * p.out.row_stride + head * p.out.head_stride;
#pragma unroll
        for (int e = 0; e < kEach; ++e) sum[e] = l == 0.0f ? 0.0f : sum[e] * inv;
        if (p.out_f32) {
            if constexpr (kEach == 4) reinterpret_cast<float4*>(at)[lane] = *reinterpret_cast<const float4*>(sum);
            else reinterpret_cast<float2*>(at)[lane] = *reinterpret_cast<const float2*>(sum);
        } else {
            if constexpr (kEach == 4) reinterpret_cast<uint2*>(at)[lane] = make_uint2(Pack<T>::pair(sum[0], sum[1]), Pack<T>::pair(sum[2], sum[3]));
            else reinterpret_cast<uint32_t*>(at)[lane] = Pack<T>::pair(sum[0], sum[1]);
        }
        if (p.lse != nullptr && lane == 0) p.lse[row * p.q_heads + head] = l == 0.0f ? -INFINITY : m * kLn2 + logf(l);
    }
}

template <typename F>
cudaError_t by_type(int dtype, F f) {  // the types of a cache
    return dtype == GFD_BF16 ? f(__nv_bfloat16()) : f(__half());
}
template <typename F>
cudaError_t by_any_type(int dtype, F f) {
    return dtype == GFD_FP32 ? f(0.0f) : by_type(dtype, f);
}

}  // namespace

cudaError_t launch_kv_append(const KvAppendParams& p, int head_dim, int dtype, int num_sms, cudaStream_t st) {
    const int rows_per_cta = p.batch.rows > 8 * num_sms ? 4 : 1;
    const dim3 grid((p.batch.rows + rows_per_cta - 1) / rows_per_cta);
    return by_type(dtype, [&](auto t) {
        using T = decltype(t);
        return head_dim == 64 ? kv_launch(kv_append_kernel<T, 64>, grid, kAppendThreads, 0, st, false, p, rows_per_cta)
                              : kv_launch(kv_append_kernel<T, 128>, grid, kAppendThreads, 0, st, false, p, rows_per_cta);
    });
}

cudaError_t launch_kv_join(const KvAttendParams& p, int head_dim, int dtype, int ctas, int slot_rows, cudaStream_t st) {
    if (ctas > kJoinCtas) return cudaErrorInvalidValue;
    // at most ctas - 1 units are cut; a warp per row
    const int64_t rows = static_cast<int64_t>(ctas - 1) * slot_rows, warps = kJoinThreads / 32;
    const int64_t all = static_cast<int64_t>(p.batch.rows) * p.q_heads;
    const int64_t want = ((rows < all ? rows : all) + warps - 1) / warps;
    const dim3 grid(static_cast<unsigned>(want < 1 ? 1 : (want > 4 * ctas ? 4 * ctas : want)));
    return by_type(dtype, [&](auto t) {
        using T = decltype(t);
        return head_dim == 64 ? kv_launch(kv_join_kernel<T, 64>, grid, kJoinThreads, 0, st, true, p, ctas, slot_rows)
                              : kv_launch(kv_join_kernel<T, 128>, grid, kJoinThreads, 0, st, true, p, ctas, slot_rows);
    });
}

cudaError_t launch_kv_merge(const KvMergeParams& p, int head_dim, int part_dtype, int out_dtype, int num_sms, bool chained,
                            cudaStream_t st) {
    const int64_t per_cta = kMergeThreads / (head_dim / 8);
    const int64_t want = (static_cast<int64_t>(p.rows) * p.heads + per_cta - 1) / per_cta;
    const dim3 grid(static_cast<unsigned>(want > 16ll * num_sms ? 16ll * num_sms : want));
    return by_any_type(part_dtype, [&](auto t) {
        return by_any_type(out_dtype, [&](auto o) {
            using T = decltype(t);
            using O = decltype(o);
            return head_dim == 64 ? kv_launch(kv_merge_kernel<T, O, 64>, grid, kMergeThreads, 0, st, chained, p)
                                  : kv_launch(kv_merge_kernel<T, O, 128>, grid, kMergeThreads, 0, st, chained, p);
        });
    });
}

}  // namespace gfdb
