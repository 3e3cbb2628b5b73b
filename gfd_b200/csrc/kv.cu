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
// Join of an attention launch's partial results: one CTA (times gridDim.y) per
// cut of the line.  Each
// thread sums 4 elements of a packed row over the unit's parts, in their order.
// ---------------------------------------------------------------------------
constexpr int kJoinThreads = 128;

template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) kv_join_kernel(const KvAttendParams p, int slot_rows) {
    const uint32_t c = blockIdx.x + 1;  // cuts 1 .. CTAs - 1
    // every CTA waits for the attention kernel, so that this grid never ends before it
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const KvPlace u = p.line.places[c];
    const KvCuts cuts(u.total, gridDim.x + 1);
    // a cut between two units joins nothing; of several inside a unit the first does
    if (c >= cuts.ctas || u.t == 0 || cuts.at(c - 1) > u.begin) return;
    const int64_t end = u.begin + u.count;
    uint32_t last = c;  // parts: CTA c - 1 (slot 1), c .. last (slot 0)
    while (last + 1 < cuts.ctas && cuts.at(last + 1) < end) ++last;
    const int64_t size = static_cast<int64_t>(slot_rows) * (D + 2);
    const float* slot1 = p.line.slots + (2 * static_cast<int64_t>(c - 1) + 1) * size;
    const float* slot0 = p.line.slots + 2 * static_cast<int64_t>(c) * size;
    const int parts = static_cast<int>(last - c) + 2;
    for (int i = blockIdx.y * kJoinThreads + threadIdx.x; i < u.packed * (D / 4); i += kJoinThreads * gridDim.y) {
        const int r = i / (D / 4), d0 = i % (D / 4) * 4;
        float m = slot1[slot_rows * D + r];
#pragma unroll 4
        for (int x = 1; x < parts; ++x) m = fmaxf(m, slot0[2 * (x - 1) * size + slot_rows * D + r]);
        float sum[4] = {}, l = 0.0f;
#pragma unroll 4
        for (int x = 0; x < parts; ++x) {
            const float* slot = x == 0 ? slot1 : slot0 + 2 * (x - 1) * size;
            const float pm = slot[slot_rows * D + r], pl = slot[slot_rows * D + slot_rows + r];
            const float4 v = *reinterpret_cast<const float4*>(slot + r * D + d0);
            const float w = pm == -INFINITY ? 0.0f : fast_exp2(pm - m);
            l += pm == -INFINITY ? pl : pl * w;  // -inf: 0, or NaN from scores that are NaN
            if (w != 0.0f) {
                sum[0] = fmaf(v.x, w, sum[0]);
                sum[1] = fmaf(v.y, w, sum[1]);
                sum[2] = fmaf(v.z, w, sum[2]);
                sum[3] = fmaf(v.w, w, sum[3]);
            }
        }
        const int packed = u.packed0 + r;
        const int64_t row = u.row0 + packed / p.group;
        const int head = u.h * p.group + packed % p.group;
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int e = 0; e < 4; ++e) sum[e] = l == 0.0f ? 0.0f : sum[e] * inv;
        kv_store_out<T>(p, row, head, d0, sum, 4);
        if (p.lse != nullptr && d0 == 0) p.lse[row * p.q_heads + head] = l == 0.0f ? -INFINITY : m * kLn2 + logf(l);
    }
}

template <typename F>
cudaError_t by_type(int dtype, F f) {
    if (dtype == GFD_BF16) return f(__nv_bfloat16());
    if (dtype == GFD_FP16) return f(__half());
    return f(0.0f);
}

}  // namespace

cudaError_t launch_kv_append(const KvAppendParams& p, int head_dim, int dtype, int num_sms, cudaStream_t st) {
    const int rows_per_cta = p.batch.rows > 8 * num_sms ? 4 : 1;
    const int grid = (p.batch.rows + rows_per_cta - 1) / rows_per_cta;
    if (dtype == GFD_BF16) {
        if (head_dim == 64) kv_append_kernel<__nv_bfloat16, 64><<<grid, kAppendThreads, 0, st>>>(p, rows_per_cta);
        else kv_append_kernel<__nv_bfloat16, 128><<<grid, kAppendThreads, 0, st>>>(p, rows_per_cta);
    } else {
        if (head_dim == 64) kv_append_kernel<__half, 64><<<grid, kAppendThreads, 0, st>>>(p, rows_per_cta);
        else kv_append_kernel<__half, 128><<<grid, kAppendThreads, 0, st>>>(p, rows_per_cta);
    }
    return cudaGetLastError();
}

cudaError_t launch_kv_join(const KvAttendParams& p, int head_dim, int dtype, int ctas, int slot_rows, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(ctas - 1, slot_rows / 16);
    cfg.blockDim = dim3(kJoinThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    if (dtype == GFD_BF16)
        return head_dim == 64 ? cudaLaunchKernelEx(&cfg, kv_join_kernel<__nv_bfloat16, 64>, p, slot_rows)
                              : cudaLaunchKernelEx(&cfg, kv_join_kernel<__nv_bfloat16, 128>, p, slot_rows);
    return head_dim == 64 ? cudaLaunchKernelEx(&cfg, kv_join_kernel<__half, 64>, p, slot_rows)
                          : cudaLaunchKernelEx(&cfg, kv_join_kernel<__half, 128>, p, slot_rows);
}

cudaError_t launch_kv_merge(const KvMergeParams& p, int head_dim, int part_dtype, int out_dtype, int num_sms,
                            cudaStream_t st) {
    const int64_t per_cta = kMergeThreads / (head_dim / 8);
    int64_t grid = (static_cast<int64_t>(p.rows) * p.heads + per_cta - 1) / per_cta;
    if (grid > 16ll * num_sms) grid = 16ll * num_sms;
    return by_type(part_dtype, [&](auto t) {
        return by_type(out_dtype, [&](auto o) {
            using T = decltype(t);
            using O = decltype(o);
            if (head_dim == 64) kv_merge_kernel<T, O, 64><<<static_cast<unsigned>(grid), kMergeThreads, 0, st>>>(p);
            else kv_merge_kernel<T, O, 128><<<static_cast<unsigned>(grid), kMergeThreads, 0, st>>>(p);
            return cudaGetLastError();
        });
    });
}

}  // namespace gfdb
