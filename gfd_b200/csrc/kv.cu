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
// neighbours when interleaved), the items above copy.  A thread keeps its item for all heads, so the
// sines and cosines of its 8 angles stay in registers while it walks the heads of a row, 2 of them
// in flight at a time.  Memory bounds the kernel: 8.5 thousand rows of 32 + 8 + 8 heads of 128 take 53 us,
// 4.9 TB/s (4 heads in flight and 8 rows a CTA: 76 us; 3 or 5 CTAs an SM: 60, 89).  A CTA takes
// kMaxRows rows (one where there are few) and forms their places and angles once.  Angles: p * inv_freq is
// exact in 64 bits up to p = 2^29, and a turn is taken off in 64 bits before the 32-bit sine, so a
// position of a million is as accurate as a small one.
constexpr int kAppendThreads = 256;
constexpr int kMaxRows = 4;

template <typename T, int D>
__global__ void __launch_bounds__(kAppendThreads, 4) kv_append_kernel(const KvAppendParams p, int rows_per_cta) {
    __shared__ float s_cos[kMaxRows][D / 2], s_sin[kMaxRows][D / 2];
    __shared__ int32_t s_seq[kMaxRows], s_block[kMaxRows], s_place[kMaxRows], s_pos[kMaxRows];
    const KvBatchView& b = p.batch;
    const int t = threadIdx.x;
    const int32_t row0 = blockIdx.x * rows_per_cta;
    const int nrows = min(rows_per_cta, b.rows - row0);
    if (t < kMaxRows) s_seq[t] = -1;
    bool bad = false;
    for (int s = t; s < b.seqs; s += kAppendThreads) {
        const int32_t a = b.row_start[s], e = b.row_start[s + 1];
        bad |= a < 0 || a > e || e > b.rows;
    }
    if (__syncthreads_or(bad) != 0) {
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
            s_seq[i] = s;
            s_place[i] = pos;
            s_pos[i] = p.positions != nullptr ? p.positions[row0 + i] : pos;
        }
    }
    __syncthreads();
    const int half = p.rot_dim / 2;
    // the places, by the last warp, while the others form the angles
    if (t >= kAppendThreads - 32) {
        const int r = t - (kAppendThreads - 32);
        if (r < nrows && s_seq[r] >= 0) {
            const int32_t token = s_place[r], bt = p.cache.block_tokens, block = b.table[s_seq[r] * b.table_stride + token / bt];
            s_place[r] = token % bt;
            s_block[r] = block >= 0 && block < p.cache.blocks ? block : -1;
            if (s_block[r] < 0) kv_report(p.status, GFD_KV_BAD_PAGE);
        }
    } else {
        for (int i = t; i < nrows * half; i += kAppendThreads - 32) {
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
    }
    __syncthreads();

    constexpr int kItems = D / 16, kHeads = kAppendThreads / kItems, kAhead = 2;  // heads of a step, steps in flight
    const int it = t % kItems, kvh = p.cache.heads, heads = p.q_heads + 2 * kvh;
    const bool turns = it < p.rot_dim / 16;
    const int e0 = turns && !p.interleaved ? it * 8 : it * 16, e1 = turns && !p.interleaved ? e0 + half : e0 + 8;
    for (int r = 0; r < nrows; ++r) {
        if (s_seq[r] < 0) continue;
        const int64_t row = row0 + r;
        float cs[8], sn[8];
        if (turns) {
            Pack<float>::load(reinterpret_cast<const char*>(&s_cos[r][it * 8]), cs);
            Pack<float>::load(reinterpret_cast<const char*>(&s_sin[r][it * 8]), sn);
        }
        const int64_t cell = s_block[r] >= 0 ? s_block[r] * p.cache.block_stride + s_place[r] * p.cache.token_stride : -1;
        for (int h0 = t / kItems; h0 < heads; h0 += kHeads * kAhead) {
            uint4 a[kAhead], c[kAhead];
            char* dst[kAhead];
#pragma unroll
            for (int y = 0; y < kAhead; ++y) {
                const int h = h0 + y * kHeads;
                const char* src = nullptr;
                dst[y] = nullptr;
                if (h < p.q_heads) {
                    src = p.q.data + row * p.q.row_stride + h * p.q.head_stride;
                    dst[y] = p.q_out.data + row * p.q_out.row_stride + h * p.q_out.head_stride;
                } else if (h < heads && cell >= 0) {
                    const bool is_v = h >= p.q_heads + kvh;
                    const int k = h - p.q_heads - (is_v ? kvh : 0);
                    src = is_v ? p.v.data + row * p.v.row_stride + k * p.v.head_stride : p.k.data + row * p.k.row_stride + k * p.k.head_stride;
                    dst[y] = const_cast<char*>(is_v ? p.cache.v : p.cache.k) + cell + k * p.cache.head_stride;
                }
                if (src == nullptr) continue;
                // V is copied: the same pieces as the rotation's, wherever they lie
                a[y] = *reinterpret_cast<const uint4*>(src + 2 * e0);
                c[y] = *reinterpret_cast<const uint4*>(src + 2 * e1);
            }
#pragma unroll
            for (int y = 0; y < kAhead; ++y) {
                if (dst[y] == nullptr) continue;
                if (!turns || h0 + y * kHeads >= p.q_heads + kvh) {
                    *reinterpret_cast<uint4*>(dst[y] + 2 * e0) = a[y];
                    *reinterpret_cast<uint4*>(dst[y] + 2 * e1) = c[y];
                    continue;
                }
                float u[8], w[8];
                Pack<T>::load(reinterpret_cast<const char*>(&a[y]), u);
                Pack<T>::load(reinterpret_cast<const char*>(&c[y]), w);
                if (p.interleaved) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float x0 = u[2 * j], y0 = u[2 * j + 1], x1 = w[2 * j], y1 = w[2 * j + 1];
                        u[2 * j] = x0 * cs[j] - y0 * sn[j];
                        u[2 * j + 1] = x0 * sn[j] + y0 * cs[j];
                        w[2 * j] = x1 * cs[4 + j] - y1 * sn[4 + j];
                        w[2 * j + 1] = x1 * sn[4 + j] + y1 * cs[4 + j];
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const float x0 = u[j], y0 = w[j];
                        u[j] = x0 * cs[j] - y0 * sn[j];
                        w[j] = x0 * sn[j] + y0 * cs[j];
                    }
                }
                Pack<T>::store(dst[y] + 2 * e0, u);
                Pack<T>::store(dst[y] + 2 * e1, w);
            }
        }
    }
}

// ---------------------------------------------------------------------------
// Merge: one group of D / 8 threads per (row, head), 8 elements a thread, 4 parts in flight at a time.
// out = sum w_i out_i / sum w_i, w_i = e^(lse_i - m), m the greatest lse.  Memory bounds it: 4 fp32 parts of 8191
// rows of 32 heads of 128 take 93 us, 6.5 TB/s (2 parts in flight: 113); 4 bf16 parts 126 us, 2.7 TB/s.
// ---------------------------------------------------------------------------
constexpr int kMergeThreads = 256;

template <typename T, typename O, int D>
__global__ void __launch_bounds__(kMergeThreads) kv_merge_kernel(const KvMergeParams p) {
    constexpr int kLanes = D / 8, kBatch = 4;
    const int64_t n = static_cast<int64_t>(p.rows) * p.heads;
    const int lane = threadIdx.x % kLanes;
    const int64_t step = static_cast<int64_t>(gridDim.x) * (kMergeThreads / kLanes);
    for (int64_t u = blockIdx.x * static_cast<int64_t>(kMergeThreads / kLanes) + threadIdx.x / kLanes; u < n; u += step) {
        const int64_t row = kv_div(u, p.heads), h = u - row * p.heads;
        float m = -INFINITY, total = 0.0f, acc[8] = {};
        const char* src = p.parts.data + row * p.parts.row_stride + h * p.parts.head_stride + lane * 8 * sizeof(T);
        for (int i0 = 0; i0 < p.part_count; i0 += kBatch) {
            float l[kBatch], f[kBatch][8];
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                l[i] = -INFINITY;
                if (i0 + i >= p.part_count) continue;
                l[i] = p.part_lse[(i0 + i) * n + u];
                Pack<T>::load(src + (i0 + i) * p.part_stride, f[i]);
            }
            float top = m;
#pragma unroll
            for (int i = 0; i < kBatch; ++i) top = fmaxf(top, l[i]);
            const float keep = m == -INFINITY ? 0.0f : expf(m - top);
            m = top;
            total *= keep;
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] *= keep;
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                if (l[i] == -INFINITY) continue;  // whatever its output holds
                const float w = expf(l[i] - top);
                total += w;
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[e] = fmaf(w, f[i][e], acc[e]);
            }
        }
        const float inv = total == 0.0f ? 0.0f : 1.0f / total;
#pragma unroll
        for (int e = 0; e < 8; ++e) acc[e] *= inv;
        Pack<O>::store(p.out.data + row * p.out.row_stride + h * p.out.head_stride + lane * 8 * sizeof(O), acc);
        if (lane == 0 && p.lse != nullptr) p.lse[u] = total == 0.0f ? -INFINITY : m + logf(total);
    }
}

// ---------------------------------------------------------------------------
// Join of an attention launch's partial results.
// ---------------------------------------------------------------------------
constexpr int kJoinThreads = 256;
constexpr int kJoinWarps = kJoinThreads / 32;
// Weight of a part whose sums are relative to 2^base, and its share of the weight sum: a part without
// keys (-inf) adds nothing but a NaN that its scores left.
__device__ __forceinline__ void part_weight(float base, float top, float* w, float* l) {
    *w = base == -INFINITY ? 0.0f : fast_exp2(base - top);
    if (base != -INFINITY) *l *= *w;
}

// Of kv_decode, with up to hundreds of parts of a few rows: a CTA per cut takes 4 rows at a time and 128 parts:
// its threads weigh them, then each warp sums every 8th part (D / 32 elements a lane), and the warps'
// sums are added in their order.
template <typename T, int D>
__global__ void __launch_bounds__(kJoinThreads) kv_join_few_kernel(const KvAttendParams p) {
    constexpr int kEach = D / 32, kSlot = kKvFewRows * (D + 2), kParts = 128;
    __shared__ float s_w[kParts][4];
    __shared__ float s_top[kJoinWarps][2], s_sum[kJoinWarps][2];
    __shared__ float s_acc[kJoinWarps][4][D];
    const int t = threadIdx.x, lane = t & 31, warp = t >> 5, c = blockIdx.x + 1;
    kv_let_next();
    kv_wait_last();
    const KvCut u = p.line.cuts[c];
    if (u.parts == 0) return;
    const float* slots = p.line.slots + 2 * static_cast<int64_t>(c - 1) * kSlot;  // part x: slot 1 for 0, else 2 x
    for (int r0 = 0; r0 < u.packed; r0 += 4) {
        const int nr = min(4, u.packed - r0);
        float m[4], l[4], acc[4][kEach];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            m[r] = -INFINITY;
            l[r] = 0.0f;
#pragma unroll
            for (int e = 0; e < kEach; ++e) acc[r][e] = 0.0f;
        }
        for (int x0 = 0; x0 < u.parts; x0 += kParts) {
            const int n = min(kParts, u.parts - x0);
            // thread t: part t % 128, rows 2 (t / 128) and the next
            const int x = x0 + t % kParts, pair = t / kParts * 2;
            float pm[2] = {-INFINITY, -INFINITY}, pl[2] = {0.0f, 0.0f};
            const float* slot = slots + static_cast<int64_t>(x == 0 ? 1 : 2 * x) * kSlot + kKvFewRows * D + r0 + pair;
#pragma unroll
            for (int y = 0; y < 2; ++y)
                if (t % kParts < n && pair + y < nr) {
                    pm[y] = slot[y];
                    pl[y] = slot[kKvFewRows + y];
                }
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                float top = pm[y];
#pragma unroll
                for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                if (lane == 0) s_top[warp][y] = top;
            }
            __syncthreads();
            float top[4];
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                top[r] = m[r];
#pragma unroll
                for (int w = 0; w < 4; ++w) top[r] = fmaxf(top[r], s_top[r / 2 * 4 + w][r & 1]);
            }
#pragma unroll
            for (int y = 0; y < 2; ++y) {
                float w;
                part_weight(pm[y], pair == 0 ? top[y] : top[2 + y], &w, &pl[y]);
                s_w[t % kParts][pair + y] = w;
#pragma unroll
                for (int o = 16; o; o >>= 1) pl[y] += __shfl_xor_sync(0xffffffffu, pl[y], o);
                if (lane == 0) s_sum[warp][y] = pl[y];
            }
            __syncthreads();
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float keep;
                part_weight(m[r], top[r], &keep, &l[r]);
                m[r] = top[r];
#pragma unroll
                for (int w = 0; w < 4; ++w) l[r] += s_sum[r / 2 * 4 + w][r & 1];
#pragma unroll
                for (int e = 0; e < kEach; ++e) acc[r][e] *= keep;
            }
#pragma unroll 2
            for (int y = warp; y < n; y += kJoinWarps) {
                const float* v = slots + static_cast<int64_t>(x0 + y == 0 ? 1 : 2 * (x0 + y)) * kSlot + r0 * D + lane * kEach;
                float f[4][kEach];
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (r < nr) {
                        if constexpr (kEach == 4) *reinterpret_cast<float4*>(f[r]) = *reinterpret_cast<const float4*>(v + r * D);
                        else *reinterpret_cast<float2*>(f[r]) = *reinterpret_cast<const float2*>(v + r * D);
                    }
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float w = s_w[y][r];
                    if (r < nr && w != 0.0f)
#pragma unroll
                        for (int e = 0; e < kEach; ++e) acc[r][e] = fmaf(f[r][e], w, acc[r][e]);
                }
            }
            __syncthreads();
        }
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int e = 0; e < kEach; ++e) s_acc[warp][r][lane * kEach + e] = acc[r][e];
        __syncthreads();
        for (int i = t; i < nr * (D / 2); i += kJoinThreads) {
            const int r = i / (D / 2), d = i % (D / 2) * 2;
            float a = 0.0f, b = 0.0f;
#pragma unroll
            for (int w = 0; w < kJoinWarps; ++w) {
                a += s_acc[w][r][d];
                b += s_acc[w][r][d + 1];
            }
            const float mr = r < 2 ? (r == 0 ? m[0] : m[1]) : (r == 2 ? m[2] : m[3]);
            const float lr = r < 2 ? (r == 0 ? l[0] : l[1]) : (r == 2 ? l[2] : l[3]);
            const float inv = lr == 0.0f ? 0.0f : 1.0f / lr;
            const int32_t of = kv_div_group(p, r0 + r);
            const int64_t row = u.row0 + of;
            const int head = u.h * p.group + r0 + r - of * p.group;
            char* at = p.out.data + row * p.out.row_stride + head * p.out.head_stride;
            if (p.out_f32) *reinterpret_cast<float2*>(at + 4 * d) = make_float2(a * inv, b * inv);
            else *reinterpret_cast<uint32_t*>(at + 2 * d) = Pack<T>::pair(a * inv, b * inv);
            if (p.lse != nullptr && d == 0) p.lse[row * p.q_heads + head] = kv_lse(p, mr, lr);
        }
        __syncthreads();
    }
}

// Of kv_prompt, with many rows: a CTA takes 32 rows of a cut, a lane one of them and a warp D / 8
// elements, so that the parts are read as they were written, 4 at a time; the results go through shared
// memory to be written row by row.
template <typename T, int D, bool kShared>
__global__ void __launch_bounds__(kJoinThreads) kv_join_many_kernel(const KvAttendParams p) {
    constexpr int kEach = D / 8, kBatch = 4;  // elements of a thread, parts side by side
    constexpr int64_t kSlot = static_cast<int64_t>(kKvManyRows) * (D + 2);
    __shared__ float s_out[32][D + 4];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = blockIdx.x + 1;
    kv_let_next();
    kv_wait_last();
    const KvCut u = p.line.cuts[c];
    const int r0 = blockIdx.y * 32;
    if (u.parts == 0 || r0 >= u.packed) return;
    const float* slots = p.line.slots + 2 * (c - 1) * kSlot;  // part x: slot 1 for 0, else 2 x
    const bool live = r0 + lane < u.packed;
    const int r = live ? r0 + lane : r0;
    const int32_t packed = u.packed0 + r, of = kv_div_group(p, packed);
    const int64_t row = u.row0 + of;
    const int head = u.h * p.group + packed - of * p.group;
    const int64_t place = row * p.q_heads + head;
    const float own_lse = kShared ? p.own_lse[place] : -INFINITY;
    float m = -INFINITY, l = 0.0f, sum[kEach] = {};
    for (int x0 = 0; x0 < u.parts; x0 += kBatch) {
        float pm[kBatch], pl[kBatch], f[kBatch][kEach];
#pragma unroll
        for (int y = 0; y < kBatch; ++y) {
            const int x = x0 + y;
            pm[y] = -INFINITY;
            pl[y] = 0.0f;
            if (x >= u.parts) continue;
            const float* slot = slots + (x == 0 ? 1 : 2 * x) * kSlot;
            pm[y] = slot[kKvManyRows * D + r];
            pl[y] = slot[kKvManyRows * D + kKvManyRows + r];
#pragma unroll
            for (int e = 0; e < kEach; e += 4)
                *reinterpret_cast<float4*>(f[y] + e) =
                    *reinterpret_cast<const float4*>(slot + (static_cast<int64_t>(warp * kEach + e) / 4 * kKvManyRows + r) * 4);
        }
        float top = m, keep;
#pragma unroll
        for (int y = 0; y < kBatch; ++y) top = fmaxf(top, pm[y]);
        part_weight(m, top, &keep, &l);
        m = top;
#pragma unroll
        for (int e = 0; e < kEach; ++e) sum[e] *= keep;
#pragma unroll
        for (int y = 0; y < kBatch; ++y) {
            float w;
            part_weight(pm[y], top, &w, &pl[y]);
            l += pl[y];
            if (w != 0.0f)
#pragma unroll
                for (int e = 0; e < kEach; ++e) sum[e] = fmaf(f[y][e], w, sum[e]);
        }
    }
    const bool valid = live && (!kShared || __float_as_uint(own_lse) != kKvSkipped);
    if (valid) {
        const KvFinish f = kv_finish<kShared>(p, m, l, own_lse);
#pragma unroll
        for (int e = 0; e < kEach; ++e) sum[e] *= f.scale;
        if (kShared && f.own != 0.0f)
#pragma unroll
            for (int e = 0; e < kEach; e += 4) {
                const float4 y = *reinterpret_cast<const float4*>(p.own_out + place * D + warp * kEach + e);
                sum[e] = fmaf(y.x, f.own, sum[e]);
                sum[e + 1] = fmaf(y.y, f.own, sum[e + 1]);
                sum[e + 2] = fmaf(y.z, f.own, sum[e + 2]);
                sum[e + 3] = fmaf(y.w, f.own, sum[e + 3]);
            }
        if (p.lse != nullptr && warp == 0) p.lse[place] = kv_lse(p, f.base, f.sum);
#pragma unroll
        for (int e = 0; e < kEach; e += 4) *reinterpret_cast<float4*>(&s_out[lane][warp * kEach + e]) = *reinterpret_cast<const float4*>(sum + e);
    }
    const unsigned ok = __ballot_sync(0xffffffffu, valid);  // the same rows in every warp
    __syncthreads();
    constexpr int kLanes = D / 8;
    for (int i = threadIdx.x / kLanes; i < 32; i += kJoinThreads / kLanes) {
        if (!((ok >> i) & 1u)) continue;
        const int32_t pk = u.packed0 + r0 + i, o = kv_div_group(p, pk);
        char* at = p.out.data + static_cast<int64_t>(u.row0 + o) * p.out.row_stride + (u.h * p.group + pk - o * p.group) * p.out.head_stride;
        const int d = threadIdx.x % kLanes * 8;
        float f[8];
        *reinterpret_cast<float4*>(f) = *reinterpret_cast<const float4*>(&s_out[i][d]);
        *reinterpret_cast<float4*>(f + 4) = *reinterpret_cast<const float4*>(&s_out[i][d + 4]);
        if (p.out_f32) Pack<float>::store(at + 4 * d, f);
        else Pack<T>::store(at + 2 * d, f);
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
    const int rows_per_cta = p.batch.rows > 4 * num_sms ? kMaxRows : 1;
    const dim3 grid((p.batch.rows + rows_per_cta - 1) / rows_per_cta);
    return by_type(dtype, [&](auto t) {
        using T = decltype(t);
        return head_dim == 64 ? kv_launch(kv_append_kernel<T, 64>, grid, kAppendThreads, 0, st, false, p, rows_per_cta)
                              : kv_launch(kv_append_kernel<T, 128>, grid, kAppendThreads, 0, st, false, p, rows_per_cta);
    });
}

cudaError_t launch_kv_join_few(const KvAttendParams& p, int head_dim, int dtype, int stretches, cudaStream_t st) {
    return by_type(dtype, [&](auto t) {
        using T = decltype(t);
        return kv_launch(head_dim == 64 ? kv_join_few_kernel<T, 64> : kv_join_few_kernel<T, 128>, dim3(stretches - 1), kJoinThreads, 0, st, true, p);
    });
}

cudaError_t launch_kv_join_many(const KvAttendParams& p, int head_dim, int dtype, int stretches, cudaStream_t st) {
    return by_type(dtype, [&](auto t) {
        using T = decltype(t);
        auto* f = p.shared_pass ? (head_dim == 64 ? kv_join_many_kernel<T, 64, true> : kv_join_many_kernel<T, 128, true>)
                                : (head_dim == 64 ? kv_join_many_kernel<T, 64, false> : kv_join_many_kernel<T, 128, false>);
        return kv_launch(f, dim3(stretches - 1, kKvManyRows / 32), kJoinThreads, 0, st, true, p);
    });
}

cudaError_t launch_kv_merge(const KvMergeParams& p, int head_dim, int part_dtype, int out_dtype, int num_sms, cudaStream_t st) {
    const int64_t per_cta = kMergeThreads / (head_dim / 8);
    const int64_t want = (static_cast<int64_t>(p.rows) * p.heads + per_cta - 1) / per_cta;
    const dim3 grid(static_cast<unsigned>(want > 16ll * num_sms ? 16ll * num_sms : want));
    return by_any_type(part_dtype, [&](auto t) {
        return by_any_type(out_dtype, [&](auto o) {
            using T = decltype(t);
            using O = decltype(o);
            return head_dim == 64 ? kv_launch(kv_merge_kernel<T, O, 64>, grid, kMergeThreads, 0, st, false, p)
                                  : kv_launch(kv_merge_kernel<T, O, 128>, grid, kMergeThreads, 0, st, false, p);
        });
    });
}

}  // namespace gfdb
