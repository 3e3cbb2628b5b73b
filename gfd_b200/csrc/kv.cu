// Paged KV-cache operators: append with rotation, merge of partial results, and the
// plain attention kernel (one CTA per row and head).

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
// Attention, plain: one CTA per (row, query head), one thread per key for the scores and
// one per element for the sums; running maximum and sum in 32 bits.
// ---------------------------------------------------------------------------
constexpr int kPlainThreads = 128;

template <typename T, typename O, int D>
__global__ void __launch_bounds__(kPlainThreads) kv_attend_plain_kernel(const KvAttendParams p) {
    __shared__ float s_q[D];
    __shared__ float s_p[kPlainThreads];
    __shared__ const char* s_v[kPlainThreads];
    __shared__ float s_red[4];
    const KvBatchView& b = p.batch;
    const int t = threadIdx.x;
    if (!kv_starts_ok(b)) {
        if (blockIdx.x == 0 && blockIdx.y == 0 && t == 0) kv_report(p.status, GFD_KV_BAD_LENGTH);
        return;
    }
    for (int64_t u = blockIdx.x; u < static_cast<int64_t>(b.seqs) * p.q_heads; u += gridDim.x) {
        const int s = static_cast<int>(u / p.q_heads), h = static_cast<int>(u % p.q_heads);
        const KvSeq q = kv_seq(b.row_start[s], b.row_start[s + 1], b.kv_len[s], b.capacity, p.max_q_len);
        if (!q.ok) {
            if (t == 0) kv_report(p.status, GFD_KV_BAD_LENGTH);
            continue;
        }
        if (p.skip_few && q.rows * p.group <= kKvFewRows) continue;
        const int32_t n = p.shared_len + q.keys;
        const int kvh = h / p.group;
        const float slope = p.alibi != nullptr ? p.alibi[h] : 0.0f;
        for (int i = blockIdx.y; i < q.rows; i += gridDim.y) {
            const int64_t row = q.row0 + i;
            const int32_t pos = n - q.rows + i;
            const KvSpan sp = kv_span(pos, n, p.prefix_len != nullptr ? p.prefix_len[s] : 0, p.window, p.causal != 0);
            __syncthreads();
            if (t < D / 8) {
                float f[8];
                Pack<T>::load(p.q.data + row * p.q.row_stride + h * p.q.head_stride + 16 * t, f);
                for (int e = 0; e < 8; ++e) s_q[8 * t + e] = f[e];
            }
            __syncthreads();
            float m = -INFINITY, l = 0.0f, acc = 0.0f;
            const int32_t seen = sp.pre + (sp.hi - sp.lo);
            for (int32_t j0 = 0; j0 < seen; j0 += kPlainThreads) {
                const int32_t c = j0 + t;
                float z = -INFINITY;
                const char* v = nullptr;
                if (c < seen) {
                    const int32_t j = c < sp.pre ? c : c - sp.pre + sp.lo;
                    int32_t place;
                    const int32_t block = kv_block(b, s, j, p.cache.block_tokens, p.shared_table, p.shared_len, &place);
                    if (block >= 0 && block < p.cache.blocks) {
                        const int64_t at = block * p.cache.block_stride + place * p.cache.token_stride + kvh * p.cache.head_stride;
                        v = p.cache.v + at;
                        float dot = 0.0f;
                        for (int e = 0; e < D; e += 8) {
                            float f[8];
                            Pack<T>::load(p.cache.k + at + 2 * e, f);
                            for (int x = 0; x < 8; ++x) dot = fmaf(f[x], s_q[e + x], dot);
                        }
                        z = dot * p.scale;
                        if (p.softcap > 0.0f) z = p.softcap * tanhf(z / p.softcap);
                        z += slope * static_cast<float>(j - pos);
                    } else {
                        kv_report(p.status, GFD_KV_BAD_PAGE);
                    }
                }
                float mx = z;
                for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
                if ((t & 31) == 0) s_red[t >> 5] = mx;
                __syncthreads();
                mx = fmaxf(fmaxf(s_red[0], s_red[1]), fmaxf(s_red[2], s_red[3]));
                const float mn = fmaxf(m, mx);
                const float keep = mn == -INFINITY ? 1.0f : __expf(m - mn);
                const float e = v == nullptr || z == -INFINITY ? 0.0f : expf(z - mn);
                s_p[t] = e;
                s_v[t] = v;
                float sum = e;
                for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                __syncthreads();
                if ((t & 31) == 0) s_red[t >> 5] = sum;
                __syncthreads();
                l = l * keep + ((s_red[0] + s_red[1]) + (s_red[2] + s_red[3]));
                m = mn;
                if (t < D) {
                    acc *= keep;
                    for (int x = 0; x < kPlainThreads; ++x)
                        if (s_v[x] != nullptr && s_p[x] != 0.0f)
                            acc = fmaf(s_p[x], static_cast<float>(reinterpret_cast<const T*>(s_v[x])[t]), acc);
                }
                __syncthreads();
            }
            const bool none = m == -INFINITY && l == 0.0f;
            if (t < D)
                reinterpret_cast<O*>(p.out.data + row * p.out.row_stride + h * p.out.head_stride)[t] =
                    static_cast<O>(none ? 0.0f : acc / l);
            if (t == 0 && p.lse != nullptr) p.lse[row * p.q_heads + h] = none ? -INFINITY : m + logf(l);
        }
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

template <typename T, typename O>
static cudaError_t attend_plain(const KvAttendParams& p, int head_dim, dim3 grid, cudaStream_t st) {
    if (head_dim == 64) kv_attend_plain_kernel<T, O, 64><<<grid, kPlainThreads, 0, st>>>(p);
    else kv_attend_plain_kernel<T, O, 128><<<grid, kPlainThreads, 0, st>>>(p);
    return cudaGetLastError();
}

cudaError_t launch_kv_attend(const KvAttendParams& p, int head_dim, int dtype, int out_dtype, int num_sms, cudaStream_t st) {
    const int64_t units = static_cast<int64_t>(p.batch.seqs) * p.q_heads;
    const dim3 grid(static_cast<unsigned>(units < 65535 ? units : 65535), p.batch.rows < 64 ? p.batch.rows : 64);
    (void)num_sms;
    if (dtype == GFD_BF16)
        return out_dtype == GFD_FP32 ? attend_plain<__nv_bfloat16, float>(p, head_dim, grid, st)
                                     : attend_plain<__nv_bfloat16, __nv_bfloat16>(p, head_dim, grid, st);
    return out_dtype == GFD_FP32 ? attend_plain<__half, float>(p, head_dim, grid, st)
                                 : attend_plain<__half, __half>(p, head_dim, grid, st);
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
