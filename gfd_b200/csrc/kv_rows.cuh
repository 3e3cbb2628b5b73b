#pragma once
// Sixteen packed rows of a warp against tiles of sixteen keys in shared memory, by warp-wide products
// (mma.m16n8k16 from ldmatrix fragments): what kv_decode does all the time, and kv_prompt for the units whose
// values hold a NaN or an infinity.

#include "kv_device.cuh"

namespace gfdb {

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
__device__ __forceinline__ void ldsm4t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}

template <typename T>
__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Bits 15 and 31: that half of w is NaN or infinite (its exponent is all ones).
template <typename T>
__device__ __forceinline__ uint32_t kv_odd(uint32_t w) {
    constexpr bool kHalf = std::is_same<T, __half>::value;
    return ((w & (kHalf ? 0x7c007c00u : 0x7f807f80u)) + (kHalf ? 0x04000400u : 0x00800080u)) & 0x80008000u;
}
// w with 0 in place of such halves
template <typename T>
__device__ __forceinline__ uint32_t kv_finite(uint32_t w) {
    return w & ~((kv_odd<T>(w) >> 15) * 0xffffu);
}

// fp16 weights reach 2^8, which keeps the small ones clear of that type's coarse steps below 2^-14.
template <typename T>
constexpr float kShift = std::is_same<T, __half>::value ? 8.0f : 0.0f;

// A lane's part of the rows: rows lane / 4 and lane / 4 + 8, and of each sum elements 8 i + 2 (lane % 4) and the
// next.  K and V of a tile: 16 rows of 2 D bytes, 16-byte piece c of row r at place c ^ (r % 8).
template <typename T, int D, bool kPlain>
struct KvRows16 {
    static constexpr int kSteps = D / 16;   // k-steps of the scores, pairs of n-tiles of the sums
    static constexpr int kTile = kKvPage;   // keys of a tile
    static constexpr int kRow = 2 * D;      // bytes of a key
    uint32_t qf[kSteps][4];
    KvSpan sp[2];
    int32_t pos[2];
    float slope[2];                // in base 2
    float m[2], l[2];              // the weights' base (2^m) and sum; l: this lane's share
    float acc[2 * kSteps][4];
    int32_t rows;                  // rows that exist
    bool spent;                    // all their sums are NaN

    __device__ __forceinline__ void begin(int32_t rows_) {
        rows = rows_;
        spent = false;
        m[0] = m[1] = -INFINITY;
        l[0] = l[1] = slope[0] = slope[1] = 0.0f;
#pragma unroll
        for (int i = 0; i < 2 * kSteps; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[i][e] = 0.0f;
    }
    // row x of the lane's two, zeros where it does not exist
    __device__ __forceinline__ void load_q(int x, const char* row, bool exists) {
        const char* src = row + 4 * (threadIdx.x & 3);
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            qf[k][x] = exists ? *reinterpret_cast<const uint32_t*>(src + 32 * k) : 0u;
            qf[k][2 + x] = exists ? *reinterpret_cast<const uint32_t*>(src + 32 * k + 16) : 0u;
        }
    }
    __device__ __forceinline__ bool sees(int x, int32_t key) const { return key < sp[x].pre || (key >= sp[x].lo && key < sp[x].hi); }
    __device__ __forceinline__ bool inside(int x, int32_t j0) const {
        return (j0 >= sp[x].lo && j0 + kTile <= sp[x].hi) || j0 + kTile <= sp[x].pre;
    }
    // some row does not see some key of the tile (the same for all lanes)
    __device__ __forceinline__ bool cut(int32_t j0) const {
        const int r = (threadIdx.x & 31) >> 2;
        return __any_sync(0xffffffffu, (r < rows && !inside(0, j0)) || (r + 8 < rows && !inside(1, j0)));
    }

    // The tile's scores, weights and sums.  dist: what turns key j into a position.  odd: keys (a bit each) whose
    // values at `raw` hold a NaN or an infinity that some rows do not see; at vb, if that is elsewhere, they are 0.
    __device__ __forceinline__ void tile(const KvAttendParams& p, uint32_t kb, uint32_t vb, int32_t j0, int32_t dist, uint32_t odd, uint32_t raw) {
        const int lane = threadIdx.x & 31;
        float z[2][4] = {};
        // piece 2 k + b of row r lies at (2 k + b) ^ (r % 8): k only flips bits of the address
        const int krow = (lane & 7) + ((lane >> 4) << 3), vrow = (lane & 7) + (((lane >> 3) & 1) << 3);
        const uint32_t ka = kb + krow * kRow + ((((lane >> 3) & 1) ^ (krow & 7)) << 4);
        const uint32_t va = vb + vrow * kRow + (((lane >> 4) ^ (vrow & 7)) << 4);
#pragma unroll
        for (int k = 0; k < kSteps; ++k) {
            uint32_t f[4];
            ldsm4(f, ka ^ (k << 5));
            mma<T>(z[0], qf[k], f[0], f[1]);
            mma<T>(z[1], qf[k], f[2], f[3]);
        }
        // z[nt][2 x + e]: row lane / 4 + 8 x, key j0 + 8 nt + 2 (lane % 4) + e.  Up to 8 rows the second half idles.
        float base[2] = {0.0f, 0.0f}, top[2] = {m[0], m[1]};
        bool grew = false;
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            if (8 * x >= rows) break;
            uint32_t y[4];  // y[2 nt + e]
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = __float_as_uint(z[e / 2][2 * x + (e & 1)]);
            const int32_t j = j0 + 2 * (lane & 3);
            const bool masked = __any_sync(0xffffffffu, !inside(x, j0));
            auto seen = [&](int e) { return sees(x, j + 8 * (e / 2) + (e & 1)); };
            if (!kPlain) {
                kv_cap<4>(p, y, masked, [&](int) { return (seen(0) ? 1u : 0u) | (seen(1) ? 2u : 0u) | (seen(2) ? 4u : 0u) | (seen(3) ? 8u : 0u); });
                if (p.alibi != nullptr) {
                    const float d = static_cast<float>(dist + j - pos[x]);
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        y[e] = __float_as_uint(fmaf(slope[x], d + static_cast<float>(8 * (e / 2) + (e & 1)), __uint_as_float(y[e])));
                }
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) y[e] = __float_as_uint(__uint_as_float(y[e]) * p.scale2);
            }
            if (masked) {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (!seen(e)) y[e] = 0xff800000u;
            }
            float mx = fmaxf(__uint_as_float(y[0]), __uint_as_float(y[1]));
#pragma unroll
            for (int e = 2; e < 4; ++e) mx = fmaxf(mx, __uint_as_float(y[e]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2)) - kShift<T>;
            grew |= mx > m[x];
            top[x] = fmaxf(mx, m[x]);
            base[x] = top[x] == -INFINITY ? 0.0f : top[x];
#pragma unroll
            for (int e = 0; e < 4; ++e) z[e / 2][2 * x + (e & 1)] = __uint_as_float(y[e]);
        }
        if (__any_sync(0xffffffffu, grew)) {
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const float keep = fast_exp2(m[x] - base[x]);
                m[x] = top[x];
                l[x] *= keep;
#pragma unroll
                for (int i = 0; i < 2 * kSteps; ++i) {
                    acc[i][2 * x] *= keep;
                    acc[i][2 * x + 1] *= keep;
                }
            }
        }
        // weights: summed in 32 bits, rounded to the cache's type for the product with V
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const bool some = 8 * x < rows;
#pragma unroll
            for (int nt = 0; nt < 2; ++nt)
#pragma unroll
                for (int e = 2 * x; e < 2 * x + 2; ++e) {
                    z[nt][e] = some ? fast_exp2(z[nt][e] - base[x]) : 0.0f;
                    l[x] += z[nt][e];
                }
        }
        if (odd != 0) {
            add_odd(raw, j0, odd);
            if (raw == vb) {
                __syncwarp();
                clear_odd(vb);
                __syncwarp();
            }
        }
        const uint32_t pf[4] = {Pack<T>::pair(z[0][0], z[0][1]), Pack<T>::pair(z[0][2], z[0][3]), Pack<T>::pair(z[1][0], z[1][1]),
                                Pack<T>::pair(z[1][2], z[1][3])};
#pragma unroll
        for (int i = 0; i < kSteps; ++i) {
            uint32_t f[4];
            ldsm4t(f, va ^ (i << 5));
            mma<T>(acc[2 * i], pf, f[0], f[1]);
            mma<T>(acc[2 * i + 1], pf, f[2], f[3]);
        }
    }

    // ---- values that are NaN or infinite, in tiles of which a row does not see every key ----
    // A weight of 0 does not keep them out of a sum, so they are taken out of the product and added to the sums
    // of the rows that see them: beside an infinity or a NaN neither the weight nor the finite values count.
    // Keys (a bit each) of the tile with such a value.
    static __device__ __forceinline__ uint32_t odd_keys(uint32_t vb) {
        const int lane = threadIdx.x & 31;
        constexpr int kLanes = D / 8, kKeys = 32 / kLanes;  // lanes of a key, keys of a step
        uint32_t keys = 0;
#pragma unroll
        for (int i = 0; i < kTile / kKeys; ++i) {
            uint32_t w[4];
            lds16(w, vb + i * 512 + lane * 16);
            const uint32_t ball = __ballot_sync(0xffffffffu, (kv_odd<T>(w[0]) | kv_odd<T>(w[1]) | kv_odd<T>(w[2]) | kv_odd<T>(w[3])) != 0);
#pragma unroll
            for (int k = 0; k < kKeys; ++k)
                if ((ball >> (k * kLanes) & ((1u << kLanes) - 1)) != 0) keys |= 1u << (i * kKeys + k);
        }
        return keys;
    }
    __device__ __forceinline__ void add_odd(uint32_t vb, int32_t j0, uint32_t keys) {
        if (spent) return;
        for (; keys != 0; keys &= keys - 1) {
            const int k = __ffs(keys) - 1;
            const bool s0 = sees(0, j0 + k), s1 = sees(1, j0 + k);
#pragma unroll
            for (int i = 0; i < 2 * kSteps; ++i) {
                uint32_t w;
                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(vb + k * kRow + ((i ^ (k & 7)) << 4) + 4 * (threadIdx.x & 3)) : "memory");
                const uint32_t odd = kv_odd<T>(w);
                if (odd == 0) continue;
                float a, b;
                Pack<T>::unpair(w, a, b);
                a = odd & 0x8000u ? a : 0.0f;
                b = odd >> 31 ? b : 0.0f;
                if (s0) acc[i][0] += a, acc[i][1] += b;
                if (s1) acc[i][2] += a, acc[i][3] += b;
            }
        }
        bool left = false;
        const int r = (threadIdx.x & 31) >> 2;
#pragma unroll
        for (int i = 0; i < 2 * kSteps; ++i) {
            if (r < rows) left |= acc[i][0] == acc[i][0] || acc[i][1] == acc[i][1];
            if (r + 8 < rows) left |= acc[i][2] == acc[i][2] || acc[i][3] == acc[i][3];
        }
        spent = !__any_sync(0xffffffffu, left);
    }
    static __device__ __forceinline__ void clear_odd(uint32_t vb) {
        for (int i = threadIdx.x & 31; i < kTile * kRow / 16; i += 32) {
            uint32_t w[4];
            lds16(w, vb + i * 16);
            sts16(vb + i * 16, kv_finite<T>(w[0]), kv_finite<T>(w[1]), kv_finite<T>(w[2]), kv_finite<T>(w[3]));
        }
    }
    static __device__ __forceinline__ void lds16(uint32_t (&w)[4], uint32_t at) {
        asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]) : "r"(at) : "memory");
    }
    static __device__ __forceinline__ void sts16(uint32_t at, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
        asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
    }
};

}  // namespace gfdb
