// The up projection of low-rank adapters for a few rows, by ordinary warps: rows of one adapter against consecutive rows of
// its B [N, r].  A handful of rows is far below what a tcgen05 tile needs, and one thread per dot product spends its issue
// slots on widening; mma.sync.m16n8k16 takes sixteen rows of B as the A operand and up to eight rows of t as B.
// The k index inside the MMAs is a permutation of the real one, applied to both operands: lane t of a quad supplies the
// eight consecutive elements 8 t ... 8 t + 7 of a 32-element step (one 16-byte load), four to each of two MMAs.
#pragma once
#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "../../include/i8f.h"

namespace i8f {

constexpr int kLowRankRows = 4;      // rows of a chunk

template <bool BF16>
__device__ __forceinline__ void widen8(const uint4& r, float (&v)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (BF16) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}

template <bool BF16>
__device__ __forceinline__ void mma_low_rank(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if constexpr (BF16) {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    } else {
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    }
}

// For each of G groups: dst[(first + m) * stride + n] = t[first + m] . b[n] for m < rows (at most 8) and n < cols, first the
// group's first row.  Called by whole warps; rows, b (NULL: the group is left alone) and the sizes are the same in all lanes.
// t: pitch ldt elements, r (a multiple of 8) in use; b: cols rows of r elements.  Each group is a product of its own, so
// nothing passes from one adapter's rows to another's.  G groups x NT blocks of sixteen columns are loaded together: what
// bounds a few rows is the latency of these loads.
template <bool BF16, int G, int NT>
__device__ __forceinline__ void low_rank_rows(const uint16_t* t, int64_t ldt, const int (&first)[G], const int (&rows)[G],
                                              const uint16_t* const (&b)[G], int cols, int r, float* dst, int64_t stride, int lane) {
    const int g = lane >> 2, q = lane & 3;
    const uint4 zero = make_uint4(0u, 0u, 0u, 0u);
#pragma unroll 1
    for (int n0 = 0; n0 < cols; n0 += 16 * NT) {
        float acc[G][NT][4];
#pragma unroll
        for (int i = 0; i < G; ++i)
#pragma unroll
            for (int u = 0; u < NT; ++u) acc[i][u][0] = acc[i][u][1] = acc[i][u][2] = acc[i][u][3] = 0.f;
#pragma unroll 1
        for (int k0 = 0; k0 < r; k0 += 32) {
            const int k = k0 + 8 * q;
            uint4 rt[G], lo[G][NT], hi[G][NT];
#pragma unroll
            for (int i = 0; i < G; ++i) {
                const bool on = b[i] != nullptr && k < r;
                rt[i] = on && g < rows[i] ? *reinterpret_cast<const uint4*>(t + (first[i] + g) * ldt + k) : zero;
#pragma unroll
                for (int u = 0; u < NT; ++u) {
                    const int n = n0 + 16 * u + g;
                    lo[i][u] = on && n < cols ? __ldg(reinterpret_cast<const uint4*>(b[i] + static_cast<int64_t>(n) * r + k)) : zero;
                    hi[i][u] = on && n + 8 < cols ? __ldg(reinterpret_cast<const uint4*>(b[i] + static_cast<int64_t>(n + 8) * r + k)) : zero;
                }
            }
#pragma unroll
            for (int i = 0; i < G; ++i) {
                if (b[i] == nullptr) continue;
#pragma unroll
                for (int u = 0; u < NT; ++u) {
                    mma_low_rank<BF16>(acc[i][u], lo[i][u].x, hi[i][u].x, lo[i][u].y, hi[i][u].y, rt[i].x, rt[i].y);
                    mma_low_rank<BF16>(acc[i][u], lo[i][u].z, hi[i][u].z, lo[i][u].w, hi[i][u].w, rt[i].z, rt[i].w);
                }
            }
        }
#pragma unroll
        for (int i = 0; i < G; ++i) {
            if (b[i] == nullptr) continue;
            // lane (g, q) holds columns n0 + g and n0 + g + 8 of rows 2 q and 2 q + 1
#pragma unroll
            for (int u = 0; u < NT; ++u) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const int m = 2 * q + (e & 1), n = n0 + 16 * u + g + 8 * (e >> 1);
                    if (m < rows[i] && n < cols) dst[(first[i] + m) * stride + n] = acc[i][u][e];
                }
            }
        }
    }
}

}  // namespace i8f
