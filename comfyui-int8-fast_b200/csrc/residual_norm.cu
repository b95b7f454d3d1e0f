// The gated residual update of a transformer block between two norms, in one pass over the rows of a batch whose rows
// belong to several requests (every request has its own gate, scale and shift):
//
//   x' = c * x + g(m) * P(y)                 h = N(x') * (1 + s(m)) + t(m)
//
// m: the request of the row.  P (after the branch) and N (before the next) are an RMS norm, v / sqrt(mean(v^2) + eps), a
// LayerNorm, (v - mean) / sqrt(mean((v - mean)^2) + eps), or (P only) nothing, P(y) = y; each may carry a weight vector (without
// a norm too: a layer scale); g may be the tanh of what is given.  h leaves in the branch's 16-bit type, as per-token int8,
// or both: q = rint(h * (1 / a)), a = max(absmax(h) / 127, 1e-30).
//
// r = 1 / sqrt(...) is the device's rsqrtf (two units in the last place).  Everything between the loads and the stores is
// fp32: h and its int8 form come from the unrounded x', so each output is
// rounded once.  Row sums are per-thread sums, a shuffle tree, then the warps in order: the same order every time.
//
// Bound by the bytes of x, y, x' and h.  Measured, inputs from HBM: 4608 x 4096 bf16 in four equal requests 32.3 us = 4.7 TB/s
// (71 % of the copy rate; some 8 us of it pass before the first rows leave, the rest streams at 6.7 TB/s), in four requests
// of 46 to 3936 rows 36.6 us (a CTA whose rows cross a border works the columns of another request out), 18432 x 4096 with an
// fp32 residual 157 us = 5.8 TB/s (88 %), 777 rows of 2305 in 11 requests 18.6 us, one row 4.3 us.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "f32x2.cuh"
#include "host_common.h"
#include "ptx_sm100.cuh"
#include "tensor_maps.h"

namespace i8f {
namespace {

constexpr float kScaleFloor = 1e-30f;
constexpr int kMaxWarps = 16;
constexpr int kRowsPerRequest = 6;
constexpr int kRingRows = 256;      // batches of at least so many rows use the ring kernel

struct NormArgs {
    const void* x;
    const void* y;
    const void* gate;            // NULL: 1
    const void* scale;           // NULL: 0
    const void* shift;           // NULL: 0
    const void* post_weight;     // NULL: 1
    const void* weight;          // NULL: 1
    const int* row_request;      // NULL: request 0
    void* x_out;
    void* h;
    int8_t* q;
    float* row_scale;
    int64_t M, ldx, ldy, ldg, lds, ldt, ldxo, ldh, ldq;
    int K;
    int post_norm, norm, gate_tanh;
    float residual_scale, eps;
};

template <int DT>
struct Elem;
template <>
struct Elem<I8F_BF16> {
    using T = __nv_bfloat16;
    static __device__ __forceinline__ float to_f(T v) { return __bfloat162float(v); }
    static __device__ __forceinline__ T from_f(float v) { return __float2bfloat16_rn(v); }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {      // one conversion for two values
        const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};
template <>
struct Elem<I8F_F16> {
    using T = __half;
    static __device__ __forceinline__ float to_f(T v) { return __half2float(v); }
    static __device__ __forceinline__ T from_f(float v) { return __float2half_rn(v); }
    static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
        const __half2 h = __floats2half2_rn(lo, hi);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
};
template <>
struct Elem<I8F_F32> {
    using T = float;
    static __device__ __forceinline__ float to_f(T v) { return v; }
    static __device__ __forceinline__ T from_f(float v) { return v; }
};

// V consecutive elements at p (V = 8: 16-byte accesses; V = 1: any alignment).
template <int DT, int V>
__device__ __forceinline__ void load_v(const void* base, int64_t i, float (&f)[V]) {
    using E = Elem<DT>;
    const typename E::T* p = static_cast<const typename E::T*>(base) + i;
    if constexpr (V == 1) {
        f[0] = E::to_f(*p);
    } else {
        constexpr int kPieces = V * static_cast<int>(sizeof(typename E::T)) / 16;
        uint4 raw[kPieces];
#pragma unroll
        for (int j = 0; j < kPieces; ++j) raw[j] = reinterpret_cast<const uint4*>(p)[j];
        const typename E::T* e = reinterpret_cast<const typename E::T*>(raw);
#pragma unroll
        for (int j = 0; j < V; ++j) f[j] = E::to_f(e[j]);
    }
}
template <int DT, int V>
__device__ __forceinline__ void store_v(void* base, int64_t i, const float (&f)[V]) {
    using E = Elem<DT>;
    typename E::T* p = static_cast<typename E::T*>(base) + i;
    if constexpr (V == 1) {
        p[0] = E::from_f(f[0]);
    } else if constexpr (DT == I8F_F32) {
        reinterpret_cast<float4*>(p)[0] = make_float4(f[0], f[1], f[2], f[3]);
        reinterpret_cast<float4*>(p)[1] = make_float4(f[4], f[5], f[6], f[7]);
    } else {
        *reinterpret_cast<uint4*>(p) = make_uint4(E::pack(f[0], f[1]), E::pack(f[2], f[3]), E::pack(f[4], f[5]), E::pack(f[6], f[7]));
    }
}

// Sum (or maximum of bit patterns) over the threads of the CTA, one barrier: the slots alternate between two halves, and
// a half is written again only after the barrier of the call in between.
template <bool WARP>
struct RowReduce {
    float* slots;      // [2][kMaxWarps]
    int flip;
    __device__ __forceinline__ float sum(float v) {
#pragma unroll
        for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
        const int warps = WARP ? 1 : blockDim.x >> 5;
        if (warps == 1) return v;
        float* s = slots + flip * kMaxWarps;
        flip ^= 1;
        if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
        __syncthreads();
        float r = s[0];
        for (int w = 1; w < warps; ++w) r += s[w];
        return r;
    }
    // of non-negative values or NaN, as bit patterns: a NaN counts as larger than everything and so survives
    __device__ __forceinline__ float max_abs(uint32_t b) {
        b = __reduce_max_sync(0xFFFFFFFFu, b);
        const int warps = WARP ? 1 : blockDim.x >> 5;
        if (warps == 1) return __uint_as_float(b);
        float* s = slots + flip * kMaxWarps;
        flip ^= 1;
        if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = __uint_as_float(b);
        __syncthreads();
        uint32_t r = __float_as_uint(s[0]);
        for (int w = 1; w < warps; ++w) r = max(r, __float_as_uint(s[w]));
        return __uint_as_float(r);
    }
};

// v <- norm(v); positions past the row hold zeros and stay zero.
template <int V, int VPT, bool WARP>
__device__ __forceinline__ void normalise(float (&v)[VPT][V], int kind, float eps, int K, int nvec, RowReduce<WARP>& red) {
    if (kind == I8F_NORM_NONE) return;
    const float inv_k = 1.0f / static_cast<float>(K);
    const int t = WARP ? threadIdx.x & 31 : threadIdx.x, T = WARP ? 32 : blockDim.x;
    if (kind == I8F_NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
            for (int j = 0; j < V; ++j) s += v[i][j];
        const float mean = red.sum(s) * inv_k;
#pragma unroll
        for (int i = 0; i < VPT; ++i)
            if (i * T + t < nvec)
#pragma unroll
                for (int j = 0; j < V; ++j) v[i][j] -= mean;
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) s = fmaf(v[i][j], v[i][j], s);
    const float r = rsqrtf(red.sum(s) * inv_k + eps);
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) v[i][j] *= r;
}

// Quantisation step of a row from its absolute maximum, divided as i8f_quant_rowwise does (a product with 1 / 127 is off by a unit
// in the last place for some of them); a NaN stays: the row is marked by its scale.
__device__ __forceinline__ float row_step(float amax) {
    const float step = __fdiv_rn(amax, 127.0f);
    return step < kScaleFloor ? kScaleFloor : step;
}
template <int V>
__device__ __forceinline__ void store_q(int8_t* dst, const float (&f)[V], float inv) {
    uint32_t b[V];
#pragma unroll
    for (int j = 0; j < V; ++j) b[j] = static_cast<uint32_t>(__float2int_rn(fminf(fmaxf(f[j] * inv, -128.f), 127.f))) & 0xFFu;
    if constexpr (V == 1) {
        dst[0] = static_cast<int8_t>(b[0]);
    } else {
        uint2 o;
        o.x = b[0] | (b[1] << 8) | (b[2] << 16) | (b[3] << 24);
        o.y = b[4] | (b[5] << 8) | (b[6] << 16) | (b[7] << 24);
        *reinterpret_cast<uint2*>(dst) = o;
    }
}

// A few rows: one CTA per row, as many threads as vectors.  WARP: many short rows, a warp for each.
template <int XDT, int YDT, int V, int VPT, bool WARP>
__global__ void __launch_bounds__(WARP ? 256 : 512)
gated_residual_norm_kernel(const NormArgs a) {
    __shared__ float s_slots[2 * kMaxWarps];
    RowReduce<WARP> red{s_slots, 0};
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const int t = WARP ? threadIdx.x & 31 : threadIdx.x, T = WARP ? 32 : blockDim.x;
    const int nvec = a.K / V;
    const bool quant = a.q != nullptr;
    const int64_t row = WARP ? static_cast<int64_t>(blockIdx.x) * 8 + (threadIdx.x >> 5) : blockIdx.x;
    if (WARP && row >= a.M) return;
    const int req = a.row_request != nullptr ? a.row_request[row] : 0;
    float x[VPT][V], y[VPT][V];
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int vec = i * T + t;
#pragma unroll
        for (int j = 0; j < V; ++j) x[i][j] = y[i][j] = 0.f;
        if (vec < nvec) {
            load_v<XDT, V>(a.x, row * a.ldx + static_cast<int64_t>(vec) * V, x[i]);
            load_v<YDT, V>(a.y, row * a.ldy + static_cast<int64_t>(vec) * V, y[i]);
        }
    }
    normalise<V, VPT, WARP>(y, a.post_norm, a.eps, a.K, nvec, red);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int vec = i * T + t;
        if (vec < nvec) {
            float g[V], w[V];
#pragma unroll
            for (int j = 0; j < V; ++j) g[j] = w[j] = 1.f;
            if (a.gate != nullptr) load_v<YDT, V>(a.gate, req * a.ldg + static_cast<int64_t>(vec) * V, g);
            if (a.post_weight != nullptr) load_v<YDT, V>(a.post_weight, static_cast<int64_t>(vec) * V, w);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float gj = a.gate_tanh ? tanhf(g[j]) : g[j];
                x[i][j] = fmaf(gj, y[i][j] * w[j], a.residual_scale * x[i][j]);
            }
            store_v<XDT, V>(a.x_out, row * a.ldxo + static_cast<int64_t>(vec) * V, x[i]);
        }
    }
    normalise<V, VPT, WARP>(x, a.norm, a.eps, a.K, nvec, red);
    uint32_t big = 0u;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
        const int vec = i * T + t;
        if (vec < nvec) {
            float w[V], s[V], sh[V];
#pragma unroll
            for (int j = 0; j < V; ++j) {
                w[j] = 1.f;
                s[j] = sh[j] = 0.f;
            }
            if (a.weight != nullptr) load_v<YDT, V>(a.weight, static_cast<int64_t>(vec) * V, w);
            if (a.scale != nullptr) load_v<YDT, V>(a.scale, req * a.lds + static_cast<int64_t>(vec) * V, s);
            if (a.shift != nullptr) load_v<YDT, V>(a.shift, req * a.ldt + static_cast<int64_t>(vec) * V, sh);
#pragma unroll
            for (int j = 0; j < V; ++j) {
                x[i][j] = fmaf(x[i][j] * w[j], 1.f + s[j], sh[j]);
                if (quant) big = max(big, __float_as_uint(x[i][j]) & 0x7FFFFFFFu);
            }
            if (a.h != nullptr) store_v<YDT, V>(a.h, row * a.ldh + static_cast<int64_t>(vec) * V, x[i]);
        }
    }
    if (quant) {
        const float step = row_step(red.max_abs(big));
        const float inv = __frcp_rn(step);
        if (t == 0) a.row_scale[row] = step;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int vec = i * T + t;
            if (vec < nvec) store_q<V>(a.q + row * a.ldq + static_cast<int64_t>(vec) * V, x[i], inv);
        }
    }
}

// ------------------------------------------------------------------ many rows
// One CTA per SM walks a contiguous share of the rows.  A producer thread keeps a ring of whole rows of x and y in flight
// with untiled bulk copies (so the loads do not depend on how many threads are resident), groups of GT threads take the
// rows in turn.  What a request contributes per column, G = g * post_weight, S = (1 + scale) * weight and T = shift, is
// worked out once per request into shared memory (the tanh and the conversions with it) and read from there by every row;
// where the three do not leave room for the ring, only G is, and S and T are read as they were given.
// A row is read from shared memory twice (statistics of y, then x and y); only x' is held in registers.
//
// SHIFT: rows that do not start at a 16-byte boundary (a row length that 8 does not divide).  The copy takes the 16-byte
// pieces that contain the row; a row that starts `o` elements behind a boundary is handled in the vectors of its memory,
// elements 8 v - o ... 8 v - o + 7, so that all but the first and the last are read and written in 16-byte pieces.  x, y
// and the outputs must lie alike (o is the same for all of them), as contiguous tensors of one shape do.
// Threads that take rows.  Five groups hide a row's chain of reductions better than four (4608 x 4096 bf16 in four equal requests:
// 32.3 us against 34.7, with int8 rows 30.8 against 33.9); fp32 rows leave room for seven slots only, and four groups serve
// them better (18432 x 4096: 162 us against 166).
template <int XDT, int GT>
constexpr int workers() { return GT == 512 ? 512 : (XDT == I8F_F32 ? 4 : 5) * GT; }
constexpr int kMaxSlots = 16;
constexpr int kRingSmem = 224 * 1024;

enum : int { kStNormEmpty = 131, kStNormFull = 132 };

__host__ __device__ constexpr int slot_bytes(int row_bytes) { return (row_bytes + 15) / 16 * 16 + 32; }

template <int GT>
struct GroupReduce {      // sums over the GT threads of a group; slots as in RowReduce
    static constexpr int kWarps = GT / 32;
    float* slots;      // [2][kWarps]
    int bar, flip;
    __device__ __forceinline__ float* publish(float v) {
        float* s = slots + kWarps * flip;
        flip ^= 1;
        if ((threadIdx.x & 31) == 0) s[(threadIdx.x >> 5) & (kWarps - 1)] = v;
        asm volatile("bar.sync %0, %1;" ::"r"(bar), "n"(GT) : "memory");
        return s;
    }
    __device__ __forceinline__ float sum(float v) {
#pragma unroll
        for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
        const float* s = publish(v);
        float r = s[0];
#pragma unroll
        for (int w = 1; w < kWarps; ++w) r += s[w];
        return r;
    }
    __device__ __forceinline__ float max_abs(uint32_t b) {
        const float* s = publish(__uint_as_float(__reduce_max_sync(0xFFFFFFFFu, b)));
        uint32_t r = __float_as_uint(s[0]);
#pragma unroll
        for (int w = 1; w < kWarps; ++w) r = max(r, __float_as_uint(s[w]));
        return __uint_as_float(r);
    }
};

// The per-request arrays.  Aligned rows: 16-byte pieces of consecutive threads side by side.  SHIFT: element e at
// e + 8 + (e + 8) / 8, so that threads eight elements apart read from different banks wherever their vectors start.
template <int GT, int VPT, bool SHIFT>
struct Columns {
    // a multiple of four floats: the ring behind the arrays starts at a 16-byte boundary
    static constexpr int kFloats = SHIFT ? ((VPT * GT * 8 + 16) * 9 / 8 + 8 + 3) / 4 * 4 : VPT * GT * 8;
    static_assert(kFloats % 4 == 0, "the bulk copies need 16-byte aligned destinations");
    static __device__ __forceinline__ int at(int e) {
        if constexpr (SHIFT) return e + 8 + ((e + 8) >> 3);
        const int vec = e >> 3, i = vec / GT, tg = vec - i * GT, half = (e >> 2) & 1;
        return ((i * 2 + half) * GT + tg) * 4 + (e & 3);
    }
    static __device__ __forceinline__ void get(const float* arr, int i, int tg, int e0, f32x2 (&f)[4]) {
        if constexpr (SHIFT) {
            const float* p = arr + at(e0 & ~7);      // the vector crosses one multiple of 8 at most
            const int c = e0 & 7;
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j] = pair_of(p[c + 2 * j + (c + 2 * j >= 8 ? 1 : 0)], p[c + 2 * j + 1 + (c + 2 * j + 1 >= 8 ? 1 : 0)]);
        } else {
            const ulonglong2* p = reinterpret_cast<const ulonglong2*>(arr) + i * 2 * GT + tg;
            const ulonglong2 a = p[0], b = p[GT];
            f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
        }
    }
};

// The rows of a vector that starts at e0 and lies partly outside [0, K) get zeros there.
template <bool SHIFT>
__device__ __forceinline__ void clear_outside(int e0, int K, f32x2 (&f)[4]) {
    if constexpr (SHIFT) {
        if (e0 < 0 || e0 + 8 > K) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float lo, hi;
                halves(f[j], lo, hi);
                const int e = e0 + 2 * j;
                f[j] = pair_of(e >= 0 && e < K ? lo : 0.f, e + 1 >= 0 && e + 1 < K ? hi : 0.f);
            }
        }
    }
}
// Eight elements from e0 of a row in shared memory, two to a register pair.
template <int DT, bool SHIFT>
__device__ __forceinline__ void get8(const typename Elem<DT>::T* row, int e0, int K, f32x2 (&f)[4]) {
    if constexpr (DT == I8F_F32) {
        const ulonglong2* p = reinterpret_cast<const ulonglong2*>(row + e0);
        const ulonglong2 a = p[0], b = p[1];
        f[0] = a.x; f[1] = a.y; f[2] = b.x; f[3] = b.y;
    } else {
        const uint4 r = *reinterpret_cast<const uint4*>(row + e0);
        const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if constexpr (DT == I8F_BF16) {
                f[j] = pair_of_bits(w[j] << 16, w[j] & 0xFFFF0000u);
            } else {
                const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&w[j]));
                f[j] = pair_of(v.x, v.y);
            }
        }
    }
    clear_outside<SHIFT>(e0, K, f);
}
__device__ __forceinline__ void unpair(const f32x2 (&p)[4], float (&f)[8]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) halves(p[j], f[2 * j], f[2 * j + 1]);
}
__device__ __forceinline__ float both(f32x2 p) {
    float lo, hi;
    halves(p, lo, hi);
    return lo + hi;
}
// larger of m and |v|, a NaN if either is one
__device__ __forceinline__ float max_abs_nan(float m, float v) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(v)));
    return r;
}
// rint(f * inv) as int8 by the addition of 1.5 * 2^23; |f * inv| is at most 127.00002 (inv is the reciprocal of the
// row's step), so there is nothing to clamp.
__device__ __forceinline__ uint2 quant8(const f32x2 (&x)[4], float inv) {
    const f32x2 magic = pair_of(12582912.0f, 12582912.0f);
    uint32_t u[8];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float lo, hi;
        halves(x[j], lo, hi);
        halves_bits(add2(pair_of(__fmul_rn(lo, inv), __fmul_rn(hi, inv)), magic), u[2 * j], u[2 * j + 1]);
    }
    return make_uint2(__byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410),
                      __byte_perm(__byte_perm(u[4], u[5], 0x0040), __byte_perm(u[6], u[7], 0x0040), 0x5410));
}
template <int DT, bool SHIFT>
__device__ __forceinline__ void put8(void* base, int64_t row0, int e0, int K, const f32x2 (&p)[4]) {
    float f[8];
    unpair(p, f);
    if (!SHIFT || (e0 >= 0 && e0 + 8 <= K)) {
        store_v<DT, 8>(base, row0 + e0, f);
    } else {
        typename Elem<DT>::T* dst = static_cast<typename Elem<DT>::T*>(base) + row0 + e0;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (e0 + j >= 0 && e0 + j < K) dst[j] = Elem<DT>::from_f(f[j]);
    }
}
// A vector of per-request or per-column values from global memory (any alignment with SHIFT).
template <int DT, bool SHIFT>
__device__ __forceinline__ void column8(const void* base, int64_t at, int e0, int K, float (&f)[8]) {
    if constexpr (SHIFT) {
        const typename Elem<DT>::T* p = static_cast<const typename Elem<DT>::T*>(base) + at + e0;
#pragma unroll
        for (int j = 0; j < 8; ++j) f[j] = (e0 + j >= 0 && e0 + j < K) ? Elem<DT>::to_f(p[j]) : 0.f;
    } else {
        load_v<DT, 8>(base, at + e0, f);
    }
}

template <int XDT, int YDT, int GT, int VPT, bool SHIFT>
__global__ void __launch_bounds__((workers<XDT, GT>() + 32), 1)
gated_residual_norm_ring_kernel(const NormArgs a, int n_slots, int all_columns, int* status) {
    using TX = typename Elem<XDT>::T;
    using TY = typename Elem<YDT>::T;
    using C = Columns<GT, VPT, SHIFT>;
    constexpr int kWorkers = workers<XDT, GT>();
    constexpr int kGroups = kWorkers / GT;
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ __align__(16) float s_part[2 * kWorkers / 32];
    // Two barriers for the arrival of a slot's rows, used in turn.  A slot passes from group to group and copies land in any
    // order, so a group may come for its row while the row before it in the slot, another group's, is still on its way: on
    // one barrier that group would take the phase before for its own (they have the same parity).  The barrier's previous
    // row is then two rounds back, and that one has been consumed: the row in between could not have been issued otherwise,
    // and it was issued before the group's own previous row (there are more slots than groups).
    __shared__ __align__(8) unsigned long long s_full[2 * kMaxSlots], s_empty[kMaxSlots];
    __shared__ int s_abort;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    float* const s_gate = reinterpret_cast<float*>(smem);
    float* const s_scale = s_gate + C::kFloats;
    float* const s_shift = s_scale + C::kFloats;
    uint8_t* const ring = smem + (all_columns ? 3 : 1) * C::kFloats * sizeof(float);
    const int x_slot = slot_bytes(a.K * static_cast<int>(sizeof(TX))), y_slot = slot_bytes(a.K * static_cast<int>(sizeof(TY)));
    const int64_t row0 = a.M * blockIdx.x / gridDim.x, row1 = a.M * (blockIdx.x + 1) / gridDim.x;
    if (threadIdx.x == 0) {
        for (int i = 0; i < n_slots; ++i) {
            mbar_init(smem_u32(&s_full[i]), 1);
            mbar_init(smem_u32(&s_full[n_slots + i]), 1);
            mbar_init(smem_u32(&s_empty[i]), 1);
        }
        s_abort = 0;
        fence_mbar_init();
        fence_proxy_async_smem();
    }
    __syncthreads();

    if (threadIdx.x >= kWorkers) {
        if (threadIdx.x == kWorkers) {
            int turn = 0;       // row number modulo 2 * n_slots
            for (int64_t row = row0; row < row1; ++row) {
                const int slot = turn < n_slots ? turn : turn - n_slots;
                if (!mbar_wait_bounded(smem_u32(&s_empty[slot]), turn < n_slots ? 1u : 0u, &s_abort, status, kStNormEmpty)) break;
                const uintptr_t px = reinterpret_cast<uintptr_t>(static_cast<const TX*>(a.x) + row * a.ldx);
                const uintptr_t py = reinterpret_cast<uintptr_t>(static_cast<const TY*>(a.y) + row * a.ldy);
                const uint32_t nx = static_cast<uint32_t>(((px & 15) + a.K * sizeof(TX) + 15) & ~uintptr_t(15));
                const uint32_t ny = static_cast<uint32_t>(((py & 15) + a.K * sizeof(TY) + 15) & ~uintptr_t(15));
                uint32_t dst = smem_u32(ring) + static_cast<uint32_t>(slot * (x_slot + y_slot));
                const uint32_t bar = smem_u32(&s_full[turn]);
                mbar_arrive_expect_tx(bar, nx + ny);
                // an fp32 row starts in the 16-byte half of its 8-element vector that its place in memory says
                const uint32_t half = XDT == I8F_F32 && SHIFT ? static_cast<uint32_t>((py & 15) / 2 - (px & 15) / 4) * 4u : 0u;
                bulk_load(dst + half, reinterpret_cast<const void*>(px & ~uintptr_t(15)), nx, bar);
                bulk_load(dst + x_slot, reinterpret_cast<const void*>(py & ~uintptr_t(15)), ny, bar);
                if (++turn == 2 * n_slots) turn = 0;
            }
        }
    } else {
        const int group = threadIdx.x / GT, tg = threadIdx.x & (GT - 1);
        const int K = a.K;
        const float inv_k = 1.0f / static_cast<float>(K);
        const bool quant = a.q != nullptr;
        GroupReduce<GT> red{s_part + group * 2 * (GT / 32), 1 + group, 0};
        int turn = group, have = -1;      // row number modulo 2 * n_slots; fewer groups than slots
        uint32_t phase = 0;
        int64_t row = row0 + group;
        for (int64_t seg0 = row0; seg0 < row1;) {
            // the rows [seg0, seg1) of the share belong to one request
            const int req = a.row_request != nullptr ? __ldg(a.row_request + seg0) : 0;
            int64_t seg1 = row1;
            if (a.row_request != nullptr) {
                for (int64_t at = seg0; at < row1; at += 32) {      // the first row of another request, 32 rows at a time
                    const int64_t mine = at + (threadIdx.x & 31);
                    const uint32_t other = __ballot_sync(0xFFFFFFFFu, mine < row1 && __ldg(a.row_request + mine) != req);
                    if (other) {
                        seg1 = at + __ffs(other) - 1;
                        break;
                    }
                }
            }
            if (req != have) {
                have = req;
                asm volatile("bar.sync 15, %0;" ::"n"(kWorkers) : "memory");      // every group is done with the request before
                // (K + 7) / 8 vectors of the row as if it were aligned
                for (int e0 = static_cast<int>(threadIdx.x) * 8; e0 < K; e0 += kWorkers * 8) {
                    float g[8], pw[8], sc[8], w[8], sh[8];
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        g[j] = pw[j] = w[j] = 1.f;
                        sc[j] = sh[j] = 0.f;
                    }
                    if (a.gate != nullptr) column8<YDT, SHIFT>(a.gate, req * a.ldg, e0, K, g);
                    if (a.post_weight != nullptr) column8<YDT, SHIFT>(a.post_weight, 0, e0, K, pw);
                    if (all_columns) {
                        if (a.scale != nullptr) column8<YDT, SHIFT>(a.scale, req * a.lds, e0, K, sc);
                        if (a.weight != nullptr) column8<YDT, SHIFT>(a.weight, 0, e0, K, w);
                        if (a.shift != nullptr) column8<YDT, SHIFT>(a.shift, req * a.ldt, e0, K, sh);
                    }
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        const int at = C::at(e0 + j);
                        s_gate[at] = (a.gate_tanh ? tanhf(g[j]) : g[j]) * pw[j];
                        if (all_columns) {
                            s_scale[at] = (1.f + sc[j]) * w[j];
                            s_shift[at] = sh[j];
                        }
                    }
                }
                asm volatile("bar.sync 15, %0;" ::"n"(kWorkers) : "memory");
            }
            for (; row < seg1; row += kGroups) {
                // After a wait that ran out the rows are walked to the end all the same (every later wait gives up at once):
                // the groups meet at barriers and may not leave one another there.
                mbar_wait_bounded(smem_u32(&s_full[turn]), phase, &s_abort, status, kStNormFull);
                __syncwarp();
                const int slot = turn < n_slots ? turn : turn - n_slots;
                const uintptr_t py = reinterpret_cast<uintptr_t>(static_cast<const TY*>(a.y) + row * a.ldy);
                const int o = SHIFT ? static_cast<int>((py >> 1) & 7) : 0;      // elements between the boundary and the row
                const TX* const sx = reinterpret_cast<const TX*>(ring + slot * (x_slot + y_slot)) + o;
                const TY* const sy = reinterpret_cast<const TY*>(ring + slot * (x_slot + y_slot) + x_slot) + o;
                float mean = 0.f, r = 1.f;
                const f32x2 zero2 = pair_of(0.f, 0.f);
                if (a.post_norm == I8F_NORM_LAYER) {
                    f32x2 s = zero2;
#pragma unroll
                    for (int i = 0; i < VPT; ++i) {
                        const int e0 = (i * GT + tg) * 8 - o;
                        if (e0 < K) {
                            f32x2 y[4];
                            get8<YDT, SHIFT>(sy, e0, K, y);
#pragma unroll
                            for (int j = 0; j < 4; ++j) s = add2(s, y[j]);
                        }
                    }
                    mean = red.sum(both(s)) * inv_k;
                }
                if (a.post_norm != I8F_NORM_NONE) {
                    f32x2 s = zero2;
                    const f32x2 mean2 = pair_of(mean, mean);
#pragma unroll
                    for (int i = 0; i < VPT; ++i) {
                        const int e0 = (i * GT + tg) * 8 - o;
                        if (e0 < K) {
                            f32x2 y[4];
                            get8<YDT, SHIFT>(sy, e0, K, y);
                            if (a.post_norm == I8F_NORM_LAYER) {
#pragma unroll
                                for (int j = 0; j < 4; ++j) y[j] = sub2(y[j], mean2);
                                clear_outside<SHIFT>(e0, K, y);
                            }
#pragma unroll
                            for (int j = 0; j < 4; ++j) s = fma2(y[j], y[j], s);
                        }
                    }
                    r = rsqrtf(red.sum(both(s)) * inv_k + a.eps);
                }
                // x' = residual_scale * x + (y - mean) * r * G, and the first sum of the second norm
                f32x2 x[VPT][4];
                f32x2 s2 = zero2;
                const bool centre = a.norm == I8F_NORM_LAYER;
                {
                    const f32x2 r2 = pair_of(r, r), mr2 = pair_of(-mean * r, -mean * r), c2 = pair_of(a.residual_scale, a.residual_scale);
                    const bool plain = a.residual_scale == 1.0f;
#pragma unroll
                    for (int i = 0; i < VPT; ++i) {
                        const int e0 = (i * GT + tg) * 8 - o;
                        if (e0 < K) {
                            f32x2 y[4], g[4];
                            get8<XDT, SHIFT>(sx, e0, K, x[i]);
                            get8<YDT, SHIFT>(sy, e0, K, y);
                            C::get(s_gate, i, tg, e0, g);
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                if (!plain) x[i][j] = mul2(c2, x[i][j]);
                                x[i][j] = fma2(fma2(y[j], r2, mr2), g[j], x[i][j]);
                            }
                            clear_outside<SHIFT>(e0, K, x[i]);
                            if (centre) {
#pragma unroll
                                for (int j = 0; j < 4; ++j) s2 = add2(s2, x[i][j]);
                            } else {
#pragma unroll
                                for (int j = 0; j < 4; ++j) s2 = fma2(x[i][j], x[i][j], s2);
                            }
                            put8<XDT, SHIFT>(a.x_out, row * a.ldxo, e0, K, x[i]);
                        }
                    }
                }
                float s = red.sum(both(s2));
                if (tg == 0) mbar_arrive(smem_u32(&s_empty[slot]));      // the barrier in sum(): every thread has read the row
                if (centre) {
                    mean = s * inv_k;
                    const f32x2 mean2 = pair_of(mean, mean);
                    s2 = zero2;
#pragma unroll
                    for (int i = 0; i < VPT; ++i) {
                        const int e0 = (i * GT + tg) * 8 - o;
                        if (e0 < K) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) x[i][j] = sub2(x[i][j], mean2);
                            clear_outside<SHIFT>(e0, K, x[i]);
#pragma unroll
                            for (int j = 0; j < 4; ++j) s2 = fma2(x[i][j], x[i][j], s2);
                        }
                    }
                    s = red.sum(both(s2));
                }
                r = rsqrtf(s * inv_k + a.eps);
                const f32x2 r2 = pair_of(r, r);
                float big = 0.f;
#pragma unroll
                for (int i = 0; i < VPT; ++i) {
                    const int e0 = (i * GT + tg) * 8 - o;
                    if (e0 < K) {
                        f32x2 sc[4], sh[4];
                        if (all_columns) {
                            C::get(s_scale, i, tg, e0, sc);
                            C::get(s_shift, i, tg, e0, sh);
                        } else {
                            float c[8], w[8], t[8];
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                c[j] = t[j] = 0.f;
                                w[j] = 1.f;
                            }
                            if (a.scale != nullptr) column8<YDT, SHIFT>(a.scale, req * a.lds, e0, K, c);
                            if (a.weight != nullptr) column8<YDT, SHIFT>(a.weight, 0, e0, K, w);
                            if (a.shift != nullptr) column8<YDT, SHIFT>(a.shift, req * a.ldt, e0, K, t);
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                sc[j] = pair_of((1.f + c[2 * j]) * w[2 * j], (1.f + c[2 * j + 1]) * w[2 * j + 1]);
                                sh[j] = pair_of(t[2 * j], t[2 * j + 1]);
                            }
                        }
#pragma unroll
                        for (int j = 0; j < 4; ++j) x[i][j] = fma2(mul2(x[i][j], r2), sc[j], sh[j]);
                        if (quant) {
                            clear_outside<SHIFT>(e0, K, x[i]);
                            float f[8];
                            unpair(x[i], f);
#pragma unroll
                            for (int j = 0; j < 8; ++j) big = max_abs_nan(big, f[j]);
                        }
                        if (a.h != nullptr) put8<YDT, SHIFT>(a.h, row * a.ldh, e0, K, x[i]);
                    }
                }
                if (quant) {
                    const float step = row_step(red.max_abs(__float_as_uint(big) & 0x7FFFFFFFu));
                    const float inv = __frcp_rn(step);
                    if (tg == 0) a.row_scale[row] = step;
#pragma unroll
                    for (int i = 0; i < VPT; ++i) {
                        const int e0 = (i * GT + tg) * 8 - o;
                        if (e0 < K) {
                            int8_t* const dst = a.q + row * a.ldq + e0;
                            const uint2 b = quant8(x[i], inv);
                            if (!SHIFT || (e0 >= 0 && e0 + 8 <= K)) {
                                *reinterpret_cast<uint2*>(dst) = b;
                            } else {
#pragma unroll
                                for (int j = 0; j < 8; ++j)
                                    if (e0 + j >= 0 && e0 + j < K) dst[j] = static_cast<int8_t>((j < 4 ? b.x >> (8 * j) : b.y >> (8 * (j - 4))) & 0xFFu);
                            }
                        }
                    }
                }
                turn += kGroups;
                if (turn >= 2 * n_slots) {
                    turn -= 2 * n_slots;
                    phase ^= 1u;
                }
            }
            seg0 = seg1;
        }
    }
    __syncthreads();
    if (s_abort)      // copies still in flight get time to land before the CTA exits
        for (int i = 0; i < 64; ++i) __nanosleep(1000);
}

// Launches the ring kernel if its columns and at least `min_slots` rows (more than there are groups, or two for a single one)
// fit an SM; *done says whether they did.
template <int XDT, int YDT, int GT, int VPT, bool SHIFT>
int launch_ring(const NormArgs& a, int min_slots, int sms, cudaStream_t st, bool* done) {
    const int slot = slot_bytes(a.K * dtype_size(XDT)) + slot_bytes(a.K * dtype_size(YDT));
    constexpr int kArray = Columns<GT, VPT, SHIFT>::kFloats * 4;
    int all_columns = 1, room = (kRingSmem - 3 * kArray) / slot;
    if (room < min_slots) {
        all_columns = 0;
        room = (kRingSmem - kArray) / slot;
    }
    *done = room >= min_slots;
    if (!*done) return I8F_OK;
    const int n_slots = room < kMaxSlots ? room : kMaxSlots;
    auto kern = gated_residual_norm_ring_kernel<XDT, YDT, GT, VPT, SHIFT>;
    static bool attr_done[64] = {false};
    const int dev = current_device();
    if (!attr_done[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kRingSmem);
        if (e != cudaSuccess) return fail(I8F_ERR_CUDA, "cudaFuncSetAttribute(smem=%d): %s", kRingSmem, cudaGetErrorString(e));
        attr_done[dev] = true;
    }
    int* status = device_status_word();
    I8F_REQUIRE(status != nullptr, I8F_ERR_CUDA, "device status word unavailable");
    const int64_t grid = a.M < sms ? a.M : sms;
    kern<<<static_cast<unsigned>(grid), (workers<XDT, GT>() + 32), (all_columns ? 3 : 1) * kArray + n_slots * slot, st>>>(a, n_slots, all_columns, status);
    return check_launch("gated_residual_norm_ring_kernel");
}

template <int XDT, int YDT, bool SHIFT>
int launch_ring_for(const NormArgs& a, int sms, cudaStream_t st, bool* done) {
    const int columns = a.K + (SHIFT ? 7 : 0);      // a shifted row may touch one more vector
    *done = false;
    if (a.M < kRingRows) return I8F_OK;
#define I8F_TRY(GT, VPT, MIN)                                                                     \
    if (columns <= GT * VPT * 8) {                                                                \
        const int rc = launch_ring<XDT, YDT, GT, VPT, SHIFT>(a, MIN, sms, st, done);              \
        if (rc != I8F_OK || *done) return rc;                                                     \
    }
    // several rows at a time up to 4096 columns, longer rows one at a time; at least one row more in flight than at work
    constexpr int kMin = workers<XDT, 128>() / 128 + 1;
    I8F_TRY(128, 1, kMin)
    I8F_TRY(128, 2, kMin)
    I8F_TRY(128, 4, kMin)
    I8F_TRY(512, 2, 2)
    I8F_TRY(512, 4, 2)
#undef I8F_TRY
    return I8F_OK;
}

template <int XDT, int YDT>
int launch_norm(const NormArgs& a, int64_t requests, bool vec8, bool alike, cudaStream_t st) {
    const int sms = sm_count();
    const unsigned grid = static_cast<unsigned>(a.M), grid8 = static_cast<unsigned>((a.M + 7) / 8);
    // Which kernel (us at K columns, bf16, measured): fewer than 256 rows one CTA each (64 rows of 4096: 4.2, in the ring 6.1;
    // 512 rows: 10.7 and 7.5).  Rows of up to 512 columns a warp each (4608 rows of 512: 8.4, in the ring 14.4; of 1024: 19.0
    // and 14.6), up to 256 where the rows are not aligned.
    // Requests of a few rows each: working a request's columns out costs the ring about 4.6 us (4608 rows of 4096, one row per
    // request: 174 us, a CTA per row 64; 18 rows per request: 40 in the ring).
    const int warp_columns = vec8 ? 512 : 256;
    if (a.M >= kRingRows && a.K > warp_columns && a.M >= kRowsPerRequest * requests) {
        bool done = false;
        const int rc = vec8 ? launch_ring_for<XDT, YDT, false>(a, sms, st, &done) : alike ? launch_ring_for<XDT, YDT, true>(a, sms, st, &done) : I8F_OK;
        if (rc != I8F_OK || done) return rc;
    }
#define I8F_NORM_GO(V, VPT, WARP, G, T) gated_residual_norm_kernel<XDT, YDT, V, VPT, WARP><<<G, T, 0, st>>>(a)
    if (vec8) {
        const int nvec = a.K / 8;
        if (a.M >= kRingRows && nvec <= 64) I8F_NORM_GO(8, 2, true, grid8, 256);
        else if (nvec <= 512) I8F_NORM_GO(8, 1, false, grid, (nvec + 31) / 32 * 32);
        else if (nvec <= 1024) I8F_NORM_GO(8, 2, false, grid, 512);
        else I8F_NORM_GO(8, 4, false, grid, 512);
    } else {
        if (a.M >= kRingRows && a.K <= 256) I8F_NORM_GO(1, 8, true, grid8, 256);
        else if (a.K <= 2048) I8F_NORM_GO(1, 8, false, grid, (a.K + 255) / 256 * 32);
        else if (a.K <= 8192) I8F_NORM_GO(1, 16, false, grid, 512);
        else I8F_NORM_GO(1, 32, false, grid, 512);
    }
#undef I8F_NORM_GO
    return check_launch("gated_residual_norm_kernel");
}

bool vec_ok(const void* p, int64_t ld, int elem) { return p == nullptr || (aligned16(p) && (ld * elem) % 16 == 0); }

}  // namespace
}  // namespace i8f

using namespace i8f;

extern "C" int i8f_gated_residual_norm(const void* x, int x_dtype, int64_t ldx, const void* y, int y_dtype, int64_t ldy,
                                       int64_t M, int64_t K, const int32_t* row_request, int64_t requests, const void* gate, int64_t ldg,
                                       int gate_tanh, float residual_scale, int post_norm, const void* post_weight, int norm,
                                       const void* weight, const void* scale, int64_t lds, const void* shift, int64_t ldt,
                                       float eps, void* x_out, int64_t ldxo, void* h, int64_t ldh, int8_t* q, int64_t ldq,
                                       float* row_scale, void* stream) {
    const char* const what = "i8f_gated_residual_norm";
    I8F_REQUIRE(y_dtype == I8F_BF16 || y_dtype == I8F_F16, I8F_ERR_UNSUPPORTED, "%s: y_dtype must be bf16 or f16", what);
    I8F_REQUIRE(x_dtype == y_dtype || x_dtype == I8F_F32, I8F_ERR_UNSUPPORTED, "%s: x_dtype must be y_dtype or f32", what);
    I8F_REQUIRE(M >= 0 && M < (1LL << 31) && K >= 0, I8F_ERR_INVALID_ARG, "%s: bad size M=%lld K=%lld", what, (long long)M, (long long)K);
    I8F_REQUIRE(K <= 16384, I8F_ERR_UNSUPPORTED, "%s: row length %lld exceeds the 16384-element limit", what, (long long)K);
    I8F_REQUIRE(post_norm >= I8F_NORM_NONE && post_norm <= I8F_NORM_LAYER && norm >= I8F_NORM_RMS && norm <= I8F_NORM_LAYER,
                I8F_ERR_INVALID_ARG, "%s: unknown norm (post_norm=%d, norm=%d)", what, post_norm, norm);
    I8F_REQUIRE(eps >= 0.f, I8F_ERR_INVALID_ARG, "%s: eps must not be negative", what);
    I8F_REQUIRE(requests >= 1, I8F_ERR_INVALID_ARG, "%s: requests must be positive", what);
    if (M == 0 || K == 0) return I8F_OK;
    I8F_REQUIRE(x != nullptr && y != nullptr && x_out != nullptr, I8F_ERR_INVALID_ARG, "%s: NULL input or output", what);
    I8F_REQUIRE(h != nullptr || q != nullptr, I8F_ERR_INVALID_ARG, "%s: h and q are both NULL", what);
    I8F_REQUIRE(q == nullptr || row_scale != nullptr, I8F_ERR_INVALID_ARG, "%s: q needs row_scale", what);
    I8F_REQUIRE(ldx >= K && ldy >= K && ldxo >= K && (h == nullptr || ldh >= K) && (q == nullptr || ldq >= K), I8F_ERR_INVALID_ARG,
                "%s: a row pitch is smaller than the row", what);
    I8F_REQUIRE((gate == nullptr || ldg == 0 || ldg >= K) && (scale == nullptr || lds == 0 || lds >= K) && (shift == nullptr || ldt == 0 || ldt >= K),
                I8F_ERR_INVALID_ARG, "%s: a modulation pitch is smaller than the row", what);
    const int xs = dtype_size(x_dtype);
    const bool vec8 = K % 8 == 0 && vec_ok(x, ldx, xs) && vec_ok(x_out, ldxo, xs) && vec_ok(y, ldy, 2) && vec_ok(h, ldh, 2) &&
                      vec_ok(gate, ldg, 2) && vec_ok(scale, lds, 2) && vec_ok(shift, ldt, 2) && vec_ok(post_weight, 0, 2) &&
                      vec_ok(weight, 0, 2) && (q == nullptr || ((reinterpret_cast<uintptr_t>(q) & 7u) == 0 && ldq % 8 == 0));
    // whether all rows of x, y and the outputs start equally far behind a boundary of eight elements
    auto lies_like_y = [&](const void* p, int64_t ld, int elem, int within) {
        return p == nullptr || (static_cast<int64_t>(reinterpret_cast<uintptr_t>(p) / elem - reinterpret_cast<uintptr_t>(y) / 2) % within == 0 &&
                                (ld - ldy) % within == 0);
    };
    const bool alike = lies_like_y(x, ldx, xs, xs == 4 ? 4 : 8) && lies_like_y(x_out, ldxo, xs, xs == 4 ? 4 : 8) && lies_like_y(h, ldh, 2, 8) &&
                       lies_like_y(q, ldq, 1, 8);
    NormArgs a{};
    a.x = x;
    a.y = y;
    a.gate = gate;
    a.scale = scale;
    a.shift = shift;
    a.post_weight = post_weight;
    a.weight = weight;
    a.row_request = row_request;
    a.x_out = x_out;
    a.h = h;
    a.q = q;
    a.row_scale = row_scale;
    a.M = M;
    a.ldx = ldx;
    a.ldy = ldy;
    a.ldg = ldg;
    a.lds = lds;
    a.ldt = ldt;
    a.ldxo = ldxo;
    a.ldh = ldh;
    a.ldq = ldq;
    a.K = static_cast<int>(K);
    a.post_norm = post_norm;
    a.norm = norm;
    a.gate_tanh = gate_tanh;
    a.residual_scale = residual_scale;
    a.eps = eps;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool f32 = x_dtype == I8F_F32;
    if (y_dtype == I8F_BF16) return f32 ? launch_norm<I8F_F32, I8F_BF16>(a, requests, vec8, alike, st) : launch_norm<I8F_BF16, I8F_BF16>(a, requests, vec8, alike, st);
    return f32 ? launch_norm<I8F_F32, I8F_F16>(a, requests, vec8, alike, st) : launch_norm<I8F_F16, I8F_F16>(a, requests, vec8, alike, st);
}
