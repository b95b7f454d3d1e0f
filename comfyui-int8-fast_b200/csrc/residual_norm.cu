// The gated residual update of a transformer block between two norms, in one pass over the rows of a batch whose rows
// belong to several requests (every request has its own gate, scale and shift):
//
//   x' = c * x + g(m) * P(y)                 h = N(x') * (1 + s(m)) + t(m)
//
// m: the request of the row.  P (after the branch) and N (before the next) are an RMS norm, v / sqrt(mean(v^2) + eps), a
// LayerNorm, (v - mean) / sqrt(mean((v - mean)^2) + eps), or (P only) nothing; each may carry a weight vector; g may be
// the tanh of what is given.  h leaves in the branch's 16-bit type, as per-token int8, or both: q = rint(h * (1 / a)),
// a = max(absmax(h) / 127, 1e-30).
//
// Everything between the loads and the stores is fp32: h and its int8 form come from the unrounded x', so each output is
// rounded once.  Row sums are per-thread sums, a shuffle tree, then the warps in order: the same order every time.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "host_common.h"

namespace i8f {
namespace {

constexpr float kScaleFloor = 1e-30f;
constexpr int kMaxWarps = 16;

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
};
template <>
struct Elem<I8F_F16> {
    using T = __half;
    static __device__ __forceinline__ float to_f(T v) { return __half2float(v); }
    static __device__ __forceinline__ T from_f(float v) { return __float2half_rn(v); }
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
    } else {
        constexpr int kPieces = V * static_cast<int>(sizeof(typename E::T)) / 16;
        uint4 raw[kPieces];
        typename E::T* e = reinterpret_cast<typename E::T*>(raw);
#pragma unroll
        for (int j = 0; j < V; ++j) e[j] = E::from_f(f[j]);
#pragma unroll
        for (int j = 0; j < kPieces; ++j) reinterpret_cast<uint4*>(p)[j] = raw[j];
    }
}

// Sum (or maximum of bit patterns) over the threads of the CTA, one barrier: the slots alternate between two halves, and
// a half is written again only after the barrier of the call in between.
struct RowReduce {
    float* slots;      // [2][kMaxWarps]
    int flip;
    __device__ __forceinline__ float sum(float v) {
#pragma unroll
        for (int d = 16; d; d >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, d);
        const int warps = blockDim.x >> 5;
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
        const int warps = blockDim.x >> 5;
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
template <int V, int VPT>
__device__ __forceinline__ void normalise(float (&v)[VPT][V], int kind, float eps, int K, int nvec, RowReduce& red) {
    if (kind == I8F_NORM_NONE) return;
    const float inv_k = 1.0f / static_cast<float>(K);
    const int t = threadIdx.x, T = blockDim.x;
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
    const float r = 1.0f / sqrtf(red.sum(s) * inv_k + eps);
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) v[i][j] *= r;
}

template <int XDT, int YDT, int V, int VPT, bool QUANT>
__global__ void __launch_bounds__(512)
gated_residual_norm_kernel(const NormArgs a) {
    __shared__ float s_slots[2 * kMaxWarps];
    RowReduce red{s_slots, 0};
    const int t = threadIdx.x, T = blockDim.x;
    const int nvec = a.K / V;
    const int64_t row = blockIdx.x;
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
    normalise<V, VPT>(y, a.post_norm, a.eps, a.K, nvec, red);
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
    normalise<V, VPT>(x, a.norm, a.eps, a.K, nvec, red);
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
                if constexpr (QUANT) big = max(big, __float_as_uint(x[i][j]) & 0x7FFFFFFFu);
            }
            if (!QUANT || a.h != nullptr) store_v<YDT, V>(a.h, row * a.ldh + static_cast<int64_t>(vec) * V, x[i]);
        }
    }
    if constexpr (QUANT) {
        const float step = red.max_abs(big) / 127.0f;
        const float sc = step < kScaleFloor ? kScaleFloor : step;      // a NaN stays: the row is marked by its scale
        const float inv = 1.0f / sc;
        if (t == 0) a.row_scale[row] = sc;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
            const int vec = i * T + t;
            if (vec < nvec) {
                uint32_t b[V];
#pragma unroll
                for (int j = 0; j < V; ++j)
                    b[j] = static_cast<uint32_t>(__float2int_rn(fminf(fmaxf(x[i][j] * inv, -128.f), 127.f))) & 0xFFu;
                int8_t* dst = a.q + row * a.ldq + static_cast<int64_t>(vec) * V;
                if constexpr (V == 1) {
                    dst[0] = static_cast<int8_t>(b[0]);
                } else {
                    uint2 o;
                    o.x = b[0] | (b[1] << 8) | (b[2] << 16) | (b[3] << 24);
                    o.y = b[4] | (b[5] << 8) | (b[6] << 16) | (b[7] << 24);
                    *reinterpret_cast<uint2*>(dst) = o;
                }
            }
        }
    }
}

template <int XDT, int YDT, bool QUANT>
int launch_norm(const NormArgs& a, bool vec8, cudaStream_t st) {
    const unsigned grid = static_cast<unsigned>(a.M);
#define I8F_NORM_GO(V, VPT, T) gated_residual_norm_kernel<XDT, YDT, V, VPT, QUANT><<<grid, T, 0, st>>>(a)
    if (vec8) {
        const int nvec = a.K / 8;
        if (nvec <= 512) I8F_NORM_GO(8, 1, (nvec + 31) / 32 * 32);
        else if (nvec <= 1024) I8F_NORM_GO(8, 2, 512);
        else I8F_NORM_GO(8, 4, 512);
    } else {
        if (a.K <= 2048) I8F_NORM_GO(1, 8, (a.K + 255) / 256 * 32);
        else if (a.K <= 8192) I8F_NORM_GO(1, 16, 512);
        else I8F_NORM_GO(1, 32, 512);
    }
#undef I8F_NORM_GO
    return check_launch("gated_residual_norm_kernel");
}

bool vec_ok(const void* p, int64_t ld, int elem) { return p == nullptr || (aligned16(p) && (ld * elem) % 16 == 0); }

}  // namespace
}  // namespace i8f

using namespace i8f;

extern "C" int i8f_gated_residual_norm(const void* x, int x_dtype, int64_t ldx, const void* y, int y_dtype, int64_t ldy,
                                       int64_t M, int64_t K, const int32_t* row_request, const void* gate, int64_t ldg,
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
    NormArgs a{};
    a.x = x;
    a.y = y;
    a.gate = gate;
    a.scale = scale;
    a.shift = shift;
    a.post_weight = post_norm == I8F_NORM_NONE ? nullptr : post_weight;
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
    if (y_dtype == I8F_BF16) {
        if (q != nullptr) return f32 ? launch_norm<I8F_F32, I8F_BF16, true>(a, vec8, st) : launch_norm<I8F_BF16, I8F_BF16, true>(a, vec8, st);
        return f32 ? launch_norm<I8F_F32, I8F_BF16, false>(a, vec8, st) : launch_norm<I8F_BF16, I8F_BF16, false>(a, vec8, st);
    }
    if (q != nullptr) return f32 ? launch_norm<I8F_F32, I8F_F16, true>(a, vec8, st) : launch_norm<I8F_F16, I8F_F16, true>(a, vec8, st);
    return f32 ? launch_norm<I8F_F32, I8F_F16, false>(a, vec8, st) : launch_norm<I8F_F16, I8F_F16, false>(a, vec8, st);
}
