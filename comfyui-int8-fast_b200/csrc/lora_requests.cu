// Low-rank adapters of many requests beside one shared int8 projection: row m of the batch belongs to a request whose
// adapter is a(m) (or to none), and
//
//   t[m]  = round(x[m] . A_a(m)^T)                   A_a [r, K], one slice of a bank [n, r, K]
//   y[m]  = base[m] + t[m] . B_a(m)^T                B_a [N, r], one slice of a bank [n, N, r]
//
// t is rounded to the 16-bit type of x (as in the single-adapter path, whose second product takes 16-bit operands); all
// sums are fp32.
//
// The rows arrive as CHUNKS of at most four consecutive rows with one adapter, so that a chunk reads its adapter's factors
// once for all of its rows.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "host_common.h"

namespace i8f {
namespace {

constexpr int kChunkRows = 4;

template <int DT>
__device__ __forceinline__ void unpack8(const uint4& r, float (&v)[8]) {
    const uint32_t w[4] = {r.x, r.y, r.z, r.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (DT == I8F_BF16) {
            v[2 * i] = __uint_as_float(w[i] << 16);
            v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
        } else {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
            v[2 * i] = f.x;
            v[2 * i + 1] = f.y;
        }
    }
}
template <int DT>
__device__ __forceinline__ void store_dt(void* out, int64_t idx, float v) {
    if constexpr (DT == I8F_BF16) static_cast<__nv_bfloat16*>(out)[idx] = __float2bfloat16_rn(v);
    else static_cast<__half*>(out)[idx] = __float2half_rn(v);
}

// One warp per (chunk, rank row): the dot products of the chunk's rows with one row of its adapter's A.  Bound by the
// bytes of A; x comes from L2.  A chunk without an adapter gets zeros.
template <int DT>
__global__ void __launch_bounds__(128)
down_chunks_kernel(const void* __restrict__ x, int64_t ldx, const void* __restrict__ bank_a, int64_t K, int64_t r,
                   const int4* __restrict__ chunks, void* __restrict__ t, int64_t ldt) {
    const int lane = threadIdx.x & 31;
    const int4 c = chunks[blockIdx.x];      // first row, rows, adapter
    const int64_t j = static_cast<int64_t>(blockIdx.y) * 4 + (threadIdx.x >> 5);
    if (j >= r) return;
    float acc[kChunkRows] = {0.f, 0.f, 0.f, 0.f};
    if (c.z >= 0) {
        const uint4* a = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(bank_a) + (c.z * r + j) * K);
        const uint16_t* x0 = static_cast<const uint16_t*>(x) + c.x * ldx;
        const int64_t nvec = K >> 3;
#pragma unroll 4
        for (int64_t v = lane; v < nvec; v += 32) {
            float fa[8];
            unpack8<DT>(__ldg(a + v), fa);
#pragma unroll
            for (int m = 0; m < kChunkRows; ++m) {
                if (m < c.y) {
                    float fx[8];
                    unpack8<DT>(__ldg(reinterpret_cast<const uint4*>(x0 + m * ldx) + v), fx);
#pragma unroll
                    for (int e = 0; e < 8; ++e) acc[m] = fmaf(fx[e], fa[e], acc[m]);
                }
            }
        }
    }
#pragma unroll
    for (int m = 0; m < kChunkRows; ++m) {
#pragma unroll
        for (int d = 16; d; d >>= 1) acc[m] += __shfl_xor_sync(0xFFFFFFFFu, acc[m], d);
        if (lane == 0 && m < c.y) store_dt<DT>(t, (static_cast<int64_t>(c.x) + m) * ldt + j, acc[m]);
    }
}

// One thread per (chunk, output column): the chunk's rows of t against one row of its adapter's B, into the fp32 addend of
// the int8 product's epilogue.  Bound by the bytes of B.  Rows without an adapter are not written.
template <int DT>
__global__ void __launch_bounds__(128)
up_chunks_kernel(const void* __restrict__ t, int64_t ldt, const void* __restrict__ bank_b, int64_t N, int64_t r,
                 const int4* __restrict__ chunks, float* __restrict__ addend, int64_t ld_addend) {
    const int4 c = chunks[blockIdx.x];
    const int64_t n = static_cast<int64_t>(blockIdx.y) * 128 + threadIdx.x;
    if (c.z < 0 || n >= N) return;
    const uint4* b = reinterpret_cast<const uint4*>(static_cast<const uint16_t*>(bank_b) + (c.z * N + n) * r);
    const uint16_t* t0 = static_cast<const uint16_t*>(t) + c.x * ldt;
    float acc[kChunkRows] = {0.f, 0.f, 0.f, 0.f};
    const int nvec = static_cast<int>(r >> 3);
    for (int v = 0; v < nvec; ++v) {
        float fb[8];
        unpack8<DT>(__ldg(b + v), fb);
#pragma unroll
        for (int m = 0; m < kChunkRows; ++m) {
            if (m < c.y) {
                float ft[8];
                unpack8<DT>(__ldg(reinterpret_cast<const uint4*>(t0 + m * ldt) + v), ft);
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[m] = fmaf(ft[e], fb[e], acc[m]);
            }
        }
    }
#pragma unroll
    for (int m = 0; m < kChunkRows; ++m)
        if (m < c.y) addend[(static_cast<int64_t>(c.x) + m) * ld_addend + n] = acc[m];
}

int check_rows(const i8f_request_rows* rows, int64_t M) {
    I8F_REQUIRE(rows != nullptr, I8F_ERR_INVALID_ARG, "rows is NULL");
    I8F_REQUIRE(rows->rows == M, I8F_ERR_INVALID_ARG, "the row plan is for %lld rows, the call has %lld", (long long)rows->rows, (long long)M);
    I8F_REQUIRE(M == 0 || (rows->row_adapter != nullptr && rows->chunks != nullptr && rows->n_chunks > 0), I8F_ERR_INVALID_ARG,
                "incomplete row plan");
    return I8F_OK;
}

int check_bank(const void* bank, int64_t adapters, int64_t r, const i8f_request_rows* rows, int dtype, const char* what) {
    I8F_REQUIRE(dtype == I8F_BF16 || dtype == I8F_F16, I8F_ERR_UNSUPPORTED, "%s: dtype must be bf16 or f16", what);
    I8F_REQUIRE(bank != nullptr && adapters > rows->max_adapter, I8F_ERR_INVALID_ARG, "%s: the rows name adapter %d, the bank has %lld", what,
                rows->max_adapter, (long long)adapters);
    I8F_REQUIRE(r > 0 && r % 8 == 0 && r <= 1024, I8F_ERR_UNSUPPORTED, "%s: the rank %lld must be a multiple of 8, at most 1024", what,
                (long long)r);
    I8F_REQUIRE(aligned16(bank), I8F_ERR_ALIGNMENT, "%s: the bank must be 16-byte aligned", what);
    return I8F_OK;
}

int64_t addend_pitch(int64_t N) { return (N + 31) / 32 * 32; }

}  // namespace
}  // namespace i8f

using namespace i8f;

extern "C" {

int i8f_lora_down_requests(const void* x, int64_t ldx, const void* bank_a, int64_t adapters, int64_t r, const i8f_request_rows* rows,
                           void* t, int64_t ldt, int dtype, int64_t M, int64_t K, void* stream) {
    int rc = check_rows(rows, M);
    if (rc != I8F_OK) return rc;
    if (M == 0) return I8F_OK;
    rc = check_bank(bank_a, adapters, r, rows, dtype, "i8f_lora_down_requests");
    if (rc != I8F_OK) return rc;
    I8F_REQUIRE(x != nullptr && t != nullptr && ldx >= K && ldt >= r && K > 0, I8F_ERR_INVALID_ARG, "bad x or t");
    I8F_REQUIRE(aligned16(x) && aligned16(t) && K % 8 == 0 && ldx % 8 == 0 && ldt % 8 == 0, I8F_ERR_ALIGNMENT,
                "x and t must be 16-byte aligned, K and both pitches multiples of 8 elements");
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const dim3 grid(static_cast<unsigned>(rows->n_chunks), static_cast<unsigned>((r + 3) / 4));
    const int4* chunks = reinterpret_cast<const int4*>(rows->chunks);
    if (dtype == I8F_BF16) down_chunks_kernel<I8F_BF16><<<grid, 128, 0, st>>>(x, ldx, bank_a, K, r, chunks, t, ldt);
    else down_chunks_kernel<I8F_F16><<<grid, 128, 0, st>>>(x, ldx, bank_a, K, r, chunks, t, ldt);
    return check_launch("down_chunks_kernel");
}

size_t i8f_lora_requests_workspace_bytes(const i8f_request_rows* rows, int64_t N) {
    if (rows == nullptr || rows->rows <= 0 || N <= 0) return 0;
    return static_cast<size_t>(rows->rows) * static_cast<size_t>(addend_pitch(N)) * sizeof(float);
}

static int up_chunks(const void* t, int64_t ldt, const void* bank_b, int64_t adapters, int64_t r, const i8f_request_rows* rows, int dtype,
                     int64_t M, int64_t N, void* workspace, size_t workspace_bytes, cudaStream_t st) {
    int rc = check_bank(bank_b, adapters, r, rows, dtype, "bank_b");
    if (rc != I8F_OK) return rc;
    I8F_REQUIRE(t != nullptr && ldt >= r, I8F_ERR_INVALID_ARG, "bad t");
    I8F_REQUIRE(aligned16(t) && ldt % 8 == 0, I8F_ERR_ALIGNMENT, "t must be 16-byte aligned, its pitch a multiple of 8 elements");
    const size_t need = i8f_lora_requests_workspace_bytes(rows, N);
    I8F_REQUIRE(workspace != nullptr && workspace_bytes >= need, I8F_ERR_WORKSPACE, "workspace too small: have %zu bytes, need %zu",
                workspace_bytes, need);
    I8F_REQUIRE(aligned16(workspace), I8F_ERR_ALIGNMENT, "workspace must be 16-byte aligned");
    const int64_t tiles_n = (N + 127) / 128;
    I8F_REQUIRE(tiles_n <= 65535, I8F_ERR_UNSUPPORTED, "N=%lld is too large", (long long)N);
    const dim3 grid(static_cast<unsigned>(rows->n_chunks), static_cast<unsigned>(tiles_n));
    const int4* chunks = reinterpret_cast<const int4*>(rows->chunks);
    float* addend = static_cast<float*>(workspace);
    if (dtype == I8F_BF16) up_chunks_kernel<I8F_BF16><<<grid, 128, 0, st>>>(t, ldt, bank_b, N, r, chunks, addend, addend_pitch(N));
    else up_chunks_kernel<I8F_F16><<<grid, 128, 0, st>>>(t, ldt, bank_b, N, r, chunks, addend, addend_pitch(N));
    return check_launch("up_chunks_kernel");
}

int i8f_linear_w8a8_lora_requests(const int8_t* a, int64_t lda, const float* a_scale, const int8_t* w, int64_t ldw, const float* w_scale,
                                  int w_scale_mode, const void* bias, int bias_dtype, const void* t, int64_t ldt, const void* bank_b,
                                  int64_t adapters, int64_t r, const i8f_request_rows* rows, void* out, int out_dtype, int64_t ldo,
                                  int64_t M, int64_t N, int64_t K, int epilogue_order, void* workspace, size_t workspace_bytes,
                                  void* stream) {
    int rc = check_rows(rows, M);
    if (rc != I8F_OK) return rc;
    if (M == 0 || N == 0) return I8F_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    for (const bool check_only : {true, false}) {     // everything is checked before anything is launched
        if (!check_only) {
            rc = up_chunks(t, ldt, bank_b, adapters, r, rows, out_dtype, M, N, workspace, workspace_bytes, st);
            if (rc != I8F_OK) return rc;
        }
        rc = linear_w8a8_addend(a, lda, a_scale, w, ldw, w_scale, w_scale_mode, bias, bias_dtype, out, out_dtype, ldo, M, N, K,
                                epilogue_order, static_cast<const float*>(workspace), addend_pitch(N), rows->row_adapter, check_only, st);
        if (rc != I8F_OK) return rc;
    }
    return I8F_OK;
}

size_t i8f_linear_w8a16_small_lora_requests_workspace_bytes(const i8f_request_rows* rows, int64_t N, int64_t r) {
    if (rows == nullptr || rows->rows <= 0 || N <= 0 || r <= 0) return 0;
    return ((static_cast<size_t>(rows->rows) * static_cast<size_t>(r) * 2 + 255) & ~size_t(255)) + i8f_lora_requests_workspace_bytes(rows, N);
}

int i8f_linear_w8a16_small_lora_requests(const void* x, int x_dtype, int64_t ldx, const int8_t* w, int64_t ldw, const float* w_scale,
                                         int w_scale_mode, const void* bias, int bias_dtype, const void* bank_a, const void* bank_b,
                                         int64_t adapters, int64_t r, const i8f_request_rows* rows, void* out, int64_t ldo, int64_t M,
                                         int64_t N, int64_t K, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_rows(rows, M);
    if (rc != I8F_OK) return rc;
    if (M == 0 || N == 0) return I8F_OK;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    rc = linear_small_addend(x, x_dtype, ldx, w, ldw, w_scale, w_scale_mode, bias, bias_dtype, out, ldo, M, N, K, nullptr, 0, nullptr, true,
                             st);
    if (rc != I8F_OK) return rc;
    rc = check_bank(bank_b, adapters, r, rows, x_dtype, "bank_b");
    if (rc != I8F_OK) return rc;
    const size_t need = i8f_linear_w8a16_small_lora_requests_workspace_bytes(rows, N, r);
    I8F_REQUIRE(workspace != nullptr && workspace_bytes >= need, I8F_ERR_WORKSPACE, "workspace too small: have %zu bytes, need %zu",
                workspace_bytes, need);
    const size_t t_bytes = need - i8f_lora_requests_workspace_bytes(rows, N);
    rc = i8f_lora_down_requests(x, ldx, bank_a, adapters, r, rows, workspace, r, x_dtype, M, K, stream);
    if (rc != I8F_OK) return rc;
    uint8_t* rest = static_cast<uint8_t*>(workspace) + t_bytes;
    rc = up_chunks(workspace, r, bank_b, adapters, r, rows, x_dtype, M, N, rest, workspace_bytes - t_bytes, st);
    if (rc != I8F_OK) return rc;
    return linear_small_addend(x, x_dtype, ldx, w, ldw, w_scale, w_scale_mode, bias, bias_dtype, out, ldo, M, N, K,
                               reinterpret_cast<const float*>(rest), addend_pitch(N), rows->row_adapter, false, st);
}

}  // extern "C"
