// Host-side helpers shared by the translation units of libi8f: thread-local
// error text, argument checks and the dtype table.
#pragma once
#include <cstdarg>
#include <cstdint>
#include <cstdio>
#include <cuda_runtime.h>

#include "../../include/i8f.h"

namespace i8f {

char* error_buffer();  // thread-local, 512 bytes (defined in api.cu)

inline int fail(int code, const char* fmt, ...) {
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(error_buffer(), 512, fmt, ap);
    va_end(ap);
    return code;
}

inline int dtype_size(int dt) {
    switch (dt) {
        case I8F_BF16: return 2;
        case I8F_F16: return 2;
        case I8F_F32: return 4;
        default: return 0;
    }
}

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

void count_launch();  // one more kernel launched by the library (defined in api.cu)

inline int check_launch(const char* what) {
    cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return fail(I8F_ERR_CUDA, "%s: %s", what, cudaGetErrorString(e));
    count_launch();
    return I8F_OK;
}

int* device_status_word();  // device address of the status word on the current device, or nullptr

// One 256-row tile of a batch of requests: its run of slots, or (addend_row >= 0) its first row in the fp32 addend.
struct RequestTile {
    int slot_begin, n_slots, addend_row, pad;
};
constexpr int kMaxTileSlots = 8;      // a dense tile's adapters whose down projection is the tile's own
// One adapter of a tile and the rows of the tile that use it (bit i of word j: row 32 j + i).  `few`: so few rows that chunks do
// their down projection.
struct RequestSlot {
    int adapter, few, pad[2];
    uint32_t rows[8];
};

// The low-rank term of a batch of requests beside the int8 product.  Where requests_need_addend() says no, the kernel works
// the rows' terms out itself beside the MMAs.  Else `tiles` say where theirs comes from (NULL: all of it is in `addend`
// [M, ld_addend]).  ld_addend is a multiple of 32, the addend 16-byte aligned.
struct RequestTerm {
    const int* row_adapter;
    const float* addend;
    int64_t ld_addend;
    const RequestTile* tiles;
    const RequestSlot* slots;
    const void* t;       // [M, r], pitch ldt, in the output type
    int64_t ldt;
    const void* b;       // [adapters, N, r]
    int64_t adapters, r;
    // the kernel before this one in the stream is the library's own and started when everything before it was complete, so
    // the weights and banks may be read beside its tail
    bool after_own;
};

// Whether the product of these sizes runs on 256-wide tiles, which have no room for rows worked out beside it: the terms of
// chunked rows have to be in the addend then.
bool requests_need_addend(int64_t M, int64_t N, int64_t K);

// i8f_linear_w8a8 with such a term; in gemm_tcgen05.cu.  With `check_only` the arguments are checked and nothing is
// launched, so that a caller can refuse a bad call before it launches what comes first.
int linear_w8a8_requests(const int8_t* a, int64_t lda, const float* a_scale, const int8_t* w, int64_t ldw, const float* w_scale,
                         int w_scale_mode, const void* bias, int bias_dtype, void* out, int out_dtype, int64_t ldo, int64_t M,
                         int64_t N, int64_t K, int epilogue_order, const RequestTerm& term, bool check_only, cudaStream_t stream);
// i8f_linear_w8a16_small with the low-rank term of each row's adapter (row_adapter, t, b, r of `term`); in linear_small_m.cu.
// The kernel before it in the stream may only be the one that writes t.
int linear_small_requests(const void* x, int x_dtype, int64_t ldx, const int8_t* w, int64_t ldw, const float* w_scale, int w_scale_mode,
                          const void* bias, int bias_dtype, void* out, int64_t ldo, int64_t M, int64_t N, int64_t K,
                          const RequestTerm& term, bool check_only, cudaStream_t stream);

}  // namespace i8f

#define I8F_REQUIRE(cond, code, ...)                    \
    do {                                                \
        if (!(cond)) return ::i8f::fail(code, __VA_ARGS__); \
    } while (0)
