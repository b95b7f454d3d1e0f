// Tensor maps of K-major operands, shared by the kernels that stage them by TMA (defined in gemm_tcgen05.cu, which keeps a
// small cache of encoded maps), and the current device with its SM count (asked for once).
#pragma once
#include <cstdint>
#include <cuda.h>

namespace i8f {

enum Kind : int { kKindI8 = 0, kKindBF16 = 1, kKindF16 = 2 };

int current_device();
int sm_count();

// [rows, k_elems] with a pitch of ld_elems, box = one 128-byte span of K x box_rows (at most 256), 128-byte swizzle.
int make_operand_map(CUtensorMap* tm, int kind, const void* base, int64_t rows, int64_t k_elems, int64_t ld_elems, int box_rows);

}  // namespace i8f
