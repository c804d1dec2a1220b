// Host-side helpers that the library's translation units share (defined in nb_attn.cu).
#pragma once

#include <cuda.h>
#include <stddef.h>
#include <stdint.h>

namespace nb {

// Binds the thread's context and sets the current device up; `sms` receives its SM count. An nb_attn_error code.
int host_prepare(int* sms);

// Tensor map of a row-major bf16 matrix [rows][cols] with `stride` elements between rows; boxes of box_rows x box_cols,
// swizzled over box_cols * 2 = 64 or 128 bytes. The matrix may be empty of use but not of size. An nb_attn_error code.
int host_matrix_map(CUtensorMap* map, const void* ptr, int64_t rows, int64_t cols, int64_t stride, int box_rows,
                    int box_cols);

}  // namespace nb
