// Tensor maps of row-major matrices of 16-bit values (defined in k2_lmhead.cu).
#pragma once
#include <cuda.h>
#include <stdint.h>

namespace tome {

// Tiles of 64 columns (128 bytes, 128-byte swizzle) x box_rows rows of a contiguous matrix
// [n_rows, cols] of 16-bit values.  ptr 16-byte aligned, cols a multiple of 8.
int32_t tensor_map_16bit(CUtensorMap* map, const void* ptr, int64_t n_rows, int64_t cols,
                         int box_rows);

}  // namespace tome
