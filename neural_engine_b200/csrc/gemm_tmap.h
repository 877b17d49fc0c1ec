// gemm_tmap.h -- tensor maps of the tcgen05 GEMM's operands and outputs
// (gemm.cu), for the translation units that launch its kernel themselves.
#pragma once
#include <cuda.h>

namespace ne {

// 2-D K-major operand [rows, K] (leading dim ld elements), 128B-swizzled box
// of 64 x box_rows.
bool make_tmap(CUtensorMap* tm, const void* ptr, int rows, int K, long long ld, int box_rows,
               int fp16);
// 2-D MN-major operand: global [K rows, MN] (MN contiguous, leading dim ld),
// boxes of 64 (MN) x 64 (K rows), 128B-swizzled.
bool make_tmap_mn(CUtensorMap* tm, const void* ptr, int mn, int K, long long ld);
// Output of a staged epilogue: [rows, cols] row-major with leading dim ld
// elements, boxes of box_cols x 32 rows whose 32-, 64- or 128-byte rows use
// the matching swizzle (the kernel writes the box in that layout).
bool make_tmap_out(CUtensorMap* tm, void* ptr, int rows, int cols, long long ld,
                   CUtensorMapDataType dt, int elem_bytes, int box_cols);

}  // namespace ne
