// Host helpers of the TMA kernels (defined in gemm_sm100.cu): tensor maps over row-major matrices.
#pragma once

#include <cuda.h>

namespace pan {
namespace gemm {

// 3-D map over `batch` row-major [rows, cols] matrices (row stride `ld` elements), box [1, box_rows, box_cols].
// Returns an error string, nullptr on success.
const char* make_map(CUtensorMap* m, const void* base, long long rows, long long cols, long long ld, int box_rows,
                     int box_cols, int batch, long long bstride, CUtensorMapDataType dtype, int esize,
                     CUtensorMapSwizzle swz);
// Output map clipped at `row_end` rows and `n` columns, 32 x 32 boxes.
const char* make_out_map(CUtensorMap* m, const void* base, int row_end, int n, long long ld, bool fp32, int batch,
                         long long bstride);
int num_sms();

}  // namespace gemm
}  // namespace pan
