// Host side of the grouped GEMM's dual tiles (grouped_gemm_dual.hip).
#pragma once

#include "grouped_gemm.hpp"

namespace fluxmi {

// Whether the dual tiles take a launch that is the macro tiles' otherwise.
bool dual_takes(const GemmParams &p, int dtype);
// few: row counts in the arguments (count > 0) and a second factor per row, as the forms for few rows take them.
int launch_grouped_gemm_dual(const GemmParams &p, const FewRowsArgs &few, int dtype, int grid, hipStream_t s);
// Scale bytes from row to row for kb blocks: rows that are not whole words are wanted as a copy with whole 16 bytes.
inline __host__ __device__ int mx_scale_row(int kb) { return kb % 4 == 0 ? kb : (kb + 15) / 16 * 16; }
// MXFP4 operands: a / b[0] packed codes of k values, a multiple of 32, a_scale / b_scale their scale bytes, mx_scale_row(k / 32) for each row; a_rows is given with and
// without gather_a; half_is_f16: 16-bit results are fp16; without splits all max_rows rows are one expert's.
bool dual_takes_mx(const GemmParams &p);
int launch_grouped_gemm_dual_mx(const GemmParams &p, int grid, hipStream_t s);

}  // namespace fluxmi
