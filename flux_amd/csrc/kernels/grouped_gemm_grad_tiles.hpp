// Gradients of the grouped product by tiles of 256 x 256 (grouped_gemm_grad_tiles.hip).
#pragma once
#include "grouped_gemm_grad.hpp"

namespace fluxmi {

// Whether the tiles take a call: operands on 16 bytes, n and k multiples of 8 (codes: k of 16), offsets within a tile's operands below 2^32.
bool grad_tiles_take(Grad g, const GradArgs &a);
// Whether they are the faster form of a call that they take.
bool grad_tiles_are_faster(Grad g, int32_t nexperts, int64_t rows, int64_t n, int64_t k);
// For the sums of tiles that are cut into parts.
size_t grad_tiles_workspace_bytes(Grad g, int32_t nexperts, int64_t rows, int64_t n, int64_t k);
int launch_grad_tiles(Grad g, bool f16, const GradArgs &a, void *stream);

}  // namespace fluxmi
