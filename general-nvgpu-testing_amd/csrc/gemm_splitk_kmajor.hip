// Partial sums of K slices with B stored [K][N], fp16 and bf16: the products of a gated layer's backward pass.
#include "gated.h"
#include "kernel_set.h"

namespace beam {

hipError_t launch_partial_kmajor(int block_m, const GemmParams& p, int dtype, hipStream_t stream) {
  const dim3 grid((unsigned)((size_t)p.tiles_m * p.tiles_n * p.splits));
  const bool bf16 = dtype == BEAM_BF16;
  if (block_m == 128)
    return bf16 ? launch_gemm<__bf16, 128, 128, 2, 4, kEpiPartial, 5, 4, true>(p, grid, stream) : launch_gemm<_Float16, 128, 128, 2, 4, kEpiPartial, 5, 4, true>(p, grid, stream);
  if (block_m == 64)
    return bf16 ? launch_gemm<__bf16, 64, 128, 2, 2, kEpiPartial, 3, 3, true, 2>(p, grid, stream) : launch_gemm<_Float16, 64, 128, 2, 2, kEpiPartial, 3, 3, true, 2>(p, grid, stream);
  return hipErrorInvalidValue;
}

}  // namespace beam
