// Launchers of the gated layer h = silu(a @ gate^T) * (a @ up^T) and of the elementwise part of its backward pass.
#pragma once

#include <hip/hip_runtime.h>

#include "../../include/beam_hip.h"
#include "gemm_kernel.h"
#include "gemm_kwave.h"
#include "kernel_set.h"

namespace beam {

// A workgroup tile of the gated kernel: block_n rows of B, half of them gate and half up rows, so block_n / 2 columns of C.
// (kGatedKwave, kGatedKwaveLines: the tile of that size of gemm_kwave.h, straight fills or whole lines.)
enum GatedDepth : int { kGatedShallow = 0, kGatedWalk = 1, kGatedDeep = 2, kGatedLines = 3, kGatedKwave = 4, kGatedKwaveLines = 5 };
struct GatedTile {
  int block_m, block_n, depth;
};
// (workgroup tile M, N, wavefronts M, N, depth, LDS slots of A, of B, K groups); wavefront tiles are at least 64 wide, since half
// of that is what a store instruction writes of a row
#define BEAM_FOR_EACH_GATED_TILE(X)              \
  X(256, 256, 2, 4, kGatedShallow, 3, 2, 1)      \
  X(224, 256, 2, 4, kGatedShallow, 3, 2, 1)      \
  X(192, 256, 2, 4, kGatedShallow, 3, 2, 1)      \
  X(256, 128, 4, 2, kGatedShallow, 3, 2, 1)      \
  X(128, 128, 2, 2, kGatedShallow, 3, 2, 1)      \
  X(128, 128, 2, 2, kGatedDeep, 5, 4, 1)         \
  X(64, 128, 2, 2, kGatedShallow, 3, 2, 1)       \
  X(64, 128, 2, 2, kGatedDeep, 3, 3, 2)
// ... whose fills take whole 128-byte lines, 2 x 2 wavefronts a group: (workgroup tile M, N, LDS slots, K groups, Form)
#define BEAM_FOR_EACH_GATED_LINES_TILE(X)  \
  X(64, 128, 6, 2, kFormLineHalves)        \
  X(96, 128, 5, 2, kFormLineHalves)        \
  X(160, 128, 4, 1, kFormLines)            \
  X(192, 128, 4, 2, kFormLineHalves)
// Tiles of gemm_kwave.h: (rows, rows of B, wavefronts)
#define BEAM_FOR_EACH_GATED_KWAVE(X) \
  X(8, 32, 4)                        \
  X(16, 32, 4)                       \
  X(32, 32, 4)                       \
  X(16, 64, 4)                       \
  X(32, 64, 4)                       \
  X(64, 32, 4)                       \
  X(64, 64, 4)

// kGatedWalk: the kernel of gemm_w4.h, 256 x 256 tiles that a workgroup on each CU walks.  K % 64 == 0, K >= kW4MinK, N % 8 == 0, C and
// gu on 16 bytes, (N + 128) * K * 2 below 2^31, N at most 2^20.
hipError_t launch_gated_w4(const GemmParams& p, int dtype, dim3 grid, hipStream_t stream);
template <typename T>
hipError_t launch_gated(const GatedTile& tile, const GemmParams& p, dim3 grid, hipStream_t stream);
template <> hipError_t launch_gated<_Float16>(const GatedTile&, const GemmParams&, dim3, hipStream_t);
template <> hipError_t launch_gated<__bf16>(const GatedTile&, const GemmParams&, dim3, hipStream_t);
template <typename T>
hipError_t launch_gated_kwave(const KwPlan& plan, const KwGatedParams& p, hipStream_t stream);
template <> hipError_t launch_gated_kwave<_Float16>(const KwPlan&, const KwGatedParams&, hipStream_t);
template <> hipError_t launch_gated_kwave<__bf16>(const KwPlan&, const KwGatedParams&, hipStream_t);

// p.ws [splits][M][N] fp32: the sums of K slices of A . B with B as [K][N], in tiles of block_m x 128, block_m 64 or 128.
hipError_t launch_partial_kmajor(int block_m, const GemmParams& p, int dtype, hipStream_t stream);

// Any sizes, element by element (what the tiled kernels refuse: K below 8 or beyond a descriptor).
hipError_t launch_gated_plain(const void* A, const void* B, void* H, void* GU, int M, int N, int K, int dtype, hipStream_t stream);

// D [M][cols_d] and DT [2 N][cols_dt] (either may be null): the gradients of gate and up factor from dH [M][N] and GU [M][2 N],
// their 2 N and M columns followed by up to 63 zeros.
hipError_t launch_gated_gradients(const void* dH, const void* GU, void* D, void* DT, int M, int N, int cols_d, int cols_dt, int dtype,
                                  hipStream_t stream);

}  // namespace beam
