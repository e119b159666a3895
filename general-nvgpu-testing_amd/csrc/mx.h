// MXFP4 (OCP microscaling, e2m1 elements with an e8m0 scale for every 32 of them) on gfx950: what its kernels share.
//
// A matrix of R rows and K columns (K a multiple of 32) is held as
//   elements  [R][K / 2] bytes, two to a byte, the even column in the low half;
//   scales    [ceil(K / 256)][R][8] bytes: that of row r, block b (columns 32 b .. + 31) is scales[b / 8][r][b % 8], and the bytes
//             behind the last block are not looked at (the quantiser writes zeros).
// 256 columns of a row are 128 bytes, the K tile that every kernel of this library walks; the scales that go with it are 8 bytes a
// row, and those of neighbouring rows lie side by side: the 16 rows of a matrix-core block take theirs from one 128-byte line.
// (With scales as [R][K / 32] they would come from 16 lines, as many as the block's elements.)
//
// v_mfma_scale_f32_16x16x128_f8f6f4: lane l supplies 32 elements (16 bytes) of row l & 15 and their scale, for K positions
// 32 (l >> 4) .. + 31 of the 128.  Which 32 columns those are is free as long as A and B agree: here lane group g = l >> 4 takes
// chunk 2 g + step of the K tile's 8 in its two steps, so that the scales of both are two neighbouring bytes, one 16-bit load;
// the bytes of two blocks share a register, and the instruction picks its byte by a constant.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/beam_hip.h"

#include "gemm_kernel.h"
#include "tile_map.h"

namespace beam {

typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr int kMxTile = 256;  // columns of a K tile
constexpr int kMxBlocks = 8;  // scales of a row in it

struct MxParams {
  const void* A;         // elements [M][K / 2]; MxKw with A16: 16-bit [M][K]
  const void* B;         // elements [N][K / 2]
  const uint8_t* sa;     // scales
  const uint8_t* sb;
  void* C;               // 16-bit [M][N]
  int M, N, K;
  int tiles_m, tiles_n, group_m;
  TileDivs divs;
  int c_store;  // StoreKind of the tiled kernel
};

// Where chunk c of a row's 8 lies in LDS before the row's XOR: lane group g reads place 4 step + g, as of 16-bit elements, for
// which that XOR is made (chunks 2 g + step in their own places: a read's groups of lanes meet in the same banks, 8192^3
// 241 us, so 235).  A fill has each lane fetch the chunk that belongs where it writes, from the same line.
BEAM_HD int mx_place_of(int chunk) { return (chunk & 1) << 2 | chunk >> 1; }
BEAM_HD int mx_chunk_at(int place) { return (place & 3) << 1 | place >> 2; }

// For the kernel of gemm_w4.h: elements and K in units of 16 bits (4 columns).
struct MxW4Params : GemmParams {
  const uint8_t* sa;
  const uint8_t* sb;
};

// The scales of four blocks of 16 rows, from 8 bytes a lane (those of row r of block g in lane (r, g)) to two registers of what a
// lane needs of each block, 16 bits (chunks 2 g and 2 g + 1 of row r): blocks 0 and 2 in the first, 1 and 3 in the second.
// Lane group j holds the four 16-bit words 0 .. 3 of its row of block j and needs word g of all four.  v_permlane32_swap makes
// (words 0, 1 of blocks j and j + 2) in groups 0 and 1, (words 2, 3) in groups 2 and 3; their low words, and their high ones, go
// into a register each; v_permlane16_swap changes the high ones of the even groups for the low ones of the odd groups.
__device__ __forceinline__ void mx_turn(i32x2 rows, int* even, int* odd) {
  const auto x = __builtin_amdgcn_permlane32_swap((unsigned)rows[0], (unsigned)rows[1], false, false);
  const unsigned lo = __builtin_amdgcn_perm(x[1], x[0], 0x05040100u), hi = __builtin_amdgcn_perm(x[1], x[0], 0x07060302u);
  const auto y = __builtin_amdgcn_permlane16_swap(lo, hi, false, false);
  *even = (int)y[0];
  *odd = (int)y[1];
}

// acc += a x b for chunk step STEP, operand registers PA, PB of the pairs that share a scale register (0: low half, 1: high).
// The first operand's rows become the columns of C, as everywhere here.
template <int STEP, int PB, int PA>
__device__ __forceinline__ f32x4 mx_mfma(i32x4 b, i32x4 a, f32x4 acc, int scale_b, int scale_a) {
  const i32x8 b8 = {b[0], b[1], b[2], b[3], 0, 0, 0, 0}, a8 = {a[0], a[1], a[2], a[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b8, a8, acc, 4, 4, 2 * PB + STEP, scale_b, 2 * PA + STEP, scale_a);
}

// The scale that a block with largest magnitude `top` gets, biased: that of the power of two at or below it over 4, so that the
// magnitude is below 8 of it; at least 2^-127.  255 (NaN) for a block with an infinity or a NaN in it.  (The bits of an fp32
// value order like its magnitude, and NaNs are above infinity, so `top_bits` is the maximum of the bits without the signs.)
__device__ __forceinline__ int mx_scale_of(unsigned top_bits) {
  const int e = (int)(top_bits >> 23);
  return e == 255 ? 255 : (e > 2 ? e - 2 : 0);
}

// Eight values x / 2^(scale - 127) as elements, value i in bits 4 i .. 4 i + 3: round to nearest, ties to the even code, 6 beyond
// 6 (v_cvt_scalef32_pk_fp4_f32 with a scale of 1; the scaling by a power of two is exact).
__device__ __forceinline__ unsigned mx_encode8(const float (&x)[8], int scale) {
  const int down = 127 - scale;
  unsigned q = 0;
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, __builtin_amdgcn_ldexpf(x[0], down), __builtin_amdgcn_ldexpf(x[1], down), 1.0f, 0);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, __builtin_amdgcn_ldexpf(x[2], down), __builtin_amdgcn_ldexpf(x[3], down), 1.0f, 1);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, __builtin_amdgcn_ldexpf(x[4], down), __builtin_amdgcn_ldexpf(x[5], down), 1.0f, 2);
  q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, __builtin_amdgcn_ldexpf(x[6], down), __builtin_amdgcn_ldexpf(x[7], down), 1.0f, 3);
  return q;
}

// A block of 32 values as 16 bytes of elements, and its biased scale.
template <typename V8>
__device__ __forceinline__ i32x4 mx_encode_block(const V8 (&x)[4], int* scale) {
  float v[4][8];
  unsigned top = 0;
#pragma unroll
  for (int c = 0; c < 4; ++c)
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[c][e] = (float)x[c][e];
      const unsigned bits = __float_as_uint(v[c][e]) & 0x7fffffffu;
      top = bits > top ? bits : top;
    }
  *scale = mx_scale_of(top);
  i32x4 o;
#pragma unroll
  for (int c = 0; c < 4; ++c) o[c] = (int)mx_encode8(v[c], *scale);
  return o;
}

// How an MXFP4 product runs: tiles of MxGemm, one workgroup to a CU or several of them with rings of fewer slots; of MxKw; of gemm_w4.h.
enum MxKind : int { kMxAlone = 0, kMxKwave = 1, kMxWalk = 2, kMxShared = 3 };
// Launchers.  Tiles of MxGemm: (rows, columns, kind, wavefronts along M and N, LDS slots); of MxKw: (rows, columns, wavefronts), those
// of 16 rows also with a16: p.A is 16-bit and K at most kMxKeptColumns.
#define BEAM_FOR_EACH_MX_TILE(X)    \
  X(64, 64, kMxAlone, 2, 2, 4)      \
  X(64, 64, kMxShared, 2, 2, 3)     \
  X(128, 64, kMxShared, 4, 2, 3)    \
  X(128, 128, kMxAlone, 4, 2, 4)    \
  X(128, 128, kMxShared, 4, 2, 2)   \
  X(256, 128, kMxAlone, 4, 2, 3)    \
  X(256, 256, kMxAlone, 2, 4, 2)
#define BEAM_FOR_EACH_MX_KWAVE(X) \
  X(16, 16, 4)                    \
  X(16, 32, 4)                    \
  X(16, 64, 4)                    \
  X(32, 32, 4)                    \
  X(32, 64, 4)                    \
  X(64, 32, 4)
template <typename T>
hipError_t launch_gemm_mx(int block_m, int block_n, int kind, const MxParams& p, hipStream_t stream);
template <> hipError_t launch_gemm_mx<_Float16>(int, int, int, const MxParams&, hipStream_t);
template <> hipError_t launch_gemm_mx<__bf16>(int, int, int, const MxParams&, hipStream_t);
// The kernel of gemm_w4.h (256 x 256 tiles, a workgroup per CU walks them): K % 256 == 0, K >= 768, N % 8 == 0, C on 16 bytes.
hipError_t launch_gemm_mx_w4(const MxW4Params& p, int dtype, dim3 grid, hipStream_t stream);
template <typename T>
hipError_t launch_gemm_mx_kwave(int rows, int cols, bool a16, const MxParams& p, hipStream_t stream);
template <> hipError_t launch_gemm_mx_kwave<_Float16>(int, int, bool, const MxParams&, hipStream_t);
template <> hipError_t launch_gemm_mx_kwave<__bf16>(int, int, bool, const MxParams&, hipStream_t);
hipError_t launch_mx_quantize(const void* X, uint8_t* elements, uint8_t* scales, int M, int K, int dtype, hipStream_t stream);
hipError_t launch_mx_dequantize(const uint8_t* elements, const uint8_t* scales, void* X, int M, int K, int dtype, hipStream_t stream);
// Largest K whose rows of A fit into LDS beside the rings of a 16-row tile with 16-bit A.
constexpr int kMxKeptColumns = 10240;

}  // namespace beam
