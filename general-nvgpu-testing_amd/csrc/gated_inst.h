// Instances of the gated layer's kernels (gemm_kernel.h: kEpiGated; gemm_kwave.h) for one element type (BEAM_T).  Included by
// gated_{fp16,bf16}.hip.
#include "gated.h"
#include "kernel_set.h"

namespace beam {

namespace {

template <int BM, int BN, int WVM, int WVN, int AST, int BST, int KG, int FORM>
hipError_t launch_gated_t(const GemmParams& p, dim3 grid, hipStream_t stream) {
  using Tile = GemmTile<BEAM_T, BM, BN, WVM, WVN, kEpiGated, AST, BST, false, KG, FORM>;
  auto kern = gemmrc_kernel<BEAM_T, BM, BN, WVM, WVN, kEpiGated, AST, BST, false, KG, FORM>;
  static std::atomic<unsigned long long> configured{0};
  constexpr int LDS = Tile::GROUPS * Tile::LDS_BYTES;
  if (hipError_t e = allow_lds_once(configured, reinterpret_cast<const void*>(kern), LDS); e != hipSuccess) return e;
  hipLaunchKernelGGL(kern, grid, dim3(KG * Tile::NT), LDS, stream, p);
  return hipGetLastError();
}

template <int AG, int CB, int NW, KwRows MODE>
hipError_t launch_gated_kw(const KwGatedParams& p, hipStream_t stream) {
  using Tile = KwTile<BEAM_T, AG, CB, NW, 2, MODE, false, true>;
  auto kern = gemm_kwave_gated_kernel<BEAM_T, AG, CB, NW, 2, MODE>;
  static std::atomic<unsigned long long> configured{0};
  if (hipError_t e = allow_lds_once(configured, reinterpret_cast<const void*>(kern), Tile::LDS_BYTES); e != hipSuccess) return e;
  hipLaunchKernelGGL(kern, dim3((unsigned)(p.tiles_m * p.tiles_n)), dim3(NW * 64), Tile::LDS_BYTES, stream, p);
  return hipGetLastError();
}

}  // namespace

template <>
hipError_t launch_gated<BEAM_T>(const GatedTile& t, const GemmParams& p, dim3 grid, hipStream_t stream) {
#define BEAM_GATED(BM, BN, WVM, WVN, DEPTH, AST, BST, KG)                    \
  if (t.block_m == BM && t.block_n == BN && t.depth == DEPTH)               \
    return launch_gated_t<BM, BN, WVM, WVN, AST, BST, KG, kFormStraight>(p, grid, stream);
  BEAM_FOR_EACH_GATED_TILE(BEAM_GATED)
#undef BEAM_GATED
#define BEAM_GATED(BM, BN, S, KG, FORM)                                     \
  if (t.block_m == BM && t.block_n == BN && t.depth == kGatedLines)         \
    return launch_gated_t<BM, BN, 2, 2, S, S, KG, FORM>(p, grid, stream);
  BEAM_FOR_EACH_GATED_LINES_TILE(BEAM_GATED)
#undef BEAM_GATED
  return hipErrorInvalidValue;
}

template <>
hipError_t launch_gated_kwave<BEAM_T>(const KwPlan& plan, const KwGatedParams& p, hipStream_t stream) {
#define BEAM_GATED(ROWS, COLS, NW)                                                    \
  if (plan.rows == ROWS && plan.cols == COLS && plan.waves == NW) {                   \
    if (!plan.shift) return launch_gated_kw<ROWS / 8, COLS / 16, NW, kKwStraight>(p, stream); \
    if constexpr (ROWS > 8) return launch_gated_kw<ROWS / 8, COLS / 16, NW, kKwShift>(p, stream); \
  }
  BEAM_FOR_EACH_GATED_KWAVE(BEAM_GATED)
#undef BEAM_GATED
  return hipErrorInvalidValue;
}

}  // namespace beam
