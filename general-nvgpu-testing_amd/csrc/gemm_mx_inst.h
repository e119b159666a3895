// Instances of the kernels of gemm_mx.h for one output type (BEAM_T).  Included by gemm_mx_{fp16,bf16}.hip.
#include "gemm_mx.h"
#include "kernel_set.h"

namespace beam {

namespace {

template <int BM, int BN, int WVM, int WVN, int ST>
hipError_t launch_mx_tile(const MxParams& p, hipStream_t stream) {
  using Tile = MxGemm<BEAM_T, BM, BN, WVM, WVN, ST>;
  auto kern = gemm_mx_kernel<BEAM_T, BM, BN, WVM, WVN, ST>;
  static std::atomic<unsigned long long> configured{0};
  if (hipError_t e = allow_lds_once(configured, reinterpret_cast<const void*>(kern), Tile::LDS_BYTES); e != hipSuccess) return e;
  hipLaunchKernelGGL(kern, dim3((unsigned)(p.tiles_m * p.tiles_n)), dim3(Tile::NT), Tile::LDS_BYTES, stream, p);
  return hipGetLastError();
}

template <int MB, int CB, int NW, bool A16>
hipError_t launch_mx_kw(const MxParams& p, hipStream_t stream) {
  using Tile = MxKw<BEAM_T, MB, CB, NW, 2, A16>;
  auto kern = gemm_mx_kwave_kernel<BEAM_T, MB, CB, NW, 2, A16>;
  static std::atomic<unsigned long long> configured{0};
  constexpr int kMost = A16 ? Tile::LDS_BYTES + kMxKeptColumns / kMxTile * Tile::KEPT : Tile::LDS_BYTES;
  static_assert(kMost <= 160 * 1024, "LDS of a CU");
  if (hipError_t e = allow_lds_once(configured, reinterpret_cast<const void*>(kern), kMost); e != hipSuccess) return e;
  const int kept = A16 ? (p.K + kMxTile - 1) / kMxTile * Tile::KEPT : 0;
  const int lds = Tile::RINGS + kept > Tile::LDS_BYTES ? Tile::RINGS + kept : Tile::LDS_BYTES;
  hipLaunchKernelGGL(kern, dim3((unsigned)(p.tiles_m * p.tiles_n)), dim3(NW * 64), lds, stream, p);
  return hipGetLastError();
}

}  // namespace

template <>
hipError_t launch_gemm_mx<BEAM_T>(int block_m, int block_n, int kind, const MxParams& p, hipStream_t stream) {
#define BEAM_MX(BM, BN, KIND, WVM, WVN, ST) \
  if (block_m == BM && block_n == BN && kind == KIND) return launch_mx_tile<BM, BN, WVM, WVN, ST>(p, stream);
  BEAM_FOR_EACH_MX_TILE(BEAM_MX)
#undef BEAM_MX
  return hipErrorInvalidValue;
}

template <>
hipError_t launch_gemm_mx_kwave<BEAM_T>(int rows, int cols, bool a16, const MxParams& p, hipStream_t stream) {
#define BEAM_MX(ROWS, COLS, NW)                                                   \
  if (rows == ROWS && cols == COLS) {                                             \
    if (!a16) return launch_mx_kw<ROWS / 16, COLS / 16, NW, false>(p, stream);    \
    if constexpr (ROWS == 16) return launch_mx_kw<ROWS / 16, COLS / 16, NW, true>(p, stream); \
  }
  BEAM_FOR_EACH_MX_KWAVE(BEAM_MX)
#undef BEAM_MX
  return hipErrorInvalidValue;
}

}  // namespace beam
