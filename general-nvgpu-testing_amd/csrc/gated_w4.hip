// The 256x256 tile of four 128x128 wavefronts (gemm_w4.h) for the gated layer, fp16 and bf16.
#include "gated.h"
#include "gemm_w4.h"

namespace beam {

template <typename T, int STORE>
static hipError_t launch_gated_w4_t(const GemmParams& p, dim3 grid, hipStream_t stream) {
  using Tile = GemmW4<T, STORE, false, 4, 8, 2, false, false, true>;
  auto kern = gemm_gated_w4_kernel<T, STORE>;
  static std::atomic<unsigned long long> configured{0};
  if (hipError_t e = allow_lds_once(configured, reinterpret_cast<const void*>(kern), Tile::LDS_BYTES); e != hipSuccess) return e;
  hipLaunchKernelGGL(kern, grid, dim3(Tile::NT), Tile::LDS_BYTES, stream, p);
  return hipGetLastError();
}

template <typename T>
static hipError_t launch_gated_w4_kind(const GemmParams& p, dim3 grid, hipStream_t stream) {
  // (Non-temporal stores, which pay in a plain product's largest outputs, do not here: 4096 x 11008 x 4096 with GU, 270 MB, 558 -> 614 us.)
  return p.c_store == kStoreThrough ? launch_gated_w4_t<T, kStoreThrough>(p, grid, stream) : launch_gated_w4_t<T, kStoreCached>(p, grid, stream);
}

hipError_t launch_gated_w4(const GemmParams& p, int dtype, dim3 grid, hipStream_t stream) {
  return dtype == BEAM_BF16 ? launch_gated_w4_kind<__bf16>(p, grid, stream) : launch_gated_w4_kind<_Float16>(p, grid, stream);
}

}  // namespace beam
