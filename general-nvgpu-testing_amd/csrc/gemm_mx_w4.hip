// The 256x256 tile of four 128x128 wavefronts (gemm_w4.h) for MXFP4 operands, fp16 and bf16 output.
#include "gemm_w4.h"
#include "kernel_set.h"

namespace beam {

template <typename T, int STORE>
static hipError_t launch_mx_w4_t(const MxW4Params& p, dim3 grid, hipStream_t stream) {
  using Tile = GemmW4<T, STORE, false, 4, 8, 2, false, true>;
  auto kern = gemm_mx_w4_kernel<T, STORE>;
  static std::atomic<unsigned long long> configured{0};
  if (hipError_t e = allow_lds_once(configured, reinterpret_cast<const void*>(kern), Tile::LDS_BYTES); e != hipSuccess) return e;
  hipLaunchKernelGGL(kern, grid, dim3(Tile::NT), Tile::LDS_BYTES, stream, p);
  return hipGetLastError();
}

template <typename T>
static hipError_t launch_mx_w4_kind(const MxW4Params& p, dim3 grid, hipStream_t stream) {
  if (p.c_store == kStoreStreaming) return launch_mx_w4_t<T, kStoreStreaming>(p, grid, stream);
  return p.c_store == kStoreCached ? launch_mx_w4_t<T, kStoreCached>(p, grid, stream) : launch_mx_w4_t<T, kStoreThrough>(p, grid, stream);
}

hipError_t launch_gemm_mx_w4(const MxW4Params& p, int dtype, dim3 grid, hipStream_t stream) {
  return dtype == BEAM_BF16 ? launch_mx_w4_kind<__bf16>(p, grid, stream) : launch_mx_w4_kind<_Float16>(p, grid, stream);
}

}  // namespace beam
