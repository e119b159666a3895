// 16-bit values to MXFP4 and back (mx.h).
#include "mx.h"

namespace beam {

namespace {

// A thread takes a block of 32 columns of a row: 64 bytes in, 16 bytes of elements and a byte of scale out, nothing to exchange.
// Bound by memory: 2 M K bytes in, 0.53 M K out.  Neighbouring threads take the 8 blocks of a K tile, then the next row's: a
// wavefront reads 512 bytes of each of 8 rows, writes 128 bytes of elements a row, and its 64 scales lie side by side.
template <typename T>
__global__ void __launch_bounds__(256) mx_quantize_kernel(const T* __restrict__ X, uint8_t* __restrict__ elements, uint8_t* __restrict__ scales,
                                                          int M, int K) {
  typedef T vec8 __attribute__((ext_vector_type(8)));
  typedef vec8 vec8_at_element __attribute__((aligned(2)));
  typedef i32x4 i32x4_at_byte __attribute__((aligned(1)));
  const int kt = blockIdx.y;
  const int b = kt * kMxBlocks + (threadIdx.x & 7);
  for (long m = (long)blockIdx.x * 32 + (threadIdx.x >> 3); m < M; m += (long)gridDim.x * 32) {
    int scale = 0;  // behind the last block
    if (b < K / 32) {
      const T* const at = X + (size_t)m * K + (size_t)b * 32;
      vec8 x[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) x[c] = *(const vec8_at_element*)(at + 8 * c);
      *(i32x4_at_byte*)(elements + (size_t)m * (K / 2) + (size_t)b * 16) = mx_encode_block(x, &scale);
    }
    scales[((size_t)kt * M + m) * kMxBlocks + (threadIdx.x & 7)] = (uint8_t)scale;
  }
}

// The values held, rounded to T (exact in bf16, and in fp16 for what was quantised from fp16); the same share of a thread.
template <typename T>
__global__ void __launch_bounds__(256) mx_dequantize_kernel(const uint8_t* __restrict__ elements, const uint8_t* __restrict__ scales,
                                                            T* __restrict__ X, int M, int K) {
  typedef T vec8 __attribute__((ext_vector_type(8)));
  typedef vec8 vec8_at_element __attribute__((aligned(2)));
  typedef i32x4 i32x4_at_byte __attribute__((aligned(1)));
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const int kt = blockIdx.y;
  const int b = kt * kMxBlocks + (threadIdx.x & 7);
  if (b >= K / 32) return;
  for (long m = (long)blockIdx.x * 32 + (threadIdx.x >> 3); m < M; m += (long)gridDim.x * 32) {
    const i32x4 q = *(const i32x4_at_byte*)(elements + (size_t)m * (K / 2) + (size_t)b * 16);
    const int scale = scales[((size_t)kt * M + m) * kMxBlocks + (threadIdx.x & 7)];
    T* const at = X + (size_t)m * K + (size_t)b * 32;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      vec8 x;
      auto two = [&](f32x2 v, int e) __attribute__((always_inline)) {
        x[e] = (T)(scale == 255 ? __builtin_nanf("") : __builtin_amdgcn_ldexpf(v[0], scale - 127));
        x[e + 1] = (T)(scale == 255 ? __builtin_nanf("") : __builtin_amdgcn_ldexpf(v[1], scale - 127));
      };
      two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4((unsigned)q[c], 1.0f, 0), 0);
      two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4((unsigned)q[c], 1.0f, 1), 2);
      two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4((unsigned)q[c], 1.0f, 2), 4);
      two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4((unsigned)q[c], 1.0f, 3), 6);
      *(vec8_at_element*)(at + 8 * c) = x;
    }
  }
}

dim3 grid_of(int M, int K) { return dim3((unsigned)(((long)M + 31) / 32), (unsigned)((K + kMxTile - 1) / kMxTile)); }

}  // namespace

hipError_t launch_mx_quantize(const void* X, uint8_t* elements, uint8_t* scales, int M, int K, int dtype, hipStream_t stream) {
  if (dtype == BEAM_BF16) hipLaunchKernelGGL(mx_quantize_kernel<__bf16>, grid_of(M, K), dim3(256), 0, stream, (const __bf16*)X, elements, scales, M, K);
  else hipLaunchKernelGGL(mx_quantize_kernel<_Float16>, grid_of(M, K), dim3(256), 0, stream, (const _Float16*)X, elements, scales, M, K);
  return hipGetLastError();
}

hipError_t launch_mx_dequantize(const uint8_t* elements, const uint8_t* scales, void* X, int M, int K, int dtype, hipStream_t stream) {
  if (dtype == BEAM_BF16) hipLaunchKernelGGL(mx_dequantize_kernel<__bf16>, grid_of(M, K), dim3(256), 0, stream, elements, scales, (__bf16*)X, M, K);
  else hipLaunchKernelGGL(mx_dequantize_kernel<_Float16>, grid_of(M, K), dim3(256), 0, stream, elements, scales, (_Float16*)X, M, K);
  return hipGetLastError();
}

}  // namespace beam
