// 16-bit values to MXFP4 and back (mx.h).
#include "mx.h"

namespace beam {

namespace {

// A thread takes 8 columns of a row, 32 neighbouring ones a K tile of it, and does so for kRows rows at once; a block's largest
// magnitude is that of four threads.  Bound by memory: 2 M K bytes in, 0.53 M K out.  Accesses are 512 and 128 contiguous bytes a row
// (a block of 64 bytes to a thread, nothing to exchange, has every access touch all of a wavefront's lines; neighbouring workgroups on
// neighbouring rows meet in the same memory channels.  8192 x 8192 fp16, both ways -> so: 46 -> 40 us, 4.3 TB/s, and back 49 -> 31).
constexpr int kRows = 4;  // of a thread, 8 apart
constexpr int kRowsPerWorkgroup = 8 * kRows;

// The largest of the four threads of a block, in each of them.
__device__ __forceinline__ unsigned largest_of_four(unsigned x) {
  const unsigned y = (unsigned)__builtin_amdgcn_mov_dpp((int)x, 0xB1, 0xf, 0xf, true);  // quad_perm 1 0 3 2
  x = x > y ? x : y;
  const unsigned z = (unsigned)__builtin_amdgcn_mov_dpp((int)x, 0x4E, 0xf, 0xf, true);  // quad_perm 2 3 0 1
  return x > z ? x : z;
}

template <typename T>
__global__ void __launch_bounds__(256) mx_quantize_kernel(const T* __restrict__ X, uint8_t* __restrict__ elements, uint8_t* __restrict__ scales,
                                                          int M, int K) {
  typedef T vec8 __attribute__((ext_vector_type(8)));
  typedef vec8 vec8_at_element __attribute__((aligned(2)));
  const unsigned tiles = (unsigned)(K + kMxTile - 1) / kMxTile;  // neighbouring workgroups: neighbouring columns
  const int kt = blockIdx.x % tiles, c = threadIdx.x & 31;
  const int col = kt * kMxTile + 8 * c;
  const bool there = col < K;  // (K is a multiple of 32: the four threads of a block agree)
  const long m0 = (long)(blockIdx.x / tiles) * kRowsPerWorkgroup + (threadIdx.x >> 5);
  vec8 x[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const long m = m0 + 8 * i < M ? m0 + 8 * i : M - 1;  // (what is not there is not stored)
    x[i] = *(const vec8_at_element*)(X + (size_t)m * K + (there ? col : 0));
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const long m = m0 + 8 * i;
    float v[8];
    unsigned top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = (float)x[i][e];
      const unsigned bits = __float_as_uint(v[e]) & 0x7fffffffu;
      top = bits > top ? bits : top;
    }
    const int scale = mx_scale_of(largest_of_four(top));
    const unsigned q = mx_encode8(v, scale);
    if (m >= M) continue;
    if (there) *(unsigned*)(elements + (size_t)m * (K / 2) + col / 2) = q;
    if ((c & 3) == 0) scales[((size_t)kt * M + m) * kMxBlocks + c / 4] = (uint8_t)(there ? scale : 0);  // (zeros behind the last block)
  }
}

// The values held, rounded to T (exact in bf16, and in fp16 for what was quantised from fp16); the same share of a thread.
template <typename T>
__global__ void __launch_bounds__(256) mx_dequantize_kernel(const uint8_t* __restrict__ elements, const uint8_t* __restrict__ scales,
                                                            T* __restrict__ X, int M, int K) {
  typedef T vec8 __attribute__((ext_vector_type(8)));
  typedef vec8 vec8_at_element __attribute__((aligned(2)));
  typedef float f32x2 __attribute__((ext_vector_type(2)));
  const unsigned tiles = (unsigned)(K + kMxTile - 1) / kMxTile;  // neighbouring workgroups: neighbouring columns
  const int kt = blockIdx.x % tiles, c = threadIdx.x & 31;
  const int col = kt * kMxTile + 8 * c;
  if (col >= K) return;
  const long m0 = (long)(blockIdx.x / tiles) * kRowsPerWorkgroup + (threadIdx.x >> 5);
  unsigned q[kRows];
  int scale[kRows];
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const long m = m0 + 8 * i < M ? m0 + 8 * i : M - 1;
    q[i] = *(const unsigned*)(elements + (size_t)m * (K / 2) + col / 2);
    scale[i] = scales[((size_t)kt * M + m) * kMxBlocks + c / 4];
  }
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const long m = m0 + 8 * i;
    if (m >= M) return;
    vec8 x;
    auto two = [&](f32x2 v, int e) __attribute__((always_inline)) {
      x[e] = (T)(scale[i] == 255 ? __builtin_nanf("") : __builtin_amdgcn_ldexpf(v[0], scale[i] - 127));
      x[e + 1] = (T)(scale[i] == 255 ? __builtin_nanf("") : __builtin_amdgcn_ldexpf(v[1], scale[i] - 127));
    };
    two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i], 1.0f, 0), 0);
    two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i], 1.0f, 1), 2);
    two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i], 1.0f, 2), 4);
    two(__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(q[i], 1.0f, 3), 6);
    *(vec8_at_element*)(X + (size_t)m * K + col) = x;
  }
}

dim3 grid_of(int M, int K) { return dim3((unsigned)(((long)M + kRowsPerWorkgroup - 1) / kRowsPerWorkgroup * ((K + kMxTile - 1) / kMxTile))); }

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
