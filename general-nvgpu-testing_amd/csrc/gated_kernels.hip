// The gated layer's kernels that are not matrix products.
#include "elementwise.h"
#include "gated.h"

namespace beam {

namespace {

// One output per thread; see launch_gated_plain.
template <typename T>
__global__ void __launch_bounds__(256) gated_plain_kernel(const T* __restrict__ A, const T* __restrict__ B, T* __restrict__ H,
                                                          T* __restrict__ GU, int M, int N, int K) {
  const size_t count = (size_t)M * N;
  for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < count; i += (size_t)gridDim.x * 256) {
    const size_t m = i / (size_t)N, n = i - m * (size_t)N;
    const T* const a = A + m * K;
    const T* const gate = B + n * K;
    const T* const up = B + (n + N) * K;
    float g = 0.0f, u = 0.0f;
    for (int k = 0; k < K; ++k) {
      g += (float)a[k] * (float)gate[k];
      u += (float)a[k] * (float)up[k];
    }
    H[i] = (T)gated_f32<T>(g, u);
    if (GU) {
      GU[m * 2 * N + n] = (T)g;
      GU[m * 2 * N + N + n] = (T)u;
    }
  }
}

// v >> bits, 0 <= bits < 128, of eight 16-bit values
template <typename V8>
__device__ __forceinline__ V8 shift_down(V8 v, int bits) {
  typedef unsigned long long u64x2 __attribute__((ext_vector_type(2)));
  const u64x2 w = __builtin_bit_cast(u64x2, v);
  const int b = bits & 63;
  const unsigned long long over = b ? w[1] << (64 - b) : 0;
  u64x2 o;
  o[0] = bits >= 64 ? w[1] >> b : w[0] >> b | over;
  o[1] = bits >= 64 ? 0 : w[1] >> b;
  return __builtin_bit_cast(V8, o);
}

// With s = 1 / (1 + exp(-g)):  dg = dh * u * s * (1 + g * (1 - s)),  du = dh * g * s, in fp32, each rounded once to 16 bits,
// which the products that follow take as operands.
//
// Bound by memory: 3 M N elements in, 2 M N out for each of D and DT.  dA = D . B wants D as rows of tokens, dB = D^T . A as rows
// of features; written both ways here, both are products that read their operands in rows.  A workgroup takes 64 x 64 outputs: a
// thread two rows of 8 columns, which go to D as they are and into LDS as pairs of rows, whose 16-byte chunks are XORed with the
// column's number over 8, so that the 8 threads of a row write to different banks; DT then leaves in 128-byte runs.
template <typename T>
__global__ void __launch_bounds__(256) gated_gradients_kernel(const T* __restrict__ dH, const T* __restrict__ GU, T* __restrict__ D,
                                                              T* __restrict__ DT, int M, int N, int cols_d, int cols_dt, int tiles_n) {
  typedef T vec8 __attribute__((ext_vector_type(8)));
  typedef T vec8_at_element __attribute__((ext_vector_type(8), aligned(2)));  // rows start at any element
  typedef T pair_t __attribute__((ext_vector_type(2)));
  constexpr int R = 64, C = 64;
  __shared__ __attribute__((aligned(16))) T turned[2 * C * R];
  const int tm = blockIdx.x / tiles_n, tn = blockIdx.x - tm * tiles_n;
  const int m0 = tm * R, n0 = tn * C;
  const int c = threadIdx.x & 7, rp = threadIdx.x >> 3;
  const int n = n0 + 8 * c;
  const bool through = (N | cols_d) % 64 == 0;
  // All loads in front of any arithmetic.  Behind the last row the last one is read again; 8 columns that do not fit are the row's
  // last 8, shifted down; what is made of columns that do not exist is not stored, and of rows only zeros, in DT.
  vec8 g[2], u[2], d[2];
  if (N >= 8) {  // (uniform)
    const int at = n < N - 8 ? n : N - 8;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const size_t m = m0 + 2 * rp + h < M ? m0 + 2 * rp + h : M - 1;
      g[h] = *(const vec8_at_element*)(GU + m * 2 * N + at);
      u[h] = *(const vec8_at_element*)(GU + m * 2 * N + N + at);
      d[h] = *(const vec8_at_element*)(dH + m * N + at);
    }
    if (n0 + C > N) {  // (uniform)
      const int bits = (n - at) < 8 ? 16 * (n - at) : 0;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        g[h] = shift_down(g[h], bits);
        u[h] = shift_down(u[h], bits);
        d[h] = shift_down(d[h], bits);
      }
    }
  } else {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const size_t m = m0 + 2 * rp + h < M ? m0 + 2 * rp + h : M - 1;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int col = n + e < N ? n + e : N - 1;
        g[h][e] = GU[m * 2 * N + col];
        u[h][e] = GU[m * 2 * N + N + col];
        d[h][e] = dH[m * N + col];
      }
    }
  }
  vec8 dg[2], du[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int m = m0 + 2 * rp + h;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float gf = (float)g[h][e], df = (float)d[h][e];
      const float s = __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(gf * -1.4426950408889634f));
      dg[h][e] = (T)(df * (float)u[h][e] * (s * (1.0f + gf * (1.0f - s))));
      du[h][e] = (T)(df * (gf * s));
    }
    if (m >= M) dg[h] = du[h] = vec8{};  // (whatever the nearest row holds)
    if (D && m < M) {
      T* const row = D + (size_t)m * cols_d + n;
      if (n + 7 < N) {
        if (through) {
          store_16<kStoreThrough>(row, __builtin_bit_cast(i32x4, dg[h]));
          store_16<kStoreThrough>(row + N, __builtin_bit_cast(i32x4, du[h]));
        } else {
          *(vec8_at_element*)row = dg[h];
          *(vec8_at_element*)(row + N) = du[h];
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (n + e < N) {
            row[e] = dg[h][e];
            row[N + e] = du[h][e];
          }
      }
    }
  }
  if (D && tn == tiles_n - 1) {  // (uniform) the zeros behind its rows
    const int more = cols_d - 2 * N;
    for (int i = threadIdx.x; i < R * more; i += 256) {
      const int row = i / more, m = m0 + row;
      if (m < M) D[(size_t)m * cols_d + 2 * N + (i - row * more)] = (T)0.0f;
    }
  }
  if (!DT) return;  // (uniform)
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int col = 8 * c + e;
    T* const row = turned + col * R + ((((rp >> 2) ^ c) << 3) | ((rp & 3) << 1));
    *(pair_t*)row = pair_t{dg[0][e], dg[1][e]};
    *(pair_t*)(row + C * R) = pair_t{du[0][e], du[1][e]};
  }
  __syncthreads();
#pragma unroll
  for (int it = 0; it < 4; ++it) {
    const int q = it * 256 + (int)threadIdx.x;
    const int chunk = q & 7, col = (q >> 3) & (C - 1), up = q >> 9;
    const int m = m0 + 8 * chunk;
    if (n0 + col >= N || m >= cols_dt) continue;
    const vec8 v = *(const vec8*)(turned + up * C * R + col * R + ((chunk ^ (col >> 3)) << 3));
    T* const out = DT + ((size_t)up * N + n0 + col) * cols_dt + m;
    if (m + 7 < cols_dt) {  // (behind M these are zeros)
      if (cols_dt % 64 == 0) store_16<kStoreThrough>(out, __builtin_bit_cast(i32x4, v));
      else *(vec8_at_element*)out = v;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (m + e < cols_dt) out[e] = v[e];
    }
  }
}

}  // namespace

hipError_t launch_gated_plain(const void* A, const void* B, void* H, void* GU, int M, int N, int K, int dtype, hipStream_t stream) {
  const size_t blocks = ((size_t)M * N + 255) / 256;
  const dim3 grid((unsigned)(blocks < 65536 ? blocks : 65536));
  if (dtype == BEAM_BF16)
    hipLaunchKernelGGL(gated_plain_kernel<__bf16>, grid, dim3(256), 0, stream, (const __bf16*)A, (const __bf16*)B, (__bf16*)H, (__bf16*)GU, M, N, K);
  else
    hipLaunchKernelGGL(gated_plain_kernel<_Float16>, grid, dim3(256), 0, stream, (const _Float16*)A, (const _Float16*)B, (_Float16*)H, (_Float16*)GU, M, N, K);
  return hipGetLastError();
}

hipError_t launch_gated_gradients(const void* dH, const void* GU, void* D, void* DT, int M, int N, int cols_d, int cols_dt, int dtype,
                                  hipStream_t stream) {
  const int tiles_n = (N + 63) / 64;
  const dim3 grid((unsigned)((size_t)((M + 63) / 64) * tiles_n));
  if (dtype == BEAM_BF16)
    hipLaunchKernelGGL(gated_gradients_kernel<__bf16>, grid, dim3(256), 0, stream, (const __bf16*)dH, (const __bf16*)GU, (__bf16*)D, (__bf16*)DT, M, N, cols_d, cols_dt, tiles_n);
  else
    hipLaunchKernelGGL(gated_gradients_kernel<_Float16>, grid, dim3(256), 0, stream, (const _Float16*)dH, (const _Float16*)GU, (_Float16*)D, (_Float16*)DT, M, N, cols_d, cols_dt, tiles_n);
  return hipGetLastError();
}

}  // namespace beam
