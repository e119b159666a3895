// c = a @ b^T of two MXFP4 operands (mx.h), fp32 accumulation on the scaled matrix instructions, 16-bit output.
//
// A K tile is 256 columns, 128 bytes of a row: the bytes that a row of 64 16-bit elements has, and an instruction of 128 columns
// takes the operand bytes and (nearly) the time that one of 32 16-bit columns takes.  So the layouts, fills and reads are those
// of gemm_kernel.h, at four times the flops for a byte, and the K loop of a given depth is a quarter as long.
//
// Scales travel with their elements: a K tile's are 8 bytes a row and lie side by side in memory (mx.h), so a fill of 256 bytes
// brings those of 32 rows into the slot of the ring that the rows themselves go to, and the wait for the one is the wait for the
// other.  (Loaded straight into registers they would have to be asked for as early as the fills, a register set for every slot:
// memory operations are waited for in the order they were issued in.)
#pragma once

#include "mx.h"

namespace beam {

// The scales of NB blocks of 16 rows for one K tile, read from the 8 bytes a row at `first` (this lane's two bytes of block 0):
// lane (r, g) has those of row r, chunks 2 g and 2 g + 1; two blocks to a register.
template <int NB>
struct MxScales {
  static constexpr int REGS = (NB + 1) / 2;
  int reg[REGS];

  __device__ __forceinline__ void read(const char* first) {
#pragma unroll
    for (int i = 0; i < REGS; ++i) {
      const int lo = *(const unsigned short*)(first + 2 * i * 128);
      const int hi = 2 * i + 1 < NB ? (int)*(const unsigned short*)(first + (2 * i + 1) * 128) : 0;
      reg[i] = lo | hi << 16;
    }
  }
  __device__ __forceinline__ void mask(int m) {
#pragma unroll
    for (int i = 0; i < REGS; ++i) reg[i] &= m;
  }
};

// What a lane of group g may look at of a K tile with `blocks` of its 8 scales: its two bytes, for both halves of a register.
// Chunks behind the end of K then have a scale of 2^-127 on both sides, and whatever a fill has put there (e2m1 has neither
// infinities nor NaNs) adds less than 2^-240.
__device__ __forceinline__ int mx_tail_mask(int blocks, int g) {
  const int m = (2 * g < blocks ? 0xff : 0) | (2 * g + 1 < blocks ? 0xff00 : 0);
  return m | m << 16;
}

// acc[i][j] += step KK of blocks i of A and j of B.
template <int KK, int FM, int FN>
__device__ __forceinline__ void mx_multiply(const i32x4 (&fa)[FM], const i32x4 (&fb)[FN], const MxScales<FM>& sa, const MxScales<FN>& sb,
                                            f32x4 (&acc)[FM][FN]) {
#pragma unroll
  for (int i = 0; i < FM; ++i)
#pragma unroll
    for (int j = 0; j < FN; ++j) {
      const int s_b = sb.reg[j >> 1], s_a = sa.reg[i >> 1];
      if ((j & 1) == 0 && (i & 1) == 0) acc[i][j] = mx_mfma<KK, 0, 0>(fb[j], fa[i], acc[i][j], s_b, s_a);
      else if ((j & 1) == 0) acc[i][j] = mx_mfma<KK, 0, 1>(fb[j], fa[i], acc[i][j], s_b, s_a);
      else if ((i & 1) == 0) acc[i][j] = mx_mfma<KK, 1, 0>(fb[j], fa[i], acc[i][j], s_b, s_a);
      else acc[i][j] = mx_mfma<KK, 1, 1>(fb[j], fa[i], acc[i][j], s_b, s_a);
    }
}

// One fill of 1 KiB (8 rows of 128 bytes) or of 256 bytes (the scales of 32 rows) by a wavefront.
__device__ __forceinline__ void mx_fill_rows(__amdgpu_buffer_rsrc_t rows, char* dst, unsigned off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rows, (__attribute__((address_space(3))) void*)dst, 16, (int)off, 0, 0, 0);
}
__device__ __forceinline__ void mx_fill_scales(__amdgpu_buffer_rsrc_t rows, char* dst, unsigned off) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rows, (__attribute__((address_space(3))) void*)dst, 4, (int)off, 0, 0, 0);
}

// Four neighbouring outputs of a row that has N of them.
template <typename T>
__device__ __forceinline__ void mx_store_quad(T* row, int n, int N, f32x4 v) {
  typedef T at_element __attribute__((ext_vector_type(4), aligned(2)));
  at_element o;
#pragma unroll
  for (int e = 0; e < 4; ++e) o[e] = (T)v[e];
  if (n + 3 < N) {
    *(at_element*)(row + n) = o;
  } else {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (n + e < N) row[n + e] = o[e];
  }
}

// Workgroup tile BM x BN of WVM x WVN wavefronts that share a ring of ST LDS slots.
template <typename T, int BM, int BN, int WVM, int WVN, int ST>
struct MxGemm {
  static constexpr int NW = WVM * WVN, NT = NW * 64;
  static constexpr int TM = BM / WVM, TN = BN / WVN;
  static constexpr int FM = TM / 16, FN = TN / 16;
  static constexpr int A_BYTES = BM * kRowBytes, B_BYTES = BN * kRowBytes;
  static constexpr int SCALES = A_BYTES + B_BYTES;  // where a slot's scales begin: A's, then B's
  static constexpr int LS = ((BM + BN) / 32 + NW - 1) / NW;  // fills of scales by a wavefront
  static constexpr int SLOT = SCALES + LS * NW * 256;
  static constexpr int LDS_BYTES = ST * SLOT;
  static constexpr int LA = BM * kChunksPerRow / NT, LB = BN * kChunksPerRow / NT;
  static constexpr int LOADS = LA + LB + LS;
  static constexpr int WAIT = (ST - 2) * LOADS;  // fills behind those of the K tile that is waited for
  static_assert(LDS_BYTES <= 160 * 1024 && WAIT < 64 && ST >= 2, "LDS, vmcnt range");
  static_assert(BM * kChunksPerRow % NT == 0 && BN * kChunksPerRow % NT == 0 && BM % 32 == 0 && BN % 32 == 0, "whole fills");

  static __device__ __forceinline__ void run(const MxParams& p, char* smem) {
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wm = wave % WVM, wn = wave / WVM;
    const int r = lane & 15, g = lane >> 4;
    const int M = p.M, N = p.N;
    const unsigned row_bytes = (unsigned)p.K / 2u;
    const TileCoord tc = tile_of_workgroup(blockIdx.x, p.tiles_m, p.tiles_n, p.group_m, p.divs);
    const int row0 = tc.tm * BM, col0 = tc.tn * BN;
    const int rows_a = M - row0 < BM ? M - row0 : BM, rows_b = N - col0 < BN ? N - col0 : BN;
    const int n_tiles = (p.K + kMxTile - 1) / kMxTile;

    // Rows that do not exist are out of their descriptor's range: nothing is fetched, and LDS gets zeros.  In the last K tile the
    // bytes behind a row's end are the next row's (MxScales::mask takes them out), behind the last row's end nothing: the whole
    // offset is the lane's, which is what the range check looks at.  Fills behind the last K tile are issued, to be counted, with
    // empty descriptors.
    unsigned voff_a[LA], voff_b[LB];
#pragma unroll
    for (int i = 0; i < (LA > LB ? LA : LB); ++i) {
      const int q = i * NT + tid, row = q >> 3;
      const unsigned off = (unsigned)row * row_bytes + (unsigned)(((q & 7) ^ swizzle_of_row(row)) << 4);
      if (i < LA) voff_a[i] = off;
      if (i < LB) voff_b[i] = off;
    }
    const char* const a_base = (const char*)p.A + (size_t)row0 * row_bytes;
    const char* const b_base = (const char*)p.B + (size_t)col0 * row_bytes;
    auto fill = [&](int t, char* slot) __attribute__((always_inline)) {
      const bool there = t < n_tiles;
      const unsigned koff = there ? (unsigned)t * kRowBytes : 0u;
      const __amdgpu_buffer_rsrc_t ra = make_rsrc(a_base, there ? (unsigned)rows_a * row_bytes : 0u);
      const __amdgpu_buffer_rsrc_t rb = make_rsrc(b_base, there ? (unsigned)rows_b * row_bytes : 0u);
#pragma unroll
      for (int i = 0; i < LA; ++i) mx_fill_rows(ra, slot + i * (NT * 16) + wave * 1024, voff_a[i] + koff);
#pragma unroll
      for (int i = 0; i < LB; ++i) mx_fill_rows(rb, slot + A_BYTES + i * (NT * 16) + wave * 1024, voff_b[i] + koff);
      const size_t kt = there ? (size_t)t : 0;
#pragma unroll
      for (int i = 0; i < LS; ++i) {
        const int part = i * NW + wave;  // of 32 rows; A's come first (and behind B's there may be an empty one)
        const bool of_a = part < BM / 32;
        const uint8_t* const base = of_a ? p.sa + (kt * M + row0) * kMxBlocks : p.sb + (kt * N + col0) * kMxBlocks;
        const __amdgpu_buffer_rsrc_t rs = make_rsrc(base, there && part < (BM + BN) / 32 ? (unsigned)(of_a ? rows_a : rows_b) * kMxBlocks : 0u);
        mx_fill_scales(rs, slot + SCALES + part * 256, (unsigned)(of_a ? part : part - BM / 32) * 256u + (unsigned)lane * 4u);
      }
    };
    const int tail_mask = mx_tail_mask(p.K / 32 - (n_tiles - 1) * kMxBlocks, g);

#pragma unroll
    for (int s = 0; s < ST - 1; ++s) fill(s, smem + s * SLOT);
    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    int frag_off[2];
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) frag_off[kk] = lds_offset(r, 2 * g + kk);
    const int scale_a = SCALES + (wm * TM + r) * kMxBlocks + 2 * g, scale_b = SCALES + (BM + wn * TN + r) * kMxBlocks + 2 * g;

    char* now = smem;
    char* next = smem + (ST - 1) * SLOT;  // the slot that K tile h - 1 was in
    for (int h = 0; h < n_tiles; ++h) {
      wait_vm_and_lds<WAIT>();
      bare_barrier();  // everyone's fills of K tile h are there, and everyone has read K tile h - 1
      fill(h + ST - 1, next);
      MxScales<FM> sa;
      MxScales<FN> sb;
      sa.read(now + scale_a);
      sb.read(now + scale_b);
      if (h == n_tiles - 1) sa.mask(tail_mask), sb.mask(tail_mask);
      const char* const at_a = now + wm * TM * kRowBytes;
      const char* const at_b = now + A_BYTES + wn * TN * kRowBytes;
      i32x4 fa[2][FM], fb[2][FN];
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
        for (int j = 0; j < FN; ++j) fb[kk][j] = *(const i32x4*)(at_b + j * 16 * kRowBytes + frag_off[kk]);
#pragma unroll
        for (int i = 0; i < FM; ++i) fa[kk][i] = *(const i32x4*)(at_a + i * 16 * kRowBytes + frag_off[kk]);
      }
      mx_multiply<0>(fa[0], fb[0], sa, sb, acc);
      mx_multiply<1>(fa[1], fb[1], sa, sb, acc);
      next = now;
      now = now + SLOT == smem + ST * SLOT ? smem : now + SLOT;
    }
    wait_vm_and_lds<0>();  // (fills behind the last K tile)
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int m = row0 + wm * TM + i * 16 + r;
      if (m >= M) continue;
#pragma unroll
      for (int j = 0; j < FN; ++j) mx_store_quad((T*)p.C + (size_t)m * N, col0 + wn * TN + j * 16 + 4 * g, N, acc[i][j]);
    }
  }
};

template <typename T, int BM, int BN, int WVM, int WVN, int ST>
__global__ void __launch_bounds__(WVM* WVN * 64, 2) gemm_mx_kernel(const MxParams p) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  MxGemm<T, BM, BN, WVM, WVN, ST>::run(p, smem);
}

// Small tiles of MB blocks of 16 rows and CB of 16 columns whose K tiles are dealt out to NW wavefronts, each with a ring of S
// slots of its own (gemm_kwave.h says why): no barrier until the fp32 sums meet in LDS, added in the wavefronts' order.
//
// A16: A is 16-bit.  The workgroup quantises its rows first, a block of 32 to a thread, while the first fills of B are on their
// way, and keeps them in LDS behind the rings, K tile by K tile as a fill would have put them: one launch instead of two for a
// few tokens, whose quantising by every workgroup again costs less than that.
template <typename T, int MB, int CB, int NW, int S, bool A16>
struct MxKw {
  using vec8 = typename ElemTraits<T>::vec8;
  static constexpr int ROWS = 16 * MB, COLS = 16 * CB, NT = NW * 64;
  static constexpr int A_BYTES = ROWS * kRowBytes, B_BYTES = COLS * kRowBytes;
  // fills of scales are 256 bytes each
  static constexpr int SA_BYTES = (MB + 1) / 2 * 256, SB_BYTES = (CB + 1) / 2 * 256;
  static constexpr int B_AT = A16 ? 0 : A_BYTES + SA_BYTES;  // a slot: A's rows and scales, B's rows and scales
  static constexpr int SLOT = B_AT + B_BYTES + SB_BYTES;
  static constexpr int SUM_BYTES = ROWS * COLS * 4;  // one wavefront's fp32 sums
  static constexpr int RINGS = NW * S * SLOT;
  static constexpr int KEPT = A_BYTES + ROWS * kMxBlocks;  // A16: a K tile of A and its scales
  static constexpr int LDS_BYTES = RINGS > NW * SUM_BYTES ? RINGS : NW * SUM_BYTES;  // A16: and KEPT for every K tile
  static constexpr int LOADS = (A16 ? 0 : 2 * MB + (MB + 1) / 2) + 2 * CB + (CB + 1) / 2;
  static constexpr int CG = COLS / 4, QUADS = ROWS * CG;
  static_assert(LDS_BYTES <= 160 * 1024 && (S - 1) * LOADS < 64, "LDS, vmcnt range");
  static_assert(CG == 4 || CG == 8 || CG == 16, "sum layout");

  static __device__ __forceinline__ int sum_slot(int row, int cg) { return row * CG + (cg ^ ((row / (16 / CG)) & (CG - 1))); }

  static __device__ __forceinline__ void run(const MxParams& p, char* smem) {
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int r = lane & 15, g = lane >> 4;
    const int M = p.M, N = p.N, K = p.K;
    const unsigned row_bytes = (unsigned)K / 2u;
    const TileCoord tc = tile_of_workgroup(blockIdx.x, p.tiles_m, p.tiles_n, p.group_m, p.divs);
    const int row0 = tc.tm * ROWS, col0 = tc.tn * COLS;
    const int rows_a = M - row0 < ROWS ? M - row0 : ROWS, rows_b = N - col0 < COLS ? N - col0 : COLS;
    const int n_tiles = (K + kMxTile - 1) / kMxTile;
    const int n = (n_tiles - wave + NW - 1) / NW;  // this wavefront's K tiles: wave, wave + NW, ...; may be none
    char* const ring = smem + wave * (S * SLOT);
    char* const kept = smem + RINGS;

    unsigned voff[2];  // of the two groups of 8 rows of a block
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int row = 8 * c + (lane >> 3);
      voff[c] = (unsigned)row * row_bytes + (unsigned)(((lane & 7) ^ swizzle_of_row(row)) << 4);
    }
    const char* const a_base = (const char*)p.A + (size_t)row0 * row_bytes;  // (not A16)
    const char* const b_base = (const char*)p.B + (size_t)col0 * row_bytes;
    auto fill = [&](int t, char* slot) __attribute__((always_inline)) {  // as MxGemm's
      const bool there = t < n;
      const size_t kt = there ? (size_t)(wave + t * NW) : 0;
      const unsigned koff = (unsigned)kt * kRowBytes;
      if constexpr (!A16) {
        const __amdgpu_buffer_rsrc_t ra = make_rsrc(a_base, there ? (unsigned)rows_a * row_bytes : 0u);
#pragma unroll
        for (int i = 0; i < 2 * MB; ++i) mx_fill_rows(ra, slot + i * 1024, voff[i & 1] + (unsigned)(i >> 1) * 16u * row_bytes + koff);
        const __amdgpu_buffer_rsrc_t rs = make_rsrc(p.sa + (kt * M + row0) * kMxBlocks, there ? (unsigned)rows_a * kMxBlocks : 0u);
#pragma unroll
        for (int i = 0; i < (MB + 1) / 2; ++i) mx_fill_scales(rs, slot + A_BYTES + i * 256, (unsigned)(i * 256 + lane * 4));
      }
      const __amdgpu_buffer_rsrc_t rb = make_rsrc(b_base, there ? (unsigned)rows_b * row_bytes : 0u);
#pragma unroll
      for (int i = 0; i < 2 * CB; ++i) mx_fill_rows(rb, slot + B_AT + i * 1024, voff[i & 1] + (unsigned)(i >> 1) * 16u * row_bytes + koff);
      const __amdgpu_buffer_rsrc_t rs = make_rsrc(p.sb + (kt * N + col0) * kMxBlocks, there ? (unsigned)rows_b * kMxBlocks : 0u);
#pragma unroll
      for (int i = 0; i < (CB + 1) / 2; ++i) mx_fill_scales(rs, slot + B_AT + B_BYTES + i * 256, (unsigned)(i * 256 + lane * 4));
    };
    auto start_rings = [&]() __attribute__((always_inline)) {
      if (n > 0) {
#pragma unroll
        for (int s = 0; s < S; ++s) fill(s, ring + s * SLOT);
      }
    };
    if constexpr (!A16) {
      start_rings();
    } else {
      // Block q of the rows that exist (the others are left as they are in LDS: they feed outputs that do not exist).  A thread's
      // first one is on its way before the fills are: memory operations are waited for in order.
      const int blocks = K / 32, count = rows_a * blocks;
      auto load = [&](int q, vec8(&x)[4]) __attribute__((always_inline)) {
        const int row = q / blocks;
        typedef vec8 vec8_at_element __attribute__((aligned(2)));
        const T* const at = (const T*)p.A + (size_t)(row0 + row) * K + 32 * (q - row * blocks);
#pragma unroll
        for (int c = 0; c < 4; ++c) x[c] = *(const vec8_at_element*)(at + 8 * c);
      };
      auto keep = [&](int q, const vec8(&x)[4]) __attribute__((always_inline)) {
        const int row = q / blocks, b = q - row * blocks;
        int scale;
        const i32x4 elements = mx_encode_block(x, &scale);
        char* const tile = kept + (b >> 3) * KEPT;
        *(i32x4*)(tile + lds_offset(row, b & 7)) = elements;
        tile[A_BYTES + row * kMxBlocks + (b & 7)] = (char)scale;
      };
      vec8 x[4];
      if (tid < count) load(tid, x);
      start_rings();
      if (tid < count) keep(tid, x);
      for (int q = tid + NT; q < count; q += NT) {
        load(q, x);
        keep(q, x);
      }
      // (a barrier for LDS alone: __syncthreads() would wait for the fills)
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      bare_barrier();
    }

    f32x4 acc[MB][CB];
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < CB; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    int frag_off[2];
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) frag_off[kk] = lds_offset(r, 2 * g + kk);
    const int scale_off = r * kMxBlocks + 2 * g;
    const int tail_mask = mx_tail_mask(K / 32 - (n_tiles - 1) * kMxBlocks, g);
    char* slot = ring;
    for (int t = 0; t < n; ++t) {
      asm volatile("" ::: "memory");
      wait_vm_and_lds<(S - 1) * LOADS>();
      asm volatile("" ::: "memory");
      const char* const at_a = A16 ? kept + (wave + t * NW) * KEPT : slot;
      const char* const at_b = slot + B_AT;
      i32x4 fa[2][MB], fb[2][CB];
      MxScales<MB> sa;
      MxScales<CB> sb;
      sa.read(at_a + A_BYTES + scale_off);
      sb.read(at_b + B_BYTES + scale_off);
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
        for (int j = 0; j < CB; ++j) fb[kk][j] = *(const i32x4*)(at_b + j * 16 * kRowBytes + frag_off[kk]);
#pragma unroll
        for (int i = 0; i < MB; ++i) fa[kk][i] = *(const i32x4*)(at_a + i * 16 * kRowBytes + frag_off[kk]);
      }
      asm volatile("" ::: "memory");
      wait_lds<0>();  // everything is read: the slot is free
      __builtin_amdgcn_sched_barrier(0);
      fill(t + S, slot);
      __builtin_amdgcn_sched_barrier(0);
      if (wave + t * NW == n_tiles - 1) sa.mask(tail_mask), sb.mask(tail_mask);
      mx_multiply<0>(fa[0], fb[0], sa, sb, acc);
      mx_multiply<1>(fa[1], fb[1], sa, sb, acc);
      slot = slot + SLOT == ring + S * SLOT ? ring : slot + SLOT;
    }
    wait_vm_and_lds<0>();  // the empty fills of the last iterations must be gone before the rings are reused,
    __syncthreads();       // everyone's: a wavefront's sums may lie in another one's ring
    char* const sums = smem + wave * SUM_BYTES;
#pragma unroll
    for (int i = 0; i < MB; ++i)
#pragma unroll
      for (int j = 0; j < CB; ++j) *(f32x4*)(sums + sum_slot(i * 16 + r, j * 4 + g) * 16) = acc[i][j];
    __syncthreads();
#pragma unroll
    for (int q0 = 0; q0 < QUADS; q0 += NT) {
      const int q = q0 + tid;
      const int m = row0 + q / CG, nn = col0 + (q % CG) * 4;
      if (q >= QUADS || m >= M || nn >= N) continue;
      const char* const at = smem + sum_slot(q / CG, q % CG) * 16;
      f32x4 v = *(const f32x4*)at;
#pragma unroll
      for (int w = 1; w < NW; ++w) v += *(const f32x4*)(at + w * SUM_BYTES);
      mx_store_quad((T*)p.C + (size_t)m * N, nn, N, v);
    }
  }
};

template <typename T, int MB, int CB, int NW, int S, bool A16>
__global__ void __launch_bounds__(NW * 64, 2) gemm_mx_kwave_kernel(const MxParams p) {
  extern __shared__ __attribute__((aligned(1024))) char smem[];
  MxKw<T, MB, CB, NW, S, A16>::run(p, smem);
}

}  // namespace beam
