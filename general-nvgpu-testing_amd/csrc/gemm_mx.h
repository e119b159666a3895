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

// The scales of NB blocks of 16 rows for one K tile in a lane (r, g): those of row r of each block, chunks 2 g and 2 g + 1, 16
// bits, two blocks to a register.
template <int NB>
struct MxScales {
  static constexpr bool QUADS = NB % 4 == 0;
  static constexpr int REGS = (NB + 1) / 2;
  int reg[REGS];
  static constexpr int reg_of(int i) { return QUADS ? 2 * (i >> 2) + (i & 1) : i >> 1; }
  static constexpr int half_of(int i) { return QUADS ? (i >> 1) & 1 : i & 1; }

  // The rows' 8 bytes lie side by side from `rows` on.  Four blocks are 64 rows: lane (r, g) reads the 8 bytes of row r of block g
  // at once, and the four lane groups exchange what they need of each other's (mx_turn); otherwise the 16 bits of each block.
  i32x2 raw[QUADS ? NB / 4 : 1];
  __device__ __forceinline__ void read(const char* rows, int lane) {
    if constexpr (QUADS) {
#pragma unroll
      for (int q = 0; q < NB / 4; ++q) raw[q] = *(const i32x2*)(rows + q * 512 + lane * 8);
    } else {
      const char* const first = rows + (lane & 15) * kMxBlocks + 2 * (lane >> 4);
#pragma unroll
      for (int i = 0; i < REGS; ++i) {
        const int lo = *(const unsigned short*)(first + 2 * i * 128);
        const int hi = 2 * i + 1 < NB ? (int)*(const unsigned short*)(first + (2 * i + 1) * 128) : 0;
        reg[i] = lo | hi << 16;
      }
    }
  }
  __device__ __forceinline__ void turn() {
    if constexpr (QUADS) {
#pragma unroll
      for (int q = 0; q < NB / 4; ++q) mx_turn(raw[q], &reg[2 * q], &reg[2 * q + 1]);
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

// acc[j] += step KK of block I of A and blocks j of B.
template <int KK, int I, int FM, int FN>
__device__ __forceinline__ void mx_multiply_row(i32x4 fa, const i32x4 (&fb)[FN], const MxScales<FM>& sa, const MxScales<FN>& sb, f32x4 (&acc)[FN]) {
  using A = MxScales<FM>;
  using B = MxScales<FN>;
  const int s_a = sa.reg[A::reg_of(I)];
#pragma unroll
  for (int j = 0; j < FN; ++j) {
    if (B::half_of(j) == 0) acc[j] = mx_mfma<KK, 0, A::half_of(I)>(fb[j], fa, acc[j], sb.reg[B::reg_of(j)], s_a);
    else acc[j] = mx_mfma<KK, 1, A::half_of(I)>(fb[j], fa, acc[j], sb.reg[B::reg_of(j)], s_a);
  }
}

// f(0), ..., f(N - 1) with the index as a constant.
template <int I, int N, typename F>
__device__ __forceinline__ void mx_static_for(F&& f) {
  if constexpr (I < N) {
    f(std::integral_constant<int, I>{});
    mx_static_for<I + 1, N>(f);
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

// Workgroup tile BM x BN of WVM x WVN wavefronts that share a ring of ST LDS slots.  Eight wavefronts to a 128 x 128 tile, two to a
// SIMD, although they read half as much again from LDS as four would: with one the chain of a K tile (barrier, reads, MFMAs) has nothing
// to hide behind (1024 x 2048 x 8192 22.2 us, so 17.6).  Or several workgroups to a CU, with rings of fewer slots (4096^3 in 128 x 128
// 53, 47 us).
//
// The K loop is gemm_kernel.h's: while the MFMAs of one half of a K tile run, the fragments of the next half are read, a few
// between the MFMAs of each row, and the fills of the K tile ST - 1 further on are issued, a row's share behind each row; of two
// wavefronts on a SIMD the older one issues all of them.  A row is closed by a scheduling fence: left alone, the compiler reads
// every fragment right in front of the MFMA that needs it (8192^3 298 us, so 270).
template <typename T, int BM, int BN, int WVM, int WVN, int ST>
struct MxGemm {
  static constexpr int NW = WVM * WVN, NT = NW * 64;
  static constexpr int LDW = NW >= 8 ? NW / 2 : NW, NTL = LDW * 64;  // wavefronts that fill LDS, their threads
  static constexpr int TM = BM / WVM, TN = BN / WVN;
  static constexpr int FM = TM / 16, FN = TN / 16;
  static constexpr int A_BYTES = BM * kRowBytes, B_BYTES = BN * kRowBytes;
  static constexpr int SCALES = A_BYTES + B_BYTES;  // where a slot's scales begin: A's, then B's
  static constexpr int LS = ((BM + BN) / 32 + LDW - 1) / LDW;  // fills of scales by a loader
  static constexpr int SLOT = SCALES + LS * LDW * 256;
  static constexpr int LDS_BYTES = ST * SLOT;
  static constexpr int LA = BM * kChunksPerRow / NTL, LB = BN * kChunksPerRow / NTL;
  static constexpr int LOADS = LA + LB + LS;
  static constexpr int WAIT = (ST - 2) * LOADS;  // fills behind those of the K tile that is waited for
  static constexpr int PER_ROW = (LOADS + 2 * FM - 1) / (2 * FM);
  static_assert(LDS_BYTES <= 160 * 1024 && WAIT < 64 && ST >= 2, "LDS, vmcnt range");
  static_assert(BM * kChunksPerRow % NTL == 0 && BN * kChunksPerRow % NTL == 0 && BM % 32 == 0 && BN % 32 == 0, "whole fills");

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
      const int q = i * NTL + tid, row = q >> 3;
      const unsigned off = (unsigned)row * row_bytes + (unsigned)(mx_chunk_at((q & 7) ^ swizzle_of_row(row)) << 4);
      if (i < LA) voff_a[i] = off;
      if (i < LB) voff_b[i] = off;
    }
    const char* const a_base = (const char*)p.A + (size_t)row0 * row_bytes;
    const char* const b_base = (const char*)p.B + (size_t)col0 * row_bytes;
    // fill l of K tile t: B's rows, A's, the scales
    auto fill = [&](int l, int t, char* slot) __attribute__((always_inline)) {
      const bool there = t < n_tiles;
      const unsigned koff = there ? (unsigned)t * kRowBytes : 0u;
      if (l < LB) {
        mx_fill_rows(make_rsrc(b_base, there ? (unsigned)rows_b * row_bytes : 0u), slot + A_BYTES + l * (NTL * 16) + wave * 1024, voff_b[l] + koff);
      } else if (l < LB + LA) {
        const int i = l - LB;
        mx_fill_rows(make_rsrc(a_base, there ? (unsigned)rows_a * row_bytes : 0u), slot + i * (NTL * 16) + wave * 1024, voff_a[i] + koff);
      } else {
        const int part = (l - LB - LA) * LDW + wave;  // of 32 rows; A's come first (and behind B's there may be an empty one)
        const bool of_a = part < BM / 32;
        const size_t kt = there ? (size_t)t : 0;
        const uint8_t* const base = of_a ? p.sa + (kt * M + row0) * kMxBlocks : p.sb + (kt * N + col0) * kMxBlocks;
        const __amdgpu_buffer_rsrc_t rs = make_rsrc(base, there && part < (BM + BN) / 32 ? (unsigned)(of_a ? rows_a : rows_b) * kMxBlocks : 0u);
        mx_fill_scales(rs, slot + SCALES + part * 256, (unsigned)(of_a ? part : part - BM / 32) * 256u + (unsigned)lane * 4u);
      }
    };
    const bool loader = LDW == NW || wave < LDW;
    if (loader) {
#pragma unroll
      for (int s = 0; s < ST - 1; ++s)
#pragma unroll
        for (int l = 0; l < LOADS; ++l) fill(l, s, smem + s * SLOT);
    }
    const int tail_mask = mx_tail_mask(p.K / 32 - (n_tiles - 1) * kMxBlocks, g);
    f32x4 acc[FM][FN];
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    int frag_off[2];
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) frag_off[kk] = lds_offset(r, 4 * kk + g);
    const int wave_a = wm * TM * kRowBytes, wave_b = A_BYTES + wn * TN * kRowBytes;
    const int wave_sa = SCALES + wm * TM * kMxBlocks, wave_sb = SCALES + (BM + wn * TN) * kMxBlocks;

    // Fragments of the halves of a K tile, and their scales: zeros to begin with, so that the first step multiplies nothing.
    i32x4 fa0[FM], fa1[FM], fb0[FN], fb1[FN];
    MxScales<FM> sa;
    MxScales<FN> sb;
#pragma unroll
    for (int i = 0; i < FM; ++i) fa1[i] = i32x4{0, 0, 0, 0};
#pragma unroll
    for (int j = 0; j < FN; ++j) fb1[j] = i32x4{0, 0, 0, 0};
#pragma unroll
    for (int i = 0; i < MxScales<FM>::REGS; ++i) sa.reg[i] = 0;
#pragma unroll
    for (int j = 0; j < MxScales<FN>::REGS; ++j) sb.reg[j] = 0;
    // Multiplies half KK with (ca, cb), reads the next half (na, nb) and issues the fills of rows ROW0 .. of K tile h + ST - 1.
    auto step = [&](auto kk_tag, auto row0_tag, auto ld_tag, const i32x4(&ca)[FM], const i32x4(&cb)[FN], i32x4(&na)[FM], i32x4(&nb)[FN], const char* slot,
                    int off, int h, char* fill_slot) __attribute__((always_inline)) {
      constexpr int KK = decltype(kk_tag)::value, ROW0 = decltype(row0_tag)::value;
      constexpr bool LD = decltype(ld_tag)::value;
      constexpr int READS = FM + FN, READ_ROWS = FM > 1 ? FM - 1 : 1, PER_READ_ROW = (READS + READ_ROWS - 1) / READ_ROWS;
      mx_static_for<0, FM>([&](auto i_tag) __attribute__((always_inline)) {
        constexpr int i = decltype(i_tag)::value;
#pragma unroll
        for (int u = 0; u < PER_READ_ROW; ++u) {
          const int n = i * PER_READ_ROW + u;
          if (i < READ_ROWS && n < READS) {
            if (n < FN) nb[n] = *(const i32x4*)(slot + wave_b + n * 16 * kRowBytes + off);
            else na[n - FN] = *(const i32x4*)(slot + wave_a + (n - FN) * 16 * kRowBytes + off);
          }
        }
        mx_multiply_row<KK, i>(ca[i], cb, sa, sb, acc[i]);
        if constexpr (LD) {
#pragma unroll
          for (int u = 0; u < PER_ROW; ++u)
            if ((ROW0 + i) * PER_ROW + u < LOADS) fill((ROW0 + i) * PER_ROW + u, h + ST - 1, fill_slot);
        }
        if constexpr (FN >= 4) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
          __builtin_amdgcn_sched_group_barrier(0x020, PER_ROW, 0);
          __builtin_amdgcn_sched_group_barrier(0x008, FN - 3, 0);
        }
        __builtin_amdgcn_sched_barrier(0);
      });
    };
    auto loop = [&](auto ld_tag) __attribute__((always_inline)) {
      constexpr bool LD = decltype(ld_tag)::value;
      char* now = smem;
      char* free = smem + (ST - 1) * SLOT;  // the slot that K tile h - 1 was in
      for (int h = 0; h < n_tiles; ++h) {
        // my fills of K tile h are there, my reads of K tile h - 1 done ...
        if constexpr (LD) wait_vm_and_lds<WAIT>();
        else wait_lds<0>();
        bare_barrier();  // ... and everyone's
        MxScales<FM> ta;
        MxScales<FN> tb;
        ta.read(now + wave_sa, lane);
        tb.read(now + wave_sb, lane);
        step(std::integral_constant<int, 1>{}, std::integral_constant<int, 0>{}, ld_tag, fa1, fb1, fa0, fb0, now, frag_off[0], h, free);
        ta.turn();
        tb.turn();
        if (h == n_tiles - 1) ta.mask(tail_mask), tb.mask(tail_mask);
        sa = ta, sb = tb;
        step(std::integral_constant<int, 0>{}, std::integral_constant<int, FM>{}, ld_tag, fa0, fb0, fa1, fb1, now, frag_off[1], h, free);
        free = now;
        now = now + SLOT == smem + ST * SLOT ? smem : now + SLOT;
      }
    };
    if (loader) loop(std::true_type{});
    else loop(std::false_type{});
    mx_static_for<0, FM>([&](auto i_tag) __attribute__((always_inline)) {  // the second half of the last K tile
      mx_multiply_row<1, decltype(i_tag)::value>(fa1[decltype(i_tag)::value], fb1, sa, sb, acc[decltype(i_tag)::value]);
    });
    wait_vm_and_lds<0>();  // (fills behind the last K tile)
    __syncthreads();       // every slot is dead
    // Through LDS, as in gemm_kernel.h, whose layout this is: 16 bytes a lane, whole rows of the wavefront's part at a time (7698 x
    // 3456 x 256, 8 bytes a lane straight from the sums 26 us, so 17.6).
    constexpr int RB = TN * 2, LPR = TN / 8, RPI = 64 / LPR;
    static_assert(NW * TM * RB <= LDS_BYTES && (RB == 64 || RB == 128), "staging area");
    auto chunk_xor = [](int row) { return RB == 64 ? (row >> 1) & 3 : row & 7; };
    // (the lane's constants here from a value that the compiler cannot see through: hoisted in front of the K loop they cost the
    // 256 x 256 tile registers that it does not have, 2048 x 4096 x 11008 78 -> 87 us)
    int ol = lane;
    asm volatile("" : "+v"(ol));
    const int wr = ol & 15, wg = ol >> 4;
    char* const stage = smem + wave * (TM * RB);
#pragma unroll
    for (int i = 0; i < FM; ++i)
#pragma unroll
      for (int j = 0; j < FN; ++j) {
        typename ElemTraits<T>::vec4 v;
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = (T)acc[i][j][e];
        *(typename ElemTraits<T>::vec4*)(stage + (i * 16 + wr) * RB + (((wg & 1) ^ (wr >> 3)) << 3) + (((2 * j + (wg >> 1)) ^ chunk_xor(wr)) << 4)) = v;
      }
    using vec8 = typename ElemTraits<T>::vec8;
    const int srow = ol / LPR, schunk = ol % LPR;
    auto store_all = [&](auto kind_tag) __attribute__((always_inline)) {
#pragma unroll
      for (int it = 0; it < TM / RPI; ++it) {
        const int row = it * RPI + srow;
        vec8 v = *(const vec8*)(stage + row * RB + schunk * 16);
        if ((row >> 3) & 1) v = vec8{v[4], v[5], v[6], v[7], v[0], v[1], v[2], v[3]};
        const int m = row0 + wm * TM + row, n = col0 + wn * TN + (schunk ^ chunk_xor(row)) * 8;
        T* const at = (T*)p.C + (size_t)m * N + n;
        if (m < M && n + 7 < N) {
          store_16<decltype(kind_tag)::value>(at, __builtin_bit_cast(i32x4, v));
        } else if (m < M && n < N) {
#pragma unroll
          for (int e = 0; e < 7; ++e)
            if (n + e < N) at[e] = v[e];
        }
      }
    };
    if (p.c_store == kStoreThrough) store_all(std::integral_constant<int, kStoreThrough>{});
    else store_all(std::integral_constant<int, kStoreCached>{});
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
      voff[c] = (unsigned)row * row_bytes + (unsigned)(mx_chunk_at((lane & 7) ^ swizzle_of_row(row)) << 4);
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
        *(i32x4*)(tile + lds_offset(row, mx_place_of(b & 7))) = elements;
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
    for (int kk = 0; kk < 2; ++kk) frag_off[kk] = lds_offset(r, 4 * kk + g);
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
      sa.read(at_a + A_BYTES, lane);
      sb.read(at_b + B_BYTES, lane);
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
      sa.turn();
      sb.turn();
      if (wave + t * NW == n_tiles - 1) sa.mask(tail_mask), sb.mask(tail_mask);
      mx_static_for<0, MB>([&](auto i_tag) __attribute__((always_inline)) {
        constexpr int i = decltype(i_tag)::value;
        mx_multiply_row<0, i>(fa[0][i], fb[0], sa, sb, acc[i]);
        mx_multiply_row<1, i>(fa[1][i], fb[1], sa, sb, acc[i]);
      });
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
