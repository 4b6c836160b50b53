// 256 x 256 output tiles of the dense layer (linear_ep.hip), bf16, eight waves that take turns.
//
// Waves 0-3 own the upper 128 rows of the tile, waves 4-7 the lower; wave (wr, wc) owns 128 x 64 of it, 8 x 4 accumulators.  A SIMD
// holds one wave of each half.  A step of 64 of the contraction is two phases per half: read the fragments of B and of the first 64
// rows of A, multiply (32 instructions), read the other 64 rows of A, multiply; barriers keep the lower half one phase behind, so
// that on every SIMD one wave multiplies while the other reads LDS and asks for the tiles to come.  What a phase read is free for
// the next fetch a phase later, so B and half of A are asked for seven phases before their first use and the rest of A six, in
// two 64-KiB stages.
//
// An element's products are summed in order of k, 32 at a time, as in the tiles of mt_gemm_tile.h: the results are the same bit for
// bit.  8192 x 8192 x 8192, forward / input gradient / weight gradient: 744 / 746 / 752 us (1470 TFLOP/s; 1618 / 1412 / 1185 for
// the library; in a training pass with GELU 784 / 725 / 761), where the 256-tile of mt_gemm_tile.h takes 873 / 995 / 969 us: its waves all read, then all multiply, and
// computing 64-bit addresses costs it as many instructions as the products.  Here the matrix cores are busy 76 % of the cycles, at
// 1.7 GHz: power, as much as the barriers, is what is left.
#pragma once
#include "mt_gemm_tile.h"

// One operand of the tile: 256 rows (K-major) or columns (MN-major) x 64 of the contraction as four blocks of 8 KiB, block b
// covering rows or columns 64 b .. 64 b + 63.  K-major block: [64 rows][64 k], chunk c of row r at c ^ (r & 7).  MN-major block:
// [64 k][64 columns], chunk c of row r at c ^ 2 f(r), f(r) = bit 1 of r + 2 bit 3 of r, which puts the eight rows x 32 bytes that
// half a wave's transposed read takes on all banks.  A wave fetches four 1-KiB pieces, two in each block of its half: piece t goes
// to block 2 (wave / 4) + t / 2.  Rows, columns and depth outside the matrix arrive as zeros through the buffer's range check.
template <bool KMAJ> struct LtOperand {
  const uint16_t* next;      // first element of the next tile
  int64_t step;
  uint32_t at[4];            // byte offset of this lane's chunk of piece t; past every range where the chunk is outside the matrix
  uint32_t bytes;            // range from `next` on
  int left, rows, pitch;     // contraction left from `next` on; rows (K-major) or columns of the tile inside the matrix; bytes per row
  __device__ __forceinline__ void start(const void* base, int ld, int mn0, int mn_lim, int KK, int wave, int lane) {
    left = KK;
    rows = mn_lim - mn0 < 256 ? mn_lim - mn0 : 256;
    pitch = ld * 2;
    next = reinterpret_cast<const uint16_t*>(base) + (KMAJ ? (int64_t)mn0 * ld : (int64_t)mn0);
    step = KMAJ ? 64 : (int64_t)64 * ld;
    bytes = KMAJ ? (uint32_t)(rows - 1) * (uint32_t)pitch + 128 : 63 * (uint32_t)pitch + (uint32_t)((rows + 7) & ~7) * 2;
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int block = (wave >> 2) * 2 + (t >> 1), r = ((wave & 3) * 2 + (t & 1)) * 8 + (lane >> 3);
      if (KMAJ) {
        at[t] = (uint32_t)(block * 64 + r) * (uint32_t)pitch + (((lane & 7) ^ (r & 7)) << 4);
      } else {
        const int c = block * 8 + ((lane & 7) ^ ((r & 2) | ((r & 8) >> 1)));
        at[t] = c * 8 < rows ? (uint32_t)r * (uint32_t)pitch + c * 16 : 0xFFFFFF00u;
      }
    }
  }
  // pieces FROM .. TO - 1 of the next tile into the blocks at LDS address `img`
  template <int FROM, int TO> __device__ __forceinline__ void fetch(uint32_t img, int wave, int lane) {
    if (FROM == 0 && left < 64) {            // the last tile, and those asked for behind it
      bytes = 0;
      if (left > 0) bytes = KMAJ ? (uint32_t)(rows - 1) * (uint32_t)pitch + (uint32_t)((left + 7) & ~7) * 2
                                 : (uint32_t)(left - 1) * (uint32_t)pitch + (uint32_t)((rows + 7) & ~7) * 2;
      if (KMAJ) {
#pragma unroll
        for (int t = 0; t < 4; ++t) at[t] = ((lane & 7) ^ (lane >> 3)) * 8 < left ? at[t] : 0xFFFFFF00u;
      }
    }
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<uint16_t*>(next), 0, bytes, 0x00027000);
#pragma unroll
    for (int t = FROM; t < TO; ++t)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rsrc, (__attribute__((address_space(3))) void*)(uintptr_t)(img + ((wave >> 2) * 2 + (t >> 1)) * 8192 + ((wave & 3) * 2 + (t & 1)) * 1024),
          16, at[t], 0, 0, 0);
    if (TO == 4) {
      next += step;
      left -= 64;
    }
  }
};
// Fragments of a block: 16 rows or columns from 16 n, 32 of the contraction (ks 0 or 1).
template <bool KMAJ> struct LtFrag {
  uint32_t lane_at;
  uint32_t at[KMAJ ? 2 : 4];        // of the present tile; what is left of an address is an instruction's offset
  __device__ __forceinline__ void start(int lane, uint32_t block) {
    if (KMAJ) {
      lane_at = block + (lane & 15) * 128 + (((lane >> 4) ^ (lane & 7)) << 4);
    } else {
      const int r = (lane >> 4) * 8 + ((lane & 15) >> 2), p = lane & 3;
      lane_at = block + r * 128 + (((p >> 1) ^ ((r & 2) | ((r & 8) >> 1))) << 4) + 8 * (p & 1);
    }
  }
  __device__ __forceinline__ void tile(uint32_t st) {
#pragma unroll
    for (int i = 0; i < (KMAJ ? 2 : 4); ++i) {
      at[i] = (lane_at ^ (i * (KMAJ ? 64 : 32))) + st;
      asm volatile("" : "+v"(at[i]));
    }
  }
  __device__ __forceinline__ bf16x8 read(int more, int n, int ks) const {
    if constexpr (KMAJ) {
      typedef const __attribute__((address_space(3))) u32x4 L;
      return __builtin_bit_cast(bf16x8, *(L*)(uintptr_t)(at[ks] + more + n * 2048));
    } else {
      typedef __attribute__((address_space(3))) s16x4 L;
      typedef __attribute__((ext_vector_type(8))) short s16x8;
      const s16x4 a = mt_read_tr((L*)(uintptr_t)(at[n] + more + ks * 4096));
      const s16x4 b = mt_read_tr((L*)(uintptr_t)(at[n] + more + ks * 4096 + 512));
      const s16x8 v = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
      return __builtin_bit_cast(bf16x8, v);
    }
  }
};
// f32 sum of a fragment's eight elements added to `sum`
__device__ __forceinline__ float lt_sum(bf16x8 f, float sum) {
  typedef __bf16 pair __attribute__((ext_vector_type(2)));
  const pair one = {(__bf16)1.f, (__bf16)1.f};
#pragma unroll
  for (int j = 0; j < 8; j += 2) sum = __builtin_amdgcn_fdot2_f32_bf16(pair{f[j], f[j + 1]}, one, sum, false);
  return sum;
}
// every wave of the workgroup is here; nothing moves across
__device__ __forceinline__ void lt_barrier() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
}

// One tile (ti, tj).  MODE 0: A [I][KK] and B [J][KK]; 1: B [KK][J]; 2: A [KK][I], B [KK][J], and with want_db the sums of A's columns
// to g.aux_out.  Leading dimensions below LT_MAX_LD keep a tile's byte offsets in 32 bits.
#define LT_MAX_LD (1 << 22)
#define LT_THREADS 512
template <int MODE>
__device__ __forceinline__ void linear_tile(const MtGemmGroup& g, int ti, int tj, bool want_db, uint8_t* lds, const MtLinearEp& ep) {
  constexpr bool A_KMAJ = MODE != 2, B_KMAJ = MODE == 0;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wr = wave >> 2, wc = wave & 3;
  const int i0 = ti * BIGT, j0 = tj * BIGT, qi0 = i0 + wr * 128, qj0 = j0 + wc * 64;
  const uint32_t base = (uint32_t)(uintptr_t)(lds_u8*)lds;
  LtOperand<A_KMAJ> A;
  LtOperand<B_KMAJ> B;
  LtFrag<A_KMAJ> fa;
  LtFrag<B_KMAJ> fb;
  A.start(g.A, g.lda, i0, g.I, g.KK, wave, lane);
  B.start(g.B, g.ldb, j0, g.J, g.KK, wave, lane);
  fa.start(lane, base + wr * 16384);
  fb.start(lane, base + 32768 + wc * 8192);
  f32x4 acc[8][4];
#pragma unroll
  for (int m = 0; m < 8; ++m)
#pragma unroll
    for (int n = 0; n < 4; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  float db[2] = {0.f, 0.f};        // column sums of A: wave column wc adds up blocks 2 wc and 2 wc + 1 of its half's eight
  const int n_it = (g.KK + BK - 1) / BK;
  auto fetch_low = [&](uint32_t st) {
    B.template fetch<0, 4>(st + 32768, wave, lane);
    A.template fetch<0, 2>(st, wave, lane);
  };
  auto fetch_high = [&](uint32_t st) { A.template fetch<2, 4>(st, wave, lane); };
  bf16x8 a[4][2], b[4][2];
  auto read_a = [&](int half) {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int m = 0; m < 4; ++m) a[m][ks] = fa.read(half * 8192, m, ks);
  };
  auto multiply = [&](int half) {
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int n = 0; n < 4; ++n)
          acc[half * 4 + m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[n][ks], a[m][ks], acc[half * 4 + m][n], 0, 0, 0);
    __builtin_amdgcn_s_setprio(0);
    if (MODE == 2 && want_db && (wc >> 1) == half) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) db[e] = lt_sum(wc & 1 ? a[2 + e][ks] : a[e][ks], db[e]);
    }
  };
  // The eight youngest pieces of this wave are of blocks that are read two phases or more from here; past the next barrier every
  // wave's pieces of the blocks to be read now have landed.  Tiles behind the last are fetched as zeros, so the count holds there.
  auto landed = [] { asm volatile("s_waitcnt vmcnt(8)" ::: "memory"); };
  fetch_low(base);
  fetch_high(base);
  fetch_low(base + BIG_STAGE_BYTES);
  landed();
  lt_barrier();
  if (wr == 1) lt_barrier();              // a phase behind
  uint32_t st = 0;
  for (int it = 0; it < n_it; ++it) {
    fa.tile(st);
    fb.tile(st);
#pragma unroll
    for (int n = 0; n < 4; ++n)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) b[n][ks] = fb.read(0, n, ks);
    read_a(0);
    const uint32_t other = st ^ BIG_STAGE_BYTES;
    fetch_high(base + other);
    if (wr == 1) landed();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    lt_barrier();
    multiply(0);
    if (wr == 0) landed();
    lt_barrier();
    read_a(1);
    fetch_low(base + st);
    if (wr == 1) landed();
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    lt_barrier();
    multiply(1);
    if (wr == 0) landed();
    lt_barrier();
    st = other;
  }
  if (wr == 0) lt_barrier();
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");        // the zeros, before the epilogue takes the stages
  lt_barrier();
  if (qi0 < g.I && qj0 < g.J) mt_linear_epilogue<8, MODE == 0>(acc, lds + wave * 16384, qi0, qj0, g, ep, lane);
  if (MODE == 2 && want_db) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float s = db[e];
      s += __shfl_xor(s, 16);
      s += __shfl_xor(s, 32);
      const int row = qi0 + (wc * 2 + e) * 16 + lane;
      if (lane < 16 && row < g.I) mt_ep_put_db(g.aux_out, row, s, ep.bias_bf16);
    }
  }
}
