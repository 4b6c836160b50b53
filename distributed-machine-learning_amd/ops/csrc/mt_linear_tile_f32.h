// 64 x 64 output tiles of the f32 dense layer (linear_ep.hip): exact f32 products on v_mfma_f32_16x16x4_f32, four waves of 32 x 32.
//
// The matrix instruction is the bound: 64 products a cycle and SIMD, an eighth of what LDS and the fetches could feed.  So a wave
// only has to have its operands in time: the fragments of one half of a step (16 of its 32) are read while the other half is
// multiplied, the one barrier of a step falls between them, and the step after the next is asked for right behind it.  Addresses are
// carried along; what is left of them are instructions' offsets.  Four workgroups share a CU (LDS is sized for that: five take turns
// worse, 224 us against 216 below).
//
// An element's products are summed in the order of mt_gemm_f32_tile.h: the results are the same bit for bit.  12800 x 512 -> 2048,
// forward (with GELU, z kept) / input gradient / weight gradient in four parts: 233 / 216 / 201 us, 174 at the matrix rate (library,
// products alone: 276 / 297 / 192); the tile of mt_gemm_f32_tile.h, which reads and then multiplies, products alone: 239 / 266 / 245.  128 x 128 tiles: 236 / 257 / 232.
#pragma once
#include "mt_bodies.h"
#include "mt_linear_ep.h"
#define LF_BK 32
#define LF_TILE 64
#define LF_THREADS 256
#define LF_LDS (40 * 1024)         // a quarter of a CU's; 32 KiB are used

// A wave's R*16 x R*16 block.  FULL: the forward pass; a gradient has no bias, z, activation or residual.
template <int R, bool FULL>
__device__ __forceinline__ void lf_epilogue(const f32x4 (&acc)[R][R], int qi0, int qj0, const MtGemmGroup& g, const MtLinearEp& ep, int lane) {
  mt_ep_for_act(FULL ? ep.act : MT_ACT_NONE, [&](auto act) {
#pragma unroll
    for (int n = 0; n < R; ++n) {
      const int col = qj0 + n * 16 + (lane >> 4) * 4;
      f32x4 bb = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (FULL && ep.bias != nullptr && col + j < g.J) bb[j] = mt_ep_bias(ep, col + j);
#pragma unroll
      for (int m = 0; m < R; ++m) {
        const int row = qi0 + m * 16 + (lane & 15);
        if (row >= g.I || col >= g.J) continue;
        if (ep.part != nullptr) {
          mt_ep_put_part(ep.part, row, col, g.J, acc[m][n]);
          continue;
        }
        const bool whole = col + 4 <= g.J;
        f32x4 v = acc[m][n] + bb;
        auto put = [&](void* base, int ld) {
          float* p = reinterpret_cast<float*>(base) + (size_t)row * ld + col;
          if (whole) __builtin_memcpy(p, &v, 16);
          else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (col + j < g.J) p[j] = v[j];
          }
        };
        if (FULL && ep.z != nullptr) put(ep.z, ep.ldz);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = mt_ep_act<false>(v[j], act.value);
        if (FULL && ep.residual != nullptr) {
          const float* p = reinterpret_cast<const float*>(ep.residual) + (size_t)row * ep.ldr + col;
          f32x4 r = {0.f, 0.f, 0.f, 0.f};
          if (whole) __builtin_memcpy(&r, p, 16);
          else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (col + j < g.J) r[j] = p[j];
          }
          v += r;
        }
        put(g.C, g.ldc);
      }
    }
  });
}

// One operand of a step: 64 rows (K-major, 32 of the contraction in 128 bytes: chunk c of row r at c ^ (r & 7)) or 32 rows of the
// contraction with 64 columns (MN-major: chunk c of row r at c ^ (r & 4)).  A wave fetches two pieces of 1 KiB.
template <bool KMAJ> struct LfOperand {
  static constexpr int T = LF_TILE;
  const float* next;         // first element of the next step
  int64_t step;
  uint32_t at[T / 32];       // byte offset of this lane's chunk of a piece; past every range where the chunk is outside the matrix
  uint32_t bytes;            // range from `next` on
  int left, rows, pitch;
  __device__ __forceinline__ void start(const void* base, int ld, int mn0, int mn_lim, int KK, int wave, int lane) {
    left = KK;
    rows = mn_lim - mn0 < T ? mn_lim - mn0 : T;
    pitch = ld * 4;
    next = reinterpret_cast<const float*>(base) + (KMAJ ? (int64_t)mn0 * ld : (int64_t)mn0);
    step = KMAJ ? LF_BK : (int64_t)LF_BK * ld;
    bytes = KMAJ ? (uint32_t)(rows - 1) * (uint32_t)pitch + 128 : (LF_BK - 1) * (uint32_t)pitch + (uint32_t)((rows + 3) & ~3) * 4;
#pragma unroll
    for (int t = 0; t < T / 32; ++t) {
      const int j = wave * (T / 32) + t;
      if (KMAJ) {
        const int r = j * 8 + (lane >> 3);
        at[t] = (uint32_t)r * (uint32_t)pitch + (((lane & 7) ^ (r & 7)) << 4);
      } else {
        const int r = j * (256 / T) + lane / (T / 4), c = (lane % (T / 4)) ^ (r & 4);
        at[t] = c * 4 < rows ? (uint32_t)r * (uint32_t)pitch + c * 16 : 0xFFFFFF00u;
      }
    }
  }
  __device__ __forceinline__ void fetch(uint32_t img, int wave, int lane) {
    if (left < LF_BK) {            // the last step, and those asked for behind it
      bytes = 0;
      if (left > 0) bytes = KMAJ ? (uint32_t)(rows - 1) * (uint32_t)pitch + (uint32_t)((left + 3) & ~3) * 4
                                 : (uint32_t)(left - 1) * (uint32_t)pitch + (uint32_t)((rows + 3) & ~3) * 4;
      if (KMAJ) {
#pragma unroll
        for (int t = 0; t < T / 32; ++t) at[t] = ((lane & 7) ^ (lane >> 3)) * 4 < left ? at[t] : 0xFFFFFF00u;
      }
    }
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<float*>(next), 0, bytes, 0x00027000);
#pragma unroll
    for (int t = 0; t < T / 32; ++t)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)(uintptr_t)(img + (wave * (T / 32) + t) * 1024), 16,
                                               at[t], 0, 0, 0);
    next += step;
    left -= LF_BK;
  }
};
// Fragments: rows or columns 16 m + (lane & 15) of the wave's block, k = 16 ks + 4 (lane / 16) + 0..3.
template <bool KMAJ> struct LfFrag {
  static constexpr int T = LF_TILE;
  uint32_t lane_at, at[2];
  __device__ __forceinline__ void start(int lane, uint32_t img, int block) {
    const int i = lane & 15, g = lane >> 4;
    if (KMAJ) lane_at = img + block * (T / 2) * 128 + i * 128 + ((g ^ (i & 7)) << 4);
    else lane_at = img + block * (T / 2) * 4 + g * 16 * T + (g & 1) * 64 + i * 4;
  }
  __device__ __forceinline__ void stage(uint32_t st) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      at[e] = (lane_at ^ (e * 64)) + st;
      asm volatile("" : "+v"(at[e]));
    }
  }
  __device__ __forceinline__ f32x4 read(int m, int ks) const {
    if constexpr (KMAJ) {
      return *(const __attribute__((address_space(3))) f32x4*)(uintptr_t)(at[ks] + m * 2048);
    } else {
      f32x4 v;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        v[e] = *(const __attribute__((address_space(3))) float*)(uintptr_t)(at[m & 1] + (m >> 1) * 128 + (16 * ks + e) * T * 4);
      return v;
    }
  }
};

// One tile (ti, tj).  MODE 0: A [I][KK] and B [J][KK]; 1: B [KK][J]; 2: A [KK][I], B [KK][J], and with want_db the sums of A's columns
// to g.aux_out.  Leading dimensions below LF_MAX_LD keep a tile's byte offsets in 32 bits.
#define LF_MAX_LD (1 << 24)
template <int MODE>
__device__ __forceinline__ void linear_tile_f32(const MtGemmGroup& g, int ti, int tj, bool want_db, uint8_t* lds, const MtLinearEp& ep) {
  constexpr bool A_KMAJ = MODE != 2, B_KMAJ = MODE == 0;
  constexpr int T = LF_TILE, R = T / 32, IMG = T * 128, STAGE = 2 * IMG;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wr = wave >> 1, wc = wave & 1;
  const int i0 = ti * T, j0 = tj * T;
  const uint32_t base = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) uint8_t*)lds;
  LfOperand<A_KMAJ> A;
  LfOperand<B_KMAJ> B;
  LfFrag<A_KMAJ> fa;
  LfFrag<B_KMAJ> fb;
  A.start(g.A, g.lda, i0, g.I, g.KK, wave, lane);
  B.start(g.B, g.ldb, j0, g.J, g.KK, wave, lane);
  fa.start(lane, base, wr);
  fb.start(lane, base + IMG, wc);
  f32x4 acc[R][R];
#pragma unroll
  for (int m = 0; m < R; ++m)
#pragma unroll
    for (int n = 0; n < R; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};
  float db[R] = {};
  const int n_it = (g.KK + LF_BK - 1) / LF_BK;
  f32x4 a[2][R], b[2][R];
  auto read = [&](int ks) {
#pragma unroll
    for (int m = 0; m < R; ++m) a[ks][m] = fa.read(m, ks);
#pragma unroll
    for (int n = 0; n < R; ++n) b[ks][n] = fb.read(n, ks);
  };
  auto multiply = [&](int ks) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int m = 0; m < R; ++m)
#pragma unroll
        for (int n = 0; n < R; ++n) acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x4f32(b[ks][n][e], a[ks][m][e], acc[m][n], 0, 0, 0);
    if (MODE == 2 && want_db) {
#pragma unroll
      for (int m = 0; m < R; ++m) db[m] += (a[ks][m][0] + a[ks][m][1]) + (a[ks][m][2] + a[ks][m][3]);
    }
  };
  A.fetch(base, wave, lane);
  B.fetch(base + IMG, wave, lane);
  A.fetch(base + STAGE, wave, lane);
  B.fetch(base + STAGE + IMG, wave, lane);
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * (T / 32)) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  fa.stage(0);
  fb.stage(0);
  read(0);
  uint32_t st = 0;
  for (int it = 0; it < n_it; ++it) {
    read(1);
    __builtin_amdgcn_sched_barrier(0);
    multiply(0);
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    A.fetch(base + st, wave, lane);
    B.fetch(base + st + IMG, wave, lane);
    st ^= STAGE;
    fa.stage(st);
    fb.stage(st);
    read(0);
    __builtin_amdgcn_sched_barrier(0);
    multiply(1);
    __builtin_amdgcn_sched_barrier(0);
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");        // the zeros behind the last step, before the workgroup ends
  const int qi0 = i0 + wr * (T / 2), qj0 = j0 + wc * (T / 2);
  lf_epilogue<R, MODE == 0>(acc, qi0, qj0, g, ep, lane);
  if (MODE == 2 && want_db && wc == 0) {
#pragma unroll
    for (int m = 0; m < R; ++m) {
      float s = db[m];
      s += __shfl_xor(s, 16);
      s += __shfl_xor(s, 32);
      const int row = qi0 + m * 16 + lane;
      if (lane < 16 && row < g.I) mt_ep_put_db(g.aux_out, row, s, ep.bias_bf16);
    }
  }
}
