// Output tiles of the bf16 MFMA GEMMs (gemm.hip describes the layout): the four-wave 128 x 128 tile, shared by the grouped
// launches of trial packs, the single-layer launches and the dense layer with its activation and residual in the epilogue
// (linear_ep.hip), and the eight-wave 256 x 256 tile of the first two.
#pragma once
#include "mt_bodies.h"
#include "mt_linear_ep.h"

#define BM 128
#define BN 128
#define BK 64
#define NTHREADS 256
#define STAGE_BYTES 32768

typedef __attribute__((address_space(3))) uint8_t lds_u8;

__device__ __forceinline__ int kmaj_off(int row, int chunk) {       // [128][64] bf16 image
  return row * 128 + ((chunk ^ (row & 7)) << 4);
}
__device__ __forceinline__ int mnmaj_off(int row, int chunk) {      // [64][128] bf16 image
  return row * 256 + ((chunk ^ (((row & 3) << 2) | ((row >> 2) & 3))) << 4);
}
__device__ __forceinline__ int ctile_off(int row, int chunk) {      // [128][128] bf16 epilogue image
  return row * 256 + ((chunk ^ (row & 15)) << 4);
}

// ---- global -> LDS by LDS-DMA (4 x 1 KiB pieces per wave per operand image) ------------------------
static __device__ __attribute__((aligned(16))) uint32_t mt_zero_chunk[4];     // source of every out-of-range chunk

template <bool KMAJOR, int PIECES = 4>      // PIECES per wave: 4 with four waves, 2 with eight
__device__ __forceinline__ void stage_tile(uint8_t* img, const uint16_t* __restrict__ base, int ld, int mn0, int mn_lim,
                                           int k0, int k_lim, int wave, int lane) {
#pragma unroll
  for (int t = 0; t < PIECES; ++t) {
    const int j = wave * PIECES + t;   // which 1-KiB piece of the 16-KiB image this instruction fills
    int row, col;
    bool ok;
    if (KMAJOR) {      // image row r = 128 B = 8 chunks; slot s of row r holds chunk s ^ (r & 7)
      const int r = j * 8 + (lane >> 3);
      const int c = (lane & 7) ^ (r & 7);
      row = mn0 + r;
      col = k0 + c * 8;
      ok = (row < mn_lim) && (col < k_lim);
    } else {           // image row r = 256 B = 16 chunks; slot s holds chunk s ^ ((r&3)<<2 | (r>>2)&3)
      const int r = j * 4 + (lane >> 4);
      const int c = (lane & 15) ^ (((r & 3) << 2) | ((r >> 2) & 3));
      row = k0 + r;
      col = mn0 + c * 8;
      ok = (row < k_lim) && (col < mn_lim);
    }
    const uint16_t* src = ok ? base + (size_t)row * ld + col : reinterpret_cast<const uint16_t*>(mt_zero_chunk);
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                     (__attribute__((address_space(3))) void*)(img + j * 1024), 16, 0, 0);
  }
}

// ---- LDS -> MFMA fragments -----------------------------------------------------------------------
// K-major: lane l holds row (l & 15), kk = 32*ks + 8*(l >> 4) + 0..7  -> one 16-B chunk.
__device__ __forceinline__ bf16x8 frag_kmajor(const uint8_t* lds, int row0, int ks, int lane) {
  const int row = row0 + (lane & 15);
  const int chunk = ks * 4 + (lane >> 4);
  return __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(lds + kmaj_off(row, chunk)));
}
// MN-major: per 16-lane group g the two transposed reads cover kk rows 32*ks + 8g + {0..3} and
// {4..7}; lane 4q+p of the group addresses row q, columns 4p..4p+3 of the 16-column block and
// receives column (l & 15) of the four rows.
__device__ __forceinline__ bf16x8 frag_mnmajor(const uint8_t* lds, int col0, int ks, int lane) {
  const int g = lane >> 4, i = lane & 15, q = i >> 2, p = i & 3;
  const int c0 = col0 >> 3;
  const int r0 = ks * 32 + g * 8 + q;
  const lds_u8* a0 = (const lds_u8*)(lds + mnmaj_off(r0, c0 + (p >> 1)) + 8 * (p & 1));
  const lds_u8* a1 = (const lds_u8*)(lds + mnmaj_off(r0 + 4, c0 + (p >> 1)) + 8 * (p & 1));
  s16x4 lo = mt_read_tr((__attribute__((address_space(3))) s16x4*)a0);
  s16x4 hi = mt_read_tr((__attribute__((address_space(3))) s16x4*)a1);
  typedef __attribute__((ext_vector_type(8))) short s16x8;
  s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  return __builtin_bit_cast(bf16x8, v);
}

// All MFMAs of one 64-deep stage for this wave's 64x64 sub-tile (operands swapped, see header).
template <bool A_KMAJ, bool B_KMAJ>
__device__ __forceinline__ void mma_stage(f32x4 (&acc)[4][4], const uint8_t* ldsA, const uint8_t* ldsB, int wr, int wc,
                                          int lane, int flags) {
#pragma unroll
  for (int ks = 0; ks < 2; ++ks) {
    bf16x8 a_[4], b_[4];
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      if constexpr (A_KMAJ) a_[m] = frag_kmajor(ldsA, wr * 64 + m * 16, ks, lane);
      else a_[m] = frag_mnmajor(ldsA, wr * 64 + m * 16, ks, lane);
    }
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      if constexpr (B_KMAJ) b_[n] = frag_kmajor(ldsB, wc * 64 + n * 16, ks, lane);
      else b_[n] = frag_mnmajor(ldsB, wc * 64 + n * 16, ks, lane);
    }
    if (!(flags & 256)) {
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int n = 0; n < 4; ++n)
          acc[m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b_[n], a_[m], acc[m][n], 0, 0, 0);
    } else {       // timing-only ablation: fragments stay live, matrix pipe idle
#pragma unroll
      for (int m = 0; m < 4; ++m) asm volatile("" ::"v"(a_[m]), "v"(b_[m]));
    }
  }
}

// Column sums of the MN-major A image (bias gradient): thread -> column (tid & 127), half of the 64 rows.
__device__ __forceinline__ float colsum_stage(const uint8_t* ldsA, int tid) {
  const int col = tid & 127, half = tid >> 7;
  float s = 0.f;
#pragma unroll 8
  for (int r = 0; r < 32; ++r) {
    const int row = half * 32 + r;
    const uint16_t v = *reinterpret_cast<const uint16_t*>(ldsA + mnmaj_off(row, col >> 3) + (col & 7) * 2);
    s += bf16_bits_to_f32(v);
  }
  return s;
}

// ---- dense-layer epilogue (linear_ep.hip) -----------------------------------------------------------
// A wave's R*16 x 64 block.  `img` is its own [R*16][64] bf16 staging image: an accumulator lane holds 4 columns of a row, so
// stores go through LDS as whole 16-byte pieces of 128-byte row segments, and the residual comes in the same way.  Rows of
// the output need no alignment (columns past J are left alone); LDS traffic stays inside the wave, which executes in order.
// FULL: the forward pass; a gradient has no bias, z, activation or residual.
template <int R, bool FULL>
__device__ __forceinline__ void mt_linear_epilogue(const f32x4 (&acc)[R][4], uint8_t* img, int qi0, int qj0, const MtGemmGroup& g,
                                                   const MtLinearEp& ep, int lane) {
  const int fq = lane >> 4, fr = lane & 15;
  if (ep.part != nullptr) {
#pragma unroll
    for (int m = 0; m < R; ++m)
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int row = qi0 + m * 16 + fr, col = qj0 + n * 16 + fq * 4;
        if (row < g.I && col < g.J) mt_ep_put_part(ep.part, row, col, g.J, acc[m][n]);
      }
    return;
  }
  auto fence = [] {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
  };
  auto flush = [&](uint16_t* dst, int ld) {
    fence();
#pragma unroll 4
    for (int t = 0; t < 2 * R; ++t) {
      const int q = lane + 64 * t, lrow = q >> 3, ch = q & 7;
      const int row = qi0 + lrow, col = qj0 + ch * 8;
      const u32x4 v = *reinterpret_cast<const u32x4*>(img + kmaj_off(lrow, ch));
      if (row >= g.I || col >= g.J) continue;
      uint16_t* p = dst + (size_t)row * ld + col;
      if (col + 8 <= g.J) {
        __builtin_memcpy(p, &v, 16);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (col + e < g.J) p[e] = (uint16_t)(v[e >> 1] >> (16 * (e & 1)));
      }
    }
    fence();
  };
  auto bias4 = [&](int n) {
    f32x4 b = {0.f, 0.f, 0.f, 0.f};
    if (FULL && ep.bias != nullptr) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int col = qj0 + n * 16 + fq * 4 + j;
        if (col < g.J) b[j] = mt_ep_bias(ep, col);
      }
    }
    return b;
  };
  const bool residual = FULL && ep.residual != nullptr;
  if (FULL && ep.z != nullptr) {
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const f32x4 b = bias4(n);
#pragma unroll
      for (int m = 0; m < R; ++m) {
        const int lrow = m * 16 + fr, lcol = n * 16 + fq * 4;
        const f32x4 v = acc[m][n] + b;
        *reinterpret_cast<u32x2*>(img + kmaj_off(lrow, lcol >> 3) + (lcol & 7) * 2) =
            u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
      }
    }
    flush(reinterpret_cast<uint16_t*>(ep.z), ep.ldz);
  }
  if (residual) {
    const uint16_t* res = reinterpret_cast<const uint16_t*>(ep.residual);
#pragma unroll 4
    for (int t = 0; t < 2 * R; ++t) {
      const int q = lane + 64 * t, lrow = q >> 3, ch = q & 7;
      const int row = qi0 + lrow, col = qj0 + ch * 8;
      u32x4 v = {0u, 0u, 0u, 0u};
      if (row < g.I && col < g.J) {
        const uint16_t* p = res + (size_t)row * ep.ldr + col;
        if (col + 8 <= g.J) {
          __builtin_memcpy(&v, p, 16);
        } else {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (col + e < g.J) v[e >> 1] |= (uint32_t)p[e] << (16 * (e & 1));
        }
      }
      *reinterpret_cast<u32x4*>(img + kmaj_off(lrow, ch)) = v;
    }
    fence();
  }
  mt_ep_for_act(FULL ? ep.act : MT_ACT_NONE, [&](auto act) {
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const f32x4 b = bias4(n);
#pragma unroll
      for (int m = 0; m < R; ++m) {
        const int lrow = m * 16 + fr, lcol = n * 16 + fq * 4;
        u32x2* at = reinterpret_cast<u32x2*>(img + kmaj_off(lrow, lcol >> 3) + (lcol & 7) * 2);
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = mt_ep_act<true>(acc[m][n][j] + b[j], act.value);
        if (residual) {
          const u32x2 r = *at;
#pragma unroll
          for (int j = 0; j < 4; ++j) v[j] += bf16_bits_to_f32((r[j >> 1] >> (16 * (j & 1))) & 0xFFFFu);
        }
        *at = u32x2{pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
      }
    }
  });
  flush(reinterpret_cast<uint16_t*>(g.C), g.ldc);
}

// One 128x128 output tile.  ksplits > 1 (wgrad only): tile.ti (int16) carries the split index in bits 8..14,
// so at most 127 splits.
template <int MODE, int NSTAGE, bool EP = false>
__device__ __forceinline__ void gemm_tile(const MtGemmGroup* __restrict__ groups, const MtTile tile, int step,
                                          int flags, int arow0, int i_override, int ksplits, size_t split_stride,
                                          uint8_t* lds, const MtLinearEp* ep = nullptr) {
  constexpr bool A_KMAJ = (MODE != 2);
  constexpr bool B_KMAJ = (MODE == 0);
  if (tile.group < 0) return;   // padding entry of an XCD-balanced tile list
  MtGemmGroup g = groups[tile.group];
  if (step >= g.active_steps) return;
  if (i_override > 0) {   // evaluation: every group reads rows [arow0, arow0 + i_override) of a shared A
    g.I = i_override;
    g.A = reinterpret_cast<const uint16_t*>(g.A) + (size_t)arow0 * g.lda;
  }
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wr = wave >> 1, wc = wave & 1;
  const int split = (MODE == 2) ? (tile.ti >> 8) : 0;
  const int i0 = (MODE == 2 ? (tile.ti & 0xFF) : (int)tile.ti) * BM, j0 = tile.tj * BN;   // only wgrad tiles carry a split index
  if (i0 >= g.I || j0 >= g.J) return;
  const uint16_t* A = reinterpret_cast<const uint16_t*>(g.A);
  const uint16_t* B = reinterpret_cast<const uint16_t*>(g.B);

  f32x4 acc[4][4];
#pragma unroll
  for (int m = 0; m < 4; ++m)
#pragma unroll
    for (int n = 0; n < 4; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};

  const bool want_db = (MODE == 2) && (flags & MT_GEMM_FLAG_DBIAS) && tile.tj == 0 && g.aux_out != nullptr;
  float db_acc = 0.f;

  const int nk_all = (g.KK + BK - 1) / BK;
  int kt_lo = 0, kt_hi = nk_all;
  if (MODE == 2 && ksplits > 1) {
    const int per = (nk_all + ksplits - 1) / ksplits;
    kt_lo = split * per;
    kt_hi = (kt_lo + per < nk_all) ? kt_lo + per : nk_all;
  }

  const int wave_u = __builtin_amdgcn_readfirstlane(wave);
  const int n_it = kt_hi - kt_lo;
  auto issue = [&](int slot, int kt) {      // 8 LDS-DMA pieces per wave: tile kt -> stage `slot`
    stage_tile<A_KMAJ>(lds + slot * STAGE_BYTES, A, g.lda, i0, g.I, kt * BK, g.KK, wave_u, lane);
    stage_tile<B_KMAJ>(lds + slot * STAGE_BYTES + 16384, B, g.ldb, j0, g.J, kt * BK, g.KK, wave_u, lane);
  };

  if constexpr (NSTAGE == 2) {
    // Two stages, two workgroups per CU (throughput form).  Tile it+2 refills the stage tile `it` just
    // vacated, so two barriers per K-step; the other workgroup on the CU covers the bubbles.
    if (n_it > 0) issue(0, kt_lo);
    if (n_it > 1) issue(1, kt_lo + 1);
    for (int it = 0; it < n_it; ++it) {
      const int cur = it & 1;
      const uint8_t* ldsA = lds + cur * STAGE_BYTES;
      // this wave's 8 pieces of tile `it` have landed once at most the 8 pieces of tile it+1 are outstanding
      if (it + 1 < n_it) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();          // ... and after the barrier so have everybody else's
      mma_stage<A_KMAJ, B_KMAJ>(acc, ldsA, ldsA + 16384, wr, wc, lane, flags);
      if (want_db) db_acc += colsum_stage(ldsA, tid);
      asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();          // every wave is done reading this stage: it may be refilled
      if (it + 2 < n_it && !(flags & 512)) issue(cur, kt_lo + it + 2);
    }
  } else {
    // NSTAGE stages, one workgroup per CU (latency form, for packs with fewer tiles than CUs): NSTAGE-1
    // tiles stay in flight and ONE barrier per K-step both publishes tile `it` and proves that everybody
    // has finished tile it-1, whose stage is refilled right away.
#pragma unroll
    for (int p = 0; p < NSTAGE - 1; ++p)
      if (p < n_it) issue(p, kt_lo + p);
    for (int it = 0; it < n_it; ++it) {
      const int ahead = (n_it - 1 - it) < (NSTAGE - 2) ? (n_it - 1 - it) : (NSTAGE - 2);
      if (ahead >= 2) asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
      else if (ahead == 1) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __builtin_amdgcn_s_barrier();
      const int nxt = it + NSTAGE - 1;
      if (nxt < n_it && !(flags & 512)) issue(nxt % NSTAGE, kt_lo + nxt);
      const uint8_t* ldsA = lds + (it % NSTAGE) * STAGE_BYTES;
      mma_stage<A_KMAJ, B_KMAJ>(acc, ldsA, ldsA + 16384, wr, wc, lane, flags);
      if (want_db) db_acc += colsum_stage(ldsA, tid);
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();            // the epilogues reuse stage 0
  }

  // ------------------------------------------------------------------------------ epilogues
  if constexpr (EP) {
    mt_linear_epilogue<4, MODE == 0>(acc, lds + wave * 8192, i0 + wr * 64, j0 + wc * 64, g, *ep, lane);
    if (want_db) {
      __syncthreads();                               // the staging images are read
      float* red = reinterpret_cast<float*>(lds);
      red[tid] = db_acc;
      __syncthreads();
      if (tid < 128 && i0 + tid < g.I) mt_ep_put_db(g.aux_out, i0 + tid, red[tid] + red[tid + 128], ep->bias_bf16);
    }
    return;
  }
  const int fq = lane >> 4, fr = lane & 15;
  if (flags & 1024) {       // timing-only: keep the accumulators alive, store nothing
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int n = 0; n < 4; ++n) asm volatile("" ::"v"(acc[m][n]));
    return;
  }
  if (MODE == 2) {
    float* C = reinterpret_cast<float*>(g.C) + (size_t)split * split_stride;
#pragma unroll
    for (int m = 0; m < 4; ++m) {
      const int row = i0 + wr * 64 + m * 16 + fr;
#pragma unroll
      for (int n = 0; n < 4; ++n) {
        const int col = j0 + wc * 64 + n * 16 + fq * 4;
        if (row < g.I) {
          float* dst = C + (size_t)row * g.ldc + col;
          if (col + 3 < g.J) *reinterpret_cast<f32x4*>(dst) = acc[m][n];
          else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              if (col + j < g.J) dst[j] = acc[m][n][j];
          }
        }
      }
    }
    if (want_db) {
      float* red = reinterpret_cast<float*>(lds);    // all waves are past the last K-step barrier
      red[tid] = db_acc;
      __syncthreads();
      if (tid < 128 && i0 + tid < g.I)
        (reinterpret_cast<float*>(g.aux_out) + (size_t)split * split_stride)[i0 + tid] = red[tid] + red[tid + 128];
    }
    return;
  }

  {
    const bool relu = (MODE == 0) && (flags & MT_GEMM_FLAG_RELU);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int lcol = wc * 64 + n * 16 + fq * 4;
      float bb[4] = {0.f, 0.f, 0.f, 0.f};
      if (MODE == 0 && g.aux != nullptr) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j0 + lcol + j < g.J) bb[j] = reinterpret_cast<const float*>(g.aux)[j0 + lcol + j];
      }
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        const int lrow = wr * 64 + m * 16 + fr;
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[j] = acc[m][n][j] + bb[j];
          if (relu) v[j] = fmaxf(v[j], 0.f);
        }
        u32x2 pk = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
        *reinterpret_cast<u32x2*>(lds + ctile_off(lrow, lcol >> 3) + (lcol & 7) * 2) = pk;
      }
    }
    __syncthreads();
    uint16_t* C = reinterpret_cast<uint16_t*>(g.C);
    const uint16_t* msk = (MODE == 1 && (flags & MT_GEMM_FLAG_MASK)) ? reinterpret_cast<const uint16_t*>(g.aux)
                                                                    : nullptr;
    u32x4 hv[8];
    if (msk != nullptr) {
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const int q = tid + NTHREADS * t;
        const int row = i0 + (q >> 4), col = j0 + (q & 15) * 8;
        const bool ok = (row < g.I && col < g.J);
        hv[t] = *reinterpret_cast<const u32x4*>(msk + (ok ? ((size_t)row * g.ldaux + col) : (size_t)0));
      }
    }
#pragma unroll
    for (int t = 0; t < 8; ++t) {
      const int q = tid + NTHREADS * t;
      const int lrow = q >> 4, ch = q & 15;
      const int row = i0 + lrow, col = j0 + ch * 8;
      u32x4 v = *reinterpret_cast<const u32x4*>(lds + ctile_off(lrow, ch));
      if (msk != nullptr) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t hw = hv[t][e];
          const uint32_t lo_ok = ((hw & 0x8000u) == 0u && (hw & 0x7FFFu) != 0u) ? 0x0000FFFFu : 0u;
          const uint32_t hi_ok = ((hw & 0x80000000u) == 0u && (hw & 0x7FFF0000u) != 0u) ? 0xFFFF0000u : 0u;
          v[e] &= (lo_ok | hi_ok);
        }
      }
      if (row < g.I && col < g.J) *reinterpret_cast<u32x4*>(C + (size_t)row * g.ldc + col) = v;
    }
  }
}

#define BIGT 256
#define BIG_STAGE_BYTES 65536

// ====================================================================================================
// 256 x 256 output tiles on EIGHT waves, fragment reads software-pipelined under the MFMAs: the form for one large GEMM
// (layers thousands wide, a data-parallel trial).  A 128-tile stages 32 KB per 2*128*128*64 flop and, with its two
// barriers per K-step, tops out near a third of the matrix peak; this tile stages half the bytes per flop, and each
// SIMD holds two waves, so one wave's ds_reads and barrier waits sit under the other's MFMAs.
//
// Waves 2 (rows) x 4 (columns): wave (wr, wc) owns rows wr*128..+128, columns wc*64..+64 = 8 x 4 accumulators (128
// registers).  A stage is the same four 16-KiB images as above [A rows 0-127 | A rows 128-255 | B cols 0-127 | B cols
// 128-255], two stages = 128 KiB, one workgroup per CU.  One K-tile (64 deep) is four groups of 16 MFMAs -- (ks, row
// half) -- and the reads of group q+1 are issued before the MFMAs of group q:
//     read A(ks0, lo), B(ks0) | MFMA(ks1, hi) of tile k-1 | read A(ks0, hi) | MFMA(ks0, lo) | read A(ks1, lo), B(ks1) |
//     MFMA(ks0, hi) | read A(ks1, hi) | MFMA(ks1, lo) | barrier | LDS-DMA of tile k+2 into the stage just read
// so every batch of ds_reads has 16 MFMAs (512 matrix-pipe cycles) to come back, and a K-tile costs ONE barrier.
// An element's contraction is still summed in K order, so results equal the 128-tile kernels' bit for bit.
#define P8_THREADS 512

template <bool A_KMAJ>
__device__ __forceinline__ void p8_read_a(bf16x8 (&a)[4], const uint8_t* imgA, int mh, int ks, int lane) {
#pragma unroll
  for (int m = 0; m < 4; ++m) {
    if constexpr (A_KMAJ) a[m] = frag_kmajor(imgA, (mh * 4 + m) * 16, ks, lane);
    else a[m] = frag_mnmajor(imgA, (mh * 4 + m) * 16, ks, lane);
  }
}
template <bool B_KMAJ>
__device__ __forceinline__ void p8_read_b(bf16x8 (&b)[4], const uint8_t* imgB, int col0, int ks, int lane) {
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    if constexpr (B_KMAJ) b[n] = frag_kmajor(imgB, col0 + n * 16, ks, lane);
    else b[n] = frag_mnmajor(imgB, col0 + n * 16, ks, lane);
  }
}
template <bool DRY = false>
__device__ __forceinline__ void p8_mma(f32x4 (&acc)[8][4], int mh, const bf16x8 (&a)[4], const bf16x8 (&b)[4]) {
  if constexpr (DRY) {       // timing-only ablation: fragments stay live, matrix pipe idle
#pragma unroll
    for (int m = 0; m < 4; ++m) asm volatile("" ::"v"(a[m]), "v"(b[m]));
    return;
  }
#pragma unroll
  for (int m = 0; m < 4; ++m)
#pragma unroll
    for (int n = 0; n < 4; ++n)
      acc[mh * 4 + m][n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[n], a[m], acc[mh * 4 + m][n], 0, 0, 0);
}

// One 256 x 256 tile (ti, tj) of the group; split: which part of the contraction (weight gradient only).
template <int MODE, int SCHED>
__device__ __forceinline__ void gemm_tile_p8(const MtGemmGroup& g, int ti, int tj, int split, int flags, int ksplits,
                                             size_t split_stride, uint8_t* lds) {
  constexpr bool A_KMAJ = (MODE != 2);
  constexpr bool B_KMAJ = (MODE == 0);
  constexpr int BASE = SCHED & 1;
  constexpr bool DRY = (SCHED & 8) != 0, NOFILL = (SCHED & 16) != 0;      // timing-only ablations
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int wr = wave >> 2, wc = wave & 3;
  const int i0 = ti * BIGT, j0 = tj * BIGT;
  if (i0 >= g.I || j0 >= g.J) return;
  const uint16_t* A = reinterpret_cast<const uint16_t*>(g.A);
  const uint16_t* B = reinterpret_cast<const uint16_t*>(g.B);
  const int qi0 = i0 + wr * 128, qj0 = j0 + wc * 64;                     // this wave's block of the output
  const bool live = (qi0 < g.I) && (qj0 < g.J);      // wave-uniform; a wave outside the matrix multiplies the zeros staged for it
  const int offA = wr * 16384, offB = 32768 + (wc >> 1) * 16384, bcol0 = (wc & 1) * 64;

  f32x4 acc[8][4];
#pragma unroll
  for (int m = 0; m < 8; ++m)
#pragma unroll
    for (int n = 0; n < 4; ++n) acc[m][n] = f32x4{0.f, 0.f, 0.f, 0.f};

  const bool want_db = (MODE == 2) && (flags & MT_GEMM_FLAG_DBIAS) && tj == 0 && g.aux_out != nullptr;
  float db_acc = 0.f;

  const int nk_all = (g.KK + BK - 1) / BK;
  int kt_lo = 0, kt_hi = nk_all;
  if (MODE == 2 && ksplits > 1) {
    const int per = (nk_all + ksplits - 1) / ksplits;
    kt_lo = split * per;
    kt_hi = (kt_lo + per < nk_all) ? kt_lo + per : nk_all;
  }
  const int wave_u = __builtin_amdgcn_readfirstlane(wave);
  const int n_it = kt_hi - kt_lo;
  auto issue = [&](int slot, int kt) {      // 8 LDS-DMA pieces per wave: tile kt -> the four images of stage `slot`
    uint8_t* st = lds + slot * BIG_STAGE_BYTES;
    int ln = lane;
    asm volatile("" : "+v"(ln));            // addresses are recomputed per tile instead of pinned across the loop
    stage_tile<A_KMAJ, 2>(st, A, g.lda, i0, g.I, kt * BK, g.KK, wave_u, ln);
    stage_tile<A_KMAJ, 2>(st + 16384, A, g.lda, i0 + 128, g.I, kt * BK, g.KK, wave_u, ln);
    stage_tile<B_KMAJ, 2>(st + 32768, B, g.ldb, j0, g.J, kt * BK, g.KK, wave_u, ln);
    stage_tile<B_KMAJ, 2>(st + 49152, B, g.ldb, j0 + 128, g.J, kt * BK, g.KK, wave_u, ln);
  };

  if constexpr (BASE == 0) {
  // Two barriers per K-tile: B1 publishes tile it, B2 (after this wave's last read of it) frees the stage, whose refill
  // then has the second half of this tile and the whole next one to land.
  if (n_it > 0) issue(0, kt_lo);
  if (n_it > 1) issue(1, kt_lo + 1);
  for (int it = 0; it < n_it; ++it) {
    const int cur = it & 1;
    const uint8_t* st = lds + cur * BIG_STAGE_BYTES;
    const uint8_t* imgA = st + offA;
    const uint8_t* imgB = st + offB;
    if (it + 1 < n_it) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    bf16x8 a0[4], a1[4], a2[4], a3[4], b0[4], b1[4];
    p8_read_a<A_KMAJ>(a0, imgA, 0, 0, lane);
    p8_read_b<B_KMAJ>(b0, imgB, bcol0, 0, lane);
    __builtin_amdgcn_sched_barrier(0);
    p8_read_a<A_KMAJ>(a1, imgA, 1, 0, lane);
    __builtin_amdgcn_sched_barrier(0);
    p8_mma<DRY>(acc, 0, a0, b0);
    __builtin_amdgcn_sched_barrier(0);
    p8_read_a<A_KMAJ>(a2, imgA, 0, 1, lane);
    __builtin_amdgcn_sched_barrier(0);
    p8_mma<DRY>(acc, 1, a1, b0);
    __builtin_amdgcn_sched_barrier(0);
    p8_read_b<B_KMAJ>(b1, imgB, bcol0, 1, lane);
    p8_read_a<A_KMAJ>(a3, imgA, 1, 1, lane);
    if (want_db) db_acc += colsum_stage(st + (tid >> 8) * 16384, tid & 255);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();              // every wave holds its fragments: the stage may be refilled
    if (!NOFILL && it + 2 < n_it) issue(cur, kt_lo + it + 2);
    __builtin_amdgcn_sched_barrier(0);
    p8_mma<DRY>(acc, 0, a2, b1);
    p8_mma<DRY>(acc, 1, a3, b1);
  }
  } else {
  // One barrier per K-tile: it publishes tile it+1 (this wave's pieces of it are back: vmcnt(0), nothing younger is in
  // flight yet) and proves that every wave has read the last fragment of tile it, whose stage is refilled right after.
  // The fourth MFMA group of a tile is held back until the first reads of the next tile have been issued.
  bf16x8 a3[4], b1[4];
#pragma unroll
  for (int m = 0; m < 4; ++m) { a3[m] = bf16x8{}; b1[m] = bf16x8{}; }      // tile "-1": adds +0 to the zeroed accumulators
  if (n_it > 0) issue(0, kt_lo);
  if (n_it > 1) issue(1, kt_lo + 1);
  if (n_it > 1) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
  else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  for (int it = 0; it < n_it; ++it) {
    const int cur = it & 1;
    const uint8_t* st = lds + cur * BIG_STAGE_BYTES;
    const uint8_t* imgA = st + offA;
    const uint8_t* imgB = st + offB;
    {
      bf16x8 a0[4], a1[4], a2[4], b0[4];
      p8_read_a<A_KMAJ>(a0, imgA, 0, 0, lane);
      p8_read_b<B_KMAJ>(b0, imgB, bcol0, 0, lane);
      __builtin_amdgcn_sched_barrier(0);
      p8_mma<DRY>(acc, 1, a3, b1);                      // (ks1, rows hi) of the previous tile
      __builtin_amdgcn_sched_barrier(0);
      p8_read_a<A_KMAJ>(a1, imgA, 1, 0, lane);
      __builtin_amdgcn_sched_barrier(0);
      p8_mma<DRY>(acc, 0, a0, b0);
      __builtin_amdgcn_sched_barrier(0);
      p8_read_a<A_KMAJ>(a2, imgA, 0, 1, lane);
      p8_read_b<B_KMAJ>(b1, imgB, bcol0, 1, lane);
      __builtin_amdgcn_sched_barrier(0);
      p8_mma<DRY>(acc, 1, a1, b0);
      __builtin_amdgcn_sched_barrier(0);
      p8_read_a<A_KMAJ>(a3, imgA, 1, 1, lane);
      __builtin_amdgcn_sched_barrier(0);
      p8_mma<DRY>(acc, 0, a2, b1);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (want_db) db_acc += colsum_stage(st + (tid >> 8) * 16384, tid & 255);
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    if (!NOFILL && it + 2 < n_it) issue(cur, kt_lo + it + 2);
  }
  p8_mma<DRY>(acc, 1, a3, b1);

  }
  // ------------------------------------------------------------------------------ epilogues
  const int fq = lane >> 4, fr = lane & 15;
  if (MODE == 2) {
    float* C = reinterpret_cast<float*>(g.C) + (size_t)split * split_stride;
    if (live) {
#pragma unroll
      for (int m = 0; m < 8; ++m) {
        const int row = qi0 + m * 16 + fr;
#pragma unroll
        for (int n = 0; n < 4; ++n) {
          const int col = qj0 + n * 16 + fq * 4;
          if (row < g.I) {
            float* dst = C + (size_t)row * g.ldc + col;
            if (col + 3 < g.J) *reinterpret_cast<f32x4*>(dst) = acc[m][n];
            else {
#pragma unroll
              for (int j = 0; j < 4; ++j)
                if (col + j < g.J) dst[j] = acc[m][n][j];
            }
          }
        }
      }
    }
    if (want_db) {
      float* red = reinterpret_cast<float*>(lds);    // all waves are past the last K-step barrier
      red[tid] = db_acc;
      __syncthreads();
      float* out = reinterpret_cast<float*>(g.aux_out) + (size_t)split * split_stride;
      const int t = tid & 255, row = i0 + (tid >> 8) * 128 + t;
      if (t < 128 && row < g.I) out[row] = red[tid] + red[tid + 128];
    }
    return;
  }
  if (!live) return;
  {
    uint8_t* img = lds + wave * 16384;       // this wave's own [128][64] bf16 staging image (wave-private: no barrier)
    const bool relu = (MODE == 0) && (flags & MT_GEMM_FLAG_RELU);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      const int lcol = n * 16 + fq * 4;
      float bb[4] = {0.f, 0.f, 0.f, 0.f};
      if (MODE == 0 && g.aux != nullptr) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (qj0 + lcol + j < g.J) bb[j] = reinterpret_cast<const float*>(g.aux)[qj0 + lcol + j];
      }
#pragma unroll
      for (int m = 0; m < 8; ++m) {
        const int lrow = m * 16 + fr;
        float v[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[j] = acc[m][n][j] + bb[j];
          if (relu) v[j] = fmaxf(v[j], 0.f);
        }
        u32x2 pk = {pack_bf16x2(v[0], v[1]), pack_bf16x2(v[2], v[3])};
        *reinterpret_cast<u32x2*>(img + kmaj_off(lrow, lcol >> 3) + (lcol & 7) * 2) = pk;
      }
    }
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    uint16_t* C = reinterpret_cast<uint16_t*>(g.C);
    const uint16_t* msk = (MODE == 1 && (flags & MT_GEMM_FLAG_MASK)) ? reinterpret_cast<const uint16_t*>(g.aux)
                                                                    : nullptr;
#pragma unroll 1
    for (int t0 = 0; t0 < 16; t0 += 8) {
      u32x4 hv[8];
      if (msk != nullptr) {
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          const int q = lane + 64 * (t0 + t);
          const int row = qi0 + (q >> 3), col = qj0 + (q & 7) * 8;
          const bool ok = (row < g.I && col < g.J);
          hv[t] = *reinterpret_cast<const u32x4*>(msk + (ok ? ((size_t)row * g.ldaux + col) : (size_t)0));
        }
      }
#pragma unroll
      for (int t = 0; t < 8; ++t) {
        const int q = lane + 64 * (t0 + t);
        const int lrow = q >> 3, ch = q & 7;
        const int row = qi0 + lrow, col = qj0 + ch * 8;
        u32x4 v = *reinterpret_cast<const u32x4*>(img + kmaj_off(lrow, ch));
        if (msk != nullptr) {
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const uint32_t hw = hv[t][e];
            const uint32_t lo_ok = ((hw & 0x8000u) == 0u && (hw & 0x7FFFu) != 0u) ? 0x0000FFFFu : 0u;
            const uint32_t hi_ok = ((hw & 0x80000000u) == 0u && (hw & 0x7FFF0000u) != 0u) ? 0xFFFF0000u : 0u;
            v[e] &= (lo_ok | hi_ok);
          }
        }
        if (row < g.I && col < g.J) *reinterpret_cast<u32x4*>(C + (size_t)row * g.ldc + col) = v;
      }
    }
  }
}

// Which single GEMMs take the 256-tile: enough tiles, a contraction of at least four K-tiles per workgroup and an output at
// least two tiles wide and high (measured at p8_limit in gemm.hip).
static inline bool mt_p8_rule(int rows, int cols, int depth, int ksplits, int least) {
  if (least <= 0) return false;
  const long n = (long)((rows + BIGT - 1) / BIGT) * ((cols + BIGT - 1) / BIGT) * ksplits;
  return rows >= 2 * BIGT && cols >= 2 * BIGT && depth / ksplits >= 4 * BK && n >= least;
}
