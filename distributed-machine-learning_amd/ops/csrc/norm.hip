// Layer norm over rows of any width, forward and backward (gfx950, f32 or bf16 rows, f32 statistics).
//
//   forward : y = (x - mean) rstd w + b,  rstd = 1 / sqrt(var + eps); {mean, rstd} kept per row for the backward pass
//   backward: with u = (x - mean) rstd and g = dy w:  dx = rstd (g - mean(g) - u mean(g u)),
//             dw = sum over rows of dy u,  db = sum over rows of dy
//
// Both directions move each element once (forward 2, backward 3 tensors, and the partial rows below) and are bound by memory.  TPR
// threads share a row and keep it in registers (NV 16-byte vectors each): the variance is the mean of the centred squares, not a difference of sums, at
// no further read.  A row group walks over rows a grid apart with w and b in registers and the next row's loads issued before
// the current row's reductions, so the loads of two rows are always in flight.  The column sums of the backward pass stay in
// the same threads' registers over all their rows; a workgroup writes one partial row of each, and a second launch adds the
// partial rows in order: no atomics, the same bits every time.
//
// TPR is 16 or 64 (a part of a wave, or a wave: rows reduce by lane exchanges alone) or the whole workgroup of up to 16 waves
// (through LDS, one barrier per reduction, alternating buffers).  Rows wider than the registers of 1024 threads are read again
// for each pass.  Vectors are loaded and stored at whatever alignment the row has (global memory takes dwordx4 at any address;
// against rows on 16-byte boundaries an odd width costs 10 to 20 %: 5001 x 10000 108 us backward, x 10007 131).
//
// Measured (one copy of 1 GiB runs at 4950 GB/s): 128000 x 512 f32 forward 98 us (5350 GB/s), backward 154 (5100);
// 16384 x 4096 bf16 53 to 59 (4530 to 5050) and 99 (4070); 20000 x 4096 f32 142 (4620) and 173 (5680, part of it from the last-level
// cache).
#include "mt_common.h"

// N columns of a row or a parameter, as they lie in memory; N is 16 bytes of the ROW type.  Values are widened where they are
// used, and reread() between two uses keeps the compiler from holding the widened copies in registers in the meantime.
template <typename T> struct NormVec { static constexpr int N = 16 / (int)sizeof(T); };
template <typename T, int N> struct NormPack {
  static constexpr int W = N * (int)sizeof(T) / 4;
  uint32_t raw[W];
  __device__ __forceinline__ float get(int e) const {
    if constexpr (sizeof(T) == 4) return __uint_as_float(raw[e]);
    else return __uint_as_float((e & 1) ? raw[e >> 1] & 0xFFFF0000u : raw[e >> 1] << 16);
  }
  __device__ __forceinline__ void put(const float (&v)[N]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int e = 0; e < N; ++e) raw[e] = __float_as_uint(v[e]);
    } else {
#pragma unroll
      for (int e = 0; e < N; e += 2) raw[e >> 1] = pack_bf16x2(v[e], v[e + 1]);
    }
  }
  __device__ __forceinline__ void reread() {
#pragma unroll
    for (int i = 0; i < W; ++i) asm volatile("" : "+v"(raw[i]));
  }
};

// Drops 16-bit units from the front, zeros follow at the back.
template <int W> __device__ __forceinline__ void norm_drop(uint32_t (&r)[W], int halves) {
  if (halves & 1) {
#pragma unroll
    for (int i = 0; i < W; ++i) r[i] = (r[i] >> 16) | (i + 1 < W ? r[i + 1] << 16 : 0u);
  }
#pragma unroll
  for (int bit = 1; bit < W; bit <<= 1)
    if ((halves >> 1) & bit) {
#pragma unroll
      for (int i = 0; i < W; ++i) r[i] = i + bit < W ? r[i + bit] : 0u;
    }
}
// Columns past d arrive as zeros: the last vector of an odd row is the row's last N columns, moved down.
template <typename T, int N>
__device__ __forceinline__ void norm_load(NormPack<T, N>& o, const T* __restrict__ p, int col, int d) {
  if (col + N <= d) {
    __builtin_memcpy(o.raw, p + col, sizeof(o.raw));
  } else if (d >= N) {
    __builtin_memcpy(o.raw, p + d - N, sizeof(o.raw));
    norm_drop(o.raw, (col + N - d) * (int)sizeof(T) / 2);
  } else {
#pragma unroll
    for (int i = 0; i < NormPack<T, N>::W; ++i) o.raw[i] = 0u;
#pragma unroll 1
    for (int e = d - 1; e >= 0; --e) {
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int i = NormPack<T, N>::W - 1; i >= 0; --i) o.raw[i] = (o.raw[i] << 16) | (i > 0 ? o.raw[i - 1] >> 16 : 0u);
        o.raw[0] |= (uint32_t)__builtin_bit_cast(uint16_t, p[e]);
      } else {
#pragma unroll
        for (int i = NormPack<T, N>::W - 1; i > 0; --i) o.raw[i] = o.raw[i - 1];
        o.raw[0] = __builtin_bit_cast(uint32_t, p[e]);
      }
    }
  }
}
template <typename T, int N>
__device__ __forceinline__ void norm_store(T* __restrict__ p, const NormPack<T, N>& o, int col, int d) {
  if (col + N <= d) {
    __builtin_memcpy(p + col, o.raw, sizeof(o.raw));
  } else {
    T v[N];
    __builtin_memcpy(v, o.raw, sizeof(o.raw));
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (col + e < d) p[col + e] = v[e];
  }
}

#define NORM_ALL 0        // TPR: the whole workgroup

// Sum of K values over the TPR threads of a row.  NORM_ALL: `red` holds 2 x K x 16 floats, `turn` alternates the halves so that
// one barrier per call is enough.
template <int TPR, int K>
__device__ __forceinline__ void norm_sum(float (&v)[K], float* red, int& turn) {
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int o = (TPR == 16 ? 16 : 64) / 2; o > 0; o >>= 1) v[k] += __shfl_xor(v[k], o, 64);
  if constexpr (TPR == NORM_ALL) {
    float* buf = red + (turn & 1) * 32;
    ++turn;
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) {
#pragma unroll
      for (int k = 0; k < K; ++k) buf[k * 16 + wave] = v[k];
    }
    __syncthreads();
    const int waves = blockDim.x >> 6;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float s = 0.f;
      for (int w = 0; w < waves; ++w) s += buf[k * 16 + w];
      v[k] = s;
    }
  }
}

template <typename T, typename P, int TPR_, int NV>
__global__ __launch_bounds__(TPR_ == NORM_ALL ? 1024 : 256, TPR_ == NORM_ALL && NV <= 2 ? 5 : 1) void mt_norm_fwd_kernel(const T* __restrict__ x, const P* __restrict__ w,
                                                                            const P* __restrict__ b, T* __restrict__ y,
                                                                            float* __restrict__ stats, int64_t rows,
                                                                            int64_t stride, int d, float eps) {
  constexpr int N = NormVec<T>::N;
  __shared__ float red[64];
  const int TPR = TPR_ == NORM_ALL ? blockDim.x : TPR_;
  const int groups = TPR_ == NORM_ALL ? 1 : blockDim.x / TPR, lane = TPR_ == NORM_ALL ? threadIdx.x : threadIdx.x & (TPR_ - 1);
  const int64_t step = (int64_t)gridDim.x * groups;
  int64_t row = (int64_t)blockIdx.x * groups + (TPR_ == NORM_ALL ? 0 : threadIdx.x / TPR);
  if (row >= rows) return;                       // whole groups only; a workgroup of one group always has its row
  int turn = 0;
  NormPack<P, N> wv[NV] = {}, bv[NV] = {};
  NormPack<T, N> cur[NV] = {}, nxt[NV] = {};
#pragma unroll
  for (int t = 0; t < NV; ++t) {
    const int col = (t * TPR + lane) * N;
    if (col >= d) continue;
    norm_load(cur[t], x + row * stride, col, d);
    if (w != nullptr) norm_load(wv[t], w, col, d);
    if (b != nullptr) norm_load(bv[t], b, col, d);
  }
  const float inv = 1.f / (float)d;
  for (; row < rows; row += step) {
    if (row + step < rows) {
#pragma unroll
      for (int t = 0; t < NV; ++t) {
        const int col = (t * TPR + lane) * N;
        if (col < d) norm_load(nxt[t], x + (row + step) * stride, col, d);
      }
    }
    float s[1] = {0.f};
#pragma unroll
    for (int t = 0; t < NV; ++t) {
      if ((t * TPR + lane) * N >= d) continue;
#pragma unroll
      for (int e = 0; e < N; ++e) s[0] += cur[t].get(e);          // columns past d were loaded as zeros
    }
    norm_sum<TPR_>(s, red, turn);
    const float mean = s[0] * inv;
    s[0] = 0.f;
#pragma unroll
    for (int t = 0; t < NV; ++t) {
      const int col = (t * TPR + lane) * N;
      if (col >= d) continue;
      cur[t].reread();
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float c = col + e < d ? cur[t].get(e) - mean : 0.f;
        s[0] = __builtin_fmaf(c, c, s[0]);
      }
    }
    norm_sum<TPR_>(s, red, turn);
    const float rstd = 1.f / sqrtf(s[0] * inv + eps);
#pragma unroll
    for (int t = 0; t < NV; ++t) {
      const int col = (t * TPR + lane) * N;
      if (col >= d) continue;
      cur[t].reread();
      wv[t].reread();
      bv[t].reread();
      NormPack<T, N> o;
      float v[N];
#pragma unroll
      for (int e = 0; e < N; ++e) {
        v[e] = (cur[t].get(e) - mean) * rstd;
        if (w != nullptr) v[e] *= wv[t].get(e);
        if (b != nullptr) v[e] += bv[t].get(e);
      }
      o.put(v);
      norm_store(y + row * d, o, col, d);
      cur[t] = nxt[t];
    }
    if (stats != nullptr && lane == 0) {
      stats[2 * row] = mean;
      stats[2 * row + 1] = rstd;
    }
  }
}

// part: [workgroups][2][d] partial sums of dw and db (null: not wanted)
template <typename T, typename P, int TPR_, int NV>
__global__ __launch_bounds__(TPR_ == NORM_ALL ? 1024 : 256, TPR_ == NORM_ALL ? 4 : 1) void mt_norm_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                                            const P* __restrict__ w,
                                                                            const float* __restrict__ stats, T* __restrict__ dx,
                                                                            float* __restrict__ part, int64_t rows,
                                                                            int64_t stride, int64_t dy_stride, int d) {
  constexpr int N = NormVec<T>::N;
  __shared__ float red[64];
  __shared__ float cols[TPR_ == NORM_ALL ? 1 : 2 * TPR_ * NV * N];
  const int TPR = TPR_ == NORM_ALL ? blockDim.x : TPR_;
  const int groups = TPR_ == NORM_ALL ? 1 : blockDim.x / TPR, lane = TPR_ == NORM_ALL ? threadIdx.x : threadIdx.x & (TPR_ - 1);
  const int mine = TPR_ == NORM_ALL ? 0 : threadIdx.x / TPR;
  const int64_t step = (int64_t)gridDim.x * groups;
  int64_t row = (int64_t)blockIdx.x * groups + mine;
  int turn = 0;
  NormPack<P, N> wv[NV] = {};
  NormPack<T, N> cx[NV] = {}, cd[NV] = {}, nx[NV] = {}, nd[NV] = {};
  float aw[NV][N], ab[NV][N];
#pragma unroll
  for (int t = 0; t < NV; ++t) {
    const int col = (t * TPR + lane) * N;
#pragma unroll
    for (int e = 0; e < N; ++e) aw[t][e] = ab[t][e] = 0.f;
    if (col >= d) continue;
    if (w != nullptr) norm_load(wv[t], w, col, d);
    if (row < rows) {
      norm_load(cx[t], x + row * stride, col, d);
      norm_load(cd[t], dy + row * dy_stride, col, d);
    }
  }
  const float inv = 1.f / (float)d;
  for (; row < rows; row += step) {
    const float mean = stats[2 * row], rstd = stats[2 * row + 1];
    if (row + step < rows) {
#pragma unroll
      for (int t = 0; t < NV; ++t) {
        const int col = (t * TPR + lane) * N;
        if (col >= d) continue;
        norm_load(nx[t], x + (row + step) * stride, col, d);
        norm_load(nd[t], dy + (row + step) * dy_stride, col, d);
      }
    }
    float s[2] = {0.f, 0.f};
#pragma unroll
    for (int t = 0; t < NV; ++t) {
      const int col = (t * TPR + lane) * N;
      if (col >= d) continue;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float g0 = cd[t].get(e), u = (cx[t].get(e) - mean) * rstd;
        const float g = w != nullptr ? g0 * wv[t].get(e) : g0;    // columns past d: dy was loaded as zero
        s[0] += g;
        s[1] = __builtin_fmaf(g, u, s[1]);
        ab[t][e] += g0;
        aw[t][e] = __builtin_fmaf(g0, u, aw[t][e]);
      }
    }
    norm_sum<TPR_>(s, red, turn);
    const float mg = s[0] * inv, mu = s[1] * inv;
#pragma unroll
    for (int t = 0; t < NV; ++t) {
      const int col = (t * TPR + lane) * N;
      if (col >= d) continue;
      cx[t].reread();
      cd[t].reread();
      wv[t].reread();
      NormPack<T, N> o;
      float v[N];
#pragma unroll
      for (int e = 0; e < N; ++e) {
        const float g0 = cd[t].get(e), u = (cx[t].get(e) - mean) * rstd;
        const float g = w != nullptr ? g0 * wv[t].get(e) : g0;
        v[e] = rstd * (g - mg - u * mu);
      }
      o.put(v);
      norm_store(dx + row * d, o, col, d);
      cx[t] = nx[t];
      cd[t] = nd[t];
    }
  }
  if (part == nullptr) return;
  float* pw = part + (int64_t)blockIdx.x * 2 * d;
  if constexpr (TPR_ != NORM_ALL) {      // the groups of a workgroup own the same columns: added in group order
    for (int g = 0; g < groups; ++g) {
      if (mine == g) {
#pragma unroll
        for (int t = 0; t < NV; ++t)
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const int at = (t * TPR + lane) * N + e;
            cols[at] = g == 0 ? aw[t][e] : cols[at] + aw[t][e];
            cols[TPR * NV * N + at] = g == 0 ? ab[t][e] : cols[TPR * NV * N + at] + ab[t][e];
          }
      }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < d; c += blockDim.x) {
      pw[c] = cols[c];
      pw[d + c] = cols[TPR * NV * N + c];
    }
  } else {
#pragma unroll
    for (int t = 0; t < NV; ++t) {
      const int col = (t * TPR + lane) * N;
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (col + e < d) {
          pw[col + e] = aw[t][e];
          pw[d + col + e] = ab[t][e];
        }
    }
  }
}

// Rows wider than the registers of one workgroup: every pass reads the row again (from the caches).
template <typename T, typename P>
__global__ __launch_bounds__(1024) void mt_norm_wide_fwd_kernel(const T* __restrict__ x, const P* __restrict__ w,
                                                                const P* __restrict__ b, T* __restrict__ y,
                                                                float* __restrict__ stats, int64_t rows, int64_t stride, int d,
                                                                float eps) {
  __shared__ float red[64];
  int turn = 0;
  const float inv = 1.f / (float)d;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* xr = x + row * stride;
    float s[1] = {0.f};
    for (int c = threadIdx.x; c < d; c += 1024) s[0] += (float)xr[c];
    norm_sum<NORM_ALL>(s, red, turn);
    const float mean = s[0] * inv;
    s[0] = 0.f;
    for (int c = threadIdx.x; c < d; c += 1024) {
      const float v = (float)xr[c] - mean;
      s[0] = __builtin_fmaf(v, v, s[0]);
    }
    norm_sum<NORM_ALL>(s, red, turn);
    const float rstd = 1.f / sqrtf(s[0] * inv + eps);
    for (int c = threadIdx.x; c < d; c += 1024) {
      float v = ((float)xr[c] - mean) * rstd;
      if (w != nullptr) v *= (float)w[c];
      if (b != nullptr) v += (float)b[c];
      y[row * d + c] = (T)v;
    }
    if (stats != nullptr && threadIdx.x == 0) {
      stats[2 * row] = mean;
      stats[2 * row + 1] = rstd;
    }
  }
}

template <typename T, typename P>
__global__ __launch_bounds__(1024) void mt_norm_wide_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                                const P* __restrict__ w, const float* __restrict__ stats,
                                                                T* __restrict__ dx, int64_t rows, int64_t stride,
                                                                int64_t dy_stride, int d) {
  __shared__ float red[64];
  int turn = 0;
  const float inv = 1.f / (float)d;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x) {
    const T *xr = x + row * stride, *gr = dy + row * dy_stride;
    const float mean = stats[2 * row], rstd = stats[2 * row + 1];
    float s[2] = {0.f, 0.f};
    for (int c = threadIdx.x; c < d; c += 1024) {
      const float g = (float)gr[c] * (w != nullptr ? (float)w[c] : 1.f);
      s[0] += g;
      s[1] = __builtin_fmaf(g, ((float)xr[c] - mean) * rstd, s[1]);
    }
    norm_sum<NORM_ALL>(s, red, turn);
    const float mg = s[0] * inv, mu = s[1] * inv;
    for (int c = threadIdx.x; c < d; c += 1024) {
      const float g = (float)gr[c] * (w != nullptr ? (float)w[c] : 1.f);
      dx[row * d + c] = (T)(rstd * (g - mg - ((float)xr[c] - mean) * rstd * mu));
    }
  }
}
// Column sums for the wide form: workgroup (column block, row chunk), a thread per column.
template <typename T>
__global__ __launch_bounds__(256) void mt_norm_wide_cols_kernel(const T* __restrict__ dy, const T* __restrict__ x,
                                                                const float* __restrict__ stats, float* __restrict__ part,
                                                                int64_t rows, int64_t stride, int64_t dy_stride, int d) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= d) return;
  const int64_t per = (rows + gridDim.y - 1) / gridDim.y, lo = per * blockIdx.y, hi = lo + per < rows ? lo + per : rows;
  float sw = 0.f, sb = 0.f;
  for (int64_t row = lo; row < hi; ++row) {
    const float g = (float)dy[row * dy_stride + c];
    sw = __builtin_fmaf(g, ((float)x[row * stride + c] - stats[2 * row]) * stats[2 * row + 1], sw);
    sb += g;
  }
  part[(int64_t)blockIdx.y * 2 * d + c] = sw;
  part[((int64_t)blockIdx.y * 2 + 1) * d + c] = sb;
}

// dw, db [d] = sums of the partial rows: 32 columns x 32 strands per workgroup, strand s adds the partial rows s, s + 32, ... in
// order, and the strands are added in order through LDS.
#define NORM_COLS 32
template <typename P>
__global__ __launch_bounds__(1024) void mt_norm_cols_kernel(const float* __restrict__ part, P* __restrict__ dw, P* __restrict__ db,
                                                            int n, int d) {
  __shared__ float strands[32][NORM_COLS + 1];
  const int cl = threadIdx.x % NORM_COLS, st = threadIdx.x / NORM_COLS;
  const int c = blockIdx.x * NORM_COLS + cl;                  // 0 .. 2 d - 1: dw, then db
  float s = 0.f;
  if (c < 2 * d) {
#pragma unroll 8
    for (int i = st; i < n; i += 32) s += part[(int64_t)i * 2 * d + c];
  }
  strands[st][cl] = s;
  __syncthreads();
  if (st == 0 && c < 2 * d) {
    s = 0.f;
#pragma unroll
    for (int i = 0; i < 32; ++i) s += strands[i][cl];
    if (c < d) {
      if (dw != nullptr) dw[c] = (P)s;
    } else if (db != nullptr) {
      db[c - d] = (P)s;
    }
  }
}

// ---- launchers ----------------------------------------------------------------------------------------------------------
struct NormShape {
  int threads, nv, tpr;      // nv 0: the wide form
};
// Rows of at most 128 (forward 256) vectors: a wave or less per row, no barriers.  Few rows: one wave per workgroup, spread over the
// chip; a backward pass with a wave per row takes four, whose column sums meet in LDS: a workgroup of one row would write as many
// bytes of partial sums as it reads (2048 x 1024 bf16, with the second launch: 20.0 us by one wave, 10.8 by four; 4095 x 512
// 24.0 / 10.7; 200 x 256 7.2 / 6.1).  Wider rows: as many waves as hold one vector per
// thread, or two; a forward pass goes on to four, a backward pass, which also holds two sums per column, does not.
static NormShape norm_shape(int64_t rows, int d, int per, bool backward) {
  const int vecs = (d + per - 1) / per;
  const int threads = rows >= 4096 || (backward && vecs > 16) ? 256 : 64;
  if (vecs <= 16) return {threads, 1, 16};
  if (vecs <= 64) return {threads, 1, 64};
  if (vecs <= 128) return {threads, 2, 64};
  if (vecs <= 256 && !backward) return {threads, 4, 64};
  if (vecs <= 1024) return {(vecs + 63) / 64 * 64, 1, NORM_ALL};
  if (vecs <= 2048) return {(vecs + 127) / 128 * 64, 2, NORM_ALL};
  if (vecs <= 4096 && !backward) return {1024, 4, NORM_ALL};
  return {1024, 0, NORM_ALL};
}
// Workgroups: each walks over several rows with its parameters in registers.  Measured over 1024 .. 16384 workgroups, forward passes
// are fastest near 64 waves per CU (16384 x 4096 bf16: 53 us, 69 with four times as many; 128000 x 512 f32: 104, 125 with half).
// A backward pass writes one partial row of column sums per workgroup and takes what is resident at 16 waves per CU, whole
// workgroups on every CU (5001 x 10007 bf16: 131 us; 191 with 307 workgroups of 10 waves, 146 with 512).
#define NORM_FWD_WAVES (256 * 64)
#define NORM_BWD_WAVES 16
static int norm_blocks(const NormShape& s, int64_t rows, bool backward) {
  const int groups = s.tpr == NORM_ALL ? 1 : s.threads / s.tpr, waves = s.threads / 64;
  const int64_t want = (rows + groups - 1) / groups;
  const int64_t most = backward ? 256 * (NORM_BWD_WAVES / waves) : NORM_FWD_WAVES / waves;
  return (int)(want < most ? want : most);
}
#define NORM_WIDE_PARTS 64

#define NORM_SHAPES(GO) \
  if (s.tpr == 16) GO(16, 1) else if (s.tpr == 64 && s.nv == 1) GO(64, 1) else if (s.tpr == 64 && s.nv == 2) GO(64, 2) \
  else if (s.nv == 1) GO(NORM_ALL, 1) else if (s.nv == 2) GO(NORM_ALL, 2)

template <typename T, typename P>
static int norm_fwd(const void* x, const void* w, const void* b, void* y, float* stats, int64_t rows, int64_t stride, int d,
                    float eps, hipStream_t stream) {
  const NormShape s = norm_shape(rows, d, NormVec<T>::N, false);
  const int blocks = norm_blocks(s, rows, false);
  const T* xt = (const T*)x;
  const P *wt = (const P*)w, *bt = (const P*)b;
  if (s.nv == 0) {
    hipLaunchKernelGGL((mt_norm_wide_fwd_kernel<T, P>), dim3(blocks), dim3(1024), 0, stream, xt, wt, bt, (T*)y, stats, rows,
                       stride, d, eps);
    return (int)hipGetLastError();
  }
#define GO(TPR, NV)                                                                                                       \
  hipLaunchKernelGGL((mt_norm_fwd_kernel<T, P, TPR, NV>), dim3(blocks), dim3(s.threads), 0, stream, xt, wt, bt, (T*)y, stats, rows, \
                     stride, d, eps);
  NORM_SHAPES(GO)
  else if (s.tpr == 64) GO(64, 4) else GO(NORM_ALL, 4)
#undef GO
  return (int)hipGetLastError();
}

template <typename T, typename P>
static int norm_bwd(const void* dy, const void* x, const void* w, const float* stats, void* dx, float* part, void* dw, void* db,
                    int64_t rows, int64_t stride, int64_t dy_stride, int d, hipStream_t stream) {
  const NormShape s = norm_shape(rows, d, NormVec<T>::N, true);
  const int blocks = norm_blocks(s, rows, true);
  const T *xt = (const T*)x, *gt = (const T*)dy;
  const P* wt = (const P*)w;
  if (s.nv == 0) {
    hipLaunchKernelGGL((mt_norm_wide_bwd_kernel<T, P>), dim3(blocks), dim3(1024), 0, stream, gt, xt, wt, stats, (T*)dx, rows,
                       stride, dy_stride, d);
    if (part != nullptr)
      hipLaunchKernelGGL((mt_norm_wide_cols_kernel<T>), dim3((d + 255) / 256, blocks < NORM_WIDE_PARTS ? blocks : NORM_WIDE_PARTS), dim3(256), 0, stream, gt,
                         xt, stats, part, rows, stride, dy_stride, d);
  } else {
#define GO(TPR, NV)                                                                                                          \
  hipLaunchKernelGGL((mt_norm_bwd_kernel<T, P, TPR, NV>), dim3(blocks), dim3(s.threads), 0, stream, gt, xt, wt, stats, (T*)dx, part, \
                     rows, stride, dy_stride, d);
    NORM_SHAPES(GO)
#undef GO
  }
  if (part != nullptr) {
    const int n = s.nv == 0 && blocks > NORM_WIDE_PARTS ? NORM_WIDE_PARTS : blocks;
    hipLaunchKernelGGL((mt_norm_cols_kernel<P>), dim3((2 * d + NORM_COLS - 1) / NORM_COLS), dim3(1024), 0, stream, part, (P*)dw, (P*)db, n, d);
  }
  return (int)hipGetLastError();
}

static bool norm_args(int64_t rows, int64_t stride, int d, int x_bf16, int w_bf16) {
  return rows >= 0 && stride >= 0 && d >= 1 && d <= (1 << 29) && (x_bf16 || !w_bf16);
}

// Rows of the partial-sum workspace [n][2][d] f32 of a backward pass.
extern "C" int mt_norm_bwd_parts(int64_t rows, int d, int x_bf16) {
  if (!norm_args(rows, 0, d, x_bf16, 0)) return -2;
  const NormShape s = norm_shape(rows, d, x_bf16 ? 8 : 4, true);
  const int blocks = norm_blocks(s, rows, true);
  return s.nv == 0 && blocks > NORM_WIDE_PARTS ? NORM_WIDE_PARTS : blocks;
}
// y [rows][d] contiguous; x rows `stride` elements apart; w, b [d] (each may be null); stats [rows][2] (may be null).
extern "C" int mt_norm_fwd_launch(const void* x, const void* w, const void* b, void* y, float* stats, int64_t rows, int64_t stride,
                                  int d, float eps, int x_bf16, int w_bf16, hipStream_t stream) {
  if (!norm_args(rows, stride, d, x_bf16, w_bf16)) return -2;
  if (rows == 0) return 0;
  if (!x || !y) return -2;      // tensors without memory (of a dispatch mode) have null addresses
  if (!x_bf16) return norm_fwd<float, float>(x, w, b, y, stats, rows, stride, d, eps, stream);
  if (!w_bf16) return norm_fwd<__bf16, float>(x, w, b, y, stats, rows, stride, d, eps, stream);
  return norm_fwd<__bf16, __bf16>(x, w, b, y, stats, rows, stride, d, eps, stream);
}
// dx [rows][d] contiguous; part as mt_norm_bwd_parts says, or null when neither dw nor db is wanted.
extern "C" int mt_norm_bwd_launch(const void* dy, const void* x, const void* w, const float* stats, void* dx, float* part, void* dw,
                                  void* db, int64_t rows, int64_t stride, int64_t dy_stride, int d, int x_bf16, int w_bf16,
                                  hipStream_t stream) {
  if (!norm_args(rows, stride, d, x_bf16, w_bf16) || dy_stride < 0) return -2;
  if (rows == 0) return 0;
  if (!dy || !x || !stats || !dx || (part != nullptr) != (dw != nullptr || db != nullptr)) return -2;
  if (!x_bf16) return norm_bwd<float, float>(dy, x, w, stats, dx, part, dw, db, rows, stride, dy_stride, d, stream);
  if (!w_bf16) return norm_bwd<__bf16, float>(dy, x, w, stats, dx, part, dw, db, rows, stride, dy_stride, d, stream);
  return norm_bwd<__bf16, __bf16>(dy, x, w, stats, dx, part, dw, db, rows, stride, dy_stride, d, stream);
}
