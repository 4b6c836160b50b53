// Dense layer with bias, activation and residual in the GEMM's epilogue (gfx950, bf16 or exact f32):
//
//   forward : z = x W^T + b,  y = act(z) + residual         x [M][K], W [N][K], y [M][N]
//   backward: dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum over rows of dz;  the residual's gradient is dy
//
// The products run on the tiles of mt_gemm_tile.h and mt_gemm_f32_tile.h.  The epilogue works on the f32 accumulators, so the
// layer's output is rounded once and no separate pass over [M][N] adds the bias, applies the activation or adds the residual.
// z is kept for the backward pass in the operands' type (for bf16 that rounds the argument of act' by at most 2^-8 of it); with
// ReLU and no residual y itself is enough.  dz is one pass over dy, written with rows of whole 16-byte pieces (zeros behind
// column N) so that both gradient GEMMs can stage it.
#include "mt_gemm_tile.h"
#include "mt_gemm_f32_tile.h"

template <int NSTAGE>
__global__ __launch_bounds__(NTHREADS) void mt_linear_fwd_kernel(MtGemmGroup g, MtLinearEp ep, int tiles_i, int tiles_j) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[NSTAGE * STAGE_BYTES];
  const int n = tiles_i * tiles_j, per = (n + 7) / 8, t = (blockIdx.x % 8) * per + blockIdx.x / 8;      // whole row panels per XCD
  if (t >= n) return;
  MtTile tile;
  tile.group = 0;
  tile.ti = (int16_t)(t / tiles_j);
  tile.tj = (int16_t)(t % tiles_j);
  gemm_tile<0, NSTAGE, true>(&g, tile, 0, 0, 0, 0, 1, 0, lds, &ep);
}
#define LINEAR_BAND 4       // 256-tiles: row tiles of a band (mt_gemm_p8_kernel)
__global__ __launch_bounds__(P8_THREADS) void mt_linear_fwd_p8_kernel(MtGemmGroup g, MtLinearEp ep, int tiles_i, int tiles_j) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[2 * BIG_STAGE_BYTES];
  const int n = tiles_i * tiles_j, per = (n + 7) / 8, t = (blockIdx.x % 8) * per + blockIdx.x / 8;
  if (t >= n) return;
  const int in_band = LINEAR_BAND * tiles_j, first = (t / in_band) * LINEAR_BAND;
  const int rows = tiles_i - first < LINEAR_BAND ? tiles_i - first : LINEAR_BAND;
  const int r = t % in_band;
  gemm_tile_p8<0, 1, true>(g, first + r % rows, r / rows, 0, 0, 1, 0, lds, &ep);
}
template <int T>
__global__ __launch_bounds__(F32_THREADS) void mt_linear_fwd_f32_kernel(MtGemmGroup g, MtLinearEp ep, int tiles_i, int tiles_j) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[2 * 2 * T * 128];
  const int n = tiles_i * tiles_j, per = (n + 7) / 8, t = (blockIdx.x % 8) * per + blockIdx.x / 8;
  if (t >= n) return;
  MtTile tile;
  tile.group = 0;
  tile.ti = (int16_t)(t / tiles_j);
  tile.tj = (int16_t)(t % tiles_j);
  f32_gemm_tile<0, 2, T, 1, 0, true>(&g, tile, 0, 0, 0, 0, 1, 0, lds, &ep);
}

// dz = dy act'(s): s is z, or (ReLU without a residual) y, whose sign is z's.  A thread takes one 16-byte piece of a dz row.
template <typename T>
__global__ __launch_bounds__(256) void mt_act_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ s, T* __restrict__ dz,
                                                         int64_t rows, int n, int64_t ld_dy, int ld_dz, int act) {
  constexpr int V = 16 / (int)sizeof(T);
  const int pieces = ld_dz / V;
  const int64_t total = rows * pieces;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const int64_t row = i / pieces;
    const int col = (int)(i - row * pieces) * V;
    T a[V], b[V], o[V];
    const T *pa = dy + row * ld_dy + col, *pb = s + row * n + col;
    if (col + V <= n) {
      __builtin_memcpy(a, pa, 16);
      __builtin_memcpy(b, pb, 16);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        a[e] = col + e < n ? pa[e] : (T)0.f;
        b[e] = col + e < n ? pb[e] : (T)0.f;
      }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float slope = mt_ep_slope((float)b[e], act);
      o[e] = act == MT_ACT_RELU ? (slope != 0.f || (float)b[e] != (float)b[e] ? a[e] : (T)0.f) : (T)((float)a[e] * slope);
    }
    __builtin_memcpy(dz + row * ld_dz + col, o, 16);
  }
}

// dW [rows][cols] and db [rows]: the f32 slabs of the split contraction added in order and rounded to the parameters' types.
// Slab s: dW with rows of ld floats, then (at db_at) db.
template <typename P, typename B>
__global__ __launch_bounds__(256) void mt_linear_wsum_kernel(const float* __restrict__ arena, P* __restrict__ dw, B* __restrict__ db,
                                                             int64_t rows, int cols, int ld, int64_t db_at, int splits, int64_t slab) {
  const int64_t total = rows * cols + (db != nullptr ? rows : 0);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    const bool is_w = i < rows * cols;
    const int64_t row = i / cols;
    const float* p = arena + (is_w ? row * ld + (i - row * cols) : db_at + (i - rows * cols));
    float v = 0.f;
    for (int s = 0; s < splits; ++s) v += p[s * slab];
    if (is_w) dw[i] = (P)v;
    else db[i - rows * cols] = (B)v;
  }
}

// ---- launchers ----------------------------------------------------------------------------------------------------------
#define LINEAR_ROWS (1 << 20)      // rows of one launch: tile coordinates are 16 bits

static MtGemmGroup linear_group(const void* A, const void* B, void* C, int I, int J, int KK, int lda, int ldb, int ldc) {
  MtGemmGroup g = {};
  g.A = A; g.B = B; g.C = C;
  g.I = I; g.J = J; g.KK = KK;
  g.lda = lda; g.ldb = ldb; g.ldc = ldc;
  g.active_steps = 1;
  return g;
}
static int linear_grid(int tiles_i, int tiles_j) { return (tiles_i * tiles_j + 7) / 8 * 8; }

// x [M][ldx], W [N][ldw]: rows of whole 16-byte pieces; K columns, a multiple of a piece.  residual, z, y: [M][N] contiguous.
extern "C" int mt_linear_fwd_launch(const void* x, const void* w, const void* bias, const void* residual, void* y, void* z, int64_t M,
                                    int N, int K, int64_t ldx, int64_t ldw, int act, int bias_bf16, int bf16, hipStream_t stream) {
  const int per = bf16 ? 8 : 4, es = bf16 ? 2 : 4;
  if (M < 0 || N < 1 || K < 1 || K % per || ldx % per || ldw % per || ldx < K || ldw < K) return -2;
  if (ldx > (1 << 28) || ldw > (1 << 28) || N > 4000000 || act < 0 || act > 2) return -2;
  if ((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w)) & 15) return -2;
  for (int64_t m0 = 0; m0 < M; m0 += LINEAR_ROWS) {
    const int m = (int)(M - m0 < LINEAR_ROWS ? M - m0 : LINEAR_ROWS);
    const size_t at = (size_t)m0 * N * es;
    MtGemmGroup g = linear_group((const uint8_t*)x + (size_t)m0 * ldx * es, w, (uint8_t*)y + at, m, N, K, (int)ldx, (int)ldw, N);
    MtLinearEp ep = {bias, residual ? (const uint8_t*)residual + at : nullptr, z ? (uint8_t*)z + at : nullptr, bias_bf16, act, N, N};
    if (bf16 && mt_p8_rule(m, N, K, 1, 256)) {
      const int ti = (m + BIGT - 1) / BIGT, tj = (N + BIGT - 1) / BIGT;
      hipLaunchKernelGGL(mt_linear_fwd_p8_kernel, dim3(linear_grid(ti, tj)), dim3(P8_THREADS), 0, stream, g, ep, ti, tj);
    } else if (bf16) {
      const int ti = (m + BM - 1) / BM, tj = (N + BN - 1) / BN;
      if (ti * tj <= 320)
        hipLaunchKernelGGL(mt_linear_fwd_kernel<4>, dim3(linear_grid(ti, tj)), dim3(NTHREADS), 0, stream, g, ep, ti, tj);
      else
        hipLaunchKernelGGL(mt_linear_fwd_kernel<2>, dim3(linear_grid(ti, tj)), dim3(NTHREADS), 0, stream, g, ep, ti, tj);
    } else {
      const int64_t n128 = (int64_t)((m + 127) / 128) * ((N + 127) / 128);
      const int T = n128 >= 512 ? 128 : 64;
      const int ti = (m + T - 1) / T, tj = (N + T - 1) / T;
      if (T == 128)
        hipLaunchKernelGGL(mt_linear_fwd_f32_kernel<128>, dim3(linear_grid(ti, tj)), dim3(F32_THREADS), 0, stream, g, ep, ti, tj);
      else
        hipLaunchKernelGGL(mt_linear_fwd_f32_kernel<64>, dim3(linear_grid(ti, tj)), dim3(F32_THREADS), 0, stream, g, ep, ti, tj);
    }
  }
  return (int)hipGetLastError();
}

// s: z or y [M][N] contiguous; dz [M][ld_dz], ld_dz a multiple of a 16-byte piece, zeros behind column N.
extern "C" int mt_linear_act_bwd_launch(const void* dy, const void* s, void* dz, int64_t M, int N, int64_t ld_dy, int ld_dz, int act,
                                        int bf16, hipStream_t stream) {
  const int per = bf16 ? 8 : 4;
  if (M < 0 || N < 1 || ld_dz % per || ld_dz < N || ld_dy < 0 || act < 1 || act > 2) return -2;
  if (M == 0) return 0;
  const int64_t blocks = (M * (ld_dz / per) + 255) / 256;
  const dim3 grid((unsigned)(blocks < 16384 ? blocks : 16384));
  if (bf16)
    hipLaunchKernelGGL(mt_act_bwd_kernel<__bf16>, grid, dim3(256), 0, stream, (const __bf16*)dy, (const __bf16*)s, (__bf16*)dz, M, N,
                       ld_dy, ld_dz, act);
  else
    hipLaunchKernelGGL(mt_act_bwd_kernel<float>, grid, dim3(256), 0, stream, (const float*)dy, (const float*)s, (float*)dz, M, N,
                       ld_dy, ld_dz, act);
  return (int)hipGetLastError();
}

// dw [rows][cols], db [rows] (may be null).
extern "C" int mt_linear_wsum_launch(const float* arena, void* dw, void* db, int64_t rows, int cols, int ld, int64_t db_at, int splits,
                                     int64_t slab, int w_bf16, int b_bf16, hipStream_t stream) {
  if (rows < 1 || cols < 1 || ld < cols || splits < 1 || slab < db_at) return -2;
  const int64_t blocks = (rows * cols + rows + 255) / 256;
  const dim3 grid((unsigned)(blocks < 16384 ? blocks : 16384));
#define GO(P, B)                                                                                                                \
  hipLaunchKernelGGL((mt_linear_wsum_kernel<P, B>), grid, dim3(256), 0, stream, arena, (P*)dw, (B*)db, rows, cols, ld, db_at, splits, \
                     slab)
  if (w_bf16 && b_bf16) GO(__bf16, __bf16);
  else if (w_bf16) GO(__bf16, float);
  else if (b_bf16) GO(float, __bf16);
  else GO(float, float);
#undef GO
  return (int)hipGetLastError();
}
