// Dense layer with bias, activation and residual in the GEMM's epilogue (gfx950, bf16 or exact f32):
//
//   forward : z = x W^T + b,  y = act(z) + residual         x [M][K], W [N][K], y [M][N]
//   backward: dz = dy act'(z),  dx = dz W,  dW = dz^T x,  db = sum over rows of dz;  the residual's gradient is dy
//
// The products run on the tiles of mt_gemm_tile.h (bf16, 128 wide), mt_linear_tile.h (bf16, 256) and mt_linear_tile_f32.h.  The
// epilogue works on the f32 accumulators, so the layer's output is rounded once and no separate pass over [M][N] adds the bias,
// applies the activation or adds the residual.
// z is kept for the backward pass in the operands' type (for bf16 that rounds the argument of act' by at most 2^-8 of it); with
// ReLU and no residual y itself is enough.  dz is one pass over dy, written with rows of whole 16-byte pieces (zeros behind
// column N) so that both gradient GEMMs can stage it.
#include "mt_linear_tile.h"
#include "mt_linear_tile_f32.h"

// MODE 0: A [I][KK] and B [J][KK] (forward); 1: B [KK][J] (input gradient).  A contraction may be split over workgroups: part `sp`
// takes its share of the columns of A (and columns or rows of B) and leaves its accumulators in ep.part.
template <int MODE, typename T>
__device__ __forceinline__ void linear_split(MtGemmGroup& g, MtLinearEp& ep, int sp, int per) {
  const int k0 = sp * per;
  g.A = reinterpret_cast<const T*>(g.A) + k0;
  g.B = reinterpret_cast<const T*>(g.B) + (MODE == 0 ? (size_t)k0 : (size_t)k0 * g.ldb);
  g.KK = g.KK - k0 < per ? g.KK - k0 : per;
  ep.part += (size_t)sp * g.I * g.J;
}
// block -> (tile, part): whole row panels per XCD, the parts of a tile side by side
#define LINEAR_PICK()                                                                                                      \
  const int all = tiles_i * tiles_j * splits, share = (all + 7) / 8, u = (blockIdx.x % 8) * share + blockIdx.x / 8; \
  if (u >= all) return;                                                                                                    \
  const int t = u / splits
template <int MODE, int NSTAGE>
__global__ __launch_bounds__(NTHREADS) void mt_linear_gemm_kernel(MtGemmGroup g, MtLinearEp ep, int tiles_i, int tiles_j, int splits,
                                                                  int per) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[NSTAGE * STAGE_BYTES];
  LINEAR_PICK();
  if (splits > 1) linear_split<MODE, uint16_t>(g, ep, u % splits, per);
  MtTile tile;
  tile.group = 0;
  tile.ti = (int16_t)(t / tiles_j);
  tile.tj = (int16_t)(t % tiles_j);
  gemm_tile<MODE, NSTAGE, true>(&g, tile, 0, 0, 0, 0, 1, 0, lds, &ep);
}
#define LINEAR_BAND 4       // 256-tiles: row tiles of a band, so that an XCD's 32 tiles at a time share 12 operand panels
template <int MODE>
__global__ __launch_bounds__(LT_THREADS) void mt_linear_big_kernel(MtGemmGroup g, MtLinearEp ep, int tiles_i, int tiles_j) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * BIG_STAGE_BYTES];
  constexpr int splits = 1;
  LINEAR_PICK();
  const int in_band = LINEAR_BAND * tiles_j, first = (t / in_band) * LINEAR_BAND;
  const int rows = tiles_i - first < LINEAR_BAND ? tiles_i - first : LINEAR_BAND;
  const int r = t % in_band;
  linear_tile<MODE>(g, first + r % rows, r / rows, false, lds, ep);
}
template <int MODE>
__global__ __launch_bounds__(LF_THREADS, 4) void mt_linear_gemm_f32_kernel(MtGemmGroup g, MtLinearEp ep, int tiles_i, int tiles_j,
                                                                           int splits, int per) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[LF_LDS];
  LINEAR_PICK();
  if (splits > 1) linear_split<MODE, float>(g, ep, u % splits, per);
  linear_tile_f32<MODE>(g, t / tiles_j, t % tiles_j, false, lds, ep);
}
// The parts of a split contraction added in order, then the epilogue; four elements per thread.
template <typename T>
__global__ __launch_bounds__(256) void mt_linear_join_kernel(const float* __restrict__ part, MtLinearEp ep, T* __restrict__ y,
                                                             int64_t total, int N, int splits) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4;
  if (i >= total) return;
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  const bool whole = i + 4 <= total;
  for (int s = 0; s < splits; ++s) {
    f32x4 p = {0.f, 0.f, 0.f, 0.f};
    const float* src = part + (int64_t)s * total + i;
    if (whole) __builtin_memcpy(&p, src, 16);
    else
      for (int e = 0; e < 4; ++e) p[e] = i + e < total ? src[e] : 0.f;
    v += p;
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if (i + e >= total) break;
    const int col = (int)((i + e) % N);
    float o = v[e] + (ep.bias != nullptr ? mt_ep_bias(ep, col) : 0.f);
    if (ep.z != nullptr) reinterpret_cast<T*>(ep.z)[i + e] = (T)o;
    o = mt_ep_act<sizeof(T) == 2>(o, ep.act);
    if (ep.residual != nullptr) o += (float)reinterpret_cast<const T*>(ep.residual)[i + e];
    y[i + e] = (T)o;
  }
}

// Weight gradient with the whole contraction in one workgroup: dW (and db) leave in their own types.
template <int NSTAGE>
__global__ __launch_bounds__(NTHREADS) void mt_linear_wgrad_kernel(MtGemmGroup g, MtLinearEp ep, int tiles_i, int tiles_j, int flags) {
  __shared__ __attribute__((aligned(16))) uint8_t lds[NSTAGE * STAGE_BYTES];
  const int n = tiles_i * tiles_j, per = (n + 7) / 8, t = (blockIdx.x % 8) * per + blockIdx.x / 8;
  if (t >= n) return;
  MtTile tile;
  tile.group = 0;
  tile.ti = (int16_t)(t % tiles_i);
  tile.tj = (int16_t)(t / tiles_i);
  gemm_tile<2, NSTAGE, true>(&g, tile, 0, flags, 0, 0, 1, 0, lds, &ep);
}
__global__ __launch_bounds__(LT_THREADS) void mt_linear_wgrad_big_kernel(MtGemmGroup g, MtLinearEp ep, int tiles_i, int tiles_j, int flags) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * BIG_STAGE_BYTES];
  const int n = tiles_i * tiles_j, per = (n + 7) / 8, t = (blockIdx.x % 8) * per + blockIdx.x / 8;
  if (t >= n) return;
  const int in_band = LINEAR_BAND * tiles_j, first = (t / in_band) * LINEAR_BAND;
  const int rows = tiles_i - first < LINEAR_BAND ? tiles_i - first : LINEAR_BAND;
  const int r = t % in_band;
  const int tj = r / rows;
  linear_tile<2>(g, first + r % rows, tj, tj == 0 && (flags & MT_GEMM_FLAG_DBIAS) && g.aux_out != nullptr, lds, ep);
}
// Part `sp` of the rows; with more than one part each leaves its accumulators and column sums in a slab of its own.
__global__ __launch_bounds__(LF_THREADS, 4) void mt_linear_wgrad_f32_kernel(MtGemmGroup g, MtLinearEp ep, int tiles_i, int tiles_j,
                                                                            int splits, int per, int64_t slab) {
  __shared__ __attribute__((aligned(1024))) uint8_t lds[LF_LDS];
  LINEAR_PICK();
  if (splits > 1) {
    const int sp = u % splits, k0 = sp * per;
    g.A = reinterpret_cast<const float*>(g.A) + (size_t)k0 * g.lda;
    g.B = reinterpret_cast<const float*>(g.B) + (size_t)k0 * g.ldb;
    g.KK = g.KK - k0 < per ? g.KK - k0 : per;
    ep.part += sp * slab;
    if (g.aux_out != nullptr) g.aux_out = reinterpret_cast<float*>(g.aux_out) + sp * slab;
  }
  const int tj = t % tiles_j;
  linear_tile_f32<2>(g, t / tiles_j, tj, tj == 0 && g.aux_out != nullptr, lds, ep);
}

// A few rows (at most 16 MT): the weight is streamed once, straight from memory into the matrix instruction's operand.  A
// workgroup owns 16 output features; its waves take equal parts of the contraction, and their sums meet in LDS in wave order.
// Lane (n = lane & 15, h = lane >> 4) loads 16 bytes of weight row n at column 4 h (f32) or 8 h (bf16) of each step, and the same
// columns of x row n; UNROLL steps are loaded before their products, which keeps 8 KB of weight per wave on its way.
#define FEW_UNROLL 8
template <typename T, int MT, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void mt_linear_few_kernel(const T* __restrict__ x, const T* __restrict__ w, MtLinearEp ep,
                                                                   T* __restrict__ y, int M, int N, int K, int64_t ldx, int64_t ldw,
                                                                   int steps_per_wave) {
  constexpr int V = 16 / (int)sizeof(T), STEP = 4 * V;
  __shared__ float part[WAVES][MT][16][17];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, h = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const T* wr = w + (int64_t)(n0 + r < N ? n0 + r : N - 1) * ldw + h * V;      // rows past the last repeat it: their sums are dropped
  const T* xr[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) xr[t] = x + (int64_t)(16 * t + r < M ? 16 * t + r : M - 1) * ldx + h * V;
  f32x4 acc[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
  auto load = [&](const T* p, int k) {
    u32x4 v = {0u, 0u, 0u, 0u};
    if (k + h * V < K) v = *reinterpret_cast<const u32x4*>(p + k);
    return v;
  };
  auto mma = [&](u32x4 a, u32x4 b, f32x4 c) {
    if constexpr (sizeof(T) == 2) {
      return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(a[e]), __uint_as_float(b[e]), c, 0, 0, 0);
      return c;
    }
  };
  const int k_lo = wave * steps_per_wave * STEP, k_all = k_lo + steps_per_wave * STEP, k_hi = k_all < K ? k_all : K;
  for (int k = k_lo; k < k_hi; k += FEW_UNROLL * STEP) {
    u32x4 a[FEW_UNROLL], b[FEW_UNROLL][MT];
#pragma unroll
    for (int s = 0; s < FEW_UNROLL; ++s) {
      const int ks = k + s * STEP < k_hi ? k + s * STEP : K;                   // K: zeros
      a[s] = load(wr, ks);
#pragma unroll
      for (int t = 0; t < MT; ++t) b[s][t] = load(xr[t], ks);
    }
#pragma unroll
    for (int s = 0; s < FEW_UNROLL; ++s)
#pragma unroll
      for (int t = 0; t < MT; ++t) acc[t] = mma(a[s], b[s][t], acc[t]);
  }
#pragma unroll
  for (int t = 0; t < MT; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) part[wave][t][r][4 * h + i] = acc[t][i];       // [row][feature]
  __syncthreads();
  for (int o = threadIdx.x; o < MT * 256; o += WAVES * 64) {
    const int t = o >> 8, row = 16 * t + ((o >> 4) & 15), col = n0 + (o & 15);
    if (row >= M || col >= N) continue;
    float v = 0.f;
#pragma unroll
    for (int q = 0; q < WAVES; ++q) v += part[q][t][(o >> 4) & 15][o & 15];
    if (ep.bias != nullptr) v += mt_ep_bias(ep, col);
    const int64_t at = (int64_t)row * N + col;
    if (ep.z != nullptr) reinterpret_cast<T*>(ep.z)[at] = (T)v;
    v = mt_ep_act<sizeof(T) == 2>(v, ep.act);
    if (ep.residual != nullptr) v += (float)reinterpret_cast<const T*>(ep.residual)[at];
    y[at] = (T)v;
  }
}

// dz = dy act'(s): s is z, or (ReLU without a residual) y, whose sign is z's; and, where dz's rounding loses something (bf16, GELU),
// the column sums of dz before it, from which db comes (sums of rounded terms would be off by half again as much).  `lanes` threads
// (a power of two) take the 16-byte pieces of a row side by side, 256 / lanes rows at a time; a workgroup walks over the rows of its
// chunk and, with column sums, leaves one partial row.
template <typename T>
__global__ __launch_bounds__(256) void mt_act_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ s, T* __restrict__ dz,
                                                         float* __restrict__ part, int64_t rows, int n, int64_t ld_dy, int ld_dz,
                                                         int act, int lanes, int per) {
  constexpr int V = 16 / (int)sizeof(T);
  __shared__ float red[256 * V];
  const int lane = threadIdx.x & (lanes - 1), group = threadIdx.x / lanes, groups = 256 / lanes;
  const int col = (blockIdx.x * lanes + lane) * V;
  const int64_t lo = (int64_t)blockIdx.y * per, hi = lo + per < rows ? lo + per : rows;
  float sum[V];
#pragma unroll
  for (int e = 0; e < V; ++e) sum[e] = 0.f;
  if (col < ld_dz) {
#pragma unroll 4
    for (int64_t row = lo + group; row < hi; row += groups) {
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
        const float g = (float)a[e], z = (float)b[e];
        // ReLU passes the gradient on where the output is not a number, as it passes the output on
        const float v = act == MT_ACT_RELU ? (z > 0.f || z != z ? g : 0.f) : g * mt_ep_slope<sizeof(T) == 2>(z, act);
        sum[e] += v;
        o[e] = (T)v;
      }
      __builtin_memcpy(dz + row * ld_dz + col, o, 16);
    }
  }
  if (part == nullptr) return;
#pragma unroll
  for (int e = 0; e < V; ++e) red[threadIdx.x * V + e] = sum[e];
  __syncthreads();
  for (int i = threadIdx.x; i < lanes * V; i += 256) {
    const int c = blockIdx.x * lanes * V + i;
    if (c >= n) break;
    float v = 0.f;
    for (int g = 0; g < groups; ++g) v += red[g * lanes * V + i];
    part[(int64_t)blockIdx.y * n + c] = v;
  }
}
// db = the partial rows added in order: 16 columns x 16 strands per workgroup, the strands added in order through LDS.
template <typename B>
__global__ __launch_bounds__(256) void mt_act_cols_kernel(const float* __restrict__ part, B* __restrict__ db, int chunks, int n) {
  __shared__ float strands[16][17];
  const int cl = threadIdx.x & 15, st = threadIdx.x >> 4, c = blockIdx.x * 16 + cl;
  float v = 0.f;
  if (c < n)
    for (int i = st; i < chunks; i += 16) v += part[(int64_t)i * n + c];
  strands[st][cl] = v;
  __syncthreads();
  if (st != 0 || c >= n) return;
  v = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) v += strands[i][cl];
  db[c] = (B)v;
}

// dW [rows][cols] and db [rows]: the f32 slabs of the split contraction added up and rounded to the parameters' types.  Slab s: dW
// with rows of ld floats, then (at db_at) db.  A thread takes four columns of a row; slab s goes to sum s % 4, so that eight loads
// are on their way, and the sums are joined in a fixed order.
__device__ __forceinline__ f32x4 linear_slabs(const float* __restrict__ p, int splits, int64_t slab) {
  f32x4 acc[4] = {};
  int s = 0;
  for (; s + 8 <= splits; s += 8) {
    f32x4 v[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = *reinterpret_cast<const f32x4*>(p + (s + k) * slab);
#pragma unroll
    for (int k = 0; k < 8; ++k) acc[k & 3] += v[k];
  }
#pragma unroll 4
  for (int k = 0; k < (splits & 7); ++k) {
    const f32x4 v = *reinterpret_cast<const f32x4*>(p + (s + k) * slab);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[e] += (k & 3) == e ? v : f32x4{0.f, 0.f, 0.f, 0.f};
  }
  return (acc[0] + acc[1]) + (acc[2] + acc[3]);
}
template <typename P> __device__ __forceinline__ void linear_put4(P* at, f32x4 v, int n) {
  const P o[4] = {(P)v[0], (P)v[1], (P)v[2], (P)v[3]};
  if (n >= 4) __builtin_memcpy(at, o, sizeof(o));
  else {
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (e < n) at[e] = o[e];
  }
}
template <typename P, typename B>
__global__ __launch_bounds__(256) void mt_linear_wsum_kernel(const float* __restrict__ arena, P* __restrict__ dw, B* __restrict__ db,
                                                             int64_t rows, int cols, int ld, int64_t db_at, int splits, int64_t slab) {
  const uint32_t per_row = (uint32_t)(cols + 3) / 4;
  const int64_t of_w = rows * per_row, total = of_w + (db != nullptr ? (rows + 3) / 4 : 0);
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < total; i += (int64_t)gridDim.x * 256) {
    if (i < of_w) {
      const int64_t row = of_w <= 0xFFFFFFFFll ? (int64_t)((uint32_t)i / per_row) : i / per_row;
      const int col = (int)(i - row * per_row) * 4;
      linear_put4(dw + row * cols + col, linear_slabs(arena + row * ld + col, splits, slab), cols - col);
    } else {
      const int64_t row = (i - of_w) * 4;
      linear_put4(db + row, linear_slabs(arena + db_at + row, splits, slab), rows - row < 4 ? (int)(rows - row) : 4);
    }
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
// Which products take the 256-tile (us, depth 2048 unless said, 256-tile against 128-tile): those that the 512 places of the
// 128-tile (two per CU) do not hold at once and whose edges cost less than half again as much matrix as 128-tiles would.
//   128 tiles of 256 (4096 x 2048): 44 against 40; 136 (4352 x 2048): 44 against 59; 256: 56 against 83; 1024: 212 against 339
//   two tiles where 128-tiles are three (65536 x 384): 111 against 134, at depth 256 34 against 32; three against five (32768 x 520): 90 against 97, at depth 256 29 against 27
static bool linear_big(int64_t rows, int64_t cols, int64_t depth, int64_t lda, int64_t ldb) {
  const int64_t big = ((rows + BIGT - 1) / BIGT) * ((cols + BIGT - 1) / BIGT), small = ((rows + BM - 1) / BM) * ((cols + BN - 1) / BN);
  return lda < LT_MAX_LD && ldb < LT_MAX_LD && depth >= 4 * BK && big > 128 && 8 * big <= 3 * small;
}
static int linear_grid(int tiles_i, int tiles_j, int splits) { return (tiles_i * tiles_j * splits + 7) / 8 * 8; }

// Few rows: as many waves per workgroup as leave each at least two unrolled groups of steps, up to about 16 waves per CU.
template <typename T, int MT>
static void linear_few(const void* x, const void* w, const MtLinearEp& ep, void* y, int M, int N, int K, int64_t ldx, int64_t ldw,
                       hipStream_t stream) {
  const int step = 64 / (int)sizeof(T), steps = (K + step - 1) / step, blocks = (N + 15) / 16;
  int waves = 4;
  while (waves < 16 && blocks * waves < 256 * 16 && steps >= 4 * FEW_UNROLL * waves) waves *= 2;
  const int per = (steps + waves - 1) / waves;
#define GO(W)                                                                                                                   \
  hipLaunchKernelGGL((mt_linear_few_kernel<T, MT, W>), dim3(blocks), dim3(W * 64), 0, stream, (const T*)x, (const T*)w, ep, (T*)y, M, \
                     N, K, ldx, ldw, per)
  if (waves == 4) GO(4);
  else if (waves == 8) GO(8);
  else GO(16);
#undef GO
}
#define LINEAR_FEW_ROWS 32

// Tile edge of a launch that does not take the 256-tile, and how many parts its contraction is split into: launches of at most half
// as many tiles as the chip has CUs, whose contraction is long enough to leave every part 512 deep.
static int linear_edge(int bf16) { return bf16 ? BM : LF_TILE; }
static int linear_splits(int mode, int64_t M, int N, int KK, int bf16, int* per) {
  const int edge = linear_edge(bf16), step = bf16 ? BK : LF_BK;
  const int64_t tiles = ((M + edge - 1) / edge) * ((N + edge - 1) / edge);
  *per = KK;
  if ((mode == 0 && M <= LINEAR_FEW_ROWS) || M > LINEAR_ROWS || tiles > 128) return 1;
  int64_t want = 256 / tiles, deep = KK / 512;
  if (deep < want) want = deep;
  if (want < 2) return 1;
  *per = ((KK + (int)want - 1) / (int)want + step - 1) / step * step;
  return (KK + *per - 1) / *per;
}
// Parts [n][M][N] f32 of workspace that mt_linear_gemm_launch wants; 1: none.
extern "C" int mt_linear_parts(int mode, int64_t M, int N, int KK, int bf16) {
  if (M < 0 || N < 1 || KK < 1 || mode < 0 || mode > 1) return -2;
  int per;
  return linear_splits(mode, M, N, KK, bf16, &per);
}

// C [M][N] = act(A B + bias) + residual, contiguous, as residual and z.  A [M][lda], KK columns.  mode 0: B [N][ldb]; mode 1: B
// [KK][ldb].  Rows of A and B start on 16-byte boundaries and are whole 16-byte pieces: what an operand holds between KK (N) and the
// end of its last piece is multiplied (zeros, or rows of the other operand that are).
extern "C" int mt_linear_gemm_launch(int mode, const void* A, const void* B, const void* bias, const void* residual, void* C, void* z,
                                     float* part, int64_t M, int N, int KK, int64_t lda, int64_t ldb, int act, int bias_bf16, int bf16,
                                     hipStream_t stream) {
  const int per16 = bf16 ? 8 : 4, es = bf16 ? 2 : 4;
  if (mode < 0 || mode > 1 || M < 0 || N < 1 || KK < 1 || lda % per16 || ldb % per16 || lda < KK || ldb < (mode == 0 ? KK : N)) return -2;
  if (mode == 0 && KK % per16) return -2;
  if (lda > (bf16 ? 1 << 28 : LF_MAX_LD - 1) || ldb > (bf16 ? 1 << 28 : LF_MAX_LD - 1) || N > 2000000 || act < 0 || act > 2) return -2;
  if ((reinterpret_cast<uintptr_t>(A) | reinterpret_cast<uintptr_t>(B)) & 15) return -2;
  if (M == 0) return 0;
  if (!A || !B || !C) return -2;      // tensors without memory (of a dispatch mode) have null addresses
  if (mode == 0 && M <= LINEAR_FEW_ROWS) {
    const MtLinearEp ep = {bias, residual, z, nullptr, bias_bf16, act, N, N};
    if (bf16 && M <= 16) linear_few<__bf16, 1>(A, B, ep, C, (int)M, N, KK, lda, ldb, stream);
    else if (bf16) linear_few<__bf16, 2>(A, B, ep, C, (int)M, N, KK, lda, ldb, stream);
    else if (M <= 16) linear_few<float, 1>(A, B, ep, C, (int)M, N, KK, lda, ldb, stream);
    else linear_few<float, 2>(A, B, ep, C, (int)M, N, KK, lda, ldb, stream);
    return (int)hipGetLastError();
  }
  int per;
  const int splits = linear_splits(mode, M, N, KK, bf16, &per);
  if (splits > 1 && part == nullptr) return -2;
  for (int64_t m0 = 0; m0 < M; m0 += LINEAR_ROWS) {
    const int m = (int)(M - m0 < LINEAR_ROWS ? M - m0 : LINEAR_ROWS);
    const size_t at = (size_t)m0 * N * es;
    MtGemmGroup g = linear_group((const uint8_t*)A + (size_t)m0 * lda * es, B, (uint8_t*)C + at, m, N, KK, (int)lda, (int)ldb, N);
    MtLinearEp ep = {bias, residual ? (const uint8_t*)residual + at : nullptr, z ? (uint8_t*)z + at : nullptr,
                     splits > 1 ? part : nullptr, bias_bf16, act, N, N};
    if (bf16 && splits == 1 && linear_big(m, N, KK, lda, ldb)) {
      const int ti = (m + BIGT - 1) / BIGT, tj = (N + BIGT - 1) / BIGT;
      const dim3 grid(linear_grid(ti, tj, 1)), block(LT_THREADS);
      if (mode == 0) hipLaunchKernelGGL(mt_linear_big_kernel<0>, grid, block, 0, stream, g, ep, ti, tj);
      else hipLaunchKernelGGL(mt_linear_big_kernel<1>, grid, block, 0, stream, g, ep, ti, tj);
      continue;
    }
    const int edge = linear_edge(bf16), ti = (m + edge - 1) / edge, tj = (N + edge - 1) / edge;
    const dim3 grid(linear_grid(ti, tj, splits)), block(256);
#define GO(K, ...) hipLaunchKernelGGL((K<__VA_ARGS__>), grid, block, 0, stream, g, ep, ti, tj, splits, per)
    if (bf16) {
      const bool deep = ti * tj * splits <= 320;      // a workgroup or less per CU: four stages, else two workgroups of two
      if (mode == 0) { if (deep) GO(mt_linear_gemm_kernel, 0, 4); else GO(mt_linear_gemm_kernel, 0, 2); }
      else { if (deep) GO(mt_linear_gemm_kernel, 1, 4); else GO(mt_linear_gemm_kernel, 1, 2); }
    } else {
      if (mode == 0) GO(mt_linear_gemm_f32_kernel, 0); else GO(mt_linear_gemm_f32_kernel, 1);
    }
#undef GO
    if (splits > 1) {
      const int64_t total = (int64_t)m * N;
      const dim3 jgrid((unsigned)((total + 1023) / 1024));
      if (bf16) hipLaunchKernelGGL(mt_linear_join_kernel<__bf16>, jgrid, dim3(256), 0, stream, part, ep, (__bf16*)g.C, total, N, splits);
      else hipLaunchKernelGGL(mt_linear_join_kernel<float>, jgrid, dim3(256), 0, stream, part, ep, (float*)g.C, total, N, splits);
    }
  }
  return (int)hipGetLastError();
}

static void linear_wgrad_f32(const MtGemmGroup& g, const MtLinearEp& ep, int splits, int64_t slab, hipStream_t stream) {
  const int ti = (g.I + LF_TILE - 1) / LF_TILE, tj = (g.J + LF_TILE - 1) / LF_TILE;
  const int per = ((g.KK + splits - 1) / splits + LF_BK - 1) / LF_BK * LF_BK;
  hipLaunchKernelGGL(mt_linear_wgrad_f32_kernel, dim3(linear_grid(ti, tj, splits)), dim3(LF_THREADS), 0, stream, g, ep, ti, tj, splits,
                     per, slab);
}

// f32 parts of dW [N][K] and db [N] of dz [M][N] and x [M][K], contiguous with widths of whole 16-byte pieces: part s takes its share
// of the rows and leaves dW at arena + s slab, db behind it.
extern "C" int mt_linear_wgrad_f32_parts_launch(const void* dz, const void* x, float* arena, int64_t M, int N, int K, int splits,
                                                int64_t slab, int with_bias, hipStream_t stream) {
  if (M < 1 || M > 0x7FFFFFFF - 256 || N < 1 || K < 1 || N % 4 || K % 4 || N >= LF_MAX_LD || K >= LF_MAX_LD) return -2;
  if (!dz || !x || !arena) return -2;
  if (splits < 2 || splits > 127 || slab % 4 || slab < (int64_t)N * K + (with_bias ? N : 0)) return -2;
  MtGemmGroup g = linear_group(dz, x, arena, N, K, (int)M, N, K, K);
  if (with_bias) g.aux_out = arena + (int64_t)N * K;
  MtLinearEp ep = {};
  ep.part = arena;
  linear_wgrad_f32(g, ep, splits, slab, stream);
  return (int)hipGetLastError();
}

// dW [N][K] and db [N] (may be null) of dz [M][ld_dz] and x [M][ldx], without a split of the contraction: the widths are multiples of
// a 16-byte piece (what lies behind N and K is zeros or not stored), the gradients contiguous and of the given types.
extern "C" int mt_linear_wgrad_launch(const void* dz, const void* x, void* dw, void* db, int64_t M, int N, int K, int ld_dz, int ldx,
                                      int db_bf16, int bf16, hipStream_t stream) {
  const int per = bf16 ? 8 : 4, es = bf16 ? 2 : 4;
  if (M < 1 || M > 0x7FFFFFFF - 256 || N < 1 || K < 1 || ld_dz % per || ldx % per || ld_dz < N || ldx < K) return -2;
  if (!dz || !x || !dw) return -2;
  const int flags = db != nullptr ? MT_GEMM_FLAG_DBIAS : 0;
  if (!bf16 && (ld_dz >= LF_MAX_LD || ldx >= LF_MAX_LD)) return -2;
  if (bf16 && (K + BN - 1) / BN > 32767) return -2;    // a 128-tile's column number is 16 bits
  const int most = bf16 ? 255 * BM : N;                // output rows of a launch: the 128-tile's numbers are 8 bits here
  for (int n0 = 0; n0 < N; n0 += most) {
    const int n = N - n0 < most ? N - n0 : most;
    MtGemmGroup g = linear_group((const uint8_t*)dz + (size_t)n0 * es, x, (uint8_t*)dw + (size_t)n0 * K * es, n, K, (int)M, ld_dz, ldx, K);
    if (db != nullptr) g.aux_out = (uint8_t*)db + (size_t)n0 * (db_bf16 ? 2 : 4);
    MtLinearEp ep = {};
    ep.bias_bf16 = db_bf16;
    if (bf16 && linear_big(n, K, M, ld_dz, ldx)) {
      const int ti = (n + BIGT - 1) / BIGT, tj = (K + BIGT - 1) / BIGT;
      hipLaunchKernelGGL(mt_linear_wgrad_big_kernel, dim3(linear_grid(ti, tj, 1)), dim3(LT_THREADS), 0, stream, g, ep, ti, tj, flags);
    } else if (bf16) {
      const int ti = (n + BM - 1) / BM, tj = (K + BN - 1) / BN;
      if (ti * tj <= 320)
        hipLaunchKernelGGL(mt_linear_wgrad_kernel<4>, dim3(linear_grid(ti, tj, 1)), dim3(NTHREADS), 0, stream, g, ep, ti, tj, flags);
      else
        hipLaunchKernelGGL(mt_linear_wgrad_kernel<2>, dim3(linear_grid(ti, tj, 1)), dim3(NTHREADS), 0, stream, g, ep, ti, tj, flags);
    } else {
      linear_wgrad_f32(g, ep, 1, 0, stream);
    }
  }
  return (int)hipGetLastError();
}

struct ActGrid {
  int lanes, strips, chunks, per;
};
static ActGrid act_grid(int64_t M, int ld_dz, int bf16, bool sums) {
  const int pieces = ld_dz / (bf16 ? 8 : 4);
  ActGrid g;
  g.lanes = 4;
  while (g.lanes < 64 && g.lanes < pieces) g.lanes *= 2;
  g.strips = (pieces + g.lanes - 1) / g.lanes;
  // About eight workgroups per CU; with column sums, each of which costs a partial row, they walk over an unrolled batch of rows or more.
  int64_t chunks = (2048 + g.strips - 1) / g.strips;
  const int64_t deep = M / ((sums ? 4 : 1) * (256 / g.lanes));
  if (chunks > deep) chunks = deep;
  if (chunks < 1) chunks = 1;
  if (chunks < M / (1 << 24)) chunks = M / (1 << 24) + 1;
  g.per = (int)((M + chunks - 1) / chunks);
  g.chunks = (int)((M + g.per - 1) / g.per);
  return g;
}
// Rows of the partial-sum workspace [n][N] f32.
extern "C" int mt_linear_act_parts(int64_t M, int ld_dz, int bf16) {
  if (M < 1 || ld_dz < 1 || ld_dz % (bf16 ? 8 : 4)) return -2;
  return act_grid(M, ld_dz, bf16, true).chunks;
}
// s: z or y [M][N] contiguous; dz [M][ld_dz], ld_dz a multiple of a 16-byte piece, zeros behind column N.  db [N] with its workspace
// `part`, or both null.
extern "C" int mt_linear_act_bwd_launch(const void* dy, const void* s, void* dz, float* part, void* db, int64_t M, int N, int64_t ld_dy,
                                        int ld_dz, int act, int db_bf16, int bf16, hipStream_t stream) {
  const int per = bf16 ? 8 : 4;
  if (M < 0 || N < 1 || ld_dz % per || ld_dz < N || ld_dz - N >= per || ld_dy < 0 || act < 1 || act > 2) return -2;
  if ((part == nullptr) != (db == nullptr)) return -2;
  if (M == 0) return 0;
  if (!dy || !s || !dz) return -2;
  const ActGrid g = act_grid(M, ld_dz, bf16, db != nullptr);
  if (g.chunks > 65535) return -2;
  const dim3 grid((unsigned)g.strips, (unsigned)g.chunks);
  if (bf16)
    hipLaunchKernelGGL(mt_act_bwd_kernel<__bf16>, grid, dim3(256), 0, stream, (const __bf16*)dy, (const __bf16*)s, (__bf16*)dz, part, M,
                       N, ld_dy, ld_dz, act, g.lanes, g.per);
  else
    hipLaunchKernelGGL(mt_act_bwd_kernel<float>, grid, dim3(256), 0, stream, (const float*)dy, (const float*)s, (float*)dz, part, M, N,
                       ld_dy, ld_dz, act, g.lanes, g.per);
  if (db != nullptr) {
    const dim3 cols((unsigned)((N + 15) / 16));
    if (db_bf16) hipLaunchKernelGGL(mt_act_cols_kernel<__bf16>, cols, dim3(256), 0, stream, part, (__bf16*)db, g.chunks, N);
    else hipLaunchKernelGGL(mt_act_cols_kernel<float>, cols, dim3(256), 0, stream, part, (float*)db, g.chunks, N);
  }
  return (int)hipGetLastError();
}

// dw [rows][cols], db [rows] (may be null).
extern "C" int mt_linear_wsum_launch(const float* arena, void* dw, void* db, int64_t rows, int cols, int ld, int64_t db_at, int splits,
                                     int64_t slab, int w_bf16, int b_bf16, hipStream_t stream) {
  if (rows < 1 || cols < 1 || ld < cols || ld % 4 || db_at % 4 || slab % 4 || splits < 1 || slab < db_at + (db != nullptr ? (rows + 3) / 4 * 4 : 0))
    return -2;
  if (!arena || !dw || (reinterpret_cast<uintptr_t>(arena) & 15)) return -2;
  const int64_t blocks = (rows * ((cols + 3) / 4) + (rows + 3) / 4 + 255) / 256;
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

// The whole backward pass of a layer in one call: dz (with db from it before its rounding, where part_at is set), dx, then dW and what
// is left of db.  Offsets into the workspace are in bytes, negative where a piece is not needed; splits 0: dW leaves in its own type;
// -1: a small f32 layer (w [rows][width] contiguous, dw wanted), whose gradients are one launch of small_linear.hip and have its padded
// widths.
struct MtLinearBwd {
  const void *dy, *s, *x, *w;
  void *dx, *dw, *db;
  uint8_t* ws;
  int64_t M, dy_ld, ldw, dz_at, part_at, dxpart_at, arena_at, slab;
  int32_t N, K, rows, width, act, bf16, dw_bf16, db_bf16, splits, small_tile;      // rows, width: N and K in whole 16-byte pieces
};
extern "C" int mt_wgrad_single_launch(const void* dY, const void* X, float* C, float* db, int M, int out, int in, int ksplits,
                                      size_t split_stride, hipStream_t stream);
extern "C" int mt_small_linear_bwd_tiled_launch(const float* X, const float* W, const float* dY, float* dX, float* dW, float* db, int R, int in,
                                                int out, int tile, hipStream_t stream);
extern "C" int mt_linear_bwd_size() { return (int)sizeof(MtLinearBwd); }
extern "C" int mt_linear_bwd_launch(const MtLinearBwd* a, hipStream_t stream) {
  if (a == nullptr) return -2;
  const MtLinearBwd p = *a;
  if (p.M < 1 || p.M > 0x7FFFFFFF - 256 || p.rows < p.N || p.width < p.K || (p.act != 0) != (p.dz_at >= 0) || (p.act == 0 && p.dy_ld != p.rows))
    return -2;
  const void* dz = p.act ? p.ws + p.dz_at : p.dy;
  void* late = p.part_at >= 0 ? nullptr : p.db;
  int rc = 0;
  if (p.act)
    rc = mt_linear_act_bwd_launch(p.dy, p.s, p.ws + p.dz_at, p.part_at >= 0 ? (float*)(p.ws + p.part_at) : nullptr,
                                  p.part_at >= 0 ? p.db : nullptr, p.M, p.N, p.dy_ld, p.rows, p.act, p.db_bf16, p.bf16, stream);
  if (p.splits < 0) {
    if (rc != 0 || p.bf16 || p.ldw != p.width) return rc != 0 ? rc : -2;
    return mt_small_linear_bwd_tiled_launch((const float*)p.x, (const float*)p.w, (const float*)dz, (float*)p.dx, (float*)p.dw, (float*)late,
                                            (int)p.M, p.width, p.rows, p.small_tile, stream);
  }
  if (rc == 0 && p.dx != nullptr)
    rc = mt_linear_gemm_launch(1, dz, p.w, nullptr, nullptr, p.dx, nullptr, p.dxpart_at >= 0 ? (float*)(p.ws + p.dxpart_at) : nullptr,
                               p.M, p.K, p.N, p.rows, p.ldw, 0, 0, p.bf16, stream);
  if (rc != 0 || p.dw == nullptr) return rc;
  if (p.splits == 0) return mt_linear_wgrad_launch(dz, p.x, p.dw, late, p.M, p.N, p.K, p.rows, p.width, p.db_bf16, p.bf16, stream);
  float* arena = (float*)(p.ws + p.arena_at);
  const int64_t db_at = (int64_t)p.rows * p.width;
  rc = p.bf16 ? mt_wgrad_single_launch(dz, p.x, arena, late != nullptr ? arena + db_at : nullptr, (int)p.M, p.rows, p.width, p.splits, p.slab, stream)
              : mt_linear_wgrad_f32_parts_launch(dz, p.x, arena, p.M, p.rows, p.width, p.splits, p.slab, late != nullptr, stream);
  if (rc != 0) return rc;
  return mt_linear_wsum_launch(arena, p.dw, late, p.N, p.K, p.width, db_at, p.splits, p.slab, p.dw_bf16, p.db_bf16, stream);
}
