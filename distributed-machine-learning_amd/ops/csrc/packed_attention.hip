// Attention over packed sequences, forward and backward (gfx950): rows of q [T][heads][dk], k [T][kv_heads][dk] and
// v [T][kv_heads][dv] hold sequences of different lengths one after the other; a query sees the keys of its own sequence,
// all of them or (causal) those up to its own position; query head i reads key / value head i / (heads / kv_heads).
//
//   forward : s_ij = c q_i.k_j (c = scale log2 e),  p_ij = 2^(s_ij - L_i),  o_i = sum_j p_ij v_j,  L_i = log2 sum_j 2^s_ij
//             one pass over the keys with the running maximum m_i and sum of a softmax; L_i is kept for the backward pass
//   backward: D_i = do_i.o_i,  ds_ij = p_ij (do_i.v_j - D_i),
//             dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,  dv_j = sum_i p_ij do_i
//
// A workgroup is four waves.  In the forward and the dq kernel a wave owns 32 queries and walks over the keys; in the dk / dv
// kernel it owns 32 keys and walks over the queries of every head of the group, so each gradient element is summed by one
// wave in a fixed order: no atomics, no workspace, and the gradients of shared heads need no second pass (but for walks longer
// than a CU's share of the launch, which two workgroups share by heads: 20 documents of up to 2048, 16 / 4 heads of 128, backward
// 412 -> 393 us).  The price is that the scores are computed again in both backward kernels (7 products where 5 are the least).
//
// Every product is v_mfma_*_32x32: the walked-over rows come from LDS as the first operand, the owned rows stay in registers
// as the second, so an accumulator lane belongs to ONE owned row: row statistics are one register, a row maximum is a chain in
// the lane and one exchange with lane ^ 32.  The accumulator of the scores then IS the second operand of the next product
// (sum over the walked-over rows): lane half h holds rows 8 g + 4 h + 0..3 of each 32, and the transposed LDS read fetches the
// other operand in that same order, so probabilities never move between lanes or through LDS.
//
// f32 operands use v_mfma_f32_32x32x2_f32 (exact f32 products) in the same layout: eight instructions where bf16 takes one.
// Scores, statistics, gradients and all sums are f32 for both types; for bf16 p and ds are rounded to bf16 (at most
// 2^-8 of the value) as operands of the second product, which is what the matrix instruction takes; where few rows meet
// (pa_few_keys), the gradients add the product of what that took off.
#include "mt_common.h"

typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef __attribute__((ext_vector_type(8))) float f32x8;
typedef __attribute__((address_space(3))) uint8_t lds_u8;

#define PA_THREADS 256
#define PA_OWN 128          // rows a workgroup owns (32 per wave)
#define PA_TILE 32          // rows a workgroup of the split form owns, and rows of its tiles

// One item of owned rows: rows [row0, row0 + len) are its sequence, `first` is the item's first row in it.  An item is PA_OWN rows,
// or in the split form PA_TILE rows unless it is `solo`.  len < 0: -len rows from row0 belong to no sequence and are filled with
// zeros.
struct MtSeqItem {
  int32_t row0, len, first, solo;
};

struct MtPackedAttn {
  const void *q, *k, *v;        // inputs, element strides below; the last dimension is contiguous
  const void *out, *dout;       // backward only: forward output (contiguous) and its gradient
  void *o, *dq, *dk, *dv;       // outputs, contiguous [T][heads or kv_heads][dk or dv]
  void* low;                    // bf16 [T][heads][dv]: what rounding took off the output's rows of few keys; may be null
  float *lse, *delta;           // [heads][rows]
  float* halves;                // what the two workgroups of a cut walk leave, [cut items][kv_heads][2][dk, dv][128][D]
  const MtSeqItem *items, *kv_items;      // items of query rows and of key rows; null: count sequences of uniform_len rows each
  int64_t q_row, q_head, k_row, k_head, v_row, v_head, do_row, do_head;
  int64_t rows;
  int32_t n_items, n_kv_items, uniform_len, count;
  int32_t heads, kv_heads, head_k, head_v, causal;
  int32_t split, kv_split;      // the launch's form: 0 shared, 1 split, 2 split with every item solo (of a uniform batch)
  int32_t cut;                  // leading key items whose walk two workgroups share, half the heads of the group each
  float scale;
};

// ---- per-type pieces ----------------------------------------------------------------------------------------------------
// A fragment is 8 elements per lane = 16 of the contraction (lane half h holds 8 of them) of row (lane & 31).
template <typename T> struct PaFrag;
template <> struct PaFrag<__bf16> { typedef bf16x8 type; };
template <> struct PaFrag<float> { typedef f32x8 type; };

__device__ __forceinline__ f32x16 pa_mma(bf16x8 a, bf16x8 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16 pa_mma(f32x8 a, f32x8 b, f32x16 c) {
#pragma unroll
  for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
  return c;
}

// sum + the fragment's elements: the row sum adds the probabilities as they are multiplied, so that rounding them moves the
// weights of a row but not their total (half the error of an output over few keys, and what makes D exact enough there).
__device__ __forceinline__ float pa_row_sum(bf16x8 f, float sum) {
  typedef __bf16 pair __attribute__((ext_vector_type(2)));
  const pair one = {(__bf16)1.f, (__bf16)1.f};
#pragma unroll
  for (int j = 0; j < 8; j += 2) sum = __builtin_amdgcn_fdot2_f32_bf16(pair{f[j], f[j + 1]}, one, sum, false);
  return sum;
}
__device__ __forceinline__ float pa_row_sum(f32x8 f, float sum) {
#pragma unroll
  for (int j = 0; j < 8; ++j) sum += f[j];
  return sum;
}

// Accumulator rows 16 s .. 16 s + 15 (eight registers per lane) as a fragment of the next product.
template <typename T> __device__ __forceinline__ typename PaFrag<T>::type pa_pack(const f32x16& a, int s);
template <> __device__ __forceinline__ bf16x8 pa_pack<__bf16>(const f32x16& a, int s) {
  const u32x4 w = {pack_bf16x2(a[8 * s], a[8 * s + 1]), pack_bf16x2(a[8 * s + 2], a[8 * s + 3]),
                   pack_bf16x2(a[8 * s + 4], a[8 * s + 5]), pack_bf16x2(a[8 * s + 6], a[8 * s + 7])};
  return __builtin_bit_cast(bf16x8, w);
}
template <> __device__ __forceinline__ f32x8 pa_pack<float>(const f32x16& a, int s) {
  return f32x8{a[8 * s], a[8 * s + 1], a[8 * s + 2], a[8 * s + 3], a[8 * s + 4], a[8 * s + 5], a[8 * s + 6], a[8 * s + 7]};
}

// What the rounding of pa_pack took off, as a fragment of its own (f32: nothing).
template <typename T> __device__ __forceinline__ typename PaFrag<T>::type pa_rest(const f32x16& a, int s, const typename PaFrag<T>::type& f) {
  if constexpr (sizeof(T) == 2) {
    const u32x4 w = __builtin_bit_cast(u32x4, f);
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      r[i] = pack_bf16x2(a[8 * s + 2 * i] - __uint_as_float(w[i] << 16), a[8 * s + 2 * i + 1] - __uint_as_float(w[i] & 0xFFFF0000u));
    return __builtin_bit_cast(bf16x8, r);
  } else {
    return f - f;
  }
}

template <typename V> __device__ __forceinline__ const __attribute__((address_space(3))) V* pa_lds(uint32_t at) {
  return (const __attribute__((address_space(3))) V*)(uintptr_t)at;
}
template <typename V> __device__ __forceinline__ __attribute__((address_space(3))) V* pa_lds_mut(uint32_t at) {
  return (__attribute__((address_space(3))) V*)(uintptr_t)at;
}
__device__ __forceinline__ uint32_t pa_lds_at(const uint8_t* p) { return (uint32_t)(uintptr_t)(const lds_u8*)p; }

// LDS image of rows of D elements: 16-byte chunk c of row r sits at chunk c ^ swz(r), so that eight rows read at one column
// (row fragments) and four rows x 32 bytes (transposed reads) both cover all banks.
template <typename T, int D> struct PaImg {
  static constexpr int ROWB = D * (int)sizeof(T);
  static constexpr int CHUNKS = ROWB / 16;
  static constexpr int EPC = 16 / (int)sizeof(T);
  static __device__ __forceinline__ int swz(int r) {
    if (sizeof(T) == 4) return r & 7;
    if (D == 128) return ((r & 3) << 2) | ((r >> 2) & 3);
    if (D == 64) return ((r & 3) << 1) | ((r >> 2) & 1);
    return (((r >> 1) & 1) << 1) | ((r >> 2) & 1);
  }
  static __device__ __forceinline__ int at(int r, int chunk) { return r * ROWB + ((chunk ^ swz(r)) << 4); }

  // Fragment reads take an LDS byte address: the image's (a multiple of 1 KiB) plus row_base or col_base of the lane, worked out
  // once.  What is left per fragment is one exclusive-or with a constant (the swizzle leaves bits above a row alone) and an
  // immediate offset.
  static __device__ __forceinline__ uint32_t row_base(int lane) {
    const int r = lane & 31, h = lane >> 5;
    return (uint32_t)at(r, sizeof(T) == 2 ? h : 2 * h);
  }
  // 16 columns 16 s + 8 h + j of row row0 + (lane & 31)
  static __device__ __forceinline__ typename PaFrag<T>::type rows(uint32_t base, int row0, int s) {
    if constexpr (sizeof(T) == 2) {
      return __builtin_bit_cast(bf16x8, *pa_lds<u32x4>((base ^ (s << 5)) + row0 * ROWB));
    } else {
      const f32x4 lo = *pa_lds<f32x4>((base ^ (s << 6)) + row0 * ROWB), hi = *pa_lds<f32x4>((base ^ (s << 6) ^ 16) + row0 * ROWB);
      return f32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    }
  }
  static __device__ __forceinline__ uint32_t col_base(int lane) {
    const int h = lane >> 5;
    if constexpr (sizeof(T) == 2) {
      const int i = lane & 15, q = i >> 2, p = i & 3;
      return (uint32_t)(at(4 * h + q, (lane & 16) / 8 + (p >> 1)) + 8 * (p & 1));
    } else {
      return (uint32_t)(at(4 * h, (lane & 31) >> 2) + 4 * (lane & 3));
    }
  }
  // column 32 b + (lane & 31) of the 16 rows row0 + 8 (j / 4) + 4 h + j % 4 (row0 a multiple of 16): the order of an
  // accumulator's rows
  static __device__ __forceinline__ typename PaFrag<T>::type cols(uint32_t base, int row0, int b) {
    if constexpr (sizeof(T) == 2) {
      constexpr int FAR = D == 128 ? 32 : 0;           // how the swizzle of row r + 8 differs from that of r
      const s16x4 lo = mt_read_tr(pa_lds_mut<s16x4>((base ^ (b << 6)) + row0 * ROWB));
      const s16x4 hi = mt_read_tr(pa_lds_mut<s16x4>((base ^ (b << 6) ^ FAR) + (row0 + 8) * ROWB));
      typedef __attribute__((ext_vector_type(8))) short s16x8;
      const s16x8 v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
      return __builtin_bit_cast(bf16x8, v);
    } else {
      f32x8 v;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = *pa_lds<float>((base ^ (b << 7) ^ ((j & 3) << 4)) + (row0 + 8 * (j >> 2) + (j & 3)) * ROWB);
      return v;
    }
  }
  // LDS-DMA of NROWS rows of `d` valid columns into an image, WAVES waves sharing the 1-KiB pieces.  `base` is the first row's
  // first element; rows at and past `valid` and columns past `d` arrive as zeros through the buffer's range check.
  template <int NROWS, int WAVES = 4>
  static __device__ __forceinline__ void stage(uint8_t* img, const T* base, int64_t row_stride, int valid, int d, int wave, int lane) {
    constexpr int ALL = NROWS * ROWB / 1024, PIECES = (ALL + WAVES - 1) / WAVES;
    static_assert(ALL * 1024 == NROWS * ROWB && (ALL % WAVES == 0 || PIECES == 1), "an image is whole pieces, shared evenly or one each");
    const int64_t stride = row_stride * (int64_t)sizeof(T);
    const int rows = valid < NROWS ? valid : NROWS;
    const uint32_t bytes = rows > 0 ? (uint32_t)((rows - 1) * stride + d * (int)sizeof(T)) : 0u;
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(const_cast<T*>(base), 0, bytes, 0x00027000);
#pragma unroll
    for (int t = 0; t < PIECES; ++t) {
      const int j = wave * PIECES + t;
      if (ALL % WAVES != 0 && j >= ALL) break;
      const int at_byte = j * 1024 + lane * 16;
      const int r = at_byte / ROWB, c = ((at_byte % ROWB) >> 4) ^ swz(r);
      const uint32_t off = c * EPC < d ? (uint32_t)(r * (uint32_t)stride + c * 16) : 0xFFFFFF00u;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)(img + j * 1024), 16, off, 0, 0, 0);
    }
  }
};

// max / sum with the lane 32 further on: one exchange of the wave's halves, no LDS
__device__ __forceinline__ float pa_half_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float pa_half_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

template <typename T> __device__ __forceinline__ typename PaFrag<T>::type pa_zero_frag() {
  typename PaFrag<T>::type f;
#pragma unroll
  for (int j = 0; j < 8; ++j) f[j] = (T)0.f;
  return f;
}
// An owned row as fragments: columns 16 s + 8 h + j, zeros past d or when the row is outside its sequence.
template <typename T, int D>
__device__ __forceinline__ void pa_own_row(typename PaFrag<T>::type (&f)[D / 16], const T* row, bool ok, int d, int lane) {
  const int h = lane >> 5;
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    f[s] = pa_zero_frag<T>();
    const int c = 16 * s + 8 * h;
    if constexpr (sizeof(T) == 2) {
      if (ok && c < d) f[s] = __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4*>(row + c));
    } else {
      f32x4 lo = {0.f, 0.f, 0.f, 0.f}, hi = lo;
      if (ok && c < d) lo = *reinterpret_cast<const f32x4*>(row + c);
      if (ok && c + 4 < d) hi = *reinterpret_cast<const f32x4*>(row + c + 4);
      f[s] = f32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    }
  }
}
// Four consecutive columns of a row; `low` (bf16 only, may be null) gets what the rounding took off.
template <typename T> __device__ __forceinline__ void pa_store4(T* at, T* low, float v0, float v1, float v2, float v3) {
  if constexpr (sizeof(T) == 2) {
    const u32x2 w = {pack_bf16x2(v0, v1), pack_bf16x2(v2, v3)};
    *reinterpret_cast<u32x2*>(at) = w;
    if (low != nullptr) {
      auto left = [](float a, float b, uint32_t r) {
        return pack_bf16x2(a - __uint_as_float(r << 16), b - __uint_as_float(r & 0xFFFF0000u));
      };
      *reinterpret_cast<u32x2*>(low) = u32x2{left(v0, v1, w[0]), left(v2, v3, w[1])};
    }
  } else {
    *reinterpret_cast<f32x4*>(at) = f32x4{v0, v1, v2, v3};
  }
}
// Store a transposed accumulator (rows = columns of the output, lane & 31 = owned row).
template <typename T, int D>
__device__ __forceinline__ void pa_store_row(T* row, const f32x16 (&acc)[D / 32], float factor, int d, int lane, T* low = nullptr) {
  const int h = lane >> 5;
#pragma unroll
  for (int b = 0; b < D / 32; ++b)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int c = 32 * b + 8 * g + 4 * h;
      if (c < d) {
        pa_store4(row + c, low != nullptr ? low + c : nullptr, acc[b][4 * g] * factor, acc[b][4 * g + 1] * factor,
                  acc[b][4 * g + 2] * factor, acc[b][4 * g + 3] * factor);
      }
    }
}
template <int N> __device__ __forceinline__ void pa_clear(f32x16 (&a)[N]) {
#pragma unroll
  for (int b = 0; b < N; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i) a[b][i] = 0.f;
}

// Which item this workgroup takes.  Items come longest first (causal: the last queries, or the first keys).
__device__ __forceinline__ MtSeqItem pa_item(const MtPackedAttn& p, const MtSeqItem* items, int i, int split, bool last_first) {
  if (items != nullptr) return items[i];
  const int rows = split == 1 ? PA_TILE : PA_OWN, n = (p.uniform_len + rows - 1) / rows;
  const int t = i / p.count, seq = i - t * p.count;
  return MtSeqItem{seq * p.uniform_len, p.uniform_len, (last_first ? n - 1 - t : t) * rows, split == 2};
}
// Zeros for `n` rows of `d` columns of one head, which belong to no sequence.
template <typename T>
__device__ __forceinline__ void pa_zero_rows(T* base, int64_t row_stride, int n, int d) {
  for (int i = threadIdx.x; i < n * d; i += blockDim.x) {
    const int r = i / d;
    base[r * row_stride + (i - r * d)] = (T)0.f;
  }
}
// This wave's LDS-DMA has landed and its reads of the other stage are back; past the barrier that holds for everybody.
__device__ __forceinline__ void pa_tile_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// The four waves' partial results of 32 rows: [wave][column][row] f32, added in wave order and stored.
template <int D>
__device__ __forceinline__ void pa_join(float* join, const f32x16 (&acc)[D / 32], float factor, int wave, int lane) {
#pragma unroll
  for (int b = 0; b < D / 32; ++b)
#pragma unroll
    for (int i = 0; i < 16; ++i)
      join[(wave * D + 32 * b + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3)) * 32 + (lane & 31)] = acc[b][i] * factor;
}
template <typename T, int D>
__device__ __forceinline__ void pa_join_store(T* base, int64_t row_stride, const float* join, int rows, int d, T* low = nullptr) {
  const int r = threadIdx.x & 31;
  if (r >= rows) return;
#pragma unroll
  for (int c0 = 0; c0 < D / 8; c0 += 4) {
    const int c = (threadIdx.x >> 5) * (D / 8) + c0;
    if (c >= d) return;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w)
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += join[(w * D + c + e) * 32 + r];
    pa_store4(base + r * row_stride + c, low != nullptr ? low + r * row_stride + c : nullptr, v[0], v[1], v[2], v[3]);
  }
}
// Rows whose output is kept with what its rounding took off (MtPackedAttn::low), those that see at most 128 keys: over few keys
// D = do . o is as large as the do . v it is subtracted from, and half a bf16 step of o would show in the gradients (two keys: 0.8 %
// of dq against 0.23 %; causal sequences of up to 2048, whose first rows have the largest gradients: 0.25 against 0.24).  `first`:
// the first of the item's rows, all of which are on the same side of 128.
#define PA_LOW_ROWS 128
__device__ __forceinline__ bool pa_few_keys(const MtPackedAttn& p, int len, int first) {
  return len <= PA_LOW_ROWS || (p.causal && first < PA_LOW_ROWS);
}
__device__ __forceinline__ bool pa_low(const MtPackedAttn& p, int len, int first) {
  return p.low != nullptr && pa_few_keys(p, len, first);
}
// Rows that see at most 128 keys, and keys that at most 128 rows see (`few`, bf16): the gradients' sums of ds and p have too few terms
// for their roundings to average out, so what those took off is multiplied too.  Error of dq and dk against 64 bits, of their norm
// (0.0017 is the rounding of the output): sequences of 2 to 16 rows 0.0025 -> 0.0019; a causal sequence of 1797, heads of 16, whose first
// rows have the largest gradients, dq 0.0025 -> 0.0022.  Those walks are so short that it costs no time.
template <typename T, typename Img, int D>
__device__ __forceinline__ void pa_add_rest(f32x16 (&acc)[D / 32], uint32_t cols, int h, const typename PaFrag<T>::type& rest) {
#pragma unroll
  for (int b = 0; b < D / 32; ++b) acc[b] = pa_mma(Img::cols(cols, 16 * h, b), rest, acc[b]);
}
// What the dq kernels hold of an owned row: q, do, L and D = do . o (stored for the dk / dv kernel by the waves with `store`).
template <typename T, int DK, int DV>
__device__ __forceinline__ void pa_dq_rows(const MtPackedAttn& p, typename PaFrag<T>::type (&qf)[DK / 16],
                                           typename PaFrag<T>::type (&df)[DV / 16], float& delta, float& lse, int64_t row, int head, bool ok,
                                           bool store, bool low, int lane) {
  pa_own_row<T, DV>(df, reinterpret_cast<const T*>(p.dout) + row * p.do_row + (int64_t)head * p.do_head, ok, p.head_v, lane);
  delta = 0.f;
  lse = INFINITY;                                       // rows outside the sequence: p = 2^(s - inf) = 0
  {
    typename PaFrag<T>::type of[DV / 16];
    pa_own_row<T, DV>(of, reinterpret_cast<const T*>(p.out) + row * ((int64_t)p.heads * p.head_v) + (int64_t)head * p.head_v, ok, p.head_v,
                      lane);
#pragma unroll
    for (int s = 0; s < DV / 16; ++s)
#pragma unroll
      for (int j = 0; j < 8; ++j) delta = __builtin_fmaf((float)df[s][j], (float)of[s][j], delta);
    if (low) {
      pa_own_row<T, DV>(of, reinterpret_cast<const T*>(p.low) + row * ((int64_t)p.heads * p.head_v) + (int64_t)head * p.head_v, ok, p.head_v,
                        lane);
#pragma unroll
      for (int s = 0; s < DV / 16; ++s)
#pragma unroll
        for (int j = 0; j < 8; ++j) delta = __builtin_fmaf((float)df[s][j], (float)of[s][j], delta);
    }
  }
  delta = pa_half_sum(delta);
  if (ok) {
    lse = p.lse[(int64_t)head * p.rows + row];
    if (store && lane < 32) p.delta[(int64_t)head * p.rows + row] = delta;
  }
  pa_own_row<T, DK>(qf, reinterpret_cast<const T*>(p.q) + row * p.q_row + (int64_t)head * p.q_head, ok, p.head_k, lane);
}

// ---- forward ------------------------------------------------------------------------------------------------------------
template <typename T, int D, int BN>
__global__ __launch_bounds__(PA_THREADS, 2) void mt_pattn_fwd_kernel(const MtPackedAttn p) {
  typedef PaImg<T, D> Img;
  typedef typename PaFrag<T>::type Frag;
  constexpr int IMG = BN * Img::ROWB;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[4 * IMG];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int it = blockIdx.x / p.heads, r = blockIdx.x - it * p.heads;
  // heads of one group are kv_heads workgroups apart: the XCDs (workgroup number mod 8) then share few key / value heads each
  const int kvh = r % p.kv_heads, head = kvh * (p.heads / p.kv_heads) + r / p.kv_heads;
  const MtSeqItem item = pa_item(p, p.items, it, 0, p.causal);
  const int64_t o_row = (int64_t)p.heads * p.head_v;
  T* o = reinterpret_cast<T*>(p.o) + item.row0 * o_row + (int64_t)head * p.head_v;
  T* low = sizeof(T) == 2 && pa_low(p, item.len, item.first) ? reinterpret_cast<T*>(p.low) + item.row0 * o_row + (int64_t)head * p.head_v : nullptr;
  if (item.len <= 0) {
    pa_zero_rows<T>(o, o_row, -item.len, p.head_v);
    return;
  }
  const int first = item.first + wave * 32, mine = first + (lane & 31);
  Frag qf[D / 16];
  pa_own_row<T, D>(qf, reinterpret_cast<const T*>(p.q) + (item.row0 + (int64_t)mine) * p.q_row + (int64_t)head * p.q_head,
                   mine < item.len, p.head_k, lane);
  const T* kb = reinterpret_cast<const T*>(p.k) + item.row0 * p.k_row + (int64_t)kvh * p.k_head;
  const T* vb = reinterpret_cast<const T*>(p.v) + item.row0 * p.v_row + (int64_t)kvh * p.v_head;
  const int keys = p.causal && item.first + PA_OWN < item.len ? item.first + PA_OWN : item.len;
  const int tiles = (keys + BN - 1) / BN;
  const float c = p.scale * 1.4426950408889634f;

  // Tiles are fetched in order: the next one's addresses are carried along, not worked out per tile ahead of its fetch.
  const T *k_next = kb, *v_next = vb;
  int left = item.len;
  const int64_t k_hop = BN * p.k_row, v_hop = BN * p.v_row;
  auto issue = [&](int t) {
    uint8_t* st = lds + (t & 1) * 2 * IMG;
    Img::template stage<BN>(st, k_next, p.k_row, left, p.head_k, wave, lane);
    Img::template stage<BN>(st + IMG, v_next, p.v_row, left, p.head_v, wave, lane);
    k_next += k_hop;
    v_next += v_hop;
    left -= BN;
  };

  f32x16 acc[D / 32];
  pa_clear(acc);
  float m = -INFINITY, sum = 0.f;
  const uint32_t lds_at = pa_lds_at(lds);
  // One tile.  Fragments are read in groups, the next group on its way while the products of one run: the scheduling barriers
  // keep that order (left alone the compiler reads each fragment right before its product and waits for it: 1.4x the time).
  auto step = [&](int t, bool masked) {
    const int k0 = t * BN;
    const uint32_t krow = lds_at + (t & 1) * 2 * IMG + Img::row_base(lane), vcol = lds_at + ((t & 1) * 2 + 1) * IMG + Img::col_base(lane);
    constexpr int U = BN / 32, KG = D / 32, PG = BN / 16;      // groups: two steps of the scores; 16 keys of the output
    Frag kf[2][2][U], vf[2][D / 32];
    auto read_k = [&](int g) {
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int u = 0; u < U; ++u) kf[g & 1][e][u] = Img::rows(krow, 32 * u, 2 * g + e);
    };
    auto read_v = [&](int g) {
#pragma unroll
      for (int b = 0; b < D / 32; ++b) vf[g & 1][b] = Img::cols(vcol, 16 * g, b);
    };
    f32x16 s[U];
    pa_clear(s);
    read_k(0);
#pragma unroll
    for (int g = 0; g < KG; ++g) {
      if (g + 1 < KG) read_k(g + 1);
      else read_v(0);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int u = 0; u < U; ++u) s[u] = pa_mma(kf[g & 1][e][u], qf[2 * g + e], s[u]);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (masked) {
      const int last = p.causal && mine < item.len ? mine : item.len - 1;
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          s[u][i] = k0 + 32 * u + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3) <= last ? s[u][i] : -INFINITY;
    }
    float mx = s[0][0];
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[u][i]);
    mx = pa_half_max(mx) * c;
    // The subtracted maximum is only moved when some row grew by more than 2^8 over it: probabilities stay within f32 (and
    // bf16 keeps its relative precision), and most tiles skip the pass over the accumulator.
    if (__any(mx > m + 8.f)) {
      const float mn = fmaxf(m, mx);
      const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      sum *= f;
#pragma unroll
      for (int b = 0; b < D / 32; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[b][i] *= f;
    }
    const float sub = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        s[u][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[u][i], c, -sub));
      }
#pragma unroll
    for (int g = 0; g < PG; ++g) {
      if (g + 1 < PG) read_v(g + 1);
      const Frag pf = pa_pack<T>(s[g >> 1], g & 1);
      sum = pa_row_sum(pf, sum);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int b = 0; b < D / 32; ++b) acc[b] = pa_mma(vf[g & 1][b], pf, acc[b]);
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  // Tiles that all of this wave's queries see whole, tiles that need the mask, and tiles it only helps to fetch.
  const int mine_end = p.causal && first + 32 < keys ? first + 32 : keys;          // keys this wave looks at
  const int own = first < item.len ? (mine_end + BN - 1) / BN : 0;
  const int whole = p.causal && first + 1 < mine_end ? (first + 1) / BN : mine_end / BN;
  issue(0);
  auto enter = [&](int t) {
    pa_tile_barrier();
    if (t + 1 < tiles) issue(t + 1);
  };
  int t = 0;
  for (; t < whole && t < own; ++t) {
    enter(t);
    step(t, false);
  }
  for (; t < own; ++t) {
    enter(t);
    step(t, true);
  }
  for (; t < tiles; ++t) enter(t);
  sum = pa_half_sum(sum);
  if (mine < item.len) {      // every row sees a key: sum is 0 only where all its scores are -inf, and the output 0 / 0 as in the formula
    pa_store_row<T, D>(o + (int64_t)mine * o_row, acc, 1.f / sum, p.head_v, lane, low != nullptr ? low + (int64_t)mine * o_row : nullptr);
    if (p.lse != nullptr && lane < 32) p.lse[(int64_t)head * p.rows + item.row0 + mine] = m + __builtin_amdgcn_logf(sum);
  }
}

// ---- backward: dq (and D = do . o, which the dk / dv kernel reads) --------------------------------------------------------
template <typename T, int D, int BN>
__global__ __launch_bounds__(PA_THREADS, sizeof(T) == 4 && D == 128 ? 1 : 2) void mt_pattn_dq_kernel(const MtPackedAttn p) {
  typedef PaImg<T, D> Img;
  typedef typename PaFrag<T>::type Frag;
  constexpr int IMG = BN * Img::ROWB;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[4 * IMG];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int it = blockIdx.x / p.heads, r = blockIdx.x - it * p.heads;
  const int kvh = r % p.kv_heads, head = kvh * (p.heads / p.kv_heads) + r / p.kv_heads;
  const MtSeqItem item = pa_item(p, p.items, it, 0, p.causal);
  const int64_t dq_row = (int64_t)p.heads * p.head_k;
  T* dq = reinterpret_cast<T*>(p.dq) + item.row0 * dq_row + (int64_t)head * p.head_k;
  if (item.len <= 0) {
    pa_zero_rows<T>(dq, dq_row, -item.len, p.head_k);
    return;
  }
  const int first = item.first + wave * 32, mine = first + (lane & 31);
  const bool ok = mine < item.len;
  Frag qf[D / 16], df[D / 16];
  float delta, lse;
  pa_dq_rows<T, D, D>(p, qf, df, delta, lse, item.row0 + (int64_t)mine, head, ok, true, pa_low(p, item.len, item.first), lane);
  const T* kb = reinterpret_cast<const T*>(p.k) + item.row0 * p.k_row + (int64_t)kvh * p.k_head;
  const T* vb = reinterpret_cast<const T*>(p.v) + item.row0 * p.v_row + (int64_t)kvh * p.v_head;
  const int keys = p.causal && item.first + PA_OWN < item.len ? item.first + PA_OWN : item.len;
  const int tiles = (keys + BN - 1) / BN;
  const float c = p.scale * 1.4426950408889634f;
  // Tiles are fetched in order: the next one's addresses are carried along, not worked out per tile ahead of its fetch.
  const T *k_next = kb, *v_next = vb;
  int left = item.len;
  const int64_t k_hop = BN * p.k_row, v_hop = BN * p.v_row;
  auto issue = [&](int t) {
    uint8_t* st = lds + (t & 1) * 2 * IMG;
    Img::template stage<BN>(st, k_next, p.k_row, left, p.head_k, wave, lane);
    Img::template stage<BN>(st + IMG, v_next, p.v_row, left, p.head_v, wave, lane);
    k_next += k_hop;
    v_next += v_hop;
    left -= BN;
  };
  f32x16 acc[D / 32];
  pa_clear(acc);
  const uint32_t lds_at = pa_lds_at(lds);
  const int last = p.causal && ok ? mine : item.len - 1;
  // 32 keys at a time; fragments in groups read one group ahead, as in the forward kernel: V, K, then K's columns
  auto step = [&](int t, int u, bool masked, bool few) {
    const uint32_t kimg = lds_at + (t & 1) * 2 * IMG, krow = kimg + Img::row_base(lane), kcol = kimg + Img::col_base(lane), vrow = krow + IMG;
    constexpr int G = D / 16 < 4 ? D / 16 : 4, NG = D / 16 / G;
    Frag fr[2][G], cf[2][D / 32];
    auto read_rows = [&](int g) {          // groups 0 .. NG - 1 of V, then of K
#pragma unroll
      for (int e = 0; e < G; ++e) fr[g & 1][e] = Img::rows(g < NG ? vrow : krow, 32 * u, (g % NG) * G + e);
    };
    auto read_cols = [&](int h) {
#pragma unroll
      for (int b = 0; b < D / 32; ++b) cf[h][b] = Img::cols(kcol, 32 * u + 16 * h, b);
    };
    f32x16 s[1], d[1];
    pa_clear(s);
    pa_clear(d);
    read_rows(0);
#pragma unroll
    for (int g = 0; g < 2 * NG; ++g) {
      if (g + 1 < 2 * NG) read_rows(g + 1);
      else read_cols(0);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int e = 0; e < G; ++e) {
        if (g < NG) d[0] = pa_mma(fr[g & 1][e], df[(g % NG) * G + e], d[0]);
        else s[0] = pa_mma(fr[g & 1][e], qf[(g % NG) * G + e], s[0]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) s[0][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][i], c, -lse)) * (d[0][i] - delta);
    if (masked) {
#pragma unroll
      for (int i = 0; i < 16; ++i) s[0][i] = t * BN + 32 * u + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3) <= last ? s[0][i] : 0.f;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (h == 0) read_cols(1);
      const Frag sf = pa_pack<T>(s[0], h);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int b = 0; b < D / 32; ++b) acc[b] = pa_mma(cf[h][b], sf, acc[b]);
      __builtin_amdgcn_sched_barrier(0);
      if (few) {
        const Frag rest = pa_rest<T>(s[0], h, sf);
#pragma unroll
        for (int b = 0; b < D / 32; ++b) acc[b] = pa_mma(cf[h][b], rest, acc[b]);
      }
    }
  };
  const int mine_end = p.causal && first + 32 < keys ? first + 32 : keys;
  const int own = first < item.len ? (mine_end + BN - 1) / BN : 0;
  const int whole = p.causal && first + 1 < mine_end ? (first + 1) / BN : mine_end / BN;
  issue(0);
  auto enter = [&](int t) {
    pa_tile_barrier();
    if (t + 1 < tiles) issue(t + 1);
  };
  int t = 0;
  if (pa_few_keys(p, item.len, item.first)) {
    for (; t < own; ++t) {
      enter(t);
      for (int u = 0; u < (BN > 32 && t * BN + 32 < mine_end ? 2 : 1); ++u) step(t, u, true, true);
    }
  }
  for (; t < whole && t < own; ++t) {
    enter(t);
    step(t, 0, false, false);
    if (BN > 32) step(t, 1, false, false);
  }
  for (; t < own; ++t) {
    enter(t);
    step(t, 0, true, false);
    if (BN > 32 && t * BN + 32 < mine_end) step(t, 1, true, false);
  }
  for (; t < tiles; ++t) enter(t);
  if (ok) pa_store_row<T, D>(dq + (int64_t)mine * dq_row, acc, p.scale, p.head_k, lane);
}

// ---- backward: dk and dv ------------------------------------------------------------------------------------------------
// Eight waves: waves w and w + 4 own the same 32 keys and take the two halves of every 64-query tile; their sums meet in LDS at
// the end.  The workgroup's keys and values stay in LDS beside the query tiles and are read again for every tile, because the
// two gradients' accumulators already take half the registers of a wave when two of them are to share a SIMD.
//
// A wave's tile is three steps: scores (A: S and dp), vector work (B: p and ds), gradients (C: dv and dk).  The two waves of a
// SIMD are the two halves of one workgroup, and in step with each other they would leave the matrix pipe idle while both do B.
// So the second half runs a step behind: between two barriers the first does A while the second does C of the tile before, then
// B and C while the second does A and B.  Each half fetches its own 32 queries of the next tile once nobody reads that buffer.
// Measured with the dq kernel, 8 x 2048 causal, 16 / 4 heads of 64: 295 us against 304 in step; at 128 wide both ways take the same
// time (2 x 4096, 16 heads: 920 us, 1046 TFLOP/s of the seven products, at 2.0 GHz: power, not the schedule, is the limit there).
#define PA_DKV_THREADS 512
template <typename T, int D>
__global__ __launch_bounds__(PA_DKV_THREADS, 2) void mt_pattn_dkv_kernel(const MtPackedAttn p) {
  typedef PaImg<T, D> Img;
  typedef typename PaFrag<T>::type Frag;
  constexpr int BQ = 64, HALF = 32 * Img::ROWB, IMG = 2 * HALF, KV = PA_OWN * Img::ROWB;
  constexpr int STAGE = 2 * IMG + 1024;                              // q rows, do rows, {L, D} of the rows of either half
  constexpr int BYTES = 2 * KV + 2 * STAGE, JOIN = 2 * 128 * D * 4;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[BYTES < JOIN ? JOIN : BYTES];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // workgroups 0 .. 2 cut kv_heads - 1: the halves of the longest walks
  const int turn = blockIdx.x / p.kv_heads, kvh = blockIdx.x - turn * p.kv_heads;
  const bool is_cut = turn < 2 * p.cut;
  const int it = is_cut ? turn >> 1 : turn - p.cut;
  const int heads_all = p.heads / p.kv_heads, head_lo = is_cut && (turn & 1) ? heads_all / 2 : 0;
  const int group = is_cut && !(turn & 1) ? heads_all / 2 : heads_all - head_lo;
  const MtSeqItem item = pa_item(p, p.kv_items, it, 0, false);
  const int64_t dk_row = (int64_t)p.kv_heads * p.head_k, dv_row = (int64_t)p.kv_heads * p.head_v;
  T* dk = reinterpret_cast<T*>(p.dk) + item.row0 * dk_row + (int64_t)kvh * p.head_k;
  T* dv = reinterpret_cast<T*>(p.dv) + item.row0 * dv_row + (int64_t)kvh * p.head_v;
  if (item.len <= 0) {
    pa_zero_rows<T>(dk, dk_row, -item.len, p.head_k);
    pa_zero_rows<T>(dv, dv_row, -item.len, p.head_v);
    return;
  }
  const int block = wave & 3, half = wave >> 2;
  const int first = item.first + block * 32, mine = first + (lane & 31);
  const int q_lo = p.causal ? item.first / BQ : 0;                  // first query tile that sees a key of this workgroup
  const int per_head = (item.len + BQ - 1) / BQ - q_lo;
  const int tiles = per_head * group;
  const float c = p.scale * 1.4426950408889634f;
  {
    const int64_t r0 = item.row0 + (int64_t)item.first;
    Img::template stage<PA_OWN, 8>(lds, reinterpret_cast<const T*>(p.k) + r0 * p.k_row + (int64_t)kvh * p.k_head, p.k_row,
                                   item.len - item.first, p.head_k, wave, lane);
    Img::template stage<PA_OWN, 8>(lds + KV, reinterpret_cast<const T*>(p.v) + r0 * p.v_row + (int64_t)kvh * p.v_head, p.v_row,
                                   item.len - item.first, p.head_v, wave, lane);
  }
  uint8_t* stages = lds + 2 * KV;
  // This half's 32 queries of the next tile, tiles in order, then heads: addresses are carried along.
  const T *q_next, *d_next;
  const float* stat_next;
  int left, todo = tiles, until = per_head;
  int64_t head_next = (int64_t)kvh * heads_all + head_lo;
  auto enter_head = [&] {
    const int q0 = q_lo * BQ + 32 * half;
    const int64_t r0 = item.row0 + (int64_t)q0;
    q_next = reinterpret_cast<const T*>(p.q) + r0 * p.q_row + head_next * p.q_head;
    d_next = reinterpret_cast<const T*>(p.dout) + r0 * p.do_row + head_next * p.do_head;
    stat_next = (block == 0 ? p.lse : p.delta) + head_next * p.rows + r0;
    left = item.len - q0;
    until = per_head;
    ++head_next;
  };
  enter_head();
  const int64_t q_hop = BQ * p.q_row, d_hop = BQ * p.do_row;
  auto issue = [&](int n) {
    if (todo-- <= 0) return;
    uint8_t* st = stages + (n & 1) * STAGE;
    if (left > 0) {                                                 // else nobody will read them
      Img::template stage<32, 4>(st + half * HALF, q_next, p.q_row, left, p.head_k, block, lane);
      Img::template stage<32, 4>(st + IMG + half * HALF, d_next, p.do_row, left, p.head_v, block, lane);
      if (block < 2) {
        const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<float*>(stat_next), 0, (uint32_t)(left < 32 ? left : 32) * 4u, 0x00027000);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (__attribute__((address_space(3))) void*)(st + 2 * IMG + half * 512 + block * 256),
                                                 4, lane * 4, 0, 0, 0);
      }
    }
    q_next += q_hop;
    d_next += d_hop;
    stat_next += BQ;
    left -= BQ;
    if (--until == 0 && todo > 0) enter_head();
  };
  f32x16 ak[D / 32], av[D / 32];
  pa_clear(ak);
  pa_clear(av);
  const uint32_t lds_at = pa_lds_at(lds), st_at = lds_at + 2 * KV;
  f32x16 s[1], d[1];
  Frag pf[2], sf[2];
  auto scores = [&](int n) {                                        // A
    const uint32_t rb = Img::row_base(lane), krow = lds_at + block * HALF + rb, qrow = st_at + (n & 1) * STAGE + half * HALF + rb;
    constexpr int G = 2, NG = D / 16 / G;
    Frag fr[2][G], kr[2][G];
    auto read_rows = [&](int g) {          // groups 0 .. NG - 1 of q and k, then of do and v
#pragma unroll
      for (int e = 0; e < G; ++e) {
        fr[g & 1][e] = Img::rows(g < NG ? qrow : qrow + IMG, 0, (g % NG) * G + e);
        kr[g & 1][e] = Img::rows(g < NG ? krow : krow + KV, 0, (g % NG) * G + e);
      }
    };
    pa_clear(s);
    pa_clear(d);
    read_rows(0);
#pragma unroll
    for (int g = 0; g < 2 * NG; ++g) {
      if (g + 1 < 2 * NG) read_rows(g + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int e = 0; e < G; ++e) {
        if (g < NG) s[0] = pa_mma(fr[g & 1][e], kr[g & 1][e], s[0]);
        else d[0] = pa_mma(fr[g & 1][e], kr[g & 1][e], d[0]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto weigh = [&](int n, int qu) {                                 // B
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      // (by address: through the array the compiler would first wait for the LDS-DMA of the next tile, which may alias)
      const uint32_t at = st_at + (n & 1) * STAGE + 2 * IMG + half * 512 + 4 * (8 * g + 4 * (lane >> 5));
      const f32x4 lse = *pa_lds<f32x4>(at), delta = *pa_lds<f32x4>(at + 256);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][4 * g + e], c, -lse[e]));
        s[0][4 * g + e] = pr;
        d[0][4 * g + e] = pr * (d[0][4 * g + e] - delta[e]);
      }
    }
    if (qu + 32 > item.len || (p.causal && qu < first + 31)) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int qi = qu + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3);
        const bool see = qi < item.len && (!p.causal || mine <= qi);
        s[0][i] = see ? s[0][i] : 0.f;
        d[0][i] = see ? d[0][i] : 0.f;
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      pf[h] = pa_pack<T>(s[0], h);
      sf[h] = pa_pack<T>(d[0], h);
    }
  };
  auto gradients = [&](int n) {                                     // C
    const uint32_t qcol = st_at + (n & 1) * STAGE + half * HALF + Img::col_base(lane);
    Frag cf[2][D / 32];
    auto read_cols = [&](int g) {          // do's columns of two times 16 rows, then q's
#pragma unroll
      for (int b = 0; b < D / 32; ++b) cf[g & 1][b] = Img::cols(g < 2 ? qcol + IMG : qcol, 16 * (g & 1), b);
    };
    read_cols(0);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      if (g < 3) read_cols(g + 1);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int b = 0; b < D / 32; ++b) {
        if (g < 2) av[b] = pa_mma(cf[g & 1][b], pf[g & 1], av[b]);
        else ak[b] = pa_mma(cf[g & 1][b], sf[g & 1], ak[b]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };
  auto sees = [&](int qu) { return qu < item.len && !(p.causal && qu + 31 < first); };
  auto middle = [&] {                      // the halves meet between their steps; the reads of the first are back
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };
  issue(0);
  const int q_end = q_lo + per_head;
  int qt = q_lo;
  if (half == 0) {
    for (int n = 0; n < tiles; ++n) {
      const int qu = qt * BQ;
      if (++qt == q_end) qt = q_lo;
      pa_tile_barrier();
      issue(n + 1);
      const bool on = sees(qu);
      if (on) scores(n);
      middle();
      if (on) {
        weigh(n, qu);
        gradients(n);
      }
    }
  } else {
    bool behind = false;
    for (int n = 0; n < tiles; ++n) {
      const int qu = qt * BQ + 32;
      if (++qt == q_end) qt = q_lo;
      pa_tile_barrier();
      if (behind) gradients(n - 1);
      middle();
      issue(n + 1);
      behind = sees(qu);
      if (behind) {
        scores(n);
        weigh(n, qu);
      }
    }
    if (behind) gradients(tiles - 1);
  }
  // [dk, dv][key block][column][key] f32 of the second halves; no LDS-DMA is in flight past the last tile's barriers
  float* join = reinterpret_cast<float*>(lds) + block * 32 * D;
  __syncthreads();
  auto each = [&](auto&& f) {
#pragma unroll
    for (int b = 0; b < D / 32; ++b)
#pragma unroll
      for (int i = 0; i < 16; ++i) f(b, i, (32 * b + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3)) * 32 + (lane & 31));
  };
  if (half == 1) each([&](int b, int i, int at) { join[at] = ak[b][i]; join[128 * D + at] = av[b][i]; });
  __syncthreads();
  if (half == 1) return;
  each([&](int b, int i, int at) { ak[b][i] += join[at]; av[b][i] += join[128 * D + at]; });
  if (is_cut) {
    float* part = p.halves + (((int64_t)it * p.kv_heads + kvh) * 2 + (turn & 1)) * 2 * PA_OWN * D + (block * 32 + (lane & 31)) * D;
    if (mine < item.len) {
      pa_store_row<float, D>(part, ak, p.scale, p.head_k, lane);
      pa_store_row<float, D>(part + PA_OWN * D, av, 1.f, p.head_v, lane);
    }
    return;
  }
  if (mine < item.len) {
    pa_store_row<T, D>(dk + (int64_t)mine * dk_row, ak, p.scale, p.head_k, lane);
    pa_store_row<T, D>(dv + (int64_t)mine * dv_row, av, 1.f, p.head_v, lane);
  }
}

// dk and dv of the cut walks: the two halves added, rounded once.  Sixteen rows per workgroup.
#define PA_HALVES_ROWS 16
template <int D>
__global__ __launch_bounds__(PA_THREADS) void mt_pattn_halves_kernel(const MtPackedAttn p) {
  const int unit = blockIdx.x / (PA_OWN / PA_HALVES_ROWS), lo = (blockIdx.x % (PA_OWN / PA_HALVES_ROWS)) * PA_HALVES_ROWS;
  const int it = unit / p.kv_heads, kvh = unit - it * p.kv_heads;
  const MtSeqItem item = pa_item(p, p.kv_items, it, 0, false);
  const int left = item.len - item.first - lo, rows = left < PA_HALVES_ROWS ? left : PA_HALVES_ROWS;
  const int64_t r0 = item.row0 + (int64_t)item.first + lo;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const int d = which ? p.head_v : p.head_k;
    __bf16* out = reinterpret_cast<__bf16*>(which ? p.dv : p.dk) + (r0 * p.kv_heads + kvh) * d;
    const float* a = p.halves + (int64_t)unit * 4 * PA_OWN * D + which * PA_OWN * D + lo * D;
    const float* b = a + 2 * PA_OWN * D;
    for (int i = threadIdx.x; i < rows * (D / 4); i += PA_THREADS) {
      const int r = i / (D / 4), c = (i - r * (D / 4)) * 4;
      if (c >= d) continue;
      const f32x4 v = *reinterpret_cast<const f32x4*>(a + r * D + c) + *reinterpret_cast<const f32x4*>(b + r * D + c);
      pa_store4<__bf16>(out + (int64_t)r * p.kv_heads * d + c, nullptr, v[0], v[1], v[2], v[3]);
    }
  }
}

// ---- the split form -----------------------------------------------------------------------------------------------------
// A workgroup owns 32 rows and its four waves share the walk: wave w takes tiles w, w + 4, ... of 32 rows, in its own part of
// LDS and without barriers, and the four partial results are joined through LDS in wave order.  Against the form above a tile
// fetched feeds 32 owned rows instead of 128, and a quarter of the longest sequence's walk is the longest any wave has to go.
// A `solo` item is 128 rows, 32 per wave, and every wave walks alone over all tiles: short sequences, whose walk split in four is
// shorter than what a workgroup costs to begin and to join.
// An image is single-buffered: it is refilled as soon as the last product that reads it has its fragments, and the other
// image's products run meanwhile.  Key and value widths have images and accumulators of their own size (DK, DV).
template <int N> __device__ __forceinline__ void pa_wait_vm() {          // at most N of this wave's loads are still in flight
  static_assert(N >= 0 && N < 64, "vmcnt is a six-bit counter");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory");
}
__device__ __forceinline__ void pa_reads_done() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
// f32 steps are eight slow instructions: those behind the head's width are skipped.  bf16 steps are one, and stay in line.
template <typename T> __device__ __forceinline__ bool pa_step(int column, int width) { return sizeof(T) == 2 || column < width; }

template <typename T, int DK, int DV> struct PaSplit {
  typedef PaImg<T, DK> IK;
  typedef PaImg<T, DV> IV;
  static constexpr int KB = PA_TILE * IK::ROWB, VB = PA_TILE * IV::ROWB;           // image bytes
  static constexpr int KP = KB / 1024, VP = VB / 1024;                             // LDS-DMA instructions of one
  static constexpr int WIDE = DK > DV ? DK : DV;
  static constexpr int lds(int joined) { return 4 * (KB + VB) < 512 * joined ? 512 * joined : 4 * (KB + VB); }
  static constexpr int WAVES = sizeof(T) == 4 && WIDE == 128 ? 1 : 2;              // per SIMD
};

template <typename T, int DK, int DV>
__global__ __launch_bounds__(PA_THREADS, (PaSplit<T, DK, DV>::WAVES)) void mt_pattn_split_fwd_kernel(const MtPackedAttn p) {
  typedef PaSplit<T, DK, DV> S;
  typedef typename S::IK IK;
  typedef typename S::IV IV;
  typedef typename PaFrag<T>::type Frag;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[S::lds(DV)];
  __shared__ float stat[2][4][32];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int it = blockIdx.x / p.heads, r = blockIdx.x - it * p.heads;
  const int kvh = r % p.kv_heads, head = kvh * (p.heads / p.kv_heads) + r / p.kv_heads;
  const MtSeqItem item = pa_item(p, p.items, it, p.split, p.causal);
  const int64_t o_row = (int64_t)p.heads * p.head_v;
  T* o = reinterpret_cast<T*>(p.o) + item.row0 * o_row + (int64_t)head * p.head_v;
  T* low = sizeof(T) == 2 && pa_low(p, item.len, item.first) ? reinterpret_cast<T*>(p.low) + item.row0 * o_row + (int64_t)head * p.head_v : nullptr;
  if (item.len <= 0) {
    pa_zero_rows<T>(o, o_row, -item.len, p.head_v);
    return;
  }
  const int first = item.first + (item.solo ? wave * 32 : 0), mine = first + (lane & 31);
  if (item.solo && first >= item.len) return;
  Frag qf[DK / 16];
  pa_own_row<T, DK>(qf, reinterpret_cast<const T*>(p.q) + (item.row0 + (int64_t)mine) * p.q_row + (int64_t)head * p.q_head,
                    mine < item.len, p.head_k, lane);
  const T* kb = reinterpret_cast<const T*>(p.k) + item.row0 * p.k_row + (int64_t)kvh * p.k_head;
  const T* vb = reinterpret_cast<const T*>(p.v) + item.row0 * p.v_row + (int64_t)kvh * p.v_head;
  const int keys = p.causal && first + 32 < item.len ? first + 32 : item.len;
  const int tiles = (keys + PA_TILE - 1) / PA_TILE, t0 = item.solo ? 0 : wave, hop = item.solo ? 1 : 4;
  const float c = p.scale * 1.4426950408889634f;
  uint8_t* kimg = lds + wave * (S::KB + S::VB);
  uint8_t* vimg = kimg + S::KB;
  const uint32_t krow = pa_lds_at(kimg) + IK::row_base(lane), vcol = pa_lds_at(vimg) + IV::col_base(lane);
  auto load_k = [&](int t) {
    IK::template stage<PA_TILE, 1>(kimg, kb + (int64_t)t * PA_TILE * p.k_row, p.k_row, item.len - t * PA_TILE, p.head_k, 0, lane);
  };
  auto load_v = [&](int t) {
    IV::template stage<PA_TILE, 1>(vimg, vb + (int64_t)t * PA_TILE * p.v_row, p.v_row, item.len - t * PA_TILE, p.head_v, 0, lane);
  };
  f32x16 acc[DV / 32];
  pa_clear(acc);
  float m = -INFINITY, sum = 0.f;
  if (t0 < tiles) {
    load_k(t0);
    load_v(t0);
  }
  for (int t = t0; t < tiles; t += hop) {
    const bool more = t + hop < tiles;
    pa_wait_vm<S::VP>();                       // K of this tile; its V may still be on the way
    f32x16 s[1];
    pa_clear(s);
#pragma unroll
    for (int ks = 0; ks < DK / 16; ++ks)
      if (pa_step<T>(16 * ks, p.head_k)) s[0] = pa_mma(IK::rows(krow, 0, ks), qf[ks], s[0]);
    pa_reads_done();
    if (more) load_k(t + hop);
    const int k0 = t * PA_TILE;
    if (k0 + PA_TILE > item.len || (p.causal && k0 + PA_TILE - 1 > first)) {
      const int last = p.causal && mine < item.len ? mine : item.len - 1;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[0][i] = k0 + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3) <= last ? s[0][i] : -INFINITY;
    }
    float mx = s[0][0];
#pragma unroll
    for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[0][i]);
    mx = pa_half_max(mx) * c;
    if (__any(mx > m + 8.f)) {
      const float mn = fmaxf(m, mx);
      const float f = mn == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      sum *= f;
#pragma unroll
      for (int b = 0; b < DV / 32; ++b)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[b][i] *= f;
    }
    const float sub = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[0][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][i], c, -sub));
    if (more) pa_wait_vm<S::KP>();             // V of this tile; the next K may still be on the way
    else pa_wait_vm<0>();
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const Frag pf = pa_pack<T>(s[0], h);
      sum = pa_row_sum(pf, sum);
#pragma unroll
      for (int b = 0; b < DV / 32; ++b)
        if (pa_step<T>(32 * b, p.head_v)) acc[b] = pa_mma(IV::cols(vcol, 16 * h, b), pf, acc[b]);
    }
    pa_reads_done();
    if (more) load_v(t + hop);
  }
  sum = pa_half_sum(sum);
  float* lse = p.lse != nullptr && mine < item.len && lane < 32 ? p.lse + (int64_t)head * p.rows + item.row0 + mine : nullptr;
  if (item.solo) {
    if (mine < item.len)
      pa_store_row<T, DV>(o + (int64_t)mine * o_row, acc, 1.f / sum, p.head_v, lane, low != nullptr ? low + (int64_t)mine * o_row : nullptr);
    if (lse != nullptr) *lse = m + __builtin_amdgcn_logf(sum);
    return;
  }
  if (lane < 32) {
    stat[0][wave][lane] = m;
    stat[1][wave][lane] = sum;
  }
  __syncthreads();                             // and every wave is done with its images
  const int q = lane & 31;
  float top = -INFINITY, total = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) top = fmaxf(top, stat[0][w][q]);
  const float sub = top == -INFINITY ? 0.f : top;
#pragma unroll
  for (int w = 0; w < 4; ++w) total += stat[1][w][q] * __builtin_amdgcn_exp2f(stat[0][w][q] - sub);
  const float f = __builtin_amdgcn_exp2f(m - sub) * (1.f / total);
  pa_join<DV>(reinterpret_cast<float*>(lds), acc, f, wave, lane);
  __syncthreads();
  pa_join_store<T, DV>(o + (int64_t)first * o_row, o_row, reinterpret_cast<const float*>(lds), item.len - first, p.head_v,
                       low != nullptr ? low + (int64_t)first * o_row : nullptr);
  if (wave == 0 && lse != nullptr) *lse = sub + __builtin_amdgcn_logf(total);
}

template <typename T, int DK, int DV>
__global__ __launch_bounds__(PA_THREADS, (PaSplit<T, DK, DV>::WAVES)) void mt_pattn_split_dq_kernel(const MtPackedAttn p) {
  typedef PaSplit<T, DK, DV> S;
  typedef typename S::IK IK;
  typedef typename S::IV IV;
  typedef typename PaFrag<T>::type Frag;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[S::lds(DK)];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int it = blockIdx.x / p.heads, r = blockIdx.x - it * p.heads;
  const int kvh = r % p.kv_heads, head = kvh * (p.heads / p.kv_heads) + r / p.kv_heads;
  const MtSeqItem item = pa_item(p, p.items, it, p.split, p.causal);
  const int64_t dq_row = (int64_t)p.heads * p.head_k;
  T* dq = reinterpret_cast<T*>(p.dq) + item.row0 * dq_row + (int64_t)head * p.head_k;
  if (item.len <= 0) {
    pa_zero_rows<T>(dq, dq_row, -item.len, p.head_k);
    return;
  }
  const int first = item.first + (item.solo ? wave * 32 : 0), mine = first + (lane & 31);
  if (item.solo && first >= item.len) return;
  Frag qf[DK / 16], df[DV / 16];
  float delta, lse;
  pa_dq_rows<T, DK, DV>(p, qf, df, delta, lse, item.row0 + (int64_t)mine, head, mine < item.len, item.solo || wave == 0,
                        pa_low(p, item.len, item.first), lane);
  const T* kb = reinterpret_cast<const T*>(p.k) + item.row0 * p.k_row + (int64_t)kvh * p.k_head;
  const T* vb = reinterpret_cast<const T*>(p.v) + item.row0 * p.v_row + (int64_t)kvh * p.v_head;
  const int keys = p.causal && first + 32 < item.len ? first + 32 : item.len;
  const int tiles = (keys + PA_TILE - 1) / PA_TILE, t0 = item.solo ? 0 : wave, hop = item.solo ? 1 : 4;
  const float c = p.scale * 1.4426950408889634f;
  uint8_t* kimg = lds + wave * (S::KB + S::VB);
  uint8_t* vimg = kimg + S::KB;
  const uint32_t krow = pa_lds_at(kimg) + IK::row_base(lane), kcol = pa_lds_at(kimg) + IK::col_base(lane),
                 vrow = pa_lds_at(vimg) + IV::row_base(lane);
  auto load_k = [&](int t) {
    IK::template stage<PA_TILE, 1>(kimg, kb + (int64_t)t * PA_TILE * p.k_row, p.k_row, item.len - t * PA_TILE, p.head_k, 0, lane);
  };
  auto load_v = [&](int t) {
    IV::template stage<PA_TILE, 1>(vimg, vb + (int64_t)t * PA_TILE * p.v_row, p.v_row, item.len - t * PA_TILE, p.head_v, 0, lane);
  };
  const bool few = sizeof(T) == 2 && pa_few_keys(p, item.len, item.first);
  f32x16 acc[DK / 32];
  pa_clear(acc);
  if (t0 < tiles) {
    load_v(t0);
    load_k(t0);
  }
  for (int t = t0; t < tiles; t += hop) {
    const bool more = t + hop < tiles;
    pa_wait_vm<S::KP>();                       // V; K may still be on the way
    f32x16 s[1], d[1];
    pa_clear(s);
    pa_clear(d);
#pragma unroll
    for (int ks = 0; ks < DV / 16; ++ks)
      if (pa_step<T>(16 * ks, p.head_v)) d[0] = pa_mma(IV::rows(vrow, 0, ks), df[ks], d[0]);
    pa_reads_done();
    if (more) {
      load_v(t + hop);
      pa_wait_vm<S::VP>();
    } else {
      pa_wait_vm<0>();
    }
#pragma unroll
    for (int ks = 0; ks < DK / 16; ++ks)
      if (pa_step<T>(16 * ks, p.head_k)) s[0] = pa_mma(IK::rows(krow, 0, ks), qf[ks], s[0]);
#pragma unroll
    for (int i = 0; i < 16; ++i) s[0][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][i], c, -lse)) * (d[0][i] - delta);
    const int k0 = t * PA_TILE;
    if (k0 + PA_TILE > item.len || (p.causal && k0 + PA_TILE - 1 > first)) {
      const int last = p.causal && mine < item.len ? mine : item.len - 1;
#pragma unroll
      for (int i = 0; i < 16; ++i) s[0][i] = k0 + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3) <= last ? s[0][i] : 0.f;
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const Frag sf = pa_pack<T>(s[0], h);
#pragma unroll
      for (int b = 0; b < DK / 32; ++b)
        if (pa_step<T>(32 * b, p.head_k)) acc[b] = pa_mma(IK::cols(kcol, 16 * h, b), sf, acc[b]);
      if (few) pa_add_rest<T, IK, DK>(acc, kcol, h, pa_rest<T>(s[0], h, sf));
    }
    pa_reads_done();
    if (more) load_k(t + hop);
  }
  if (item.solo) {
    if (mine < item.len) pa_store_row<T, DK>(dq + (int64_t)mine * dq_row, acc, p.scale, p.head_k, lane);
    return;
  }
  __syncthreads();
  pa_join<DK>(reinterpret_cast<float*>(lds), acc, p.scale, wave, lane);
  __syncthreads();
  pa_join_store<T, DK>(dq + (int64_t)first * dq_row, dq_row, reinterpret_cast<const float*>(lds), item.len - first, p.head_k);
}

template <typename T, int DK, int DV>
__global__ __launch_bounds__(PA_THREADS, DK + DV > 96 ? 1 : 2) void mt_pattn_split_dkv_kernel(const MtPackedAttn p) {
  typedef PaSplit<T, DK, DV> S;
  typedef typename S::IK IK;
  typedef typename S::IV IV;
  typedef typename PaFrag<T>::type Frag;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[S::lds(S::WIDE)];
  __shared__ __attribute__((aligned(16))) float stat[4][64];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int it = blockIdx.x / p.kv_heads, kvh = blockIdx.x - it * p.kv_heads, group = p.heads / p.kv_heads;
  const MtSeqItem item = pa_item(p, p.kv_items, it, p.kv_split, false);
  const int64_t dk_row = (int64_t)p.kv_heads * p.head_k, dv_row = (int64_t)p.kv_heads * p.head_v;
  T* dk = reinterpret_cast<T*>(p.dk) + item.row0 * dk_row + (int64_t)kvh * p.head_k;
  T* dv = reinterpret_cast<T*>(p.dv) + item.row0 * dv_row + (int64_t)kvh * p.head_v;
  if (item.len <= 0) {
    pa_zero_rows<T>(dk, dk_row, -item.len, p.head_k);
    pa_zero_rows<T>(dv, dv_row, -item.len, p.head_v);
    return;
  }
  const int first = item.first + (item.solo ? wave * 32 : 0), mine = first + (lane & 31);
  if (item.solo && first >= item.len) return;
  const bool ok = mine < item.len;
  const int64_t row = item.row0 + (int64_t)mine;
  Frag kf[DK / 16], vf[DV / 16];
  pa_own_row<T, DK>(kf, reinterpret_cast<const T*>(p.k) + row * p.k_row + (int64_t)kvh * p.k_head, ok, p.head_k, lane);
  pa_own_row<T, DV>(vf, reinterpret_cast<const T*>(p.v) + row * p.v_row + (int64_t)kvh * p.v_head, ok, p.head_v, lane);
  const int q_lo = p.causal ? first / PA_TILE : 0;
  const int per_head = (item.len + PA_TILE - 1) / PA_TILE - q_lo, tiles = per_head * group;
  const int t0 = item.solo ? 0 : wave, hop = item.solo ? 1 : 4;
  const float c = p.scale * 1.4426950408889634f;
  uint8_t* qimg = lds + wave * (S::KB + S::VB);
  uint8_t* dimg = qimg + S::KB;
  const uint32_t qrow = pa_lds_at(qimg) + IK::row_base(lane), qcol = pa_lds_at(qimg) + IK::col_base(lane);
  const uint32_t drow = pa_lds_at(dimg) + IV::row_base(lane), dcol = pa_lds_at(dimg) + IV::col_base(lane);
  auto at = [&](int n, int& head, int& q0) {
    const int hg = n / per_head;
    head = kvh * group + hg;
    q0 = (q_lo + n - hg * per_head) * PA_TILE;
  };
  auto load_q = [&](int n) {
    int head, q0;
    at(n, head, q0);
    IK::template stage<PA_TILE, 1>(qimg, reinterpret_cast<const T*>(p.q) + (item.row0 + (int64_t)q0) * p.q_row + (int64_t)head * p.q_head,
                                   p.q_row, item.len - q0, p.head_k, 0, lane);
  };
  float ahead = 0.f;      // L (lanes 0-31) and D (32-63) of the rows of the tile that load_d fetched last
  auto load_d = [&](int n) {
    int head, q0;
    at(n, head, q0);
    const int qi = q0 + (lane & 31);
    const float* src = lane < 32 ? p.lse : p.delta;
    ahead = qi < item.len ? src[(int64_t)head * p.rows + item.row0 + qi] : 0.f;
    IV::template stage<PA_TILE, 1>(dimg, reinterpret_cast<const T*>(p.dout) + (item.row0 + (int64_t)q0) * p.do_row + (int64_t)head * p.do_head,
                                   p.do_row, item.len - q0, p.head_v, 0, lane);
  };
  const bool few = sizeof(T) == 2 && item.len <= PA_LOW_ROWS;
  f32x16 ak[DK / 32], av[DV / 32];
  pa_clear(ak);
  pa_clear(av);
  if (t0 < tiles) {
    load_d(t0);
    load_q(t0);
  }
  for (int n = t0; n < tiles; n += hop) {
    const bool more = n + hop < tiles;
    int head, q0;
    at(n, head, q0);
    pa_wait_vm<S::KP>();                       // do, L and D; q may still be on the way
    stat[wave][lane] = ahead;                  // read back four rows at a time
    f32x16 s[1], d[1];
    pa_clear(s);
    pa_clear(d);
#pragma unroll
    for (int ks = 0; ks < DV / 16; ++ks)
      if (pa_step<T>(16 * ks, p.head_v)) d[0] = pa_mma(IV::rows(drow, 0, ks), vf[ks], d[0]);
    pa_wait_vm<0>();
#pragma unroll
    for (int ks = 0; ks < DK / 16; ++ks)
      if (pa_step<T>(16 * ks, p.head_k)) s[0] = pa_mma(IK::rows(qrow, 0, ks), kf[ks], s[0]);
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int rr = 8 * g + 4 * (lane >> 5);
      const f32x4 lse = *reinterpret_cast<const f32x4*>(&stat[wave][rr]), delta = *reinterpret_cast<const f32x4*>(&stat[wave][32 + rr]);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float pr = __builtin_amdgcn_exp2f(__builtin_fmaf(s[0][4 * g + e], c, -lse[e]));
        s[0][4 * g + e] = pr;
        d[0][4 * g + e] = pr * (d[0][4 * g + e] - delta[e]);
      }
    }
    if (q0 + PA_TILE > item.len || (p.causal && q0 < first + 31)) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const int qr = q0 + 8 * (i >> 2) + 4 * (lane >> 5) + (i & 3);
        const bool see = qr < item.len && (!p.causal || mine <= qr);
        s[0][i] = see ? s[0][i] : 0.f;
        d[0][i] = see ? d[0][i] : 0.f;
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const Frag pf = pa_pack<T>(s[0], h);
#pragma unroll
      for (int b = 0; b < DV / 32; ++b)
        if (pa_step<T>(32 * b, p.head_v)) av[b] = pa_mma(IV::cols(dcol, 16 * h, b), pf, av[b]);
      if (few) pa_add_rest<T, IV, DV>(av, dcol, h, pa_rest<T>(s[0], h, pf));
    }
    pa_reads_done();
    if (more) load_d(n + hop);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const Frag sf = pa_pack<T>(d[0], h);
#pragma unroll
      for (int b = 0; b < DK / 32; ++b)
        if (pa_step<T>(32 * b, p.head_k)) ak[b] = pa_mma(IK::cols(qcol, 16 * h, b), sf, ak[b]);
      if (few) pa_add_rest<T, IK, DK>(ak, qcol, h, pa_rest<T>(d[0], h, sf));
    }
    pa_reads_done();
    if (more) load_q(n + hop);
  }
  if (item.solo) {
    if (ok) {
      pa_store_row<T, DK>(dk + (int64_t)mine * dk_row, ak, p.scale, p.head_k, lane);
      pa_store_row<T, DV>(dv + (int64_t)mine * dv_row, av, 1.f, p.head_v, lane);
    }
    return;
  }
  float* join = reinterpret_cast<float*>(lds);
  __syncthreads();
  pa_join<DK>(join, ak, p.scale, wave, lane);
  __syncthreads();
  pa_join_store<T, DK>(dk + (int64_t)first * dk_row, dk_row, join, item.len - first, p.head_k);
  __syncthreads();
  pa_join<DV>(join, av, 1.f, wave, lane);
  __syncthreads();
  pa_join_store<T, DV>(dv + (int64_t)first * dv_row, dv_row, join, item.len - first, p.head_v);
}

// ---- launchers ----------------------------------------------------------------------------------------------------------
template <int D>
static void pa_launch_shared(const MtPackedAttn& p, int pass, hipStream_t stream) {
  const dim3 grid((unsigned)(pass == 2 ? (p.n_kv_items + p.cut) * p.kv_heads : p.n_items * p.heads)), block(PA_THREADS);
  if (pass == 0) hipLaunchKernelGGL((mt_pattn_fwd_kernel<__bf16, D, 64>), grid, block, 0, stream, p);
  else if (pass == 1) hipLaunchKernelGGL((mt_pattn_dq_kernel<__bf16, D, 64>), grid, block, 0, stream, p);
  else {
    hipLaunchKernelGGL((mt_pattn_dkv_kernel<__bf16, D>), grid, dim3(PA_DKV_THREADS), 0, stream, p);
    if (p.cut > 0) hipLaunchKernelGGL((mt_pattn_halves_kernel<D>), dim3((unsigned)(p.cut * p.kv_heads * (PA_OWN / PA_HALVES_ROWS))), block, 0, stream, p);
  }
}
template <typename T, int DK, int DV>
static void pa_launch_split(const MtPackedAttn& p, int pass, hipStream_t stream) {
  const dim3 grid((unsigned)(pass == 2 ? p.n_kv_items * p.kv_heads : p.n_items * p.heads)), block(PA_THREADS);
  if (pass == 0) hipLaunchKernelGGL((mt_pattn_split_fwd_kernel<T, DK, DV>), grid, block, 0, stream, p);
  else if (pass == 1) hipLaunchKernelGGL((mt_pattn_split_dq_kernel<T, DK, DV>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((mt_pattn_split_dkv_kernel<T, DK, DV>), grid, block, 0, stream, p);
}
// Widths: both at most 32, 64 or 128 elements, or keys of at most 32 beside values of at most 64 (key_dim_scaling 0.5), whose smaller
// accumulators let two f32 waves of the dk / dv kernel share a SIMD.
template <typename T>
static void pa_launch_split_width(const MtPackedAttn& p, int pass, hipStream_t stream) {
  if (p.head_k <= 32 && p.head_v <= 32) pa_launch_split<T, 32, 32>(p, pass, stream);
  else if (p.head_k <= 32 && p.head_v <= 64) pa_launch_split<T, 32, 64>(p, pass, stream);
  else if (p.head_k <= 64 && p.head_v <= 64) pa_launch_split<T, 64, 64>(p, pass, stream);
  else pa_launch_split<T, 128, 128>(p, pass, stream);
}

extern "C" int mt_packed_attn_sizes(int* item_bytes, int* own_rows, int* split_rows, int* low_rows) {
  *item_bytes = (int)sizeof(MtSeqItem);
  *own_rows = PA_OWN;
  *split_rows = PA_TILE;
  *low_rows = PA_LOW_ROWS;
  return (int)sizeof(MtPackedAttn);
}

// backward: 0 forward; 1 dq and D, then dk and dv.  bf16: 0 = f32 operands (split form only), 1 = bf16.  Rows are read in 16-byte
// pieces.
extern "C" int mt_packed_attn_launch(const MtPackedAttn* a, int backward, int bf16, hipStream_t stream) {
  if (a == nullptr) return -2;
  const MtPackedAttn p = *a;
  if (p.n_items <= 0) return 0;
  const int es = bf16 ? 2 : 4, per = 16 / es;
  if (!p.q || !p.k || !p.v) return -2;      // tensors without memory (of a dispatch mode) have null addresses
  if (backward ? !p.out || !p.dout || !p.dq || !p.dk || !p.dv || !p.lse || !p.delta : !p.o) return -2;
  if (p.head_k < 1 || p.head_v < 1 || p.head_k > 128 || p.head_v > 128 || p.head_k % per || p.head_v % per) return -2;
  if (p.heads < 1 || p.kv_heads < 1 || p.heads % p.kv_heads || p.n_kv_items < 0) return -2;
  if (p.split < 0 || p.split > 2 || p.kv_split < 0 || p.kv_split > 2 || (!bf16 && (p.split == 0 || p.kv_split == 0))) return -2;
  if (p.items == nullptr || p.kv_items == nullptr) {      // a uniform batch: the numbers of items follow from its shape
    if (p.uniform_len < 1 || p.count < 1 || p.items != p.kv_items) return -2;
    for (int i = 0; i < 2; ++i) {
      const int rows = (i ? p.kv_split : p.split) == 1 ? PA_TILE : PA_OWN;
      if ((int64_t)((p.uniform_len - 1) / rows + 1) * p.count != (i ? p.n_kv_items : p.n_items)) return -2;
    }
  }
  if (p.cut != 0 && (p.cut < 0 || (int64_t)p.cut * p.kv_heads * (PA_OWN / PA_HALVES_ROWS) > 0x7FFFFFFF || p.cut > p.n_kv_items || p.halves == nullptr || p.kv_split != 0 || p.heads < 2 * p.kv_heads)) return -2;
  // a launch has fewer than 2^32 threads
  const int64_t kv_threads = ((int64_t)p.n_kv_items + p.cut) * p.kv_heads * (p.kv_split ? PA_THREADS : PA_DKV_THREADS);
  if ((int64_t)p.n_items * p.heads * PA_THREADS > 0xFFFFFFFFll || (backward && kv_threads > 0xFFFFFFFFll)) return -2;
  if (!(p.scale > 0.f)) return -2;
  const int64_t strides[8] = {p.q_row, p.q_head, p.k_row, p.k_head, p.v_row, p.v_head, p.do_row, p.do_head};
  for (int i = 0; i < 8; ++i)      // 32-bit byte offsets inside a staged tile of at most 128 rows
    if (strides[i] < 0 || strides[i] % per || strides[i] * es > (1 << 24)) return -2;
  const void* ptrs[10] = {p.q, p.k, p.v, p.out, p.dout, p.o, p.dq, p.dk, p.dv, p.low};
  for (int i = 0; i < 10; ++i)
    if (reinterpret_cast<uintptr_t>(ptrs[i]) & 15) return -2;
  const int widest = p.head_k > p.head_v ? p.head_k : p.head_v;
  for (int pass = backward ? 1 : 0; pass <= (backward ? 2 : 0); ++pass) {
    if (!bf16) pa_launch_split_width<float>(p, pass, stream);
    else if (pass == 2 ? p.kv_split : p.split) pa_launch_split_width<__bf16>(p, pass, stream);
    else if (widest <= 32) pa_launch_shared<32>(p, pass, stream);
    else if (widest <= 64) pa_launch_shared<64>(p, pass, stream);
    else pa_launch_shared<128>(p, pass, stream);
  }
  return (int)hipGetLastError();
}
