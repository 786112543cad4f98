// What the attention kernels share: arguments, tiles in LDS, matrix fragments.
//
// All products keep one operand's rows in the lanes' columns: with the tile that runs through LDS as the matrix instruction's rows and the
// rows that a wavefront owns as its columns, every column of a 32x32 result lies in one lane and its partner 32 lanes on.  Row statistics
// then need one exchange, and a result's registers are already the second operand of the product that follows, if that product takes its
// 16 (or 2) terms in the order in which the registers hold them: the order of a sum's terms is free, so its first operand is read in that
// order.  Nothing goes back to LDS between the two products.
#ifndef SINGA_AMD_CSRC_ATTN_H_
#define SINGA_AMD_CSRC_ATTN_H_

#include <type_traits>

#include "common.h"
#include "rows.h"

namespace attn {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef __amdgpu_buffer_rsrc_t rsrc_t;

constexpr float kLog2e = 1.44269504088896341f, kLn2 = 0.693147180559945309f;
constexpr float kNegInf = -__builtin_inff();
constexpr int kOOB = 0x7ffffff0;   // an offset behind every buffer: loads give zeros
constexpr int kBlock = 256;

// Sizes, masks and the position bias of a call (sgh_attn_geom and the tensors of lengths), in every kernel's arguments
struct Shape {
  int q_len, k_len, heads, kv_heads, dim, causal;
  float scale;
  const int32_t *q_lengths, *k_lengths, *q_starts;
  // the band of distances [-reach, reach] beyond which the bias is that of its ends; 0 buckets: no bias
  int buckets, bidirectional, reach;
  const float *table;
};
// where bucket e + 1, e + 2, ... of one direction begin
struct Bounds {
  int n;
  int at[SGH_ATTN_MAX_BUCKETS];
};

struct Span {
  int q, k, start;   // rows of a sequence that count, and the position of its first query
};
__device__ __forceinline__ Span span_of(const Shape &s, int b) {
  Span r{s.q_len, s.k_len, s.k_len - s.q_len};
  if (s.q_lengths) r.q = min(max(s.q_lengths[b], 0), s.q_len);
  if (s.k_lengths) r.k = min(max(s.k_lengths[b], 0), s.k_len);
  if (s.q_starts) r.start = min(max(s.q_starts[b], -(1 << 30)), 1 << 30);
  return r;
}

// the bucket of a key `distance` behind its query
__device__ __forceinline__ int bucket_of(const Shape &s, const Bounds &bounds, int distance) {
  const int n = s.bidirectional ? abs(distance) : max(-distance, 0);
  int lo = 0, hi = bounds.n;   // bounds at or below n
  while (lo < hi) {
    const int m = (lo + hi) >> 1;
    if (bounds.at[m] <= n) lo = m + 1;
    else hi = m;
  }
  return s.bidirectional && distance > 0 ? lo + s.buckets / 2 : lo;
}

// ------------------------------------------------------------------------------------ storage types

struct F32 {
  typedef float elem;
  typedef StF32 St;
  static constexpr int VEC = 4;
  static constexpr bool half = false;
};
struct F16 {
  typedef uint16_t elem;
  typedef StF16 St;
  static constexpr int VEC = 8;
  static constexpr bool half = true;
  static __device__ __forceinline__ unsigned pack(float a, float b) { return sgh_pack2_f16(a, b); }
  static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
};
struct BF16 {
  typedef uint16_t elem;
  typedef StBF16 St;
  static constexpr int VEC = 8;
  static constexpr bool half = true;
  static __device__ __forceinline__ unsigned pack(float a, float b) { return sgh_pack2_bf16(a, b); }
  static __device__ __forceinline__ f32x16 mfma(u32x4 a, u32x4 b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  }
};

// 16 bytes of the results of two products' order: T::VEC values of a row
typedef u32x4 frag_t;

// ------------------------------------------------------------------------------------ tiles in LDS

// A tile holds rows of DP values, 16-byte chunks [row][RS], RS a power of two.  Chunk c of row r lies at place c ^ turn(r), so that
// neither the reads of one chunk of 32 rows nor those of 64 bytes of four rows meet in a bank.
template <class T, int DP>
struct Tile {
  static constexpr int CH = DP / T::VEC;                       // chunks of a row that are used
  static constexpr int RS = CH <= 4 ? 4 : CH <= 8 ? 8 : CH <= 16 ? 16 : 32;
  static constexpr int BYTES_OF_ROW = RS * 16;
  static __device__ __forceinline__ int turn(int r) {
    if constexpr (!T::half) return RS >= 16 ? (((r >> 2) & 1) << 3) | ((r & 3) << 1) | ((r >> 3) & 1) : (r >> 1) & (RS - 1);
    if constexpr (RS == 16) return ((r & 3) << 2) | ((r >> 2) & 3);
    if constexpr (RS == 8) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
    return (r >> 2) & 3;
  }
  static __device__ __forceinline__ int place(int r, int c) { return (r * RS + (c ^ turn(r))) * 16; }
};

typedef __attribute__((address_space(3))) void lds_void;
// 16 bytes for each lane, one behind the other from `lds` on
__device__ __forceinline__ void load_lds16(rsrc_t rs, lds_void *lds, int voff) {
#ifdef __HIP_DEVICE_COMPILE__   // (the host's pass takes this size for an error, and then drops kernels that call it, without a word)
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, lds, 16, voff, 0, 0, 0);
#endif
}

// Copies rows of a matrix into a tile.  Rows from `rows` on and values from `dim` on become zeros, whatever lies there.
template <class T, int DP, int ROWS>
struct Stage {
  typedef typename T::elem elem;
  typedef Tile<T, DP> L;
  static constexpr int N = ROWS * L::RS / kBlock;   // chunks of a thread
  static_assert(N * kBlock == ROWS * L::RS, "whole rounds");
  int voff[N];
  size_t stride;   // elements from row to row
  int dim;
  bool direct;
  // (`direct`: rows of whole 16-byte chunks at multiples of 16 bytes; loads then write LDS without a register)
  __device__ __forceinline__ void init(size_t stride_, int dim_, bool direct_) {
    stride = stride_, dim = dim_, direct = direct_;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int p = j * kBlock + int(threadIdx.x), r = p / L::RS, c = (p % L::RS) ^ L::turn(r);
      voff[j] = c * T::VEC < dim ? int((r * stride + size_t(c) * T::VEC) * sizeof(elem)) : kOOB;
    }
  }
  __device__ __forceinline__ void operator()(char *lds, const elem *p, int rows) const {
    rows = min(rows, ROWS);
    if (direct) {
      const int bytes = rows > 0 ? int(((rows - 1) * stride + dim) * sizeof(elem)) : 0;
      const rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(const_cast<elem *>(p), 0, bytes, 0x00020000);
      char *at = lds + __builtin_amdgcn_readfirstlane(int(threadIdx.x) >> 6) * 1024;
#pragma unroll
      for (int j = 0; j < N; ++j) load_lds16(rs, (lds_void *)(at + j * kBlock * 16), voff[j]);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int q = j * kBlock + int(threadIdx.x), r = q / L::RS, c = (q % L::RS) ^ L::turn(r);
        *reinterpret_cast<u32x4 *>(lds + q * 16) = chunk(p + r * stride, c * T::VEC, r < rows ? dim : 0);
      }
    }
  }
  // values [at, at + VEC) of a row of `n`, zeros behind it
  static __device__ __forceinline__ u32x4 chunk(const elem *row, int at, int n) {
    u32x4 v = {0, 0, 0, 0};
    if (at + T::VEC <= n) {
      __builtin_memcpy(&v, row + at, 16);
    } else if (at < n) {
      alignas(16) elem e[T::VEC] = {};
#pragma unroll
      for (int i = 0; i < T::VEC; ++i)
        if (at + i < n) e[i] = row[at + i];
      __builtin_memcpy(&v, e, 16);
    }
    return v;
  }
};
// tiles that the block's threads have requested are there, and everybody is done with what was read before
__device__ __forceinline__ void tiles_arrive() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// ------------------------------------------------------------------------------------ products

// The columns' fragments: chunk (2 k + hi) of the lane's row, k = 0 .. STEPS - 1
template <class T, int DP>
constexpr int kSteps = DP / (2 * T::VEC);
template <class T, int DP>
using cols_t = frag_t[kSteps<T, DP>];

template <class T, int DP>
__device__ __forceinline__ void load_columns(cols_t<T, DP> &f, const typename T::elem *row, int dim, int hi, bool direct) {
#pragma unroll
  for (int k = 0; k < kSteps<T, DP>; ++k) {
    const int at = (2 * k + hi) * T::VEC;
    if (direct) f[k] = at < dim ? *reinterpret_cast<const u32x4 *>(row + at) : u32x4{0, 0, 0, 0};
    else f[k] = Stage<T, DP, 64>::chunk(row, at, dim);
  }
}

// c += (one chunk pair of 32 rows) x (columns)
template <class T>
__device__ __forceinline__ f32x16 mul_step(frag_t a, frag_t b, f32x16 c) {
  if constexpr (T::half) {
    return T::mfma(a, b, c);
  } else {
    const sgh_v4f x = __builtin_bit_cast(sgh_v4f, a), y = __builtin_bit_cast(sgh_v4f, b);
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x[i], y[i], c, 0, 0, 0);
    return c;
  }
}

// c[q] += rows [row0, row0 + 32) of the tile x columns f[q]
template <class T, int DP, int Q>
__device__ __forceinline__ void mul_rows(const char *tile, int row0, const cols_t<T, DP> (&f)[Q], f32x16 (&c)[Q], int lane) {
  typedef Tile<T, DP> L;
  const int r = row0 + (lane & 31), hi = lane >> 5;
#pragma unroll
  for (int k = 0; k < kSteps<T, DP>; ++k) {
    const frag_t a = *reinterpret_cast<const frag_t *>(tile + L::place(r, 2 * k + hi));
#pragma unroll
    for (int q = 0; q < Q; ++q) c[q] = mul_step<T>(a, f[q][k], c[q]);
  }
}

// Row of register i of a 32x32 result, without the 4 * (lane / 32)
__device__ __forceinline__ constexpr int row_of(int i) { return (i & 3) + 8 * (i >> 2); }

// The registers of a 32x32 result as the second operand of a product over its rows
template <class T>
struct Terms {
  u32x4 v[2];
  __device__ __forceinline__ void set(const f32x16 &x) {
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int j = 0; j < 4; ++j) v[s][j] = T::pack(x[8 * s + 2 * j], x[8 * s + 2 * j + 1]);
  }
};
template <>
struct Terms<F32> {
  f32x16 v;
  __device__ __forceinline__ void set(const f32x16 &x) { v = x; }
};

// c[q][n] += (rows [row0, row0 + 32) of the tile, transposed: values 32 n ..) x t[q]
template <class T, int DP, int Q>
__device__ __forceinline__ void mul_transposed(const char *tile, int row0, const Terms<T> (&t)[Q], f32x16 (&c)[Q][DP / 32], int lane) {
  typedef Tile<T, DP> L;
  const int hi = lane >> 5;
  if constexpr (T::half) {
    // 16 lanes take four rows of 16 values and return them by columns
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    const int r = 4 * hi + ((lane >> 2) & 3), sub = (lane >> 4) & 1;
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int n = 0; n < DP / 32; ++n) {
        const int c0 = 4 * n + 2 * sub + ((lane >> 1) & 1), within = (lane & 1) * 8;
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(tile + L::place(row0 + 16 * s + r, c0) + within));
        const s16x4 up = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(tile + L::place(row0 + 16 * s + 8 + r, c0) + within));
        const u32x2 l = __builtin_bit_cast(u32x2, lo), u = __builtin_bit_cast(u32x2, up);
        const frag_t a = {l[0], l[1], u[0], u[1]};
#pragma unroll
        for (int q = 0; q < Q; ++q) c[q][n] = T::mfma(a, t[q].v[s], c[q][n]);
      }
  } else {
    const int d = lane & 31;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      const int r = row0 + row_of(i) + 4 * hi;
#pragma unroll
      for (int n = 0; n < DP / 32; ++n) {
        const float a = *reinterpret_cast<const float *>(tile + L::place(r, 8 * n + (d >> 2)) + (d & 3) * 4);
#pragma unroll
        for (int q = 0; q < Q; ++q) c[q][n] = __builtin_amdgcn_mfma_f32_32x32x2f32(a, t[q].v[i], c[q][n], 0, 0, 0);
      }
    }
  }
}

// The value of the lane 32 lanes on or back, together with the lane's own
__device__ __forceinline__ float max_of_pair(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
  return fmaxf(__builtin_bit_cast(float, unsigned(r[0])), __builtin_bit_cast(float, unsigned(r[1])));
}
__device__ __forceinline__ float sum_of_pair(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
  return __builtin_bit_cast(float, unsigned(r[0])) + __builtin_bit_cast(float, unsigned(r[1]));
}

template <int N>
__device__ __forceinline__ void zero(f32x16 (&c)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) c[n][i] = 0.f;
}

// Stores a lane's column (values 32 n + row of c[n]) times f as a row of `dim` values
template <class T, int DP>
__device__ __forceinline__ void store_column(typename T::elem *row, const f32x16 (&c)[DP / 32], float f, int dim, int hi, bool direct) {
#pragma unroll
  for (int n = 0; n < DP / 32; ++n)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * n + 8 * g + 4 * hi;
      float x[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = c[n][4 * g + i] * f;
      if (direct) {
        if (d < dim) {
          if constexpr (T::half) *reinterpret_cast<u32x2 *>(row + d) = u32x2{T::pack(x[0], x[1]), T::pack(x[2], x[3])};
          else *reinterpret_cast<sgh_v4f *>(row + d) = sgh_v4f{x[0], x[1], x[2], x[3]};
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (d + i < dim) T::St::st(row + d + i, x[i]);
      }
    }
}
// The same as 32-bit partial results: rows of DP values
template <int DP>
__device__ __forceinline__ void store_partial(float *row, const f32x16 (&c)[DP / 32], float f, int hi) {
#pragma unroll
  for (int n = 0; n < DP / 32; ++n)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      sgh_v4f x;
#pragma unroll
      for (int i = 0; i < 4; ++i) x[i] = c[n][4 * g + i] * f;
      *reinterpret_cast<sgh_v4f *>(row + 32 * n + 8 * g + 4 * hi) = x;
    }
}

// The bias of distances -reach .. reach for head h, times log2(e), in LDS
__device__ __forceinline__ void expand_bias(const Shape &s, const Bounds &bounds, int h, float *band) {
  for (int i = threadIdx.x; i <= 2 * s.reach; i += kBlock)
    band[i] = s.table[size_t(bucket_of(s, bounds, i - s.reach)) * s.heads + h] * kLog2e;
}

// Where a call's blocks lie: block w runs on the XCD w % 8, so the blocks of one head of keys, which read the same rows, go to one XCD where
// their number allows it
__device__ __forceinline__ void block_at(unsigned w, unsigned tiles, unsigned units, unsigned *tile, unsigned *unit) {
  if (units % 8 == 0) {
    const unsigned l = w / 8;
    *unit = (l / tiles) * 8 + w % 8, *tile = l % tiles;
  } else {
    *unit = w / tiles, *tile = w % tiles;
  }
}

}  // namespace attn

#endif  // SINGA_AMD_CSRC_ATTN_H_
