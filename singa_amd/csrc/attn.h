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
  if (s.causal) r.k = min(r.k, max(r.start + r.q, 0));   // (keys behind the last query are seen by none: not looked at)
  return r;
}

// the bucket of a key `distance` behind its query
__device__ __forceinline__ int bucket_of(const Shape &s, const Bounds &bounds, int distance) {
  const int n = s.bidirectional ? abs(distance) : max(-distance, 0);
  int lo = 0;
  for (int m = 0; m < bounds.n; ++m) lo += bounds.at[m] <= n;   // (the same for all lanes: scalar loads, and none waits for another)
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

// A tile holds rows of DP values, 16-byte chunks [row][RS], RS a power of two, in groups of 1024 bytes (what one load of a wavefront writes) that
// are 1040 bytes apart.  Chunk c of row r lies at place c ^ turn(r) of its row.  With both, the two ways in which a tile is read meet in no bank
// (64 of 4 bytes): one chunk of 16 rows, and four chunks of four rows.  turn() moves two bits of a chunk's number and is the same 8 rows on
// (but for the shortest rows), so that a lane has a handful of addresses, and all others are those and a constant.  (Without the 16 bytes, by three
// turned bits, half of the LDS's cycles were conflicts.)
template <class T, int DP>
struct Tile {
  static constexpr int CH = DP / T::VEC;                       // chunks of a row that are used
  static constexpr int RS = CH <= 4 ? 4 : CH <= 8 ? 8 : CH <= 16 ? 16 : 32;
  static constexpr int G = 64 / RS, GROUP = 1040;              // rows of a group
  static constexpr int bytes(int rows) { return rows / G * GROUP; }
  static __device__ __forceinline__ constexpr int turn(int r) {
    if constexpr (RS == 4) return (r >> 2) & 3;
    if constexpr (RS == 8) return ((r >> 1) & 1) << 2 | ((r >> 2) & 1) << 1;
    if constexpr (RS == 16) return (r & 3) << 2;
    return (r & 1) << 3;
  }
  static __device__ __forceinline__ int place(int r, int c) { return r / G * GROUP + (r % G * RS + (c ^ turn(r))) * 16; }
};

// Loads that write LDS: what the compiler knows of them it waits for in front of every transposed read, whichever tile that reads, so they are
// assembly (with no register to wait for), and tiles_arrive() waits for them.
typedef unsigned rsrc4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ rsrc4_t buffer_of(const void *p, int bytes) {
  const unsigned long long a = reinterpret_cast<unsigned long long>(p);
  return rsrc4_t{unsigned(a), unsigned(a >> 32) & 0xffffu, unsigned(bytes), 0x00020000u};   // (the same for all lanes)
}
__device__ __forceinline__ unsigned lds_offset(const void *lds) {
  typedef __attribute__((address_space(3))) const void lds_void;
  return unsigned(size_t((lds_void *)lds));
}
// 16 (4) bytes for each lane, one behind the other from `lds` on, the same for the whole wavefront; offsets behind the buffer give zeros
// (m0 is reserved: the compiler sets it in front of what needs it and, told that it is written here, again behind.  It warns of every such register.)
#pragma clang diagnostic push
#pragma clang diagnostic ignored "-Winline-asm"
__device__ __forceinline__ void load_lds16(rsrc4_t buffer, unsigned lds, int offset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(__builtin_amdgcn_readfirstlane(int(lds))), "v"(offset), "s"(buffer)
               : "memory", "m0");
}
__device__ __forceinline__ void load_lds4(rsrc4_t buffer, unsigned lds, int offset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"s"(__builtin_amdgcn_readfirstlane(int(lds))), "v"(offset), "s"(buffer)
               : "memory", "m0");
}
#pragma clang diagnostic pop

// Copies rows of a matrix into a tile.  Rows from `rows` on and values from `dim` on become zeros, whatever lies there.
template <class T, int DP, int ROWS, int NT = kBlock>
struct Stage {
  typedef typename T::elem elem;
  typedef Tile<T, DP> L;
  static constexpr int N = (ROWS * L::RS + NT - 1) / NT;   // chunks of a thread
  static_assert(ROWS * L::RS % SGH_WAVE == 0, "whole wavefronts");
  static constexpr bool kPart = N * NT != ROWS * L::RS;    // (the last wavefronts have one less)
  int voff[N];
  size_t stride;   // elements from row to row
  int dim, self;   // self: which of the NT threads that copy together
  bool direct;
  // (`direct`: rows of whole 16-byte chunks at multiples of 16 bytes; loads then write LDS without a register)
  __device__ __forceinline__ void init(size_t stride_, int dim_, bool direct_, int self_ = int(threadIdx.x)) {
    stride = stride_, dim = dim_, direct = direct_, self = self_;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const int p = j * NT + self, r = p / L::RS, c = (p % L::RS) ^ L::turn(r);
      voff[j] = c * T::VEC < dim ? int((r * stride + size_t(c) * T::VEC) * sizeof(elem)) : kOOB;
    }
  }
  // loads of a wavefront
  __device__ __forceinline__ int loads(int wave) const {
    int n = 0;
#pragma unroll
    for (int j = 0; j < N; ++j) n += !kPart || j * NT + wave * SGH_WAVE < ROWS * L::RS;
    return n;
  }
  __device__ __forceinline__ void operator()(char *lds, const elem *p, int rows) const {
    rows = min(rows, ROWS);
    if (direct) {
      const int bytes = rows > 0 ? ((rows - 1) * int(stride) + dim) * int(sizeof(elem)) : 0;   // (heads * dim is at most 2^20)
      rsrc4_t buffer = buffer_of(p, bytes);
      if constexpr (NT == SGH_WAVE)   // (one wavefront's: the compiler cannot tell that its lanes agree)
        for (int i = 0; i < 3; ++i) buffer[i] = unsigned(__builtin_amdgcn_readfirstlane(int(buffer[i])));
      const unsigned to = lds_offset(lds);
      const int wave = __builtin_amdgcn_readfirstlane(self >> 6);
#pragma unroll
      for (int j = 0; j < N; ++j)
        if (!kPart || j * NT + wave * SGH_WAVE < ROWS * L::RS) load_lds16(buffer, to + (wave + j * NT / SGH_WAVE) * L::GROUP, voff[j]);
    } else {
#pragma unroll
      for (int j = 0; j < N; ++j) {
        const int q = j * NT + self, r = q / L::RS, c = (q % L::RS) ^ L::turn(r);
        if (!kPart || q < ROWS * L::RS) *reinterpret_cast<u32x4 *>(lds + q / SGH_WAVE * L::GROUP + q % SGH_WAVE * 16) = chunk(p + r * stride, c * T::VEC, r < rows ? dim : 0);
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
// Loads into registers have arrived (vmcnt(0)).  In front of a loop that requests tiles: the compiler would otherwise wait for them inside, where they are used,
// and with that for every tile on its way.
__device__ __forceinline__ void registers_arrive() { __builtin_amdgcn_s_waitcnt(0x0f70); }

// A wavefront's own tiles are there, but for up to `behind` later loads (0 to 63 of them)
__device__ __forceinline__ void own_tiles_arrive(int behind) {
#define SGH_WAIT(N) case N: asm volatile("s_waitcnt vmcnt(" #N ") lgkmcnt(0)" ::: "memory"); break;
  switch (behind) {   // (every multiple of 2 that a kernel here asks for; others wait for all)
    SGH_WAIT(2) SGH_WAIT(4) SGH_WAIT(6) SGH_WAIT(8) SGH_WAIT(12) SGH_WAIT(16) SGH_WAIT(24) SGH_WAIT(32) SGH_WAIT(48)
    default: asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  }
#undef SGH_WAIT
}
// The wavefront's reads of LDS are done (what they read may be written over)
__device__ __forceinline__ void own_reads_end() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }
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

// Row of register i of a 32x32 result, without the 4 * (lane / 32)
__device__ __forceinline__ constexpr int row_of(int i) { return (i & 3) + 8 * (i >> 2); }

// The registers of a 32x32 result as the second operand of a product over its rows.  The 16-bit products take 16-bit operands: probabilities and
// the gradients of the scores are rounded to the tensors' type, once.  A result then has the error of two roundings for one: 2.1e-3 for the 1.6e-3 of
// fp32 terms (bfloat16, 4096 places), backwards 2.4e-3 for 1.7e-3.  Terms in two parts would bring that back for twice the products.
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

// Nothing is moved across: the loads in front are issued before what follows uses the first of them.  (Left to itself the compiler loaded one
// fragment, waited for it, used it and loaded the next.)
__device__ __forceinline__ void pin() { __builtin_amdgcn_sched_barrier(0); }

// A lane's places in a tile, and the products that read it
template <class T, int DP>
struct Reader {
  typedef Tile<T, DP> L;
  // Row reads take chunk 2 k + hi of row lane % 32: of the bits of k, those that turn() moves make an address, the others are a constant
  static constexpr int LOW = L::RS >= 32 ? 4 : L::RS == 16 ? 2 : 1;   // what k counts before its first turned bit
  static constexpr int ROWS = L::RS >= 32 ? 2 : L::RS == 4 ? 2 : 4;
  int row[ROWS];
  static __device__ __forceinline__ constexpr int which(int k) { return k / LOW % ROWS; }
  static __device__ __forceinline__ constexpr int beyond(int k) { return (k % LOW + k / (LOW * ROWS) * (LOW * ROWS)) * 32; }
  // Transposed reads.  16-bit: 16 lanes take four rows of 16 values and get them by columns, for values 32 n and on; fp32: a value of row i + 4 hi
  static constexpr int COLS = T::half ? (L::RS == 4 ? 1 : L::RS == 8 ? 2 : 4) : L::RS == 8 ? 1 : 2;
  int col[T::half ? (L::RS == 4 ? 2 : 1) : 4][COLS];
  __device__ __forceinline__ explicit Reader(int lane) {
    const int hi = lane >> 5;
#pragma unroll
    for (int k = 0; k < ROWS; ++k) row[k] = L::place(lane & 31, 2 * k * LOW + hi);
#pragma unroll
    for (int n = 0; n < COLS; ++n)
      if constexpr (T::half) {
        const int r = 4 * hi + ((lane >> 2) & 3), c = 4 * n + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
        col[0][n] = L::place(r, c) + (lane & 1) * 8;
        if constexpr (L::RS == 4) col[1][n] = L::place(r + 8, c) + (lane & 1) * 8;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) col[i][n] = L::place(i + 4 * hi, 8 * n + ((lane & 31) >> 2)) + (lane & 3) * 4;
      }
  }
  // What a product reads of a tile: rows [row0, row0 + 32), or the same rows transposed.  Loaded apart from the product where the order of
  // the loads matters (pin()).
  struct Rows {
    frag_t v[kSteps<T, DP>];
  };
  struct Cols {
    typename std::conditional<T::half, frag_t, float>::type v[T::half ? 2 : 16][DP / 32];
  };
  __device__ __forceinline__ frag_t row_chunk(const char *tile, int row0, int k) const {
    return *reinterpret_cast<const frag_t *>(tile + row[which(k)] + (row0 / L::G * L::GROUP + beyond(k)));
  }
  template <class V>
  __device__ __forceinline__ void col_chunk(const char *tile, int row0, int s, int n, V *v) const {
    if constexpr (T::half) {
      typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
      const char *at = tile + (row0 + 16 * s) / L::G * L::GROUP;
      const char *on = L::RS == 4 ? at + col[L::RS == 4][n] : at + col[0][n] + 8 / L::G * L::GROUP;
      const u32x2 l = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)(at + col[0][n])));
      const u32x2 u = __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4 *)on));
      *v = frag_t{l[0], l[1], u[0], u[1]};
    } else {
      *v = *reinterpret_cast<const float *>(tile + col[s & 3][n % COLS] + ((row0 + (s >> 2) * 8) / L::G * L::GROUP + n / COLS * COLS * 128));
    }
  }
  __device__ __forceinline__ void load(const char *tile, int row0, Rows &a) const {
#pragma unroll
    for (int k = 0; k < kSteps<T, DP>; ++k) a.v[k] = row_chunk(tile, row0, k);
  }
  __device__ __forceinline__ void load(const char *tile, int row0, Cols &a) const {
#pragma unroll
    for (int s = 0; s < (T::half ? 2 : 16); ++s)
#pragma unroll
      for (int n = 0; n < DP / 32; ++n) col_chunk(tile, row0, s, n, &a.v[s][n]);
  }
  // c += rows x columns f
  static __device__ __forceinline__ void mul(const Rows &a, const cols_t<T, DP> &f, f32x16 &c) {
#pragma unroll
    for (int k = 0; k < kSteps<T, DP>; ++k) c = mul_step<T>(a.v[k], f[k], c);
  }
  // c[n] += (rows, transposed: values 32 n ..) x t
  static __device__ __forceinline__ void mul(const Cols &a, const Terms<T> &t, f32x16 (&c)[DP / 32]) {
#pragma unroll
    for (int s = 0; s < (T::half ? 2 : 16); ++s)
#pragma unroll
      for (int n = 0; n < DP / 32; ++n) {
        if constexpr (T::half) c[n] = T::mfma(a.v[s][n], t.v[s], c[n]);
        else c[n] = __builtin_amdgcn_mfma_f32_32x32x2f32(a.v[s][n], t.v[s], c[n], 0, 0, 0);
      }
  }
  __device__ __forceinline__ void rows(const char *tile, int row0, const cols_t<T, DP> &f, f32x16 &c) const {
    Rows a;
    load(tile, row0, a);
    if constexpr (T::half && DP <= 64) pin();   // (bfloat16 heads of 64, 8 x 12 of 1024 places, bias, backward: 163 -> 159 us; of 128 1750 -> 1920)
    mul(a, f, c);
  }
  // The same with few registers: four chunk pairs at a time, the columns' last ones (from HELD on) from another tile, of 32 values
  template <int HELD>
  __device__ __forceinline__ void rows_by_four(const char *tile, int row0, const frag_t (&f)[HELD], const Reader<T, 32> &rest, const char *columns,
                                               f32x16 &c) const {
    constexpr int STEP = kSteps<T, DP> < 4 ? kSteps<T, DP> : 4;
#pragma unroll
    for (int k0 = 0; k0 < kSteps<T, DP>; k0 += STEP) {
      frag_t a[STEP], b[STEP];
#pragma unroll
      for (int k = 0; k < STEP; ++k)
        if (k0 + k < kSteps<T, DP>) {
          a[k] = row_chunk(tile, row0, k0 + k);
          if (k0 + k >= HELD) b[k] = rest.row_chunk(columns, 0, k0 + k - HELD);
        }
      pin();
#pragma unroll
      for (int k = 0; k < STEP; ++k)
        if (k0 + k < kSteps<T, DP>) c = mul_step<T>(a[k], k0 + k < HELD ? f[k0 + k < HELD ? k0 + k : 0] : b[k], c);
      pin();
    }
  }
  __device__ __forceinline__ void transposed_by_four(const char *tile, int row0, const Terms<T> &t, f32x16 (&c)[DP / 32]) const {
#pragma unroll
    for (int s = 0; s < (T::half ? 2 : 16); ++s) {
      typename std::conditional<T::half, frag_t, float>::type a[DP / 32];
#pragma unroll
      for (int n = 0; n < DP / 32; ++n) col_chunk(tile, row0, s, n, &a[n]);
      if (T::half || s % 4 == 3) pin();
#pragma unroll
      for (int n = 0; n < DP / 32; ++n) {
        if constexpr (T::half) c[n] = T::mfma(a[n], t.v[s], c[n]);
        else c[n] = __builtin_amdgcn_mfma_f32_32x32x2f32(a[n], t.v[s], c[n], 0, 0, 0);
      }
    }
  }
  // c += rows [row0, row0 + 32) of the tile x rows [own, own + 32) of another one as columns, four chunk pairs at a time
  __device__ __forceinline__ void rows(const char *tile, int row0, const char *columns, int own, f32x16 &c) const {
    constexpr int STEP = kSteps<T, DP> < 4 ? kSteps<T, DP> : DP == 128 ? 2 : 4;
#pragma unroll
    for (int k0 = 0; k0 < kSteps<T, DP>; k0 += STEP) {
      frag_t a[STEP], b[STEP];
#pragma unroll
      for (int k = 0; k < STEP; ++k)
        if (k0 + k < kSteps<T, DP>) a[k] = row_chunk(tile, row0, k0 + k), b[k] = row_chunk(columns + own / L::G * L::GROUP, 0, k0 + k);
      pin();
#pragma unroll
      for (int k = 0; k < STEP; ++k)
        if (k0 + k < kSteps<T, DP>) c = mul_step<T>(a[k], b[k], c);
      pin();
    }
  }
  __device__ __forceinline__ void transposed(const char *tile, int row0, const Terms<T> &t, f32x16 (&c)[DP / 32]) const {
    Cols a;
    load(tile, row0, a);
    mul(a, t, c);
  }
};
// The value of the lane 32 lanes on or back, together with the lane's own
__device__ __forceinline__ float max_of_pair(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
  return fmaxf(__builtin_bit_cast(float, unsigned(r[0])), __builtin_bit_cast(float, unsigned(r[1])));
}
__device__ __forceinline__ float sum_of_pair(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, x), __builtin_bit_cast(unsigned, x), false, false);
  return __builtin_bit_cast(float, unsigned(r[0])) + __builtin_bit_cast(float, unsigned(r[1]));
}

__device__ __forceinline__ void zero(f32x16 &c) {
#pragma unroll
  for (int i = 0; i < 16; ++i) c[i] = 0.f;
}
template <int N>
__device__ __forceinline__ void zero(f32x16 (&c)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) zero(c[n]);
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
  for (int i = threadIdx.x; i <= 2 * s.reach; i += int(blockDim.x))
    band[i] = s.table[size_t(bucket_of(s, bounds, i - s.reach)) * s.heads + h] * kLog2e;
}

// Rows of `dim` values anywhere as rows of `wide` (whole 16-byte chunks) at multiples of 16 bytes, zeros behind them.  What the kernels read many
// times is copied so first: loads of 16 bytes then write LDS without a register.
struct PadArgs {
  const void *from[4];
  void *to[4];
  size_t rows[4];
  int dim, wide;
};
template <class T>
__global__ __launch_bounds__(kBlock) void k_attn_pad(PadArgs a) {
  const int chunks = a.wide / T::VEC, which = blockIdx.y;
  const size_t n = a.rows[which] * chunks, step = size_t(gridDim.x) * kBlock;
  for (size_t i = size_t(blockIdx.x) * kBlock + threadIdx.x; i < n; i += step) {
    const size_t row = i / unsigned(chunks);
    const int c = int(i - row * chunks);
    const u32x4 v = Stage<T, 32, 64>::chunk(static_cast<const typename T::elem *>(a.from[which]) + row * a.dim, c * T::VEC, a.dim);
    reinterpret_cast<u32x4 *>(a.to[which])[i] = v;
  }
}

// Where a call's blocks lie: block w runs on the XCD w % 8, so the blocks of one head of keys, which read the same rows, go to one XCD where
// their number allows it.  Splits lie one behind the other.  Under a causal mask the tiles are of different lengths: long ones come first
// (`down`: the last ones), but where all blocks run at once every other 256 of them go the other way, so that a CU gets a short one with
// each long one (8 x 8 heads, 512 tokens, fp32 backward: 156 -> 123 us).
struct Where {
  unsigned tile, unit, split;
};
__device__ __forceinline__ Where block_at(unsigned tiles, unsigned units, unsigned splits, bool down) {
  const unsigned n = tiles * units, split = blockIdx.x / n, w = blockIdx.x % n;
  Where r = {0, 0, split};
  unsigned round;
  if (units % 8 == 0) {
    const unsigned l = w / 8, group = l / tiles;
    r.unit = group * 8 + w % 8, r.tile = l % tiles, round = group * tiles * 8;
  } else {
    r.unit = w / tiles, r.tile = w % tiles, round = r.unit * tiles;
  }
  const bool other = n * splits <= 512 && ((split * n + round) / 256) % 2 != 0;
  if (down != other) r.tile = tiles - 1 - r.tile;
  return r;
}

}  // namespace attn

#endif  // SINGA_AMD_CSRC_ATTN_H_
