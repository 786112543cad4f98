// Token vectors: rows of a table by id, and the table's gradient.
//
//   y[t]  = scale * W[ids[t]]
//   dW[v] = add[v] + scale * sum over t with ids[t] = v of dy[t],  t ascending
//
// Both are bound by memory: the forward pass reads the rows asked for and writes as many, the gradient reads dy once and writes the
// whole table.  The order of the gradient's sums is fixed by the ids alone, so its bits do not change from run to run: no floating-point
// atomics.  A token that is padding or has no row of the table takes part in nothing (it becomes the id `vocab`, behind every row).
#include "common.h"
#include "rows.h"

namespace {

constexpr int kBlock = 256;
constexpr int kWaves = kBlock / SGH_WAVE;

__device__ int g_index_errors = 0;

// How the lanes of a wavefront lie over rows of `dim` elements: `lanes` of them on one row (a power of two; 64 / lanes rows at once),
// `slices` times over where a row is longer than 64 vectors.
struct RowLanes {
  int epl, lanes, slices;
};
RowLanes row_lanes(size_t dim, int vec) {   // vec: elements of 16 bytes
  RowLanes r;
  r.epl = dim < size_t(vec) ? 1 : vec;
  const size_t vecs = (dim + r.epl - 1) / r.epl;
  r.lanes = 1;
  while (r.lanes < SGH_WAVE && size_t(r.lanes) < vecs) r.lanes *= 2;
  r.slices = int((vecs + SGH_WAVE - 1) / SGH_WAVE);
  return r;
}

// ------------------------------------------------------------------------------------ forward

// A wavefront takes 64 / lanes tokens and PER slices of their rows, all loads in flight before the first store.  Bound by memory: 16384 tokens of
// 4096 bfloat16 elements 32 us, 78 MB read past the die's caches and 134 written, 6.7 TB/s; 32 tokens are a launch, 3.3 us.
template <class S, int EPL, int PER, bool STREAM>
__global__ __launch_bounds__(kBlock) void k_embed_fwd(const int32_t *__restrict__ ids, const typename S::elem *__restrict__ W,
                                                      typename S::elem *__restrict__ y, size_t tokens, size_t vocab, size_t dim,
                                                      float scale, int pad, int lanes) {
  const int lane = threadIdx.x & (SGH_WAVE - 1), per_wave = SGH_WAVE / lanes;
  const size_t vecs = (dim + EPL - 1) / EPL;
  const size_t first = size_t(blockIdx.y) * PER * SGH_WAVE + (lane & (lanes - 1));
  const size_t step = size_t(gridDim.x) * kWaves * per_wave;
  for (size_t t = (size_t(blockIdx.x) * kWaves + (threadIdx.x >> 6)) * per_wave + lane / lanes; t < tokens; t += step) {
    const int id = ids[t];
    const bool pads = id == pad, found = !pads && id >= 0 && size_t(id) < vocab;
    if (!pads && !found && first == 0) atomicAdd(&g_index_errors, 1);
    const typename S::elem *row = W + (found ? size_t(id) : 0) * dim;
    float v[PER][EPL];
    size_t at[PER];
#pragma unroll
    for (int p = 0; p < PER; ++p) {
      const size_t vec = first + size_t(p) * SGH_WAVE;
      at[p] = vec * EPL + EPL > dim ? dim - EPL : vec * EPL;
#pragma unroll
      for (int j = 0; j < EPL; ++j) v[p][j] = 0.f;
      if (found && vec < vecs) sgh_load_any<S, EPL>(row + at[p], v[p]);
    }
#pragma unroll
    for (int p = 0; p < PER; ++p) {
#pragma unroll
      for (int j = 0; j < EPL; ++j) v[p][j] = found ? v[p][j] * scale : 0.f;
      if (first + size_t(p) * SGH_WAVE < vecs) sgh_store_any<S, EPL, STREAM>(y + t * dim + at[p], v[p]);
    }
  }
}

template <class S, int EPL, int PER>
int launch_fwd(const int32_t *ids, const typename S::elem *W, typename S::elem *y, size_t tokens, size_t vocab, size_t dim,
               float scale, int pad, const RowLanes &r, hipStream_t s) {
  const size_t per_block = size_t(kWaves) * (SGH_WAVE / r.lanes);
  size_t blocks = (tokens + per_block - 1) / per_block;
  if (blocks > (1u << 22)) blocks = 1u << 22;
  const int ny = (r.slices + PER - 1) / PER;
  const dim3 grid{unsigned(blocks), unsigned(ny)};
  // (134 MB, 16384 tokens of 4096 16-bit elements: 44.6 us through the caches, 32.2 past them)
  if (tokens * dim * sizeof(typename S::elem) >= kStreamBytes)
    SGH_LAUNCH_TIMED((k_embed_fwd<S, EPL, PER, true>), grid, dim3(kBlock), 0, s, ids, W, y, tokens, vocab, dim, scale, pad, r.lanes);
  else
    SGH_LAUNCH_TIMED((k_embed_fwd<S, EPL, PER, false>), grid, dim3(kBlock), 0, s, ids, W, y, tokens, vocab, dim, scale, pad, r.lanes);
  SGH_LAUNCH_CHECK();
  return SGH_OK;
}

constexpr size_t kMostDim = size_t(1) << 21;   // (the slices of a row, of 64 elements or more, are a grid's second dimension: at most 65535)

bool sizes_ok(size_t tokens, size_t vocab, size_t dim) {
  return tokens <= 0x7fffffffu && vocab <= 0x7fffffffu && dim <= kMostDim;
}

template <class S>
int embed_fwd(const int32_t *ids, const typename S::elem *W, typename S::elem *y, size_t tokens, size_t vocab, size_t dim, float scale,
              int pad, void *stream) {
  if (!sizes_ok(tokens, vocab, dim)) return SGH_EINVAL;
  if (tokens == 0 || dim == 0) return SGH_OK;
  constexpr size_t e = sizeof(typename S::elem);
  if (!ids || (!W && vocab != 0) || !y) return SGH_EINVAL;
  if (sgh_ranges_meet(y, tokens * dim * e, W, vocab * dim * e) || sgh_ranges_meet(y, tokens * dim * e, ids, tokens * 4)) return SGH_EINVAL;
  hipStream_t s = sgh_stream_of(stream);
  sgh_note_write(y, tokens * dim * e);
  sgh_prof_kernel_scope prof("embedding_fwd/k_embed_fwd", double(tokens) * (4 + 2.0 * dim * e), s);
  const RowLanes r = row_lanes(dim, S::VEC);
  if (r.epl == 1) return launch_fwd<S, 1, 1>(ids, W, y, tokens, vocab, dim, scale, pad, r, s);
  return launch_fwd<S, S::VEC, 4>(ids, W, y, tokens, vocab, dim, scale, pad, r, s);
}

// ------------------------------------------------------------------------------------ the gradient

// A token in the sorted list: its id (`vocab` where it takes part in nothing) and its place
struct alignas(8) Token {
  unsigned key, place;
};

// A call's tensors and how they are cut
template <class T>
struct Bwd {
  const int32_t *ids;
  const T *dy, *add;
  T *dW;
  const Token *sorted;
  unsigned *tail;                  // of every tile: the first of the sums that its last row is to be joined from, if any
  float *partial;                  // [tiles][2][pitch]: sums of a row's tokens that hold whole tiles: a tile's head or all of it, its tail
  size_t pitch;
  size_t dim, vocab;
  unsigned tokens, tile, stretch;  // sorted tokens of a tile, of a workgroup
  float scale;
  int pad, lanes, slices;
};

// One vector of a row of `add` (zeros without one), asked for before the sums so that the two waits are one, and the store of acc * scale on
// top of it.  The row's last vector is moved back to end with the row (at != vec * EPL): its first elements are the vector's before it,
// which may be stored already where `add` is the result itself, and are left alone.
template <class S, int EPL>
__device__ __forceinline__ void load_add(const Bwd<typename S::elem> &a, size_t row, size_t at, float *g) {
#pragma unroll
  for (int j = 0; j < EPL; ++j) g[j] = 0.f;
  if (a.add) sgh_load_any<S, EPL>(a.add + row * a.dim + at, g);
}
template <class S, int EPL, bool STREAM>
__device__ __forceinline__ void store_row(const Bwd<typename S::elem> &a, size_t row, size_t at, size_t vec, float *acc, const float *g) {
  typename S::elem *out = a.dW + row * a.dim + at;
#pragma unroll
  for (int j = 0; j < EPL; ++j) acc[j] = acc[j] * a.scale + g[j];
  if (at == vec * EPL) {
    sgh_store_any<S, EPL, STREAM>(out, acc);
  } else {
#pragma unroll
    for (int j = 0; j < EPL; ++j)
      if (at + j >= vec * EPL) S::st(out + j, acc[j]);
  }
}

// Sum of rows place[from .. to) of dy, ascending, on top of acc
template <class S, int EPL, bool STREAM>
__device__ __forceinline__ void add_tokens(const typename S::elem *dy, size_t dim, size_t at, const unsigned *place, unsigned from,
                                           unsigned to, float *acc) {
  constexpr int U = 4;   // (8: 97 -> 99 us for 131072 tokens of 1024 16-bit elements)
  unsigned i = from;
  // (no branch around any of a group's loads: it would wait there.  All in guarded groups: 68 -> 60.5 us for 131072 tokens of 512, 9.1 -> 6.5 for
  // 1024 of 4096 in 200 rows)
  for (; i + U <= to; i += U) {
    float v[U][EPL];
#pragma unroll
    for (int u = 0; u < U; ++u) sgh_load_any<S, EPL, STREAM>(dy + size_t(place[i + u]) * dim + at, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < EPL; ++j) acc[j] += v[u][j];
  }
  for (; i < to; ++i) {
    float v[EPL];
    sgh_load_any<S, EPL, STREAM>(dy + size_t(place[i]) * dim + at, v);
#pragma unroll
    for (int j = 0; j < EPL; ++j) acc[j] += v[j];
  }
}

// LDS as the wavefront's lanes left it, before and after
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// Inclusive sum over the lanes in front
__device__ __forceinline__ unsigned wave_upto(unsigned v) {
  const int lane = threadIdx.x & (SGH_WAVE - 1);
#pragma unroll
  for (int o = 1; o < SGH_WAVE; o <<= 1) {
    const unsigned u = __shfl_up(v, o, SGH_WAVE);
    if (lane >= o) v += u;
  }
  return v;
}

// How many of the lanes in `mask` are in front of this one
__device__ __forceinline__ int lanes_below(unsigned long long mask) {
  return __builtin_amdgcn_mbcnt_hi(unsigned(mask >> 32), __builtin_amdgcn_mbcnt_lo(unsigned(mask), 0));
}

// Lanes of the wavefront (those with `there`) whose value agrees with this lane's in its low BITS bits
template <int BITS>
__device__ __forceinline__ unsigned long long same_lanes(unsigned v, bool there) {
  const unsigned long long all = __ballot(there);
  unsigned lo = unsigned(all), hi = unsigned(all >> 32);
#pragma unroll
  for (int b = 0; b < BITS; ++b) {
    const unsigned mine = unsigned(int(v << (31 - b)) >> 31);   // all ones where the bit is set
    const unsigned long long set = __ballot(int(mine) < 0);
    lo &= ~(unsigned(set) ^ mine);
    hi &= ~(unsigned(set >> 32) ^ mine);
  }
  return (static_cast<unsigned long long>(hi) << 32) | lo;
}

// ------------------------------------------------------------------------------------ few tokens

constexpr int kMostRows = 256;           // rows of a workgroup
constexpr unsigned kScanTokens = 512;

// Up to kScanTokens tokens, in one launch: a workgroup has a few consecutive rows, looks through all ids for theirs, sorts those in LDS and
// sums and stores its rows, or slices of them; rows without a token become zero, or `add`.  A launch that waits for another costs more than the
// ids, which every workgroup reads: 512 tokens, 10007 rows of 201 binary16 elements 7.8 us; 131072 rows of 64: 8.0, sorted 14.  (32 KB of the result
// for a workgroup.  Beyond kScanTokens a call waits for the rows of the commonest ids, which few workgroups have: 1024 tokens of text, 32000
// rows of 512: 29.7 us, sorted 21.4; 512: 17.0 and 19.6; ids that are all one: 112 and 24, 57 and 21.)
template <class S, int EPL, bool STREAM>
__global__ __launch_bounds__(kBlock) void k_embed_rows(Bwd<typename S::elem> a, int rows_each) {
  __shared__ unsigned begin[kMostRows], end[kMostRows];
  __shared__ unsigned found[kScanTokens];    // places of the rows' tokens, by row
  __shared__ unsigned listed[kScanTokens];   // (row, place) in the order of the places
  __shared__ unsigned sums[kWaves];
  const int tid = threadIdx.x, lane = tid & (SGH_WAVE - 1), wave = tid >> 6;
  const size_t row0 = size_t(blockIdx.x) * rows_each;
  const int rows = a.vocab - row0 < size_t(rows_each) ? int(a.vocab - row0) : rows_each;
  for (int r = tid; r < rows; r += kBlock) begin[r] = end[r] = 0;
  constexpr int P = kScanTokens / kBlock;   // a thread's tokens are neighbours: one prefix sum keeps the order
  unsigned mine[P], n = 0;
#pragma unroll
  for (int p = 0; p < P; ++p) {
    const unsigned t = tid * P + p;
    mine[p] = 0xffffffffu;
    if (t < a.tokens) {
      const int id = a.ids[t];
      if (id != a.pad && (id < 0 || size_t(id) >= a.vocab)) {
        if (blockIdx.x == 0 && blockIdx.y == 0) atomicAdd(&g_index_errors, 1);
      } else if (id != a.pad && size_t(id) >= row0 && size_t(id) < row0 + rows) {
        mine[p] = unsigned(size_t(id) - row0);
        ++n;
      }
    }
  }
  const unsigned upto = wave_upto(n);
  if (lane == SGH_WAVE - 1) sums[wave] = upto;
  __syncthreads();
  unsigned slot = upto - n, total = 0;
  for (int w = 0; w < kWaves; ++w) {
    if (w < wave) slot += sums[w];
    total += sums[w];
  }
#pragma unroll
  for (int p = 0; p < P; ++p)
    if (mine[p] != 0xffffffffu) {
      listed[slot++] = (mine[p] << 16) | unsigned(tid * P + p);
      atomicAdd(&end[mine[p]], 1u);
    }
  __syncthreads();
  if (wave == 0) {   // a stable counting sort by row: end[] holds the counts
    unsigned carry = 0;
    for (int r = lane; r - lane < rows; r += SGH_WAVE) {
      const unsigned c = r < rows ? end[r] : 0, up = wave_upto(c);
      if (r < rows) begin[r] = end[r] = carry + up - c;
      carry += __shfl(up, SGH_WAVE - 1, SGH_WAVE);
    }
    wave_sync();
    for (unsigned i = lane; i - lane < total; i += SGH_WAVE) {
      const bool there = i < total;
      const unsigned e = there ? listed[i] : 0, r = e >> 16;
      const unsigned long long same = same_lanes<8>(r, there);
      const int ahead = lanes_below(same);
      const unsigned old = there ? end[r] : 0;
      wave_sync();
      if (there) found[old + ahead] = e & 0xffffu;
      if (there && ahead == 0) end[r] = old + __popcll(same);
      wave_sync();
    }
  }
  __syncthreads();
  const size_t vecs = (a.dim + EPL - 1) / EPL;
  const int per_wave = SGH_WAVE / a.lanes, groups = (rows + per_wave - 1) / per_wave;
  for (size_t unit = size_t(blockIdx.y) * kWaves + wave; unit < size_t(groups) * a.slices; unit += size_t(gridDim.y) * kWaves) {
    const int group = a.slices == 1 ? int(unit) : int(unit / unsigned(a.slices));
    const size_t vec = (unit - size_t(group) * a.slices) * SGH_WAVE + (lane & (a.lanes - 1));
    const int r = group * per_wave + lane / a.lanes;
    if (r >= rows || vec >= vecs) continue;
    const size_t at = vec * EPL + EPL > a.dim ? a.dim - EPL : vec * EPL;
    const unsigned b = begin[r], e = end[r];
    if (b == e && a.add == a.dW) continue;
    float acc[EPL];
#pragma unroll
    for (int j = 0; j < EPL; ++j) acc[j] = 0.f;
    add_tokens<S, EPL, false>(a.dy, a.dim, at, found, b, e, acc);
    float g[EPL];
    load_add<S, EPL>(a, row0 + r, at, g);
    store_row<S, EPL, STREAM>(a, row0 + r, at, vec, acc, g);
  }
}

// ------------------------------------------------------------------------------------ many tokens

// 1. The tokens are sorted by id, stable.  Up to kRankTokens each token counts those that belong in front of it, in one launch.  More are sorted
//    in passes of at most 9 bits from the lowest: a pass counts the digits of each workgroup's stretch of tokens, turns the counts into the
//    place of every stretch's first token with a digit, and moves the tokens there.  Sorting leaves the memory idle: beside it, in the same
//    launches, other workgroups store the rows that have no token.
// 2. Tiles of sorted tokens: a wavefront goes through the tokens of a tile (and a slice of the rows' elements), and stores each row whose
//    tokens begin there.  Where a row's tokens hold a whole tile, that tile's sum is kept instead,
// 3. and the tile in which they begin joins the sums.

constexpr unsigned kNoKey = 0xffffffffu;
constexpr int kDigitBits = 9, kBins = 1 << kDigitBits;
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / SGH_WAVE;
constexpr int kItems = 2;                              // tokens of a thread at a time
constexpr unsigned kStretch = kSortThreads * kItems;
constexpr int kMostStretches = 64;                     // each workgroup reads the counts of all
// (Counting is quadratic.  The whole gradient for a table of 131072 rows of 64 bfloat16 elements: 20.6 us for 8192 tokens counted, 29.4 sorted in
// passes; 33.8 and 31.5 for 16384.)
constexpr unsigned kRankTokens = 8192;
constexpr unsigned kFillRows = 8192;                   // rows that a workgroup looks out for

struct Sort {
  const int32_t *ids;                  // first pass
  const Token *in;                     // later ones
  Token *out;
  unsigned *counts;                    // [stretches][bins]
  unsigned tokens, vocab, per_stretch;
  int pad, shift, bins, stretches;
};
// Rows without a token: `rows` of them are looked after by each workgroup, the share `launch` of `launches` in this launch
enum class Taken {
  kIds,      // the rows that have one are found by looking through all ids,
  kClear,    // or they are marked: the first launch clears the marks (and stores nothing), the first move sets them,
  kMarks,    // the later launches read them;
  kCounts    // with one digit they are in the counts
};
struct Fill {
  unsigned rows;
  int launch, launches;
  Taken from;
  unsigned char *taken;        // [vocab] or null
};

struct SortSpace {
  unsigned next[kBins];                  // where the next token with a digit goes
  uint16_t in_wave[kSortWaves][kBins];   // tokens with a digit of each wavefront, then those of the wavefronts in front
  unsigned sums[kSortWaves];
};

__device__ __forceinline__ unsigned key_of(int id, unsigned vocab, int pad) {
  return id < 0 || unsigned(id) >= vocab || id == pad ? vocab : unsigned(id);
}

__device__ __forceinline__ void count_digits(const Sort &s, unsigned from, unsigned to, unsigned *h) {
  constexpr unsigned U = 2;
  for (size_t i = size_t(from) + threadIdx.x; i < to; i += U * kSortThreads) {
    unsigned k[U];
#pragma unroll
    for (unsigned u = 0; u < U; ++u) {
      const size_t j = i + u * kSortThreads;
      k[u] = j < to ? (s.ids ? unsigned(s.ids[j]) : s.in[j].key) : 0;
    }
#pragma unroll
    for (unsigned u = 0; u < U; ++u)
      if (i + u * kSortThreads < to) {
        if (s.ids) k[u] = key_of(int(k[u]), s.vocab, s.pad);
        atomicAdd(&h[(k[u] >> s.shift) & (s.bins - 1)], 1u);
      }
  }
}

// All tokens with a digit below this thread's, from every digit's total in thread `digit`
__device__ __forceinline__ unsigned lower_digits(SortSpace &sp, unsigned total) {
  const int lane = threadIdx.x & (SGH_WAVE - 1), wave = threadIdx.x >> 6;
  const unsigned upto = wave_upto(total);
  if (lane == SGH_WAVE - 1) sp.sums[wave] = upto;
  __syncthreads();
  unsigned lower = upto - total;
  for (int w = 0; w < wave; ++w) lower += sp.sums[w];
  return lower;
}

// Up to ITEMS * 64 tokens of every wavefront, neighbours each
template <int ITEMS>
struct Held {
  unsigned key[ITEMS], place[ITEMS], rank[ITEMS];
};
constexpr unsigned kNoPlace = 0xffffffffu;

// Ranks the held tokens among those of the wavefront with their digit, whose counts go to in_wave (zero before)
template <int ITEMS>
__device__ __forceinline__ void sort_rank(const Sort &s, unsigned per_wave, SortSpace &sp, Held<ITEMS> &h) {
  const int wave = threadIdx.x >> 6;
#pragma unroll
  for (int u = 0; u < ITEMS; ++u)
    if (u * SGH_WAVE < per_wave) {
      const bool there = h.place[u] != kNoPlace;
      const unsigned digit = (h.key[u] >> s.shift) & (s.bins - 1);
      const unsigned long long same = same_lanes<kDigitBits>(digit, there);
      const int ahead = lanes_below(same);
      const unsigned old = sp.in_wave[wave][digit];
      h.rank[u] = old + ahead;
      wave_sync();   // (every lane has read the count before one of them writes it)
      if (there && ahead == 0) sp.in_wave[wave][digit] = uint16_t(old + __popcll(same));
      wave_sync();
    }
}
__device__ __forceinline__ void clear_counts(SortSpace &sp) {
  unsigned *w = reinterpret_cast<unsigned *>(&sp.in_wave[0][0]);
  for (int i = threadIdx.x; i < kSortWaves * kBins / 2; i += kSortThreads) w[i] = 0;
}
// in_wave from counts to those of the wavefronts in front: thread `digit`; returns the digit's total
__device__ __forceinline__ unsigned front_counts(SortSpace &sp) {
  unsigned at = 0;
#pragma unroll
  for (int w = 0; w < kSortWaves; ++w) {
    const unsigned c = sp.in_wave[w][threadIdx.x];
    sp.in_wave[w][threadIdx.x] = uint16_t(at);
    at += c;
  }
  return at;
}
__device__ __forceinline__ unsigned place_of(const Sort &s, const SortSpace &sp, unsigned key, unsigned rank) {
  const unsigned digit = (key >> s.shift) & (s.bins - 1);
  return sp.next[digit] + sp.in_wave[threadIdx.x >> 6][digit] + rank;
}
__device__ __forceinline__ unsigned counted_key(const Sort &s, int id, bool there) {
  const unsigned k = key_of(id, s.vocab, s.pad);
  if (there && k == s.vocab && id != s.pad) atomicAdd(&g_index_errors, 1);
  return k;
}

// The rows that have no token: zero, or `add`
template <class S, int EPL, bool STREAM>
__device__ __forceinline__ void fill_rows(const Bwd<typename S::elem> &a, const Sort &s, const Fill &f, unsigned part, unsigned char *taken) {
  const size_t row0 = size_t(part) * f.rows;
  const unsigned rows = a.vocab - row0 < f.rows ? unsigned(a.vocab - row0) : f.rows, threads = kSortThreads;
  const unsigned tid = threadIdx.x, lane = tid & (SGH_WAVE - 1), wave = tid >> 6;
  const unsigned lo = rows * f.launch / f.launches, hi = rows * (f.launch + 1) / f.launches;   // its share
  if (f.from == Taken::kClear) {
    for (unsigned r = tid; r < rows; r += threads) f.taken[row0 + r] = 0;
    return;
  }
  if (f.from == Taken::kIds) {
    for (unsigned r = tid; r < rows; r += threads) taken[r] = 0;
    __syncthreads();
    constexpr unsigned U = 8;
    for (size_t i = tid; i < a.tokens; i += U * threads) {
      int id[U];
#pragma unroll
      for (unsigned u = 0; u < U; ++u) id[u] = i + u * threads < a.tokens ? a.ids[i + u * threads] : a.pad;
#pragma unroll
      for (unsigned u = 0; u < U; ++u) {
        const size_t r = size_t(id[u]) - row0;   // (an id below the rows, or below 0, is a large number)
        if (id[u] >= 0 && r < rows && id[u] != a.pad) taken[r] = 1;
      }
    }
  } else if (f.from == Taken::kMarks) {
    for (unsigned r = lo + tid; r < hi; r += threads) taken[r] = f.taken[row0 + r];
  } else {
    for (unsigned r = lo + tid; r < hi; r += threads) {
      unsigned n = 0;
      for (int b = 0; b < s.stretches; ++b) n |= s.counts[b * s.bins + row0 + r];
      taken[r] = n != 0;
    }
  }
  __syncthreads();
  const size_t vecs = (a.dim + EPL - 1) / EPL;
  const unsigned per_wave = SGH_WAVE / a.lanes;
  constexpr int U = 4;
  const unsigned waves = threads / SGH_WAVE;
  for (unsigned r0 = lo + wave; r0 < hi; r0 += threads) {   // every `waves`-th row is a wavefront's, a lane asks for each of 64
    const unsigned asked = r0 + lane * waves;
    const unsigned long long free = __ballot(asked < hi && !taken[asked]);
    for (unsigned i = lane / a.lanes; i < SGH_WAVE && r0 + i * waves < hi; i += per_wave) {
      if (!(free >> i & 1)) continue;
      const size_t row = (row0 + r0 + i * waves) * a.dim;
      for (size_t vec = lane & (a.lanes - 1); vec < vecs; vec += U * SGH_WAVE) {
        float v[U][EPL];
        size_t at[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const size_t n = vec + u * SGH_WAVE;
          at[u] = row + (n * EPL + EPL > a.dim ? a.dim - EPL : n * EPL);
#pragma unroll
          for (int j = 0; j < EPL; ++j) v[u][j] = 0.f;
          if (a.add && n < vecs) sgh_load_any<S, EPL, STREAM>(a.add + at[u], v[u]);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
          if (vec + u * SGH_WAVE < vecs) sgh_store_any<S, EPL, STREAM>(a.dW + at[u], v[u]);
      }
    }
  }
}

// Up to kRankTokens tokens: the place of a token in the sorted list is the number of those with a smaller key, or with the same one further in
// front.  A workgroup has all keys in LDS, where a wavefront goes through them for M tokens at a time, its lanes four neighbouring keys each:
// two instructions for 64 comparisons, T^2 of these: 4.5 us for 1025 tokens, 6.3 for 4096, 8.4 for 8192.  (Passes by one workgroup, the tokens
// in its registers: 12 us for 2048, 19 for 8192.)
constexpr unsigned kChunk = 4 * SGH_WAVE;   // keys that a wavefront looks at at once
union RankLds {
  sgh_v4u keys[kRankTokens / 4];
  unsigned char taken[kFillRows];
};
template <int M>
__device__ __forceinline__ void rank_tokens(const Sort &s, const RankLds &lds, unsigned first) {
  const unsigned *all = reinterpret_cast<const unsigned *>(lds.keys), lane = threadIdx.x & (SGH_WAVE - 1);
  const sgh_v4u *keys = lds.keys + lane;
  unsigned key[M], n[M];
#pragma unroll
  for (int m = 0; m < M; ++m) {
    key[m] = __builtin_amdgcn_readfirstlane(all[first + m]);   // (kNoKey behind the last token)
    n[m] = 0;
  }
  // `more`: 1 where equal keys are in front
  auto count = [&](unsigned from, unsigned to, unsigned more) {
#pragma unroll 4
    for (unsigned c = from; c < to; ++c) {
      const sgh_v4u k = keys[c * SGH_WAVE];
#pragma unroll
      for (int m = 0; m < M; ++m)
#pragma unroll
        for (int e = 0; e < 4; ++e) n[m] += k[e] < key[m] + more;
    }
  };
  const unsigned here = first / kChunk, chunks = (s.tokens + kChunk - 1) / kChunk;   // (M divides kChunk and `first`)
  count(0, here, 1);
  count(here, chunks, 0);
  const sgh_v4u k = keys[here * SGH_WAVE];
#pragma unroll
  for (int m = 0; m < M; ++m) {
#pragma unroll
    for (int e = 0; e < 4; ++e) n[m] += k[e] == key[m] && here * kChunk + lane * 4 + e < first + m;
#pragma unroll
    for (int o = 1; o < SGH_WAVE; o <<= 1) n[m] += __shfl_xor(n[m], o, SGH_WAVE);
  }
#pragma unroll
  for (int m = 0; m < M; ++m)
    if (int(lane) == m && first + m < s.tokens) {
      if (key[m] == s.vocab && s.ids[first + m] != s.pad) atomicAdd(&g_index_errors, 1);
      s.out[n[m]] = Token{key[m], first + m};
    }
}
template <class S, int EPL, bool STREAM>
__global__ __launch_bounds__(kSortThreads) void k_embed_rank(Bwd<typename S::elem> a, Sort s, int per_wave, Fill f) {
  __shared__ RankLds lds;
  if (blockIdx.x >= unsigned(s.stretches)) return fill_rows<S, EPL, STREAM>(a, s, f, blockIdx.x - s.stretches, lds.taken);
  unsigned *all = reinterpret_cast<unsigned *>(lds.keys);
  const unsigned room = (s.tokens + kChunk - 1) / kChunk * kChunk;
  constexpr unsigned U = 8;
  for (unsigned i = threadIdx.x; i < room; i += U * kSortThreads) {
    int id[U];
#pragma unroll
    for (unsigned u = 0; u < U; ++u) id[u] = i + u * kSortThreads < s.tokens ? s.ids[i + u * kSortThreads] : 0;
#pragma unroll
    for (unsigned u = 0; u < U; ++u) {
      const unsigned at = i + u * kSortThreads;
      if (at < room) all[at] = at < s.tokens ? key_of(id[u], s.vocab, s.pad) : kNoKey;
    }
  }
  __syncthreads();
  const unsigned first = __builtin_amdgcn_readfirstlane((blockIdx.x * kSortWaves + (threadIdx.x >> 6)) * per_wave);
  if (first >= s.tokens) return;
  if (per_wave == 1) rank_tokens<1>(s, lds, first);
  else if (per_wave == 2) rank_tokens<2>(s, lds, first);
  else rank_tokens<4>(s, lds, first);
}

union SortLds {
  SortSpace sort;
  unsigned char taken[kFillRows];
};

template <class S, int EPL, bool STREAM>
__global__ __launch_bounds__(kSortThreads) void k_embed_count(Bwd<typename S::elem> a, Sort s, Fill f) {
  __shared__ SortLds lds;
  if (blockIdx.x >= unsigned(s.stretches)) return fill_rows<S, EPL, STREAM>(a, s, f, blockIdx.x - s.stretches, lds.taken);
  unsigned *h = lds.sort.next;
  for (int d = threadIdx.x; d < s.bins; d += kSortThreads) h[d] = 0;
  __syncthreads();
  const unsigned from = blockIdx.x * s.per_stretch, left = s.tokens - from;
  count_digits(s, from, from + (left < s.per_stretch ? left : s.per_stretch), h);
  __syncthreads();
  for (int d = threadIdx.x; d < s.bins; d += kSortThreads) s.counts[blockIdx.x * s.bins + d] = h[d];
}

template <class S, int EPL, bool STREAM>
__global__ __launch_bounds__(kSortThreads) void k_embed_move(Bwd<typename S::elem> a, Sort s, Fill f) {
  __shared__ SortLds lds;
  if (blockIdx.x >= unsigned(s.stretches)) return fill_rows<S, EPL, STREAM>(a, s, f, blockIdx.x - s.stretches, lds.taken);
  SortSpace &sp = lds.sort;
  const int tid = threadIdx.x;
  const unsigned from = blockIdx.x * s.per_stretch, left = s.tokens - from;
  const size_t to = size_t(from) + (left < s.per_stretch ? left : s.per_stretch);
  const unsigned lane = tid & (SGH_WAVE - 1), wave = tid >> 6, per_wave = SGH_WAVE * kItems;
  Held<kItems> h;
  auto ask = [&](size_t base) {
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
      const size_t i = base + wave * per_wave + u * SGH_WAVE + lane;
      Token t = {0, kNoPlace};
      if (i < to) t = s.ids ? Token{unsigned(s.ids[i]), unsigned(i)} : s.in[i];
      h.key[u] = t.key, h.place[u] = t.place;
    }
  };
  ask(from);
  // all tokens of a digit, and those of the stretches in front, by the threads that share it
  const int digit = tid & (s.bins - 1), share = tid / s.bins, shares = kSortThreads / s.bins;
  unsigned all = 0, before = 0;
#pragma unroll 8
  for (int b = share; b < s.stretches; b += shares) {
    const unsigned c = s.counts[b * s.bins + digit];
    all += c;
    before += b < int(blockIdx.x) ? c : 0;
  }
  unsigned *of_thread = reinterpret_cast<unsigned *>(&sp.in_wave[0][0]);   // two values of every thread
  of_thread[tid] = all;
  of_thread[kSortThreads + tid] = before;
  __syncthreads();
  if (tid < s.bins)
    for (int o = 1; o < shares; ++o) all += of_thread[o * s.bins + tid], before += of_thread[kSortThreads + o * s.bins + tid];
  before += lower_digits(sp, tid < s.bins ? all : 0);
  __syncthreads();
  if (tid < s.bins) sp.next[tid] = before;
  for (size_t base = from; base < to; base += kStretch) {
    clear_counts(sp);
    if (s.ids) {
#pragma unroll
      for (int u = 0; u < kItems; ++u) {
        h.key[u] = counted_key(s, int(h.key[u]), h.place[u] != kNoPlace);
        if (f.taken && h.place[u] != kNoPlace && h.key[u] < s.vocab) f.taken[h.key[u]] = 1;
      }
    }
    __syncthreads();
    sort_rank(s, per_wave, sp, h);
    __syncthreads();
    const unsigned total = tid < s.bins ? front_counts(sp) : 0;
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kItems; ++u)
      if (h.place[u] != kNoPlace) s.out[place_of(s, sp, h.key[u], h.rank[u])] = Token{h.key[u], h.place[u]};
    ask(base + kStretch);
    __syncthreads();
    if (tid < s.bins) sp.next[tid] += total;
  }
}

// Where a wavefront's lanes are: a tile of its own for every `lanes` of them, and a vector of the rows
__host__ __device__ inline unsigned slices_at_once(int slices) { return slices < kWaves ? slices : kWaves; }   // of a workgroup
__host__ __device__ inline unsigned tiles_at_once(int lanes, int slices) { return kWaves / slices_at_once(slices) * (SGH_WAVE / lanes); }
struct Spot {
  unsigned tile;   // of the workgroup's
  size_t vec;
};
template <class T>
__device__ __forceinline__ Spot spot_of(const Bwd<T> &a) {
  const unsigned lane = threadIdx.x & (SGH_WAVE - 1), wave = threadIdx.x >> 6, each = slices_at_once(a.slices);
  return {wave / each * (SGH_WAVE / a.lanes) + lane / a.lanes,
          (size_t(blockIdx.y) * each + wave % each) * SGH_WAVE + (lane & (a.lanes - 1))};
}

// A workgroup has `a.stretch` neighbours of the sorted list (whole tiles).  Its threads first work out the jobs that begin there, each a sum
// of neighbouring tokens that becomes a row of the result or is kept for joining: the tokens of a row that hold no whole tile (they may end
// in the next one), or a row's piece of a tile.  Then the wavefronts take the jobs in turn, `lanes` lanes and a vector of each to a job.
// (One wavefront that goes through a tile's tokens with loads of several jobs in flight needs its store once for each of them: the code no
// longer fits the instruction cache, 6 -> 13 us at 2048 tokens of 64.)  Bound by dy: 65536 tokens of 2048 bfloat16 elements 91 us, 319 MB read and
// 84 written; few tokens by five loads one behind the other, 6 to 8 us.
template <class S, int EPL, bool STREAM, bool STREAM_DY>
__global__ __launch_bounds__(kBlock) void k_embed_tiles(Bwd<typename S::elem> a) {
  extern __shared__ unsigned lds[];   // one key in front, the stretch, two tiles behind it; their places; the jobs
  __shared__ unsigned jobs;
  const unsigned room = a.stretch + 2 * a.tile;
  unsigned *keys = lds + 1, *places = keys + room, *from_ = places + room, *to_ = from_ + a.stretch, *dest_ = to_ + a.stretch;
  const size_t base = size_t(blockIdx.x) * a.stretch;
  const unsigned count = a.tokens - base < room ? unsigned(a.tokens - base) : room;   // known keys
  const unsigned mine = count < a.stretch ? count : a.stretch;
  if (threadIdx.x == 0) {
    lds[0] = base ? a.sorted[base - 1].key : kNoKey;
    jobs = 0;
  }
  for (unsigned i = threadIdx.x; i < room; i += kBlock) {
    const Token t = i < count ? a.sorted[base + i] : Token{kNoKey, 0};
    keys[i] = t.key, places[i] = t.place;
  }
  const unsigned ahead = base >= a.tile ? a.sorted[base - a.tile].key : kNoKey;   // the first key of the tile in front
  __syncthreads();
  constexpr unsigned kRow = 0x80000000u;   // a job's destination: a row of the result (else one of the kept sums)
  for (unsigned i = threadIdx.x; i < mine; i += kBlock) {
    const unsigned k = keys[i], first = i & ~(a.tile - 1), tile = unsigned(base / a.tile) + first / a.tile;
    if (i == first + a.tile - 1 || i + 1 == mine) {   // the tile's last row: does it begin here, hold a whole tile and go on?
      const bool whole = i == first + a.tile - 1 && keys[first] == k;
      const bool joined = keys[int(first) - 1] != k && k < a.vocab && i == first + a.tile - 1 &&
                          (whole ? keys[i + 1] == k : keys[i + a.tile] == k);
      if (blockIdx.y == 0) a.tail[tile] = joined ? 2 * tile + (whole ? 0 : 1) : kNoKey;
    }
    if (k >= a.vocab) continue;
    const bool begins = keys[int(i) - 1] != k;
    if (!begins && i != first) continue;
    const unsigned next = begins ? (i + a.tile - 1) & ~(a.tile - 1) : i;   // where a whole tile could begin
    const bool whole = keys[next + a.tile - 1] == k;
    unsigned to, dest;
    if (whole && next != i) {   // up to the first whole tile
      to = next, dest = 2 * tile + 1;
    } else {
      if (whole) {
        to = i + a.tile;
      } else {
        unsigned lo = i + 1, hi = next + a.tile - 1;   // the first token behind: keys[hi] is one
        while (lo < hi) {
          const unsigned mid = (lo + hi) / 2;
          if (keys[mid] == k) lo = mid + 1;
          else hi = mid;
        }
        to = lo;
      }
      if (begins && !(whole && keys[to] == k)) {
        dest = kRow;
      } else {
        if (!whole && (first ? keys[first - a.tile] : ahead) != k) continue;   // taken by the tile in front
        dest = 2 * tile;
      }
    }
    const unsigned slot = atomicAdd(&jobs, 1u);
    from_[slot] = i, to_[slot] = to, dest_[slot] = dest;
  }
  __syncthreads();
  const unsigned lane = threadIdx.x & (SGH_WAVE - 1), n = jobs, per_wave = SGH_WAVE / a.lanes;
  const size_t vec = size_t(blockIdx.y) * SGH_WAVE + (lane & (a.lanes - 1));
  if (vec * EPL >= a.dim) return;
  const size_t at = vec * EPL + EPL > a.dim ? a.dim - EPL : vec * EPL;
  for (unsigned j = (threadIdx.x >> 6) * per_wave + lane / a.lanes; j < n; j += kWaves * per_wave) {
    const unsigned from = from_[j], dest = dest_[j];
    float acc[EPL], g[EPL];
#pragma unroll
    for (int e = 0; e < EPL; ++e) acc[e] = 0.f;
    if (dest == kRow) load_add<S, EPL>(a, keys[from], at, g);
    add_tokens<S, EPL, STREAM_DY>(a.dy, a.dim, at, places, from, to_[j], acc);
    if (dest == kRow) {
      store_row<S, EPL, STREAM>(a, keys[from], at, vec, acc, g);
    } else {
      float *out = a.partial + size_t(dest) * a.pitch + at;
#pragma unroll
      for (int e = 0; e < EPL; ++e) out[e] = acc[e];
    }
  }
}

// Rows whose tokens hold whole tiles, from the tile in which they begin: the sum of their tokens there, of the whole tiles, and of the tokens
// behind.  Bound by the commonest row's chain of sums, 16 loads in flight: 10.6 us for 65536 tokens of 2048, 1.4 to 4.5 for fewer.
template <class S, int EPL, bool STREAM>
__global__ __launch_bounds__(kBlock) void k_embed_join(Bwd<typename S::elem> a) {
  const unsigned tiles = tiles_at_once(a.lanes, a.slices);
  const Spot sp = spot_of(a);
  const size_t index = size_t(blockIdx.x) * tiles + sp.tile;
  if (sp.tile >= tiles || index * a.tile >= a.tokens) return;
  const unsigned from = a.tail[index];
  if (from == kNoKey) return;
  const unsigned lane = threadIdx.x & (SGH_WAVE - 1), of_tile = lane & (a.lanes - 1);
  const size_t at = sp.vec * EPL + EPL > a.dim ? a.dim - EPL : sp.vec * EPL;
  const unsigned row = a.sorted[(index + 1) * a.tile - 1].key;
  // tiles behind this one that begin with a token of the row: a lane asks for one
  size_t more = 0;
  for (;;) {
    const size_t begin = (index + 1 + more + of_tile) * a.tile;
    const unsigned long long is = __ballot(begin < a.tokens && a.sorted[begin].key == row) >> (lane - of_tile);
    const unsigned n = ~is ? unsigned(__builtin_ctzll(~is)) : SGH_WAVE;
    more += n < unsigned(a.lanes) ? n : a.lanes;
    if (n < unsigned(a.lanes)) break;
  }
  if (sp.vec * EPL >= a.dim) return;
  float acc[EPL];
#pragma unroll
  for (int j = 0; j < EPL; ++j) acc[j] = 0.f;
  float g[EPL];
  load_add<S, EPL>(a, row, at, g);
  const float *p = a.partial + size_t(from) * a.pitch + at;
#pragma unroll
  for (int j = 0; j < EPL; ++j) acc[j] += p[j];
  p = a.partial + (index + 1) * 2 * a.pitch + at;
  constexpr int U = EPL == 8 ? 8 : 16;
  for (size_t t = 0; t < more; t += U, p += U * 2 * a.pitch) {
    float v[U][EPL];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (t + u < more) {
#pragma unroll
        for (int j = 0; j < EPL; ++j) v[u][j] = p[u * 2 * a.pitch + j];
      }
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (t + u < more) {
#pragma unroll
        for (int j = 0; j < EPL; ++j) acc[j] += v[u][j];
      }
  }
  store_row<S, EPL, STREAM>(a, row, at, sp.vec, acc, g);
}

struct BwdPlan {
  bool scan, rank;
  unsigned tile, tiles;
  int passes, digit_bits, stretches;
  unsigned per_stretch;
  size_t other, counts, tail, taken, partial, bytes;   // offsets into the workspace
};
size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

BwdPlan bwd_plan(size_t tokens, size_t vocab, size_t dim) {
  BwdPlan p = {};
  p.scan = tokens <= kScanTokens;
  if (p.scan) return p;
  p.rank = tokens <= kRankTokens;
  p.tile = tokens <= 16384 ? 16 : 32;   // few, so that neither a tile nor the tiles of one row are a long sum
  p.tiles = unsigned((tokens + p.tile - 1) / p.tile);
  int bits = 1;
  while ((vocab >> bits) != 0) ++bits;   // (the largest key is `vocab`)
  p.passes = (bits + kDigitBits - 1) / kDigitBits;
  p.digit_bits = (bits + p.passes - 1) / p.passes;
  const size_t stretches = (tokens + kStretch - 1) / kStretch;
  const size_t each = (stretches + kMostStretches - 1) / kMostStretches;
  p.per_stretch = unsigned(each * kStretch);
  p.stretches = int((stretches + each - 1) / each);
  const size_t list = up256(tokens * sizeof(Token));
  p.other = list;
  p.counts = p.rank ? list : 2 * list;
  p.tail = p.counts + (p.rank ? 0 : up256(size_t(p.stretches) * kBins * 4));
  p.taken = p.tail + up256(size_t(p.tiles) * 4);
  p.partial = p.taken + (p.rank || p.passes == 1 ? 0 : up256(vocab));
  p.bytes = p.partial + 2 * size_t(p.tiles) * up256(dim * 4);
  return p;
}

template <class S, int EPL, bool STREAM>
int launch_scan(const Bwd<typename S::elem> &a, hipStream_t s) {
  // about 32 KB of the result for a workgroup, the whole chip busy where the table is large enough
  const size_t per_wave = SGH_WAVE / a.lanes, cus = size_t(sgh_num_cus());
  size_t rows = (size_t(32) << 10) / (a.dim * sizeof(typename S::elem));
  const size_t spread = a.vocab / (cus * 8);
  if (rows > spread) rows = spread;
  if (rows < per_wave) rows = per_wave;
  while ((a.vocab + rows - 1) / rows > (1u << 23)) rows *= 2;
  if (rows > size_t(kMostRows)) rows = kMostRows;   // (2^31 rows at the most: 2^23 workgroups)
  const size_t blocks = (a.vocab + rows - 1) / rows;
  const size_t units = (rows + per_wave - 1) / per_wave * size_t(a.slices);
  size_t ny = blocks >= cus * 4 ? 1 : (cus * 4 + blocks - 1) / blocks;
  if (ny > (units + kWaves - 1) / kWaves) ny = (units + kWaves - 1) / kWaves;
  hipLaunchKernelGGL((k_embed_rows<S, EPL, STREAM>), dim3(unsigned(blocks), unsigned(ny)), dim3(kBlock), 0, s, a, int(rows));
  SGH_LAUNCH_CHECK();
  return SGH_OK;
}

template <class S, int EPL, bool STREAM>
int launch_bwd(Bwd<typename S::elem> a, const BwdPlan &p, void *workspace, hipStream_t s) {
  if (p.scan) return launch_scan<S, EPL, STREAM>(a, s);
  char *ws = static_cast<char *>(workspace);
  auto at = [&](size_t off) { return reinterpret_cast<unsigned *>(ws + off); };
  Token *sorted = reinterpret_cast<Token *>(ws), *other = reinterpret_cast<Token *>(ws + p.other);
  a.sorted = sorted, a.tail = at(p.tail);
  a.partial = reinterpret_cast<float *>(ws + p.partial);
  a.tile = p.tile, a.pitch = up256(a.dim * 4) / 4;
  // The rows without a token, spread over the launches that sort and know them: at least 64 KB of the result for a workgroup and launch.
  // (Leaving a part for the launch of the tiles, whose own traffic they would run beside, was slower: 44.8 -> 48.9 and 337 -> 400 us for 8192
  // tokens of 1024 fp32 elements and 65536 of 2048 bfloat16.  Looking through the ids takes a workgroup 15 us for 131072 tokens; so the
  // rows of more than kRankTokens are marked on the way: 82 -> 68 us for 131072 tokens, 32000 rows of 512 bfloat16.)
  const bool marked = !p.rank && p.passes > 1;
  Fill f = {0, 0, marked ? 2 * p.passes - 2 : 1, p.rank ? Taken::kIds : marked ? Taken::kClear : Taken::kCounts, nullptr};
  Sort so = {};
  so.ids = a.ids, so.counts = at(p.counts), so.tokens = a.tokens, so.vocab = unsigned(a.vocab), so.pad = a.pad;
  so.bins = 1 << p.digit_bits, so.stretches = p.stretches, so.per_stretch = p.per_stretch;
  const size_t cus = size_t(sgh_num_cus());
  // Tokens that a wavefront ranks: one, or two where that leaves a workgroup for every CU; beside a table that takes longer to fill, four, for more
  // room there (8192 tokens, 50000 rows of 1024 bfloat16: 34.5 -> 29.7 us; of 41 MB: 34.9 -> 36.6)
  const size_t table = a.vocab * a.dim * sizeof(typename S::elem);
  const int per_wave = a.add != a.dW && table >= size_t(64) << 20 ? 4 : a.tokens > cus * kSortWaves ? 2 : 1;
  if (p.rank) so.stretches = int((a.tokens + kSortWaves * per_wave - 1) / (kSortWaves * per_wave));
  unsigned fill_blocks = 0;
  if (a.add != a.dW) {
    size_t want = (table >> 16) / f.launches;
    const size_t most = 2 * cus - (p.rank ? size_t(so.stretches) : 0);   // (two workgroups fit a CU)
    if (want > most) want = most;
    if (want < 1) want = 1;
    size_t rows = (a.vocab + want - 1) / want;
    if (rows > kFillRows) rows = kFillRows;
    f.rows = unsigned(rows);
    fill_blocks = unsigned((a.vocab + rows - 1) / rows);
    if (marked) f.taken = reinterpret_cast<unsigned char *>(ws + p.taken);
  }
  if (p.rank) {
    so.out = sorted;
    hipLaunchKernelGGL((k_embed_rank<S, EPL, STREAM>), dim3(so.stretches + fill_blocks), dim3(kSortThreads), 0, s, a, so, per_wave, f);
    SGH_LAUNCH_CHECK();
  } else {
    for (int pass = 0; pass < p.passes; ++pass) {
      so.out = (p.passes - 1 - pass) & 1 ? other : sorted;
      so.shift = pass * p.digit_bits;
      // the first count clears the marks, the first move sets them, or stores the rows if it is the last
      const unsigned beside_count = pass != 0 || marked ? fill_blocks : 0, beside_move = pass != 0 || !marked ? fill_blocks : 0;
      hipLaunchKernelGGL((k_embed_count<S, EPL, STREAM>), dim3(p.stretches + beside_count), dim3(kSortThreads), 0, s, a, so, f);
      SGH_LAUNCH_CHECK();
      if (pass != 0) ++f.launch;
      hipLaunchKernelGGL((k_embed_move<S, EPL, STREAM>), dim3(p.stretches + beside_move), dim3(kSortThreads), 0, s, a, so, f);
      SGH_LAUNCH_CHECK();
      if (pass != 0) ++f.launch;
      if (marked) f.from = Taken::kMarks;
      so.ids = nullptr, so.in = so.out;
    }
  }
  Bwd<typename S::elem> t = a;
  if (t.lanes < 8) t.lanes = 8;   // (LDS holds the tokens of a workgroup)
  // Jobs a wavefront takes one after the other, more where the workgroups' own start counts (bf16, 65536 tokens of 2048: 351 us with 4, 337 with 8;
  // f32, 8192 of 1024: 44.8 and 48.3), one while that leaves CUs without work (bf16, 1025 tokens of 64: 16.3 -> 14.3)
  const unsigned takers = kWaves * (SGH_WAVE / t.lanes);
  const size_t at_once = size_t(a.tokens) / takers * a.slices;   // workgroups of one job for each taker
  t.stretch = takers * (at_once > cus * 128 ? 8 : at_once > cus * 2 ? 4 : 1);
  if (t.stretch < t.tile) t.stretch = t.tile;
  const unsigned lds = (2 * (t.stretch + 2 * t.tile) + 3 * t.stretch + 1) * 4, blocks = (t.tokens + t.stretch - 1) / t.stretch;
  // (dy past the caches: 65536 tokens of 2048 16-bit elements 321 -> 308 us; 33 MB of it, 39.6 -> 41.3)
  const dim3 stretches{blocks, unsigned(a.slices)};
  if (EPL != 1 && size_t(a.tokens) * a.dim * sizeof(typename S::elem) >= kStreamBytes)
    hipLaunchKernelGGL((k_embed_tiles<S, EPL, STREAM, EPL != 1>), stretches, dim3(kBlock), lds, s, t);
  else
    hipLaunchKernelGGL((k_embed_tiles<S, EPL, STREAM, false>), stretches, dim3(kBlock), lds, s, t);
  SGH_LAUNCH_CHECK();
  const unsigned tiles = tiles_at_once(t.lanes, t.slices), each = slices_at_once(t.slices);
  const dim3 grid{(p.tiles + tiles - 1) / tiles, (t.slices + each - 1) / each};
  hipLaunchKernelGGL((k_embed_join<S, EPL, STREAM>), grid, dim3(kBlock), 0, s, t);
  SGH_LAUNCH_CHECK();
  return SGH_OK;
}

template <class S>
int embed_bwd(const int32_t *ids, const typename S::elem *dy, const typename S::elem *add, typename S::elem *dW, size_t tokens,
              size_t vocab, size_t dim, float scale, int pad, void *workspace, size_t ws_bytes, void *stream) {
  if (!sizes_ok(tokens, vocab, dim)) return SGH_EINVAL;
  if (vocab == 0 || dim == 0) return SGH_OK;
  constexpr size_t e = sizeof(typename S::elem);
  const size_t bytes = vocab * dim * e;
  if ((tokens != 0 && (!ids || !dy)) || !dW) return SGH_EINVAL;
  if (sgh_ranges_meet(dW, bytes, dy, tokens * dim * e) || sgh_ranges_meet(dW, bytes, ids, tokens * 4)) return SGH_EINVAL;
  if (add && add != dW && sgh_ranges_meet(dW, bytes, add, bytes)) return SGH_EINVAL;
  const BwdPlan p = bwd_plan(tokens, vocab, dim);
  if (p.bytes != 0 && (!workspace || ws_bytes < p.bytes)) return SGH_EWORKSPACE;
  if (reinterpret_cast<uintptr_t>(workspace) % alignof(Token) != 0) return SGH_EINVAL;
  hipStream_t s = sgh_stream_of(stream);
  sgh_note_write(dW, bytes);
  sgh_prof_scope prof("embedding_bwd", double(tokens) * (4 + double(dim) * e) + double(bytes) * (add ? 2 : 1), s);
  const RowLanes r = row_lanes(dim, S::VEC);
  Bwd<typename S::elem> a = {};
  a.dy = dy, a.add = add, a.dW = dW, a.ids = ids, a.dim = dim, a.vocab = vocab, a.tokens = unsigned(tokens), a.tile = 1;
  a.scale = scale, a.pad = pad, a.lanes = r.lanes, a.slices = r.slices;
  if (r.epl == 1) return launch_bwd<S, 1, false>(a, p, workspace, s);
  // The result past the caches where it would push much dy out of the last of them, or is larger than that and of whole lines: those that are stored in
  // two parts cost more there.  (131 MB, with 33 MB of dy: 36.9 us past, 42.2 through, with 8: 33.8 and 30.7; 262 and 8: 77.5 and 68.7; 410 and
  // 80: 115 and 130; 525 and 2, rows of 4002 bytes: 136 and 115.)
  const bool past = bytes >= kStreamBytes && (tokens * dim * e * 12 > bytes || (bytes >= 3 * kStreamBytes && dim * e % 128 == 0));
  return past ? launch_bwd<S, S::VEC, true>(a, p, workspace, s) : launch_bwd<S, S::VEC, false>(a, p, workspace, s);
}

}  // namespace

extern "C" {

#define SGH_EMBEDDING(SFX, S, T)                                                                                                  \
  int sgh_embedding_fwd_##SFX(const int32_t *ids, const T *W, T *y, size_t tokens, size_t vocab, size_t dim, float scale,         \
                              int padding_idx, void *stream) {                                                                    \
    return embed_fwd<S>(ids, W, y, tokens, vocab, dim, scale, padding_idx, stream);                                               \
  }                                                                                                                               \
  int sgh_embedding_bwd_##SFX(const int32_t *ids, const T *dy, const T *add, T *dW, size_t tokens, size_t vocab, size_t dim,      \
                              float scale, int padding_idx, void *workspace, size_t ws_bytes, void *stream) {                     \
    return embed_bwd<S>(ids, dy, add, dW, tokens, vocab, dim, scale, padding_idx, workspace, ws_bytes, stream);                   \
  }
SGH_EMBEDDING(f32, StF32, float)
SGH_EMBEDDING(f16, StF16, uint16_t)
SGH_EMBEDDING(bf16, StBF16, uint16_t)
#undef SGH_EMBEDDING

size_t sgh_embedding_bwd_workspace_bytes(size_t tokens, size_t vocab, size_t dim) {
  return sizes_ok(tokens, vocab, dim) && vocab != 0 && dim != 0 ? bwd_plan(tokens, vocab, dim).bytes : 0;
}

int sgh_embedding_index_errors(void *stream, int *count) {
  if (!count) return SGH_EINVAL;
  void *counter;
  SGH_HIP_TRY(hipGetSymbolAddress(&counter, HIP_SYMBOL(g_index_errors)));
  return sgh_take_count(static_cast<int *>(counter), sgh_stream_of(stream), count);
}

}  // extern "C"
