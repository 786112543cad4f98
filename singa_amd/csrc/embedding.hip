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
template <class S>
RowLanes row_lanes(size_t dim) {
  RowLanes r;
  r.epl = dim < size_t(S::VEC) ? 1 : S::VEC;
  const size_t vecs = (dim + r.epl - 1) / r.epl;
  r.lanes = 1;
  while (r.lanes < SGH_WAVE && size_t(r.lanes) < vecs) r.lanes *= 2;
  r.slices = int((vecs + SGH_WAVE - 1) / SGH_WAVE);
  return r;
}

// ------------------------------------------------------------------------------------ forward

// A wavefront takes 64 / lanes tokens and PER slices of their rows, all loads in flight before the first store.
template <class S, int EPL, int PER>
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
      if (first + size_t(p) * SGH_WAVE < vecs) sgh_store_any<S, EPL>(y + t * dim + at[p], v[p]);
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
  SGH_LAUNCH_TIMED((k_embed_fwd<S, EPL, PER>), dim3(unsigned(blocks), unsigned(ny)), dim3(kBlock), 0, s, ids, W, y, tokens, vocab,
                   dim, scale, pad, r.lanes);
  SGH_LAUNCH_CHECK();
  return SGH_OK;
}

constexpr size_t kMostDim = size_t(1) << 24;   // (the slices of a row are a grid's second dimension: at most 65535)

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
  const RowLanes r = row_lanes<S>(dim);
  if (r.epl == 1) return launch_fwd<S, 1, 1>(ids, W, y, tokens, vocab, dim, scale, pad, r, s);
  return launch_fwd<S, S::VEC, 4>(ids, W, y, tokens, vocab, dim, scale, pad, r, s);
}

// ------------------------------------------------------------------------------------ the order of the tokens

// Stable sort of (id, place) by id: passes of at most 9 bits from the lowest.  A pass counts the digits of each workgroup's stretch of
// tokens, turns the counts into the place of every stretch's first token with a digit, and moves the tokens there.
constexpr int kDigitBits = 9, kBins = 1 << kDigitBits;
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / SGH_WAVE;
constexpr int kItems = 4;                              // tokens of a thread at a time
constexpr int kStretch = kSortThreads * kItems;
constexpr int kMostStretches = 64;                     // workgroups of a pass: each reads all their counts

// LDS as the wavefront's lanes left it, before and after
__device__ __forceinline__ void wave_sync() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

__device__ __forceinline__ unsigned key_of(int id, unsigned vocab, int pad) {
  return id < 0 || unsigned(id) >= vocab || id == pad ? vocab : unsigned(id);
}

__global__ __launch_bounds__(kSortThreads) void k_embed_count(const int32_t *__restrict__ ids, const unsigned *__restrict__ keys,
                                                              unsigned tokens, unsigned vocab, int pad, int shift, int bins,
                                                              unsigned per_block, unsigned *__restrict__ counts) {
  __shared__ unsigned h[kBins];
  for (int d = threadIdx.x; d < bins; d += kSortThreads) h[d] = 0;
  __syncthreads();
  const size_t from = size_t(blockIdx.x) * per_block, to = from + per_block < tokens ? from + per_block : tokens;
  for (size_t i = from + threadIdx.x; i < to; i += kSortThreads) {
    unsigned k;
    if (ids) {
      const int id = ids[i];
      k = key_of(id, vocab, pad);
      if (k == vocab && id != pad) atomicAdd(&g_index_errors, 1);
    } else {
      k = keys[i];
    }
    atomicAdd(&h[(k >> shift) & (bins - 1)], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < bins; d += kSortThreads) counts[size_t(blockIdx.x) * bins + d] = h[d];
}

__global__ __launch_bounds__(kSortThreads) void k_embed_move(const int32_t *__restrict__ ids, const unsigned *__restrict__ keys,
                                                             const unsigned *__restrict__ places, unsigned tokens, unsigned vocab,
                                                             int pad, int shift, int bins, unsigned per_block,
                                                             const unsigned *__restrict__ counts, unsigned *__restrict__ keys_out,
                                                             unsigned *__restrict__ places_out) {
  __shared__ unsigned next[kBins];               // where the next token with a digit goes
  __shared__ unsigned in_wave[kSortWaves][kBins];
  __shared__ unsigned sums[kSortWaves];
  const int tid = threadIdx.x, lane = tid & (SGH_WAVE - 1), wave = tid >> 6;
  // all tokens with a lower digit, then this digit's of the stretches in front
  {
    unsigned all = 0, before = 0;
    if (tid < bins)
      for (unsigned b = 0; b < gridDim.x; ++b) {
        const unsigned c = counts[size_t(b) * bins + tid];
        all += c;
        if (b < blockIdx.x) before += c;
      }
    unsigned upto = all;
#pragma unroll
    for (int o = 1; o < SGH_WAVE; o <<= 1) {
      const unsigned u = __shfl_up(upto, o, SGH_WAVE);
      if (lane >= o) upto += u;
    }
    if (lane == SGH_WAVE - 1) sums[wave] = upto;
    __syncthreads();
    unsigned lower = 0;
    for (int w = 0; w < wave; ++w) lower += sums[w];
    if (tid < bins) next[tid] = lower + upto - all + before;
  }
  const size_t from = size_t(blockIdx.x) * per_block, to = from + per_block < tokens ? from + per_block : tokens;
  for (size_t base = from; base < to; base += kStretch) {
    for (int i = tid; i < kSortWaves * bins; i += kSortThreads) in_wave[i / bins][i % bins] = 0;
    __syncthreads();
    unsigned key[kItems], place[kItems], rank[kItems];
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
      const size_t i = base + size_t(wave) * (SGH_WAVE * kItems) + u * SGH_WAVE + lane;
      const bool there = i < to;
      key[u] = there ? (ids ? key_of(ids[i], vocab, pad) : keys[i]) : 0;
      place[u] = there ? (ids ? unsigned(i) : places[i]) : 0xffffffffu;
    }
#pragma unroll
    for (int u = 0; u < kItems; ++u) {
      const bool there = place[u] != 0xffffffffu;
      const unsigned digit = (key[u] >> shift) & (bins - 1);
      unsigned long long same = __ballot(there);   // lanes with this digit
#pragma unroll
      for (int b = 0; b < kDigitBits; ++b) {
        const bool bit = (digit >> b) & 1;
        const unsigned long long set = __ballot(bit);
        same &= bit ? set : ~set;
      }
      const int ahead = __popcll(same & ((1ull << lane) - 1));
      const unsigned old = in_wave[wave][digit];
      rank[u] = old + ahead;
      wave_sync();   // (every lane has read the count before one of them writes it)
      if (there && ahead == 0) in_wave[wave][digit] = old + __popcll(same);
      wave_sync();
    }
    __syncthreads();
    if (tid < bins) {
      unsigned at = next[tid];
      for (int w = 0; w < kSortWaves; ++w) {
        const unsigned c = in_wave[w][tid];
        in_wave[w][tid] = at;
        at += c;
      }
      next[tid] = at;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kItems; ++u)
      if (place[u] != 0xffffffffu) {
        const unsigned to_ = in_wave[wave][(key[u] >> shift) & (bins - 1)] + rank[u];
        keys_out[to_] = key[u];
        places_out[to_] = place[u];
      }
    __syncthreads();
  }
}

// ------------------------------------------------------------------------------------ the gradient

// Rows of the gradient that take part in a call, and where their tokens are found
template <class T>
struct Rows {
  const T *dy, *add;
  T *dW;
  const unsigned *keys, *places;   // sorted
  const int32_t *ids;              // few tokens: as they came
  float *partial;                  // sums of whole tiles of one row, [tiles][dim]
  size_t dim, vocab;
  unsigned tokens, tile;           // tokens of a tile, a power of two
  float scale;
  int pad, lanes, slices, rows;    // rows: of a workgroup
};

// Sum of rows place[from .. to) of dy, ascending, on top of acc
template <class S, int EPL>
__device__ __forceinline__ void add_tokens(const typename S::elem *dy, size_t dim, size_t at, const unsigned *place, unsigned from,
                                           unsigned to, float *acc) {
  constexpr int U = 8;
  unsigned i = from;
  for (; i + U <= to; i += U) {
    float v[U][EPL];
#pragma unroll
    for (int u = 0; u < U; ++u) sgh_load_any<S, EPL>(dy + size_t(place[i + u]) * dim + at, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int j = 0; j < EPL; ++j) acc[j] += v[u][j];
  }
  for (; i < to; ++i) {
    float v[EPL];
    sgh_load_any<S, EPL>(dy + size_t(place[i]) * dim + at, v);
#pragma unroll
    for (int j = 0; j < EPL; ++j) acc[j] += v[j];
  }
}

// Tiles of `tile` sorted tokens that are all of one row: their sums, so that a row with many tokens is not one wavefront's work
template <class S, int EPL>
__global__ __launch_bounds__(kBlock) void k_embed_tiles(Rows<typename S::elem> a) {
  const unsigned first = blockIdx.x * a.tile, last = first + a.tile - 1;   // (only whole tiles are launched)
  const unsigned key = a.keys[first];
  if (key >= a.vocab || a.keys[last] != key) return;
  const int lane = threadIdx.x & (SGH_WAVE - 1);
  const size_t vecs = (a.dim + EPL - 1) / EPL;
  for (size_t sl = blockIdx.y * kWaves + (threadIdx.x >> 6); sl < size_t(a.slices); sl += gridDim.y * kWaves) {
    const size_t vec = sl * SGH_WAVE + lane;
    if (vec >= vecs) continue;
    const size_t at = vec * EPL + EPL > a.dim ? a.dim - EPL : vec * EPL;
    float acc[EPL];
#pragma unroll
    for (int j = 0; j < EPL; ++j) acc[j] = 0.f;
    add_tokens<S, EPL>(a.dy, a.dim, at, a.places, first, last + 1, acc);
    float *out = a.partial + size_t(blockIdx.x) * a.dim + at;
#pragma unroll
    for (int j = 0; j < EPL; ++j) out[j] = acc[j];
  }
}

// First of the sorted keys that is not below x, by a wavefront: 64 probes a step
__device__ __forceinline__ unsigned lower_bound(const unsigned *keys, unsigned n, unsigned x) {
  unsigned lo = 0, hi = n;
  const unsigned lane = threadIdx.x & (SGH_WAVE - 1);
  while (lo < hi) {
    const unsigned step = (hi - lo + SGH_WAVE - 1) / SGH_WAVE;
    const size_t probe = size_t(lo) + size_t(lane + 1) * step - 1;   // the last of each of 64 stretches
    const bool below = probe < hi && keys[probe] < x;
    const unsigned whole = unsigned(__popcll(__ballot(below)));
    const size_t start = size_t(lo) + size_t(whole) * step, stop = start + step - 1;
    lo = start < hi ? unsigned(start) : hi;
    hi = stop < hi ? unsigned(stop) : hi;
  }
  return lo;
}

constexpr int kMostRows = 256;        // of a workgroup
constexpr unsigned kScanTokens = 1024;   // up to here a workgroup looks through the ids itself

// Workgroup: a few consecutive rows of the gradient.  It finds their tokens -- in the sorted list, or (SCAN) among all ids -- and every
// wavefront sums and stores rows, or slices of them; rows without a token become zero, or `add`.
template <class S, int EPL, bool SCAN>
__global__ __launch_bounds__(kBlock) void k_embed_rows(Rows<typename S::elem> a) {
  typedef typename S::elem T;
  __shared__ unsigned begin[kMostRows], end[kMostRows];
  __shared__ unsigned found[SCAN ? kScanTokens : 2];   // SCAN: places of the rows' tokens, by row; else the bounds of the rows' tokens
  __shared__ unsigned listed[SCAN ? kScanTokens : 1];  // (row, place) in the order of the places
  __shared__ unsigned sums[kWaves];
  const int tid = threadIdx.x, lane = tid & (SGH_WAVE - 1), wave = tid >> 6;
  const size_t row0 = size_t(blockIdx.x) * a.rows;
  const int rows = a.vocab - row0 < size_t(a.rows) ? int(a.vocab - row0) : a.rows;
  for (int r = tid; r < rows; r += kBlock) begin[r] = end[r] = 0;
  if constexpr (SCAN) {
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
    unsigned upto = n;
#pragma unroll
    for (int o = 1; o < SGH_WAVE; o <<= 1) {
      const unsigned u = __shfl_up(upto, o, SGH_WAVE);
      if (lane >= o) upto += u;
    }
    if (lane == SGH_WAVE - 1) sums[wave] = upto;
    __syncthreads();
    unsigned at = upto - n, total = 0;
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) at += sums[w];
      total += sums[w];
    }
#pragma unroll
    for (int p = 0; p < P; ++p)
      if (mine[p] != 0xffffffffu) {
        listed[at++] = (mine[p] << 16) | unsigned(tid * P + p);
        atomicAdd(&end[mine[p]], 1u);
      }
    __syncthreads();
    if (wave == 0) {   // a stable counting sort by row: end[] holds the counts
      unsigned carry = 0;
      for (int r = lane; r - lane < rows; r += SGH_WAVE) {
        const unsigned c = r < rows ? end[r] : 0;
        unsigned up = c;
#pragma unroll
        for (int o = 1; o < SGH_WAVE; o <<= 1) {
          const unsigned u = __shfl_up(up, o, SGH_WAVE);
          if (lane >= o) up += u;
        }
        if (r < rows) begin[r] = end[r] = carry + up - c;
        carry += __shfl(up, SGH_WAVE - 1, SGH_WAVE);
      }
      wave_sync();
      for (unsigned i = lane; i - lane < total; i += SGH_WAVE) {
        const bool there = i < total;
        const unsigned e = there ? listed[i] : 0, r = e >> 16;
        unsigned long long same = __ballot(there);
#pragma unroll
        for (int b = 0; b < 8; ++b) {
          const bool bit = (r >> b) & 1;
          const unsigned long long set = __ballot(bit);
          same &= bit ? set : ~set;
        }
        const int ahead = __popcll(same & ((1ull << lane) - 1));
        const unsigned old = there ? end[r] : 0;
        wave_sync();
        if (there) found[old + ahead] = e & 0xffffu;
        if (there && ahead == 0) end[r] = old + __popcll(same);
        wave_sync();
      }
    }
    __syncthreads();
  } else {
    if (wave < 2) {
      const unsigned b = a.tokens ? lower_bound(a.keys, a.tokens, unsigned(row0 + (wave ? rows : 0))) : 0;
      if (lane == 0) found[wave] = b;
    }
    __syncthreads();
    const unsigned lo = found[0], hi = found[1];
    for (unsigned i = lo + tid; i < hi; i += kBlock) {
      const unsigned k = a.keys[i], r = unsigned(k - row0);
      if (i == lo || a.keys[i - 1] != k) begin[r] = i;
      if (i + 1 == hi || a.keys[i + 1] != k) end[r] = i + 1;
    }
    __syncthreads();
  }
  const unsigned *place = SCAN ? found : a.places;
  const size_t vecs = (a.dim + EPL - 1) / EPL;
  const int per_wave = SGH_WAVE / a.lanes, groups = (rows + per_wave - 1) / per_wave;
  for (size_t unit = size_t(blockIdx.y) * kWaves + wave; unit < size_t(groups) * a.slices; unit += size_t(gridDim.y) * kWaves) {
    const int group = a.slices == 1 ? int(unit) : int(unit / unsigned(a.slices));
    const size_t vec = (unit - size_t(group) * a.slices) * SGH_WAVE + (lane & (a.lanes - 1));
    const int r = group * per_wave + lane / a.lanes;
    if (r >= rows || vec >= vecs) continue;
    const bool moved = vec * EPL + EPL > a.dim;   // the row's last vector, moved back
    const size_t at = moved ? a.dim - EPL : vec * EPL;
    const unsigned b = begin[r], e = end[r];
    T *out = a.dW + (row0 + r) * a.dim + at;
    const T *add = a.add ? a.add + (row0 + r) * a.dim + at : nullptr;
    if (b == e && add == out) continue;
    float acc[EPL];
#pragma unroll
    for (int j = 0; j < EPL; ++j) acc[j] = 0.f;
    if (!SCAN && e - b >= a.tile) {
      const unsigned t0 = (b + a.tile - 1) / a.tile, t1 = e / a.tile;   // whole tiles of this row
      if (t0 < t1) {
        add_tokens<S, EPL>(a.dy, a.dim, at, place, b, t0 * a.tile, acc);
        for (unsigned t = t0; t < t1; ++t) {
          const float *p = a.partial + size_t(t) * a.dim + at;
#pragma unroll
          for (int j = 0; j < EPL; ++j) acc[j] += p[j];
        }
        add_tokens<S, EPL>(a.dy, a.dim, at, place, t1 * a.tile, e, acc);
      } else {
        add_tokens<S, EPL>(a.dy, a.dim, at, place, b, e, acc);
      }
    } else {
      add_tokens<S, EPL>(a.dy, a.dim, at, place, b, e, acc);
    }
#pragma unroll
    for (int j = 0; j < EPL; ++j) acc[j] *= a.scale;
    if (moved) {   // only what the vector before it leaves: `add` may be the result itself
#pragma unroll
      for (int j = 0; j < EPL; ++j)
        if (at + j >= vec * EPL) S::st(out + j, add ? S::ld(add + j) + acc[j] : acc[j]);
    } else {
      if (add) {
        float g[EPL];
        sgh_load_any<S, EPL>(add, g);
#pragma unroll
        for (int j = 0; j < EPL; ++j) acc[j] += g[j];
      }
      sgh_store_any<S, EPL>(out, acc);
    }
  }
}

struct BwdPlan {
  bool scan;
  unsigned tile, tiles;             // whole tiles
  int passes, digit_bits, stretches;
  unsigned per_stretch;
  size_t keys, places, keys2, places2, counts, partial, bytes;   // offsets into the workspace
};
size_t up256(size_t n) { return (n + 255) & ~size_t(255); }

BwdPlan bwd_plan(size_t tokens, size_t vocab, size_t dim) {
  BwdPlan p = {};
  p.scan = tokens <= kScanTokens;
  if (p.scan) return p;
  p.tile = 64;   // near the root of the tokens: neither the tokens of a tile nor the tiles of a row are a long sum
  while (size_t(p.tile) * p.tile * 16 < tokens) p.tile *= 2;
  p.tiles = unsigned(tokens / p.tile);
  int bits = 1;
  while ((vocab >> bits) != 0) ++bits;   // (the largest key is `vocab`)
  p.passes = (bits + kDigitBits - 1) / kDigitBits;
  p.digit_bits = (bits + p.passes - 1) / p.passes;
  const size_t stretches = (tokens + kStretch - 1) / kStretch;
  const size_t each = (stretches + kMostStretches - 1) / kMostStretches;
  p.per_stretch = unsigned(each * kStretch);
  p.stretches = int((stretches + each - 1) / each);
  const size_t list = up256(tokens * 4);
  p.places = list;
  p.keys2 = 2 * list;
  p.places2 = 3 * list;
  p.counts = 4 * list;
  p.partial = p.counts + up256(size_t(p.stretches) * kBins * 4);
  p.bytes = p.partial + up256(size_t(p.tiles) * dim * 4);
  return p;
}

template <class S, int EPL>
int launch_bwd(Rows<typename S::elem> a, const BwdPlan &p, void *workspace, hipStream_t s) {
  constexpr size_t e = sizeof(typename S::elem);
  if (!p.scan) {
    char *ws = static_cast<char *>(workspace);
    auto at = [&](size_t off) { return reinterpret_cast<unsigned *>(ws + off); };
    const unsigned *keys = nullptr, *places = nullptr;
    unsigned *counts = at(p.counts);
    for (int pass = 0; pass < p.passes; ++pass) {
      const int32_t *ids = pass == 0 ? a.ids : nullptr;
      unsigned *k = at(pass % 2 ? p.keys2 : 0), *pl = at(pass % 2 ? p.places2 : p.places);
      const int shift = pass * p.digit_bits, bins = 1 << p.digit_bits;
      hipLaunchKernelGGL(k_embed_count, dim3(p.stretches), dim3(kSortThreads), 0, s, ids, keys, a.tokens, unsigned(a.vocab), a.pad, shift,
                         bins, p.per_stretch, counts);
      SGH_LAUNCH_CHECK();
      hipLaunchKernelGGL(k_embed_move, dim3(p.stretches), dim3(kSortThreads), 0, s, ids, keys, places, a.tokens, unsigned(a.vocab), a.pad,
                         shift, bins, p.per_stretch, counts, k, pl);
      SGH_LAUNCH_CHECK();
      keys = k, places = pl;
    }
    a.keys = keys, a.places = places;
    a.partial = reinterpret_cast<float *>(ws + p.partial);
    a.tile = p.tile;
    const int ny = (a.slices + kWaves - 1) / kWaves;
    hipLaunchKernelGGL((k_embed_tiles<S, EPL>), dim3(p.tiles, ny), dim3(kBlock), 0, s, a);
    SGH_LAUNCH_CHECK();
  }
  // about 32 KB of the result for a workgroup, the whole chip busy where the table is large enough
  const int per_wave = SGH_WAVE / a.lanes;
  size_t rows = (size_t(32) << 10) / (a.dim * e);
  const size_t spread = a.vocab / (size_t(sgh_num_cus()) * 8);
  if (rows > spread) rows = spread;
  if (rows < size_t(per_wave)) rows = per_wave;
  if (rows > size_t(kMostRows)) rows = kMostRows;
  while ((a.vocab + rows - 1) / rows > (1u << 23)) rows *= 2;   // (2^31 rows at the most: 2^8 of them suffice)
  if (rows > size_t(kMostRows)) rows = kMostRows;
  a.rows = int(rows);
  const size_t blocks = (a.vocab + rows - 1) / rows;
  const size_t units = (rows + per_wave - 1) / per_wave * size_t(a.slices);
  size_t ny = blocks >= size_t(sgh_num_cus()) * 4 ? 1 : (size_t(sgh_num_cus()) * 4 + blocks - 1) / blocks;
  if (ny > (units + kWaves - 1) / kWaves) ny = (units + kWaves - 1) / kWaves;
  if (p.scan)
    hipLaunchKernelGGL((k_embed_rows<S, EPL, true>), dim3(unsigned(blocks), unsigned(ny)), dim3(kBlock), 0, s, a);
  else
    hipLaunchKernelGGL((k_embed_rows<S, EPL, false>), dim3(unsigned(blocks), unsigned(ny)), dim3(kBlock), 0, s, a);
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
  hipStream_t s = sgh_stream_of(stream);
  sgh_note_write(dW, bytes);
  sgh_prof_scope prof("embedding_bwd", double(tokens) * (4 + double(dim) * e) + double(bytes) * (add ? 2 : 1), s);
  const RowLanes r = row_lanes<S>(dim);
  Rows<typename S::elem> a = {};
  a.dy = dy, a.add = add, a.dW = dW, a.ids = ids, a.dim = dim, a.vocab = vocab, a.tokens = unsigned(tokens), a.tile = 1;
  a.scale = scale, a.pad = pad, a.lanes = r.lanes, a.slices = r.slices;
  return r.epl == 1 ? launch_bwd<S, 1>(a, p, workspace, s) : launch_bwd<S, S::VEC>(a, p, workspace, s);
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
  SGH_HIP_TRY(hipStreamSynchronize(sgh_stream_of(stream)));
  int v = 0;
  SGH_HIP_TRY(hipMemcpyFromSymbol(&v, HIP_SYMBOL(g_index_errors), sizeof(int), 0, hipMemcpyDeviceToHost));
  const int zero = 0;
  SGH_HIP_TRY(hipMemcpyToSymbol(HIP_SYMBOL(g_index_errors), &zero, sizeof(int), 0, hipMemcpyHostToDevice));
  *count = v;
  return SGH_OK;
}

}  // extern "C"
