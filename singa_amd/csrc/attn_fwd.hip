// Forward pass of attention: o = softmax(scale q k^T + bias) v in one pass over the keys, and the logarithm of every row's sum.
//
// s and the probabilities of a 32x32 block live in one wavefront's registers, queries in the lanes: a running maximum m and sum l for each query,
// o rescaled when m grows.  Exponentials are powers of two (scale and bias times log2 e).
//
// A block is four wavefronts of 32 queries; tiles of 64 keys and values (fp32: 32) lie twice in LDS, one pair being filled while the other is
// used.  With one query to a lane a row's maximum and sum cost one exchange of two lanes, and the probabilities are where the product with the
// values wants them; 64 queries to a wavefront left no registers for a second one on its SIMD.  Bound by the chain in each wavefront,
// product, exponentials and conversions, product: with two of them on a SIMD the matrix units are 43 % busy.  bfloat16, 4 x 32 heads of 128 over 4096
// places, groups of 4, causal, ragged: 387 to 409 us, 830 to 880 TFLOP/s of the pairs that are seen; fp32, 4 x 16 heads of 128 over 2048 places, causal:
// 875 us, 78 TFLOP/s.
#include "attn.h"
#include "attn_run.h"

namespace {

using namespace attn;

struct FwdArgs {
  Shape s;
  const void *q, *k, *v;
  void *o;
  float *lse;
  float *part;        // [splits][units][rows][DP + 1]: results of a part of the keys, and the logarithms of their sums
  unsigned tiles, units, splits;
  int pack;           // heads of a group that share a tile: row r is query r / pack, head r % pack of the group
  int keys_each;      // keys of a split, a multiple of 64
  bool direct;        // of keys and values, rows of s.dim
  int io_dim;         // q and o have rows of io_dim
  bool io_direct;
};

// m moves only when a row's maximum has grown by more than 2^8: the terms then stay within 2^8 of one, and o is rescaled seldom
constexpr float kGrowth = 8.f;
constexpr int kRows = 128, kFewRows = 32;   // queries of a block

template <class T, int DP, bool BIAS>
__global__ __launch_bounds__(kBlock, 2) void k_attn_fwd(FwdArgs a, Bounds bounds) {
  typedef typename T::elem elem;
  typedef Tile<T, DP> L;
  constexpr int KT = T::half ? 64 : 32, SUB = KT / 32, ND = DP / 32, ROWS = kRows;
  constexpr int TILE = L::bytes(KT);
  // binary16: terms from 2^-14 to 2^14 with all their bits
  constexpr float kShift = std::is_same<T, F16>::value ? 6.f : 0.f;
  extern __shared__ __align__(16) char lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hi = lane >> 5;
  const Shape &s = a.s;
  const Where at = block_at(a.tiles, a.units, a.splits, true);
  const unsigned tile = at.tile, unit = at.unit, split = at.split;
  const int per_batch = s.heads / a.pack, b = unit / per_batch, head0 = int(unit % per_batch) * a.pack;
  const int kv = head0 / (s.heads / s.kv_heads);
  const Span span = span_of(s, b);
  const int rows = s.q_len * a.pack, row0 = int(tile) * ROWS + wave * 32;

  // the lane's query: keys [0, limit) are seen
  const int r = row0 + (lane & 31), query = a.pack == 1 ? r : r / a.pack, head = a.pack == 1 ? head0 : head0 + r % a.pack;
  const int limit = r < rows && query < span.q ? (s.causal ? min(span.k, max(span.start + query + 1, 0)) : span.k) : 0;
  int most = limit, least = limit;
  cols_t<T, DP> qf;
  load_columns<T, DP>(qf, static_cast<const elem *>(a.q) + ((size_t(b) * s.q_len + query) * s.heads + head) * a.io_dim,
                      limit ? a.io_dim : 0, hi, a.io_direct);
  for (int m = 1; m < 32; m *= 2) most = max(most, __shfl_xor(most, m)), least = min(least, __shfl_xor(least, m));
  most = __builtin_amdgcn_readfirstlane(most), least = __builtin_amdgcn_readfirstlane(least);
  // of the whole block: the last row's
  int end = span.k;
  if (s.causal) {
    const int last = min(int(tile + 1) * ROWS, rows) - 1;
    end = min(end, max(span.start + min(last / a.pack, span.q - 1) + 1, 0));
  }
  if (int(tile) * ROWS >= span.q * a.pack) end = 0;
  const int begin = int(split) * a.keys_each;
  end = min(end, begin + a.keys_each);

  float *band = reinterpret_cast<float *>(lds + 4 * TILE);
  const int band_len = 2 * s.reach + 1;
  if constexpr (BIAS)
    for (int g = 0; g < a.pack; ++g) expand_bias(s, bounds, head0 + g, band + g * band_len);

  const size_t stride = size_t(s.kv_heads) * s.dim;
  Stage<T, DP, KT> stage;
  stage.init(stride, s.dim, a.direct);
  const elem *kp = static_cast<const elem *>(a.k) + (size_t(b) * s.k_len * s.kv_heads + kv) * s.dim;
  const elem *vp = static_cast<const elem *>(a.v) + (size_t(b) * s.k_len * s.kv_heads + kv) * s.dim;

  f32x16 acc[ND];
  zero(acc);
  float m = -3e38f, l = 0.f;
  // (maxima are taken before the scale, which is therefore made positive: the products are multiplied by -1 or 0 first if it is not)
  const float factor = s.scale * kLog2e;
  const float turned = BIAS || factor > 0.f ? 1.f : factor < 0.f ? -1.f : 0.f, c = BIAS || factor != 0.f ? (BIAS ? factor : __builtin_fabsf(factor)) : 1.f;
  const Reader<T, DP> reader(lane);
  auto request = [&](int k0, int slot) {
    stage(lds + slot * 2 * TILE, kp + k0 * stride, span.k - k0);
    stage(lds + slot * 2 * TILE + TILE, vp + k0 * stride, span.k - k0);
  };
  registers_arrive();
  if (begin < end) request(begin, 0);
  int slot = 0;
  for (int k0 = begin; k0 < end; k0 += KT, slot ^= 1) {
    tiles_arrive();
    if (k0 + KT < end) request(k0 + KT, slot ^ 1);
    const char *kt = lds + slot * 2 * TILE, *vt = kt + TILE;
    if (k0 >= most) continue;   // (no row of this wavefront sees any of them)
    f32x16 p[SUB];
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      zero(p[u]);
      reader.rows(kt, 32 * u, qf, p[u]);
    }
    // Scores: in units of log2 with a bias; else as the products are, and the maximum is multiplied.  -inf where the mask is.
    if (!BIAS && turned != 1.f) {
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i) p[u][i] *= turned;
    }
    float top = kNegInf;
    if constexpr (BIAS) {
      const int first = k0 - (span.start + query);   // the distance of key k0
      const int lo = k0 - (span.start + (row0 + 31) / a.pack), up = k0 + KT - 1 - (span.start + row0 / a.pack);
      const float *mine = band + (head - head0) * band_len + s.reach;
      if (up <= -s.reach || lo >= s.reach) {   // far away the bias is one number
        const float far = mine[up <= -s.reach ? -s.reach : s.reach];
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
          for (int i = 0; i < 16; ++i) p[u][i] = __builtin_fmaf(p[u][i], c, far);
      } else {
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int d = first + 32 * u + row_of(i) + 4 * hi;
            p[u][i] = __builtin_fmaf(p[u][i], c, mine[min(max(d, -s.reach), s.reach)]);
          }
      }
    }
    if (k0 + KT > least) {
      const int left = limit - k0 - 4 * hi;
#pragma unroll
      for (int u = 0; u < SUB; ++u)
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (32 * u + row_of(i) >= left) p[u][i] = kNegInf;
    }
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, p[u][i]);
    top = max_of_pair(top);
    if (!BIAS) top *= c;
    if (__ballot(top > m + kGrowth)) {
      const float now = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - now);
      m = now, l *= f;
#pragma unroll
      for (int n = 0; n < ND; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[n][i] *= f;
    }
    const float from = m - kShift;
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < SUB; ++u)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        p[u][i] = __builtin_amdgcn_exp2f(BIAS ? p[u][i] - from : __builtin_fmaf(p[u][i], c, -from));
        sum += p[u][i];
      }
    l += sum;
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      Terms<T> terms;
      terms.set(p[u]);
      reader.transposed(vt, 32 * u, terms, acc);
    }
  }

  if (r >= rows) return;
  const float sum = sum_of_pair(l);
  // (a row that sees nothing has o = 0 and the logarithm of 0)
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (sum == 0.f) zero(acc);
  const float lse = sum == 0.f ? kNegInf : (m - kShift + __builtin_amdgcn_logf(sum)) * kLn2;
  if (a.splits == 1) {
    store_column<T, DP>(static_cast<elem *>(a.o) + ((size_t(b) * s.q_len + query) * s.heads + head) * a.io_dim, acc, inv, a.io_dim, hi,
                        a.io_direct);
    if (hi == 0) a.lse[(size_t(b) * s.heads + head) * s.q_len + query] = lse;
  } else {
    const size_t n = size_t(a.units) * rows, at = split * n + size_t(unit) * rows + r;
    store_partial<DP>(a.part + at * DP, acc, inv, hi);
    if (hi == 0) a.part[a.splits * n * DP + at] = lse;
  }
}

// Few queries (32 with the heads of a group): the wavefronts of a block share the keys, 32 at a time, each with tiles of its own in LDS that
// nobody else waits for, and join what they have in the end.  Bound by the way of keys and values from memory; in the kernel above one wavefront
// would have all the products, and three wait.  (16 sequences of up to 16384 places, 4 heads of keys of 64, binary16, bias: 52 us, and
// its join 5; fp32, 5 x 8 heads of keys of 128, 16180 places: 216 -> 126, 5.2 TB/s.)
template <class T, int DP>
struct Few {
  static constexpr int KT = 32, TILE = Tile<T, DP>::bytes(KT), WAVE = 2 * TILE;   // a wavefront's keys and values
  static constexpr int SLOTS = 4 * 4 * WAVE <= (132 << 10) ? 4 : 4 * 2 * WAVE <= (132 << 10) ? 2 : 1;
  static constexpr bool ONE = SLOTS == 1;   // rows of over 256 bytes: the next keys are requested over those just used, then the values alike
  static constexpr int AHEAD = ONE ? 1 : SLOTS - 1;
  static constexpr int ROW = DP + 4;                                             // floats of a row of results in LDS
  static constexpr size_t kTiles = 4 * SLOTS * WAVE, kResults = (4 * 32 * ROW + 8 * 32) * sizeof(float);
  static constexpr size_t kBytes = kTiles > kResults ? kTiles : kResults;
};
template <class T, int DP, bool BIAS>
__global__ __launch_bounds__(kBlock, 1) void k_attn_few(FwdArgs a, Bounds bounds) {
  typedef typename T::elem elem;
  typedef Few<T, DP> F;
  static_assert(F::kBytes + kMostBand <= (156 << 10), "LDS");
  constexpr int ND = DP / 32;
  constexpr float kShift = std::is_same<T, F16>::value ? 6.f : 0.f;
  extern __shared__ __align__(16) char lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hi = lane >> 5;
  const Shape &s = a.s;
  const Where at = block_at(1, a.units, a.splits, true);
  const int unit = int(at.unit), per_batch = s.heads / a.pack, b = unit / per_batch, head0 = unit % per_batch * a.pack;
  const int kv = head0 / (s.heads / s.kv_heads);
  const Span span = span_of(s, b);
  const int rows = s.q_len * a.pack, r = lane & 31, query = r / a.pack, head = head0 + r % a.pack;
  const int limit = r < rows && query < span.q ? (s.causal ? min(span.k, max(span.start + query + 1, 0)) : span.k) : 0;
  cols_t<T, DP> qf;
  load_columns<T, DP>(qf, static_cast<const elem *>(a.q) + ((size_t(b) * s.q_len + query) * s.heads + head) * a.io_dim, limit ? a.io_dim : 0, hi,
                      a.io_direct);
  int most = limit, least = r < rows ? limit : 1 << 30;
  for (int m = 1; m < 32; m *= 2) most = max(most, __shfl_xor(most, m)), least = min(least, __shfl_xor(least, m));
  most = __builtin_amdgcn_readfirstlane(most), least = __builtin_amdgcn_readfirstlane(least);
  // the split's part of the keys that are seen, in whole rounds of the block
  const int each = ((most + int(a.splits) - 1) / int(a.splits) + 4 * F::KT - 1) / (4 * F::KT) * (4 * F::KT);
  const int begin = min(most, int(at.split) * each), end = min(most, begin + each);

  float *band = reinterpret_cast<float *>(lds + F::kBytes);
  const int band_len = 2 * s.reach + 1;
  if constexpr (BIAS)
    for (int g = 0; g < a.pack; ++g) expand_bias(s, bounds, head0 + g, band + g * band_len);

  const size_t stride = size_t(s.kv_heads) * s.dim;
  Stage<T, DP, F::KT, SGH_WAVE> stage;
  stage.init(stride, s.dim, a.direct, lane);
  const elem *kp = static_cast<const elem *>(a.k) + (size_t(b) * s.k_len * s.kv_heads + kv) * s.dim;
  const elem *vp = static_cast<const elem *>(a.v) + (size_t(b) * s.k_len * s.kv_heads + kv) * s.dim;
  char *const mine = lds + wave * F::SLOTS * F::WAVE;
  f32x16 acc[ND];
  zero(acc);
  float m = -3e38f, l = 0.f;
  const float c = s.scale * kLog2e;
  const Reader<T, DP> reader(lane);
  auto request_keys = [&](int k0, int slot) { stage(mine + slot * F::WAVE, kp + k0 * stride, span.k - k0); };
  auto request_values = [&](int k0, int slot) { stage(mine + slot * F::WAVE + F::TILE, vp + k0 * stride, span.k - k0); };
  registers_arrive();
  __syncthreads();   // (the bias)
  const int first_key = begin + wave * F::KT, turns = first_key < end ? (end - first_key + 4 * F::KT - 1) / (4 * F::KT) : 0;
  const int loads = a.direct ? stage.loads(0) : 0;   // of a tile
  for (int i = 0; i < F::AHEAD && i < turns; ++i) request_keys(first_key + i * 4 * F::KT, i), request_values(first_key + i * 4 * F::KT, i);
  int slot = 0, ahead_slot = F::AHEAD;
  for (int turn = 0; turn < turns; ++turn) {
    own_tiles_arrive(F::ONE ? loads : 2 * loads * min(F::AHEAD - 1, turns - 1 - turn));
    const int k0 = first_key + turn * 4 * F::KT, ahead = k0 + F::AHEAD * 4 * F::KT;
    const bool more = turn + F::AHEAD < turns;
    if (!F::ONE && more) {
      request_keys(ahead, ahead_slot), request_values(ahead, ahead_slot);
      ahead_slot = ahead_slot == F::SLOTS - 1 ? 0 : ahead_slot + 1;
    }
    const char *kt = mine + slot * F::WAVE, *vt = kt + F::TILE;
    slot = slot == F::SLOTS - 1 ? 0 : slot + 1;
    f32x16 p;
    zero(p);
    reader.rows(kt, 0, qf, p);
    if constexpr (F::ONE) {
      own_reads_end();
      if (more) request_keys(ahead, 0);
    }
    float top = kNegInf;
    if constexpr (BIAS) {
      const float *centre = band + (r < rows ? head - head0 : 0) * band_len + s.reach;
      const int first = k0 - (span.start + query) + 4 * hi;
#pragma unroll
      for (int i = 0; i < 16; ++i) p[i] = __builtin_fmaf(p[i], c, centre[min(max(first + row_of(i), -s.reach), s.reach)]);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) p[i] *= c;
    }
    if (k0 + F::KT > least) {
      const int left = limit - k0 - 4 * hi;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (row_of(i) >= left) p[i] = kNegInf;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, p[i]);
    top = max_of_pair(top);
    if (__ballot(top > m + kGrowth)) {
      const float now = fmaxf(m, top), f = __builtin_amdgcn_exp2f(m - now);
      m = now, l *= f;
#pragma unroll
      for (int n = 0; n < ND; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[n][i] *= f;
    }
    const float from = m - kShift;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      p[i] = __builtin_amdgcn_exp2f(p[i] - from);
      l += p[i];
    }
    Terms<T> terms;
    terms.set(p);
    if constexpr (F::ONE) own_tiles_arrive(more ? loads : 0);
    reader.transposed(vt, 0, terms, acc);
    if constexpr (F::ONE) {
      own_reads_end();
      if (more) request_values(ahead, 0);
    }
  }

  // what the four have: sums relative to their own maxima
  float *const results = reinterpret_cast<float *>(lds), *const tops = results + 4 * 32 * F::ROW, *const totals = tops + 4 * 32;
  l = sum_of_pair(l);
  __syncthreads();
  store_partial<DP>(results + (wave * 32 + r) * F::ROW, acc, 1.f, hi);
  if (hi == 0) tops[wave * 32 + r] = m, totals[wave * 32 + r] = l;
  __syncthreads();
  for (int i = tid; i < rows * (DP / 4); i += kBlock) {
    const int row = i / (DP / 4), d = i % (DP / 4) * 4, q = row / a.pack, h = head0 + row % a.pack;
    float top = tops[row], sum = 0.f;
#pragma unroll
    for (int w = 1; w < 4; ++w) top = fmaxf(top, tops[w * 32 + row]);
    sgh_v4f o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      const float total = totals[w * 32 + row], f = total == 0.f ? 0.f : __builtin_amdgcn_exp2f(tops[w * 32 + row] - top);
      sum += total * f;
      if (total != 0.f) o += *reinterpret_cast<const sgh_v4f *>(results + (w * 32 + row) * F::ROW + d) * f;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum, lse = sum == 0.f ? kNegInf : (top - kShift + __builtin_amdgcn_logf(sum)) * kLn2;
    if (a.splits == 1) {
      elem *out = static_cast<elem *>(a.o) + ((size_t(b) * s.q_len + q) * s.heads + h) * a.io_dim;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (d + e < a.io_dim) T::St::st(out + d + e, o[e] * inv);
      if (d == 0) a.lse[(size_t(b) * s.heads + h) * s.q_len + q] = lse;
    } else {
      const size_t n = size_t(a.units) * rows, to = at.split * n + size_t(unit) * rows + row;
      *reinterpret_cast<sgh_v4f *>(a.part + to * DP + d) = o * inv;
      if (d == 0) a.part[a.splits * n * DP + to] = lse;
    }
  }
}

// Joins the parts of the keys, a block to a row: o = sum e^(lse_s - lse) o_s.  DP / 4 lanes have four values each, the groups of so many lanes
// share the parts (16 rows of 128 values in 235 parts: one group to a row 100 us).
template <class T, int DP>
__global__ __launch_bounds__(kBlock) void k_attn_join(FwdArgs a) {
  typedef typename T::elem elem;
  constexpr int TEAM = DP / 4, GROUPS = kBlock / TEAM;
  __shared__ float least[4], total[GROUPS];
  __shared__ sgh_v4f sums[GROUPS][TEAM];
  const Shape &s = a.s;
  const size_t rows = size_t(s.q_len) * a.pack, n = a.units * rows, at = blockIdx.x;
  const float *lses = a.part + a.splits * n * DP + at;
  float top = kNegInf;
  for (unsigned i = threadIdx.x; i < a.splits; i += kBlock) top = fmaxf(top, lses[i * n]);
#pragma unroll
  for (int m = 1; m < SGH_WAVE; m *= 2) top = fmaxf(top, __shfl_xor(top, m));
  if (threadIdx.x % SGH_WAVE == 0) least[threadIdx.x / SGH_WAVE] = top;
  __syncthreads();
  top = fmaxf(fmaxf(least[0], least[1]), fmaxf(least[2], least[3]));
  const int g = threadIdx.x / TEAM, d = int(threadIdx.x % TEAM) * 4;
  if (g < GROUPS) {
    float sum = 0.f;
    sgh_v4f o = {0.f, 0.f, 0.f, 0.f};
    for (unsigned i = g; i < a.splits; i += GROUPS) {
      const float lse = lses[i * n];
      const float f = lse == kNegInf ? 0.f : __builtin_amdgcn_exp2f((lse - top) * kLog2e);   // (a NaN stays one)
      sum += f;
      o += *reinterpret_cast<const sgh_v4f *>(a.part + (i * n + at) * DP + d) * f;
    }
    sums[g][threadIdx.x % TEAM] = o;
    if (d == 0) total[g] = sum;
  }
  __syncthreads();
  if (threadIdx.x >= TEAM) return;
  sgh_v4f o = sums[0][threadIdx.x];
  float sum = total[0];
#pragma unroll
  for (int k = 1; k < GROUPS; ++k) o += sums[k][threadIdx.x], sum += total[k];
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const size_t unit = at / rows;
  const int r = int(at % rows), per_batch = s.heads / a.pack, b = int(unit / per_batch);
  const int query = r / a.pack, head = int(unit % per_batch) * a.pack + r % a.pack;
  elem *out = static_cast<elem *>(a.o) + ((size_t(b) * s.q_len + query) * s.heads + head) * a.io_dim;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (d + i < a.io_dim) T::St::st(out + d + i, o[i] * inv);
  if (d == 0) a.lse[(size_t(b) * s.heads + head) * s.q_len + query] = sum == 0.f ? kNegInf : top + __builtin_amdgcn_logf(sum) * kLn2;
}

template <class T, int DP>
int join(const FwdArgs &a, hipStream_t s) {
  if (a.splits > 1) {
    hipLaunchKernelGGL((k_attn_join<T, DP>), dim3(unsigned(size_t(a.units) * a.s.q_len * a.pack)), dim3(kBlock), 0, s, a);
    SGH_LAUNCH_CHECK();
  }
  return SGH_OK;
}
template <class T, int DP, bool BIAS>
int launch(const FwdArgs &a, const Bounds &bounds, size_t band, hipStream_t s) {
  static std::atomic<unsigned long long> asked{0};
  constexpr int KT = T::half ? 64 : 32;
  SGH_HIP_TRY(sgh_allow_lds(reinterpret_cast<const void *>(k_attn_fwd<T, DP, BIAS>), asked));
  SGH_LAUNCH_TIMED((k_attn_fwd<T, DP, BIAS>), dim3(a.tiles * a.units * a.splits), dim3(kBlock), (4 * Tile<T, DP>::bytes(KT)) + band, s, a, bounds);
  SGH_LAUNCH_CHECK();
  return join<T, DP>(a, s);
}
template <class T, int DP, bool BIAS>
int launch_few(const FwdArgs &a, const Bounds &bounds, size_t band, hipStream_t s) {
  static std::atomic<unsigned long long> asked{0};
  SGH_HIP_TRY(sgh_allow_lds(reinterpret_cast<const void *>(k_attn_few<T, DP, BIAS>), asked));
  SGH_LAUNCH_TIMED((k_attn_few<T, DP, BIAS>), dim3(a.units * a.splits), dim3(kBlock), (Few<T, DP>::kBytes) + band, s, a, bounds);
  SGH_LAUNCH_CHECK();
  return join<T, DP>(a, s);
}

// How a forward pass is cut
struct Plan {
  int dp, pack;
  unsigned tiles, units, splits;
  int keys_each;
  bool few;     // queries: k_attn_few
  bool pad;     // keys and values of rows that are not whole chunks are copied first
  size_t part, ws;
};
// (elem_bytes: fp32 never needs less of the workspace than the others)
Plan plan_of(const sgh_attn_geom *g, size_t elem_bytes) {
  Plan p;
  p.dp = (g->dim + 31) / 32 * 32;
  const int group = g->heads / g->kv_heads;
  // few queries: the heads of a group read their keys together
  p.pack = size_t(g->q_len) * group <= kRows && band_bytes(g) * group <= kMostBand ? group : 1;
  p.tiles = unsigned((size_t(g->q_len) * p.pack + kRows - 1) / kRows);
  p.units = unsigned(size_t(g->batch) * (g->heads / p.pack));
  // Few queries: wavefronts that share the keys, whose tiles take most of a CU's LDS (binary16, 45 units of 27 rows, heads of 128: 260 keys
  // 11.8 -> 9.9 us, 100 keys 7.9 -> 7.8, 64 keys 6.6 -> 7.6; more units than CUs, 400 with a bias: 250 keys 17 -> 22, 512 without one, 2000
  // keys: 100 -> 96).
  const size_t cus = size_t(sgh_num_cus());
  p.few = size_t(g->q_len) * p.pack <= size_t(kFewRows) && g->k_len > (p.units <= cus ? 64 : 512);
  // Few rows: several blocks to the keys of each (the launch that joins them takes 4 us and more, 64 keys of a block 1.2, of fp32 four times that).
  // Wavefronts that share keys keep the way to memory full with one block to a CU (16 x 4 heads over 16384 keys: 56 us, two 68, four 92),
  // others with four (the kernel above on fp32, 16 x 8 heads of 128, 2000 keys: 82 us, one 152).  More than 512 keys (fp32: 256) are shared, in
  // parts of up to 512, or 256 where blocks are few (bfloat16, 100 queries of 8 heads over 900 keys: 20 -> 14 us, 2 x 8 heads, 400 places 12 -> 20;
  // fp32, 2 x 4 heads of 128, 512 places 74 -> 48).
  p.splits = 1, p.keys_each = 1 << 30;
  const size_t blocks = size_t(p.tiles) * p.units, want = (p.few ? 1 : 4) * cus;
  const bool rare = !p.few && blocks * 2 <= cus;
  if (blocks * 2 <= want && g->k_len > (rare && elem_bytes == 4 ? 256 : 512)) {
    const size_t part = rare ? 256 : 512;
    size_t n = want / blocks, most = (size_t(g->k_len) + part - 1) / part;
    if (n > most) n = most;
    p.keys_each = int(((size_t(g->k_len) + n - 1) / n + 63) / 64 * 64);
    p.splits = unsigned((g->k_len + p.keys_each - 1) / p.keys_each);
  }
  p.part = p.splits > 1 ? (size_t(p.splits) * p.units * g->q_len * p.pack * (p.dp + 1) * sizeof(float) + 15) / 16 * 16 : 0;
  // where several blocks read them (4 x 16 heads of 61, 2048 tokens: 88 us, read as they are 228)
  p.pad = p.tiles * (group / p.pack) >= 2;
  p.ws = p.part + (p.pad ? 2 * wide_bytes(g->dim, size_t(g->batch) * g->k_len * g->kv_heads) : 0);
  return p;
}

template <class T, int DP>
int run_dim(const FwdArgs &a, const Bounds &bounds, bool few, hipStream_t s) {
  const size_t band = a.s.buckets ? a.pack * (2 * a.s.reach + 1) * sizeof(float) : 0;
  if (few) {
    if (a.s.buckets) return launch_few<T, DP, true>(a, bounds, band, s);
    return launch_few<T, DP, false>(a, bounds, band, s);
  }
  if (a.s.buckets) return launch<T, DP, true>(a, bounds, band, s);
  return launch<T, DP, false>(a, bounds, band, s);
}

template <class T>
int forward(const sgh_attn_geom *g, const void *q, const void *k, const void *v, const float *table, const int32_t *q_lengths,
            const int32_t *k_lengths, const int32_t *q_starts, void *o, float *lse, void *workspace, size_t ws_bytes, void *stream) {
  const int rc = check_geom(g);
  if (rc != SGH_OK) return rc;
  if (g->batch == 0 || g->q_len == 0) return SGH_OK;
  const size_t e = sizeof(typename T::elem), bq = size_t(g->batch) * g->q_len * g->heads, qn = bq * g->dim * e;
  const size_t kn = size_t(g->batch) * g->k_len * g->kv_heads * g->dim * e;
  if (!q || !o || !lse || (g->k_len != 0 && (!k || !v)) || (g->buckets != 0 && !table)) return SGH_EINVAL;
  const Plan p = plan_of(g, e);
  if (p.ws && (!workspace || ws_bytes < p.ws)) return SGH_EWORKSPACE;
  if (p.ws && !sgh_aligned16(workspace)) return SGH_EINVAL;
  const sgh_extent results[] = {{o, qn}, {lse, bq * 4}, {workspace, p.ws}};
  const sgh_extent arguments[] = {{q, qn}, {k, kn}, {v, kn}, {table, g->buckets ? size_t(g->buckets) * g->heads * 4 : 0},
                              {q_lengths, q_lengths ? size_t(g->batch) * 4 : 0}, {k_lengths, k_lengths ? size_t(g->batch) * 4 : 0},
                              {q_starts, q_starts ? size_t(g->batch) * 4 : 0}};
  if (sgh_any_overlap(results, arguments)) return SGH_EINVAL;
  FwdArgs a;
  a.s = shape_of(g, table, q_lengths, k_lengths, q_starts);
  a.q = q, a.k = k, a.v = v, a.o = o, a.lse = lse, a.part = static_cast<float *>(workspace);
  a.tiles = p.tiles, a.units = p.units, a.splits = p.splits, a.pack = p.pack, a.keys_each = p.keys_each;
  a.io_dim = g->dim;
  a.io_direct = g->dim % T::VEC == 0 && sgh_aligned16(q) && sgh_aligned16(o);
  a.direct = g->dim % T::VEC == 0 && sgh_aligned16(k) && sgh_aligned16(v);
  Bounds bounds;
  bounds_of(g, &bounds);
  hipStream_t s = sgh_stream_of(stream);
  sgh_note_write(o, qn);
  sgh_prof_kernel_scope prof("attn_fwd/k_attn_fwd", 4.0 * g->batch * g->heads * g->q_len * double(g->k_len) * g->dim, s);
  const int wide = p.pad ? wide_of(g->dim, e) : 0;
  if (p.splits > 1 || wide) prof.span();
  if (wide) {
    const size_t rows = size_t(g->batch) * g->k_len * g->kv_heads;
    char *at = static_cast<char *>(workspace) + p.part;
    const PadArgs pad = {{k, v}, {at, at + rows * wide * e}, {rows, rows}, g->dim, wide};
    const int r = pad_rows<T>(pad, 2, s);
    if (r != SGH_OK) return r;
    a.k = pad.to[0], a.v = pad.to[1], a.s.dim = wide, a.direct = true;
  }
  switch (p.dp) {
    case 32: return run_dim<T, 32>(a, bounds, p.few, s);
    case 64: return run_dim<T, 64>(a, bounds, p.few, s);
    case 96: return run_dim<T, 96>(a, bounds, p.few, s);
    default: return run_dim<T, 128>(a, bounds, p.few, s);
  }
}

}  // namespace

extern "C" {

size_t sgh_attn_fwd_workspace_bytes(const sgh_attn_geom *g) {
  return check_geom(g) == SGH_OK && g->batch != 0 && g->q_len != 0 ? plan_of(g, sizeof(float)).ws : 0;
}

#define SGH_ATTN_FWD(SFX, S, E)                                                                                                        \
  int sgh_attn_fwd_##SFX(const sgh_attn_geom *g, const E *q, const E *k, const E *v, const float *table, const int32_t *q_lengths,     \
                         const int32_t *k_lengths, const int32_t *q_starts, E *o, float *lse, void *workspace, size_t ws_bytes,        \
                         void *stream) {                                                                                               \
    return forward<S>(g, q, k, v, table, q_lengths, k_lengths, q_starts, o, lse, workspace, ws_bytes, stream);                         \
  }
SGH_ATTN_FWD(f32, F32, float)
SGH_ATTN_FWD(f16, F16, uint16_t)
SGH_ATTN_FWD(bf16, BF16, uint16_t)
#undef SGH_ATTN_FWD

}  // extern "C"
