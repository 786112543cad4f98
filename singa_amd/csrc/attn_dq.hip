// First half of attention's backward pass: the gradients of the queries and of the position bias, and delta = do . o for the second half
// (attn_dkv.hip).  A wavefront owns queries, keys and values run through LDS; the probabilities are computed anew from the logarithms of the row
// sums:  p = e^(s - lse),  ds = p (do . v - delta),  dq = scale sum ds k.
//
// As the forward pass, with three products for its two: a tile of values is read by rows only, a tile of keys by rows and by columns.  Bound by
// the chain of products and exponentials in each wavefront, two to a SIMD (matrix units 61 % busy with bfloat16 heads of 128, 53 % with fp32 heads of
// 64): bfloat16, 2 x 16 heads of 128, 8192 places, causal: 727 us; fp32, 8 x 8 heads of 64, 512 places: 64 us.  A bias adds a look-up for each
// pair near the diagonal and the buckets' sums: bfloat16, 8 x 12 heads of 64, 1024 places: 91 us.
#include "attn_bwd.h"

namespace {

using namespace attn;

template <class T, int DP, bool BIAS>
__global__ __launch_bounds__(kBlock, (T::half || DP <= 64 ? 2 : 1)) void k_attn_dq(BwdArgs a, Bounds bounds) {
  typedef typename T::elem elem;
  typedef Tile<T, DP> L;
  constexpr int KT = T::half ? 64 : 32, SUB = KT / 32, ND = DP / 32, ROWS = kRows;
  constexpr int TILE = L::bytes(KT);
  extern __shared__ __align__(16) char lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hi = lane >> 5;
  const Shape &s = a.s;
  const Where place = block_at(a.q_tiles, a.q_units, a.q_splits, true);
  const unsigned tile = place.tile, unit = place.unit, split = place.split;
  const int per_batch = s.heads / a.pack, b = unit / per_batch, head0 = int(unit % per_batch) * a.pack;
  const int kv = head0 / (s.heads / s.kv_heads);
  const Span span = span_of(s, b);
  const int rows = s.q_len * a.pack, row0 = int(tile) * ROWS + wave * 32;

  // The 16-bit matrix products' sums are rounded a little downwards (by a thirtieth of a place on the average), which 10^8 terms of a bucket add
  // up to: odd queries have the gradient of their result negated, so that it goes both ways (13 x 8 heads, 2833 places, table's gradient: 4.4e-6 off,
  // so 5.0e-7; fp32 products show none of it).
  constexpr bool kFlip = BIAS && T::half;
  const float flip = kFlip && (lane & 1) ? -1.f : 1.f;
  const int r = row0 + (lane & 31), query = a.pack == 1 ? r : r / a.pack, head = a.pack == 1 ? head0 : head0 + r % a.pack;
  const int limit = r < rows && query < span.q ? (s.causal ? min(span.k, max(span.start + query + 1, 0)) : span.k) : 0;
  int most = limit, least = limit;
  const size_t at = ((size_t(b) * s.q_len + query) * s.heads + head) * s.dim;
  const size_t stat = (size_t(b) * s.heads + head) * s.q_len + query;
  const int n = limit ? s.dim : 0;
  cols_t<T, DP> qf, df;
  load_columns<T, DP>(qf, static_cast<const elem *>(a.q) + at, n, hi, a.direct);
  load_columns<T, DP>(df, static_cast<const elem *>(a.dout) + at, n, hi, a.direct);
  // (with a bias a natural logarithm: the product with log2 e is rounded with the sum, which the bias's gradient is told by)
  float lse = limit ? a.lse[stat] : kNegInf;
  if (lse == kNegInf) lse = -kNegInf;
  const float lse2 = lse * kLog2e;
  if (!BIAS) lse = lse2;
  float x = 0.f;
  cols_t<T, DP> of;
  load_columns<T, DP>(of, static_cast<const elem *>(a.o) + ((size_t(b) * s.q_len + query) * s.heads + head) * a.io_dim, n ? a.io_dim : 0, hi,
                      a.io_direct);
#pragma unroll
  for (int k = 0; k < kSteps<T, DP>; ++k) {
    float o[T::VEC], d[T::VEC];
    T::St::template load16<false>(reinterpret_cast<const elem *>(&of[k]), o);
    T::St::template load16<false>(reinterpret_cast<const elem *>(&df[k]), d);
#pragma unroll
    for (int i = 0; i < T::VEC; ++i) x = __builtin_fmaf(o[i], d[i], x);
  }
  float delta = sum_of_pair(x);
  if (r < rows && hi == 0 && split == 0) {
    a.stats[stat] = lse2 - term_bits<T>();
    a.stats[size_t(a.q_units) * rows + stat] = -delta;
  }
  if constexpr (kFlip) {   // (rows are queries here: with a bias no heads share a tile)
    delta *= flip;
    if (lane & 1)
#pragma unroll
      for (int k = 0; k < kSteps<T, DP>; ++k)
#pragma unroll
        for (int i = 0; i < 4; ++i) df[k][i] ^= 0x80008000u;
  }
  for (int m = 1; m < 32; m *= 2) most = max(most, __shfl_xor(most, m)), least = min(least, __shfl_xor(least, m));
  most = __builtin_amdgcn_readfirstlane(most), least = __builtin_amdgcn_readfirstlane(least);
  int end = span.k;
  if (s.causal) {
    const int last = min(int(tile + 1) * ROWS, rows) - 1;
    end = min(end, max(span.start + min(last / a.pack, span.q - 1) + 1, 0));
  }
  if (int(tile) * ROWS >= span.q * a.pack) end = 0;
  const int begin = int(split) * a.keys_each;
  end = min(end, begin + a.keys_each);

  const int band_len = 2 * s.reach + 1;
  float *band = reinterpret_cast<float *>(lds + 4 * TILE), *sums = band + band_len + wave * band_len;   // sums: a wavefront's own
  float far_back = 0.f, far_on = 0.f;
  if constexpr (BIAS) {
    expand_bias(s, bounds, head0, band);
    for (int i = lane; i < band_len; i += SGH_WAVE) sums[i] = 0.f;
  }

  const size_t stride = size_t(s.kv_heads) * s.dim;
  Stage<T, DP, KT> stage;
  stage.init(stride, s.dim, a.direct);
  const elem *kp = static_cast<const elem *>(a.k) + (size_t(b) * s.k_len * s.kv_heads + kv) * s.dim;
  const elem *vp = static_cast<const elem *>(a.v) + (size_t(b) * s.k_len * s.kv_heads + kv) * s.dim;
  f32x16 acc[ND];
  Range<T> range;
  zero(acc);
  const float c = s.scale * kLog2e;
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
    if (k0 >= most) continue;
#pragma unroll
    for (int u = 0; u < SUB; ++u) {
      f32x16 p, ds;
      zero(p);
      reader.rows(kt, 32 * u, qf, p);
      if constexpr (T::half) pin();   // (one product's loads under way at a time: 2 x 16 heads of 128, 8192 places, 1870 -> 1720 us, fp32 heads of 64 125 -> 128)
      // (the product starts from -delta)
#pragma unroll
      for (int i = 0; i < 16; ++i) ds[i] = -delta;
      reader.rows(vt, 32 * u, df, ds);
      const int k1 = k0 + 32 * u;
      const int first = k1 - (span.start + query) + 4 * hi;
      if constexpr (BIAS) {
        const int lo = k1 - (span.start + row0 + 31), up = k1 + 31 - (span.start + row0);
        const float *mine = band + s.reach;
        if (up <= -s.reach || lo >= s.reach) {
          const float far = __builtin_fmaf(-lse, kLog2e, mine[up <= -s.reach ? -s.reach : s.reach]);
#pragma unroll
          for (int i = 0; i < 16; ++i) p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[i], c, far));
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i)
            p[i] = __builtin_amdgcn_exp2f(
                __builtin_fmaf(p[i], c, __builtin_fmaf(-lse, kLog2e, mine[min(max(first + row_of(i), -s.reach), s.reach)])));
        }
      } else {
#pragma unroll
        for (int i = 0; i < 16; ++i) p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[i], c, -lse));
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) ds[i] *= p[i];
      if (k1 + 32 > least) {
        const int left = limit - k1 - 4 * hi;
#pragma unroll
        for (int i = 0; i < 16; ++i)
          if (row_of(i) >= left) ds[i] = 0.f;
      }
      if constexpr (BIAS) {
        const int lo = k1 - (span.start + row0 + 31), up = k1 + 31 - (span.start + row0);
        if (up <= -s.reach || lo >= s.reach) {
          float x = 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) x += ds[i];
          x *= flip;
          if (up <= -s.reach) far_back += x;
          else far_on += x;
        } else {
          // Sums of the diagonals.  Lane j gets from row r the column (r - j) mod 32, whose distance is j or j - 32 on from the block's
          // corner: two sums for each lane, in the order of the rows.
          float on = 0.f, back = 0.f;
          const int j = lane & 31;
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int r = row_of(i) + 4 * hi;
            const float x = __shfl(ds[i], ((r - j) & 31) + 32 * hi);
            const float y = kFlip && row_of(i) & 1 ? -x : x;   // (column r - j: its sign is the row's times this lane's)
            if (r >= j) on += y;
            else back += y;
          }
          on = sum_of_pair(on) * flip, back = sum_of_pair(back) * flip;
          const int d = lo + 31 + (hi ? j - 32 : j);
          const float x = hi ? back : on;
          if (d < -s.reach) far_back += x;
          else if (d > s.reach) far_on += x;
          else sums[d + s.reach] += x;
          __builtin_amdgcn_wave_barrier();
        }
      }
      range.fit(ds, acc);
      Terms<T> terms;
      terms.set(ds);
      reader.transposed(kt, 32 * u, terms, acc);
    }
  }

  if (r < rows) {
    if (!limit) zero(acc);
    const float f = s.scale * range.inverse() * flip;
    if (a.q_splits == 1) {
      store_column<T, DP>(static_cast<elem *>(a.dq) + ((size_t(b) * s.q_len + query) * s.heads + head) * a.io_dim, acc, f, a.io_dim, hi,
                          a.io_direct);
    } else {
      const size_t n = size_t(a.q_units) * rows;
      store_partial<DP>(a.q_part + (split * n + size_t(unit) * rows + r) * DP, acc, f, hi);
    }
  }
  if constexpr (BIAS) {
    // the block's sums of the buckets: distances in order, the wavefronts' sums of each one behind the other
    for (int m = 1; m < SGH_WAVE; m *= 2) far_back += __shfl_xor(far_back, m), far_on += __shfl_xor(far_on, m);
    __builtin_amdgcn_wave_barrier();
    if (lane == 0) sums[0] += far_back, sums[2 * s.reach] += far_on;
    __syncthreads();
    float *out = a.bias_part + (size_t(head0) * a.bias_blocks + (size_t(b) * a.q_tiles + tile) * a.q_splits + split) * s.buckets;
    float *all = band + band_len;
    for (int d = tid; d < band_len; d += kBlock) all[d] = (all[d] + all[band_len + d]) + (all[2 * band_len + d] + all[3 * band_len + d]);
    __syncthreads();
    all += s.reach;
    for (int e = tid; e < s.buckets; e += kBlock) {
      const int half = s.bidirectional ? s.buckets / 2 : s.buckets, n = e % half, sign = e < half ? -1 : 1;
      const int from = n == 0 ? 0 : bounds.at[n - 1], to = n == half - 1 ? s.reach : min(bounds.at[n] - 1, s.reach);
      float x = 0.f;
      for (int m = max(from, sign > 0); m <= to; ++m) x += all[sign * m];
      if (!s.bidirectional && n == 0)   // (one direction: all keys in front have the bucket of distance 0)
        for (int d = 1; d <= s.reach; ++d) x += all[d];
      out[e] = x;
    }
  }
}

// dq of keys in parts: the parts' sum
template <class T, int DP>
__global__ __launch_bounds__(kBlock) void k_attn_dq_join(BwdArgs a) {
  constexpr int TEAM = DP / 4, PER = kBlock / TEAM;
  const Shape &s = a.s;
  const size_t rows = size_t(s.q_len) * a.pack, n = a.q_units * rows, at = size_t(blockIdx.x) * PER + threadIdx.x / TEAM;
  const int d = int(threadIdx.x % TEAM) * 4;
  if (threadIdx.x >= PER * TEAM || at >= n) return;
  sgh_v4f x = {0.f, 0.f, 0.f, 0.f};
  for (unsigned i = 0; i < a.q_splits; ++i) x += *reinterpret_cast<const sgh_v4f *>(a.q_part + (i * n + at) * DP + d);
  const size_t unit = at / rows;
  const int r = int(at % rows), per_batch = s.heads / a.pack, b = int(unit / per_batch);
  const int query = r / a.pack, head = int(unit % per_batch) * a.pack + r % a.pack;
  typename T::elem *out = static_cast<typename T::elem *>(a.dq) + ((size_t(b) * s.q_len + query) * s.heads + head) * a.io_dim;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (d + i < a.io_dim) T::St::st(out + d + i, x[i]);
}

// dtable[e][h]: the sum over all blocks of head h, each thread's in order, then the threads' by halves
__global__ __launch_bounds__(kBlock) void k_attn_dtable(BwdArgs a, float *dtable) {
  __shared__ float part[kBlock];
  const int h = blockIdx.x, e = blockIdx.y;
  const float *p = a.bias_part + size_t(h) * a.bias_blocks * a.s.buckets + e;
  float x = 0.f;
  for (size_t i = threadIdx.x; i < a.bias_blocks; i += kBlock) x += p[i * a.s.buckets];
  part[threadIdx.x] = x;
  for (int m = kBlock / 2; m > 0; m /= 2) {
    __syncthreads();
    if (int(threadIdx.x) < m) part[threadIdx.x] += part[threadIdx.x + m];
  }
  if (threadIdx.x == 0) dtable[size_t(e) * a.s.heads + h] = part[0];
}

template <class T, int DP, bool BIAS>
int launch(const BwdArgs &a, const Bounds &bounds, float *dtable, hipStream_t s) {
  constexpr int KT = T::half ? 64 : 32;
  const size_t lds = 4 * Tile<T, DP>::bytes(KT) + (BIAS ? 5 * (2 * a.s.reach + 1) * sizeof(float) : 0);
  static std::atomic<unsigned long long> asked{0};
  SGH_HIP_TRY(sgh_allow_lds(reinterpret_cast<const void *>(k_attn_dq<T, DP, BIAS>), asked));
  hipLaunchKernelGGL((k_attn_dq<T, DP, BIAS>), dim3(a.q_tiles * a.q_units * a.q_splits), dim3(kBlock), lds, s, a, bounds);
  SGH_LAUNCH_CHECK();
  if (a.q_splits > 1) {
    const size_t n = size_t(a.q_units) * a.s.q_len * a.pack, per = kBlock / (DP / 4);
    hipLaunchKernelGGL((k_attn_dq_join<T, DP>), dim3(unsigned((n + per - 1) / per)), dim3(kBlock), 0, s, a);
    SGH_LAUNCH_CHECK();
  }
  if (BIAS) {
    hipLaunchKernelGGL(k_attn_dtable, dim3(unsigned(a.s.heads), unsigned(a.s.buckets)), dim3(kBlock), 0, s, a, dtable);
    SGH_LAUNCH_CHECK();
  }
  return SGH_OK;
}
template <class T, int DP>
int run_dim(const BwdArgs &a, const Bounds &bounds, float *dtable, hipStream_t s) {
  if (a.s.buckets) return launch<T, DP, true>(a, bounds, dtable, s);
  return launch<T, DP, false>(a, bounds, dtable, s);
}

}  // namespace

namespace attn {

template <class T>
int run_dq(const BwdArgs &a, const Bounds &bounds, float *dtable, hipStream_t s) {
  switch ((a.s.dim + 31) / 32) {
    case 1: return run_dim<T, 32>(a, bounds, dtable, s);
    case 2: return run_dim<T, 64>(a, bounds, dtable, s);
    case 3: return run_dim<T, 96>(a, bounds, dtable, s);
    default: return run_dim<T, 128>(a, bounds, dtable, s);
  }
}
template int run_dq<F32>(const BwdArgs &, const Bounds &, float *, hipStream_t);
template int run_dq<F16>(const BwdArgs &, const Bounds &, float *, hipStream_t);
template int run_dq<BF16>(const BwdArgs &, const Bounds &, float *, hipStream_t);

}  // namespace attn
