// Second half of attention's backward pass: the gradients of the keys and values.  A wavefront owns keys; the queries, the gradients of their
// results and the statistics that the first half left run through LDS, for one head of the group after the other:
//   dv = sum p do,  dk = scale sum ds q.
// Each sum is one wavefront's, in the order of the heads and queries: the same bits every time, and nothing is added in memory.
//
// Four products of a tile: the scores and do . v once more, then dv and dk.  Bound by their chain with the exponentials between them, in two
// wavefronts to a SIMD: matrix units 56 % busy with bfloat16 heads of 128 (2 x 16 heads, 8192 places, causal: 1000 to 1070 us), 59 % with fp32 heads of
// 64 (8 x 8 heads, 512 places: 58 us).  Scores and do . v once for both halves would need dq added up in memory, in an order that changes, or a dq for
// each block of keys.  Two wavefronts to a group of keys, each with half the queries, were slower.
#include "attn_bwd.h"

namespace {

using namespace attn;

constexpr int kStats = SGH_WAVE;   // places of a tile's statistics of a kind: a load writes one for each lane

// A block's form.  VL: its values lie in LDS, where registers for two wavefronts of a SIMD would not do otherwise; the tiles are then 32 rows.
template <class T, int DP>
struct Form {
  static constexpr bool VL = T::half ? DP >= 96 : DP >= 64;
  static constexpr int QR = T::half && !VL ? 64 : 32;
  static constexpr int TILE = Tile<T, DP>::bytes(QR), SLOT = 2 * TILE + 2 * kStats * 4;
  static constexpr int VALUES = VL ? Tile<T, DP>::bytes(kRows) : 0;
  // of the longest rows the last 32 values of a key as well
  static constexpr bool KL = T::half && DP == 128;
  static constexpr int HELD = KL ? kSteps<T, DP> - kSteps<T, 32> : kSteps<T, DP>, REST = KL ? Tile<T, 32>::bytes(kRows) : 0;
  static constexpr int PER_SIMD = T::half || DP <= 64 ? 2 : 1;
  static constexpr size_t lds(int reach, bool bias) { return 2 * SLOT + VALUES + REST + (bias ? (2 * reach + 1) * sizeof(float) : 0); }
};

template <class T, int DP, bool BIAS>
__global__ __launch_bounds__(kBlock, (Form<T, DP>::PER_SIMD)) void k_attn_dkv(BwdArgs a, Bounds bounds) {
  typedef typename T::elem elem;
  typedef Form<T, DP> F;
  constexpr int QR = F::QR, SUB = QR / 32, ND = DP / 32, KEYS = kRows, TILE = F::TILE, SLOT = F::SLOT;
  constexpr bool VL = F::VL;
  extern __shared__ __align__(16) char lds[];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), hi = lane >> 5;
  const Shape &s = a.s;
  const Where place = block_at(a.k_tiles, a.k_units, a.k_splits, false);
  const unsigned tile = place.tile, unit = place.unit, split = place.split;
  const int b = unit / s.kv_heads, kv = unit % s.kv_heads, group = s.heads / s.kv_heads;
  const Span span = span_of(s, b);
  const int key0 = int(tile) * KEYS + wave * 32, key = key0 + (lane & 31);

  frag_t kf[F::HELD];
  cols_t<T, DP> vf;
  const size_t first_value = ((size_t(b) * s.k_len + key) * s.kv_heads + kv) * s.dim;
  const int values_of_key = key < span.k ? s.dim : 0;
  load_columns<T, F::HELD * 2 * T::VEC>(kf, static_cast<const elem *>(a.k) + first_value, values_of_key, hi, a.direct);
  if (!VL) load_columns<T, DP>(vf, static_cast<const elem *>(a.v) + first_value, values_of_key, hi, a.direct);
  // queries [from, span.q) see a key of the block, [mine, span.q) one of the wavefront
  const int from = s.causal ? max(int(tile) * KEYS - span.start, 0) / QR * QR : 0;
  const int mine = s.causal ? key0 - span.start : 0, all_see = s.causal ? key0 + 31 - span.start : 0;
  const int turns_of_head = int(tile) * KEYS < span.k && from < span.q ? (span.q - from + QR - 1) / QR : 0;
  const int turns = turns_of_head * group, each = (turns + int(a.k_splits) - 1) / int(a.k_splits);
  const int begin = min(turns, int(split) * each), end = min(turns, begin + each);

  char *const values = lds + 2 * SLOT;
  char *const rest = values + F::VALUES;
  float *band = reinterpret_cast<float *>(rest + F::REST);
  const size_t stride = size_t(s.heads) * s.dim;
  Stage<T, DP, QR> stage;
  stage.init(stride, s.dim, a.direct);
  const size_t first_row = (size_t(b) * s.q_len * s.heads + size_t(kv) * group) * s.dim;
  const elem *qp = static_cast<const elem *>(a.q) + first_row, *dp = static_cast<const elem *>(a.dout) + first_row;
  const float *lse = a.stats + (size_t(b) * s.heads + size_t(kv) * group) * s.q_len;
  const float *delta = lse + size_t(s.q_len) * s.heads * (a.k_units / s.kv_heads);

  f32x16 dk[ND], dv[ND];
  Range<T> range;
  zero(dk), zero(dv);
  const float c = s.scale * kLog2e;
  const Reader<T, DP> reader(lane);
  const Reader<T, 32> short_reader(lane);
  // A turn is QR queries of a head of the group.  Where the next one to be requested begins in the matrices and the statistics:
  int head = 0, q0 = 0, ahead_head = 0, ahead_q0 = 0, slot = 0;
  size_t skip = 0, stat = 0;
  auto request = [&](int slot) {
    char *at = lds + slot * SLOT;
    const int rows = span.q - ahead_q0;
    stage(at, qp + skip, rows);
    stage(at + TILE, dp + skip, rows);
    if (wave < 2)   // (rows behind the last query: 0, beside rows of zeros)
      load_lds4(buffer_of((wave ? delta : lse) + stat, rows * 4), lds_offset(at) + 2 * TILE + wave * kStats * 4, lane < QR ? lane * 4 : kOOB);
    ahead_q0 += QR, skip += QR * stride, stat += QR;
    if (ahead_q0 >= span.q) {
      ahead_q0 = from, ++ahead_head;
      skip = size_t(ahead_head) * s.dim + from * stride, stat = size_t(ahead_head) * s.q_len + from;
    }
  };
  bool other_head = true;
  registers_arrive();
  if (begin < end) {
    if constexpr (VL) {
      Stage<T, DP, KEYS> all;
      all.init(size_t(s.kv_heads) * s.dim, s.dim, a.direct);
      all(values, static_cast<const elem *>(a.v) + ((size_t(b) * s.k_len + size_t(tile) * KEYS) * s.kv_heads + kv) * s.dim, span.k - int(tile) * KEYS);
    }
    if constexpr (F::KL) {
      Stage<T, 32, KEYS> last;
      last.init(size_t(s.kv_heads) * s.dim, s.dim - (DP - 32), a.direct);
      last(rest, static_cast<const elem *>(a.k) + ((size_t(b) * s.k_len + size_t(tile) * KEYS) * s.kv_heads + kv) * s.dim + (DP - 32),
           span.k - int(tile) * KEYS);
    }
    ahead_head = head = begin / turns_of_head, ahead_q0 = q0 = from + begin % turns_of_head * QR;
    skip = size_t(head) * s.dim + q0 * stride, stat = size_t(head) * s.q_len + q0;
    request(0);
  }
  for (int turn = begin; turn < end; ++turn, slot ^= 1) {
    tiles_arrive();
    const int next_head = q0 + QR < span.q ? head : head + 1, next_q0 = q0 + QR < span.q ? q0 + QR : from;
    if (turn + 1 < end) request(slot ^ 1);
    if constexpr (BIAS)
      if (other_head) {
        expand_bias(s, bounds, kv * group + head, band);
        __syncthreads();
      }
    other_head = next_head != head;
    const char *qt = lds + slot * SLOT, *dt = qt + TILE;
    const float *st = reinterpret_cast<const float *>(dt + TILE);
    if (q0 + QR > mine) {
#pragma unroll
      for (int u = 0; u < SUB; ++u) {
        f32x16 p, ds;
        zero(p);
        if constexpr (VL) reader.rows_by_four(qt, 32 * u, kf, short_reader, rest + wave * 32 / Tile<T, 32>::G * Tile<T, 32>::GROUP, p);
        else reader.rows(qt, 32 * u, kf, p);
#pragma unroll
        for (int g = 0; g < 4; ++g) {   // (the product starts from -delta)
          const sgh_v4f x = *reinterpret_cast<const sgh_v4f *>(st + kStats + 32 * u + 8 * g + 4 * hi);
#pragma unroll
          for (int i = 0; i < 4; ++i) ds[4 * g + i] = x[i];
        }
        if constexpr (VL) reader.rows(dt, 32 * u, values, wave * 32, ds);
        else reader.rows(dt, 32 * u, vf, ds);
        float row_lse[16];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const sgh_v4f x = *reinterpret_cast<const sgh_v4f *>(st + 32 * u + 8 * g + 4 * hi);
#pragma unroll
          for (int i = 0; i < 4; ++i) row_lse[4 * g + i] = x[i];
        }
        const int q1 = q0 + 32 * u;
        if constexpr (BIAS) {
          const int first = key - (span.start + q1) - 4 * hi;   // distance in row 0
          const int lo = key0 - (span.start + q1 + 31), up = key0 + 31 - (span.start + q1);
          const float *centre = band + s.reach;
          if (up <= -s.reach || lo >= s.reach) {
            const float far = centre[up <= -s.reach ? -s.reach : s.reach];
#pragma unroll
            for (int i = 0; i < 16; ++i) p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[i], c, far) - row_lse[i]);
          } else {
#pragma unroll
            for (int i = 0; i < 16; ++i)
              p[i] = __builtin_amdgcn_exp2f(
                  __builtin_fmaf(p[i], c, centre[min(max(first - row_of(i), -s.reach), s.reach)]) - row_lse[i]);
          }
        } else {
#pragma unroll
          for (int i = 0; i < 16; ++i) p[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[i], c, -row_lse[i]));
        }
        if (s.causal && q1 < all_see) {
          const int seen_from = key - span.start - q1 - 4 * hi;   // first row that sees the lane's key
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (row_of(i) < seen_from) p[i] = 0.f;
        }
        if (BIAS && q1 + 32 > span.q) {   // (rows behind the last query are zeros, but e^bias may leave the type, and 0 times infinity is NaN)
          const int left = span.q - q1 - 4 * hi;
#pragma unroll
          for (int i = 0; i < 16; ++i)
            if (row_of(i) >= left) p[i] = 0.f;
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) ds[i] *= p[i];
        Terms<T> terms;
        terms.set(p);
        if constexpr (VL) reader.transposed_by_four(dt, 32 * u, terms, dv);
        else reader.transposed(dt, 32 * u, terms, dv);
        range.fit(ds, dk);
        terms.set(ds);
        if constexpr (VL) reader.transposed_by_four(qt, 32 * u, terms, dk);
        else reader.transposed(qt, 32 * u, terms, dk);
      }
    }
    head = next_head, q0 = next_q0;
  }

  if (key >= s.k_len) return;
  if (key >= span.k) zero(dk), zero(dv);   // (what lies behind a sequence gets zeros)
  constexpr float down = std::is_same<T, F16>::value ? 0x1p-14f : 1.f;
  const float f = key < span.k ? s.scale * range.inverse() * down : 0.f;
  if (a.k_splits == 1) {
    const size_t at = ((size_t(b) * s.k_len + key) * s.kv_heads + kv) * a.io_dim;
    store_column<T, DP>(static_cast<elem *>(a.dk) + at, dk, f, a.io_dim, hi, a.io_direct);
    store_column<T, DP>(static_cast<elem *>(a.dv) + at, dv, down, a.io_dim, hi, a.io_direct);
  } else {
    const size_t n = size_t(a.k_units) * s.k_len, at = 2 * split * n + size_t(unit) * s.k_len + key;
    store_partial<DP>(a.k_part + at * DP, dk, f, hi);
    store_partial<DP>(a.k_part + (at + n) * DP, dv, down, hi);
  }
}

// dk and dv of queries in parts: the parts' sums
template <class T, int DP>
__global__ __launch_bounds__(kBlock) void k_attn_dkv_join(BwdArgs a) {
  constexpr int TEAM = DP / 4, PER = kBlock / TEAM;
  const Shape &s = a.s;
  const size_t n = size_t(a.k_units) * s.k_len, at = size_t(blockIdx.x) * PER + threadIdx.x / TEAM;
  const int d = int(threadIdx.x % TEAM) * 4;
  if (threadIdx.x >= PER * TEAM || at >= 2 * n) return;
  sgh_v4f x = {0.f, 0.f, 0.f, 0.f};
  for (unsigned i = 0; i < a.k_splits; ++i) x += *reinterpret_cast<const sgh_v4f *>(a.k_part + (2 * i * n + at) * DP + d);
  const size_t row = at % n, unit = row / s.k_len, key = row % s.k_len, b = unit / s.kv_heads, kv = unit % s.kv_heads;
  typename T::elem *out = static_cast<typename T::elem *>(at < n ? a.dk : a.dv) + ((b * s.k_len + key) * s.kv_heads + kv) * a.io_dim;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (d + i < a.io_dim) T::St::st(out + d + i, x[i]);
}

template <class T, int DP, bool BIAS>
int launch(const BwdArgs &a, const Bounds &bounds, hipStream_t s) {
  const size_t lds = Form<T, DP>::lds(a.s.reach, BIAS);
  static std::atomic<unsigned long long> asked{0};
  SGH_HIP_TRY(sgh_allow_lds(reinterpret_cast<const void *>(k_attn_dkv<T, DP, BIAS>), asked));
  hipLaunchKernelGGL((k_attn_dkv<T, DP, BIAS>), dim3(a.k_tiles * a.k_units * a.k_splits), dim3(kBlock), lds, s, a, bounds);
  SGH_LAUNCH_CHECK();
  if (a.k_splits > 1) {
    const size_t n = 2 * size_t(a.k_units) * a.s.k_len, per = kBlock / (DP / 4);
    hipLaunchKernelGGL((k_attn_dkv_join<T, DP>), dim3(unsigned((n + per - 1) / per)), dim3(kBlock), 0, s, a);
    SGH_LAUNCH_CHECK();
  }
  return SGH_OK;
}
template <class T, int DP>
int run_dim(const BwdArgs &a, const Bounds &bounds, hipStream_t s) {
  if (a.s.buckets) return launch<T, DP, true>(a, bounds, s);
  return launch<T, DP, false>(a, bounds, s);
}

template <class T>
int run_dkv(const BwdArgs &a, const Bounds &bounds, hipStream_t s) {
  switch ((a.s.dim + 31) / 32) {
    case 1: return run_dim<T, 32>(a, bounds, s);
    case 2: return run_dim<T, 64>(a, bounds, s);
    case 3: return run_dim<T, 96>(a, bounds, s);
    default: return run_dim<T, 128>(a, bounds, s);
  }
}

// How a backward pass is cut
struct Plan {
  BwdArgs a;
  size_t stats, q_part, bias_part, k_part, wide;   // bytes
  size_t bytes() const { return stats + q_part + bias_part + k_part + wide; }
};
size_t up16(size_t n) { return (n + 15) / 16 * 16; }
// (elem_bytes: fp32 never needs less of the workspace than the others)
Plan plan_of(const sgh_attn_geom *g, size_t elem_bytes) {
  Plan p;
  BwdArgs &a = p.a;
  const size_t dp = size_t(g->dim + 31) / 32 * 32, cus = size_t(sgh_num_cus());
  const int group = g->heads / g->kv_heads;
  a.pack = !g->buckets && size_t(g->q_len) * group <= size_t(kRows) ? group : 1;
  a.q_tiles = unsigned((size_t(g->q_len) * a.pack + kRows - 1) / kRows);
  a.q_units = unsigned(size_t(g->batch) * (g->heads / a.pack));
  a.k_tiles = unsigned((size_t(g->k_len) + kRows - 1) / kRows);
  a.k_units = unsigned(size_t(g->batch) * g->kv_heads);
  // Few blocks: several to the keys of a block of queries, and to the queries of a block of keys.  The parts are the smaller the fewer blocks
  // there are (fp32, 2 x 8 heads of 64, 400 places: parts of up to 512 keys 111 us, of 256 99; 8 x 8 heads, 512 places, a block to a CU: one part
  // 148, two 156; bfloat16 heads of 128 there: 65 and 75).
  a.q_splits = a.k_splits = 1, a.keys_each = 1 << 30;
  const size_t q_blocks = size_t(a.q_tiles) * a.q_units, k_blocks = size_t(a.k_tiles) * a.k_units;
  const size_t part = q_blocks * 2 <= cus ? 256 : 512;
  if (q_blocks && q_blocks <= cus && size_t(g->k_len) > part) {
    size_t n = 2 * cus / q_blocks, most = (size_t(g->k_len) + part - 1) / part;
    if (n > most) n = most;
    a.keys_each = int(((size_t(g->k_len) + n - 1) / n + 63) / 64 * 64);
    a.q_splits = unsigned((g->k_len + a.keys_each - 1) / a.keys_each);
  }
  // (64 queries of fp32 cost four times those of 16 bits, the join the same: parts of two turns and more, fp32, 2 x 8 heads of 64, 400 places 99 ->
  // 72 us, of 128, 300 places 148 -> 115; bfloat16, 2 x 8 heads, 400 places 28 -> 31)
  const size_t turns = size_t(group) * ((size_t(g->q_len) + 63) / 64), least = elem_bytes == 4 && k_blocks * 2 <= cus ? 2 : 4;
  if (k_blocks && k_blocks <= cus && turns >= 2 * least) {
    size_t n = 2 * cus / k_blocks, most = turns / least;
    a.k_splits = unsigned(n < most ? n : most);
  }
  a.bias_blocks = size_t(g->batch) * a.q_tiles * a.q_splits;
  p.stats = up16(2 * sizeof(float) * g->batch * g->heads * size_t(g->q_len));
  p.q_part = a.q_splits > 1 ? a.q_splits * a.q_units * size_t(g->q_len) * a.pack * dp * sizeof(float) : 0;
  p.bias_part = g->buckets ? up16(a.bias_blocks * g->heads * g->buckets * sizeof(float)) : 0;
  // rows that are not whole chunks are copied first, unless each is read once
  const size_t q_rows = size_t(g->batch) * g->q_len * g->heads, k_rows = size_t(g->batch) * g->k_len * g->kv_heads;
  p.wide = a.q_tiles * (group / a.pack) >= 2 || a.k_tiles >= 2 ? 2 * wide_bytes(g->dim, q_rows) + 2 * wide_bytes(g->dim, k_rows) : 0;
  p.k_part = a.k_splits > 1 ? 2 * a.k_splits * a.k_units * size_t(g->k_len) * dp * sizeof(float) : 0;
  return p;
}

template <class T>
int backward(const sgh_attn_geom *g, const void *dout, const void *q, const void *k, const void *v, const void *o, const float *lse,
             const float *table, const int32_t *q_lengths, const int32_t *k_lengths, const int32_t *q_starts, void *dq, void *dk, void *dv,
             float *dtable, void *workspace, size_t ws_bytes, void *stream) {
  const int rc = check_geom(g);
  if (rc != SGH_OK) return rc;
  if (g->batch == 0) {   // (nothing but the table)
    if (g->buckets == 0) return SGH_OK;
    return dtable ? sgh_memset_f32(dtable, 0.f, size_t(g->buckets) * g->heads, stream) : SGH_EINVAL;
  }
  const size_t e = sizeof(typename T::elem), bq = size_t(g->batch) * g->q_len * g->heads, qn = bq * g->dim * e;
  const size_t kn = size_t(g->batch) * g->k_len * g->kv_heads * g->dim * e, tn = g->buckets ? size_t(g->buckets) * g->heads * 4 : 0;
  if (qn != 0 && (!dout || !q || !o || !lse || !dq)) return SGH_EINVAL;
  if (kn != 0 && (!k || !v || !dk || !dv)) return SGH_EINVAL;
  if (g->buckets != 0 && (!table || !dtable)) return SGH_EINVAL;
  Plan p = plan_of(g, e);
  if (p.bytes() && (!workspace || ws_bytes < p.bytes())) return SGH_EWORKSPACE;
  if (p.bytes() && !sgh_aligned16(workspace)) return SGH_EINVAL;
  const sgh_extent results[] = {{dq, qn}, {dk, kn}, {dv, kn}, {dtable, tn}, {workspace, p.bytes()}};
  const sgh_extent arguments[] = {{dout, qn}, {q, qn}, {k, kn}, {v, kn}, {o, qn}, {lse, bq * 4}, {table, tn},
                              {q_lengths, q_lengths ? size_t(g->batch) * 4 : 0}, {k_lengths, k_lengths ? size_t(g->batch) * 4 : 0},
                              {q_starts, q_starts ? size_t(g->batch) * 4 : 0}};
  if (sgh_any_overlap(results, arguments)) return SGH_EINVAL;
  BwdArgs &a = p.a;
  a.s = shape_of(g, table, q_lengths, k_lengths, q_starts);
  a.q = q, a.k = k, a.v = v, a.o = o, a.dout = dout, a.lse = lse, a.dq = dq, a.dk = dk, a.dv = dv;
  char *at = static_cast<char *>(workspace);
  a.stats = reinterpret_cast<float *>(at), at += p.stats;
  a.q_part = reinterpret_cast<float *>(at), at += p.q_part;
  a.bias_part = reinterpret_cast<float *>(at), at += p.bias_part;
  a.k_part = reinterpret_cast<float *>(at), at += p.k_part;
  a.io_dim = g->dim;
  a.direct = a.io_direct = g->dim % T::VEC == 0;
  for (const void *x : {dout, q, k, v}) a.direct = a.direct && sgh_aligned16(x);
  for (const void *x : {o, (const void *)dq, (const void *)dk, (const void *)dv}) a.io_direct = a.io_direct && sgh_aligned16(x);
  Bounds bounds;
  bounds_of(g, &bounds);
  hipStream_t s = sgh_stream_of(stream);
  sgh_note_write(dq, qn), sgh_note_write(dk, kn), sgh_note_write(dv, kn), sgh_note_write(dtable, tn);
  sgh_prof_kernel_scope prof("attn_bwd/k_attn_dq+k_attn_dkv", 10.0 * g->batch * g->heads * g->q_len * double(g->k_len) * g->dim, s);
  prof.span();
  const int wide = p.wide ? wide_of(g->dim, e) : 0;
  if (wide) {
    const size_t q_rows = bq, k_rows = size_t(g->batch) * g->k_len * g->kv_heads, row = size_t(wide) * e;
    const PadArgs pad = {{q, dout, k, v}, {at, at + q_rows * row, at + 2 * q_rows * row, at + (2 * q_rows + k_rows) * row}, {q_rows, q_rows, k_rows, k_rows},
                         g->dim, wide};
    const int r = pad_rows<T>(pad, 4, s);
    if (r != SGH_OK) return r;
    a.q = pad.to[0], a.dout = pad.to[1], a.k = pad.to[2], a.v = pad.to[3], a.s.dim = wide, a.direct = true;
  }
  if (g->q_len != 0) {
    const int r = run_dq<T>(a, bounds, dtable, s);
    if (r != SGH_OK) return r;
  } else if (g->buckets != 0) {
    const int r = sgh_memset_f32(dtable, 0.f, size_t(g->buckets) * g->heads, stream);
    if (r != SGH_OK) return r;
  }
  return g->k_len != 0 ? run_dkv<T>(a, bounds, s) : SGH_OK;
}

}  // namespace

extern "C" {

size_t sgh_attn_bwd_workspace_bytes(const sgh_attn_geom *g) {
  return attn::check_geom(g) == SGH_OK && g->batch != 0 ? plan_of(g, sizeof(float)).bytes() : 0;
}

#define SGH_ATTN_BWD(SFX, S, E)                                                                                                        \
  int sgh_attn_bwd_##SFX(const sgh_attn_geom *g, const E *dout, const E *q, const E *k, const E *v, const E *o, const float *lse,      \
                         const float *table, const int32_t *q_lengths, const int32_t *k_lengths, const int32_t *q_starts, E *dq,       \
                         E *dk, E *dv, float *dtable, void *workspace, size_t ws_bytes, void *stream) {                                \
    return backward<S>(g, dout, q, k, v, o, lse, table, q_lengths, k_lengths, q_starts, dq, dk, dv, dtable, workspace, ws_bytes,       \
                       stream);                                                                                                        \
  }
SGH_ATTN_BWD(f32, F32, float)
SGH_ATTN_BWD(f16, F16, uint16_t)
SGH_ATTN_BWD(bf16, BF16, uint16_t)
#undef SGH_ATTN_BWD

}  // extern "C"
