// Distillation from a teacher's top logits: the loss of a row of student logits x against a short list (id, teacher logit) and a label,
// and its gradient.
//
//   p_k  = softmax of teacher_k / tau over the row's list
//   loss = w (soft tau^2 sum_k p_k (log p_k - log q_k) + hard (log S_1 - (x_label - m)))
//   dx_j = scale w (soft tau (q_j - sum_{k at j} p_k) + hard (r_j - [j = label]))
//   q_j  = exp((x_j - m) / tau) / S_tau,  r_j = exp(x_j - m) / S_1,  log q_k = (x_k - m) / tau - log S_tau
//
// with m the row's maximum, S_tau and S_1 the sums of the exponentials.  The vocabulary is long and the lists are short: what counts is how
// often the logits pass through memory.  The forward pass reads them once (running maximum and sums), the gradient reads them once more and
// is written once; both in one call write the gradient behind the statistics of the same row.  Nothing of the size of the logits is kept.
// Differences to the maximum are taken before they are scaled: they are exact where they matter, and a row at the type's lowest value is
// an ordinary one.
#include "common.h"
#include "rows.h"

namespace {

constexpr int kBlock = 256;
constexpr size_t kMostDim = size_t(1) << 28;   // a row's bytes and what is asked for behind it count in 32 bits
constexpr float kLog2e = 1.44269504088896340736f;

__device__ int g_list_errors = 0;

template <class T>
struct Rows {
  const T *x;
  T *dx;
  const int32_t *top;        // [batch, k] or null
  const float *teacher;
  const int32_t *labels;     // [batch] or null
  const float *weights;      // [batch] or null
  float *loss;
  float *stats;              // [batch, 3]: m, S_tau, S_1
  size_t batch, dim;
  int k;
  float tau, soft, hard, scale;
  float inv_tau;
  bool in_place;             // dx is x
  float4 *parts;             // few long rows: of each a record, then its parts' maxima and sums
  int per_row;               // parts of a row, or 0
};
constexpr int kMostParts = SGH_WAVE;   // (a lane each where they are joined)

__device__ __forceinline__ float exp2_(float v) { return __builtin_amdgcn_exp2f(v); }

// Over 16 neighbouring lanes without LDS, then over the four sixteens through scalar registers: every lane gets the result.  (Six shuffles
// through LDS take ten times as long, and a row of a short vocabulary waits for a dozen of these.)
template <int CTRL>
__device__ __forceinline__ float lanes_of(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
constexpr int kSwap1 = 0xb1, kSwap2 = 0x4e, kHalfMirror = 0x141, kMirror = 0x140;   // lane ^ 1, ^ 2, 7 - lane of eight, 15 - lane of sixteen
__device__ __forceinline__ float lane_value(float v, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, v), lane));
}
__device__ __forceinline__ float sum16(float v) {
  v += lanes_of<kSwap1>(v);
  v += lanes_of<kSwap2>(v);
  v += lanes_of<kHalfMirror>(v);
  return v + lanes_of<kMirror>(v);
}
__device__ __forceinline__ float max16(float v) {
  v = fmaxf(v, lanes_of<kSwap1>(v));
  v = fmaxf(v, lanes_of<kSwap2>(v));
  v = fmaxf(v, lanes_of<kHalfMirror>(v));
  return fmaxf(v, lanes_of<kMirror>(v));
}
__device__ __forceinline__ float wave_sum(float v) {
  v = sum16(v);
  return (lane_value(v, 0) + lane_value(v, 16)) + (lane_value(v, 32) + lane_value(v, 48));
}
__device__ __forceinline__ float wave_max(float v) {
  v = max16(v);
  return fmaxf(fmaxf(lane_value(v, 0), lane_value(v, 16)), fmaxf(lane_value(v, 32), lane_value(v, 48)));
}

// NT threads share a row: a wavefront (a workgroup then has several rows), or the workgroup; kAny: whatever the workgroup's size
constexpr int kAny = 0, kMostThreads = 1024;
constexpr int kHeld = 16;   // vectors of a row that a thread holds
template <int NT>
struct Team {
  static constexpr int kPerBlock = NT == SGH_WAVE ? kBlock / SGH_WAVE : 1;
  static constexpr int kThreads = NT == SGH_WAVE ? kBlock : NT == kAny ? kMostThreads : NT;   // at the most
  static constexpr int kWaves = (NT == kAny ? kMostThreads : NT) / SGH_WAVE;
  static __device__ __forceinline__ unsigned size() { return NT == kAny ? blockDim.x : unsigned(NT); }
  static constexpr int kLists = NT == SGH_WAVE ? 1 : 2;   // a row's list may still be read where the next one's is fetched
  // (known to be the same for a wavefront's lanes: so are its row and what follows from that)
  static __device__ __forceinline__ int id() { return NT == SGH_WAVE ? __builtin_amdgcn_readfirstlane(int(threadIdx.x >> 6)) : 0; }
  static __device__ __forceinline__ int tid() { return NT == SGH_WAVE ? threadIdx.x & 63 : threadIdx.x; }
  // what the team's threads stored (LDS and global memory) is seen by all of them behind this
  static __device__ __forceinline__ void sync() {
    if constexpr (NT == SGH_WAVE) {
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup");
      __builtin_amdgcn_wave_barrier();
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup");
    } else {
      __syncthreads();
    }
  }
};

// A row's list beyond 64 entries, in LDS; entry k is the label
struct List {
  int *at;       // column, -1: no entry
  float *p, *x;  // the teacher's logit, later its share; the student's logit
};
__device__ __forceinline__ size_t list_bytes(int k) { return size_t(k + 1) * 12; }
__device__ __forceinline__ List list_at(char *lds, int k) {
  List l;
  l.at = reinterpret_cast<int *>(lds);
  l.p = reinterpret_cast<float *>(l.at + k + 1);
  l.x = l.p + k + 1;
  return l;
}

// What the teacher's list comes to: whether there is an entry, its largest logit, the sum of exp((logit - most) / tau)
struct Teacher {
  bool any;
  float most, sum;
};

// The label of a row, or -1; `count`: those out of range
template <class T>
__device__ __forceinline__ int checked_label(const Rows<T> &a, int label, bool count) {
  if (label < -1 || (label >= 0 && size_t(label) >= a.dim)) {
    if (count) atomicAdd(&g_list_errors, 1);
    return -1;
  }
  return label;
}

// A row's list is seen to by one wavefront of its team, in three steps, so that nothing else waits for its loads (the entries, then the student's
// logits there).  Up to 64 entries are a lane's each, in registers; a longer list goes to LDS, where the whole team ends up with it.
template <class T>
struct Entry {
  int at = -1;
  float v = 0.f, x = 0.f, p = 0.f;   // the teacher's logit, the student's, the teacher's share
  int label = -1;
  float label_x = 0.f;               // (lane 0)
  T x_raw = 0, label_raw = 0;        // as they are loaded: nothing waits for them before step 3
};
__host__ __device__ inline bool short_list(int k) { return k <= SGH_WAVE; }
// 1: the entries are asked for
template <class T>
__device__ __forceinline__ void ask_list(const Rows<T> &a, size_t row, Entry<T> &e) {
  const int lane = threadIdx.x & (SGH_WAVE - 1);
  if (a.soft != 0.f && lane < a.k) e.at = a.top[row * a.k + lane], e.v = a.teacher[row * a.k + lane];
}
// 2: they are there, and the student's logits are asked for; whether there is an entry.  `count`: those out of range
template <class T>
__device__ __forceinline__ int checked_entry(const Rows<T> &a, int at, float v, bool count) {
  if (at < -1 || (at >= 0 && size_t(at) >= a.dim)) {
    if (count) atomicAdd(&g_list_errors, 1);
    return -1;
  }
  return v == -__builtin_inff() ? -1 : at;   // (no share)
}
template <class S>
__device__ __forceinline__ bool gather_list(const Rows<typename S::elem> &a, size_t row, int label, bool count, const List &l,
                                            Entry<typename S::elem> &e) {
  const int lane = threadIdx.x & (SGH_WAVE - 1);
  const typename S::elem *x = a.x + row * a.dim;
  e.label = label;
  if (lane == 0 && label >= 0) e.label_raw = x[label];
  e.at = checked_entry(a, e.at, e.v, count);
  if (e.at >= 0) e.x_raw = x[e.at];
  bool present = e.at >= 0;
  if (!short_list(a.k)) {
    if (lane == 0) l.at[a.k] = label, l.p[a.k] = 1.f;
    l.at[lane] = e.at, l.p[lane] = e.v;
    for (int k = lane + SGH_WAVE; k < a.k; k += SGH_WAVE) {
      int at = -1;
      if (a.soft != 0.f) {
        const float v = a.teacher[row * a.k + k];
        at = checked_entry(a, a.top[row * a.k + k], v, count);
        l.p[k] = v;
        if (at >= 0) l.x[k] = S::ld(x + at), present = true;
      }
      l.at[k] = at;
    }
  }
  return __ballot(present) != 0;
}
// 3: those are there; what the teacher's logits come to
template <class S>
__device__ __forceinline__ Teacher finish_list(const Rows<typename S::elem> &a, bool any, const List &l, Entry<typename S::elem> &e) {
  if (e.at >= 0) e.x = S::ld(&e.x_raw);
  if (e.label >= 0) e.label_x = S::ld(&e.label_raw);
  const int lane = threadIdx.x & (SGH_WAVE - 1);
  Teacher t = {any, -__builtin_inff(), 0.f};
  const float c = kLog2e * a.inv_tau;
  if (short_list(a.k)) {
    if (!any) return t;
    t.most = wave_max(e.at >= 0 ? e.v : -__builtin_inff());
    t.sum = wave_sum(e.at >= 0 ? exp2_((e.v - t.most) * c) : 0.f);
    return t;
  }
  l.x[lane] = e.x;
  if (lane == 0) l.x[a.k] = e.label_x;
  if (!any) return t;
  for (int k = lane; k < a.k; k += SGH_WAVE)
    if (l.at[k] >= 0) t.most = fmaxf(t.most, l.p[k]);
  t.most = wave_max(t.most);
  for (int k = lane; k < a.k; k += SGH_WAVE)
    if (l.at[k] >= 0) t.sum += exp2_((l.p[k] - t.most) * c);
  t.sum = wave_sum(t.sum);
  return t;
}

// The teacher's shares, by the same wavefront; returns the divergence (LOSS)
template <bool LOSS, class T>
__device__ __forceinline__ float teacher_shares(const Rows<T> &a, const Teacher &t, float m, float log_st, const List &l, Entry<T> &e) {
  const int lane = threadIdx.x & (SGH_WAVE - 1);
  const float log_sum = logf(t.sum), inv = 1.f / t.sum;
  float kl = 0.f;
  auto share = [&](float v, float x) {
    const float d = (v - t.most) * a.inv_tau, p = exp2_((v - t.most) * (kLog2e * a.inv_tau)) * inv;
    if (LOSS && p != 0.f) kl += p * (d - log_sum - ((x - m) * a.inv_tau - log_st));
    return p;
  };
  if (short_list(a.k)) {
    e.p = e.at >= 0 ? share(e.v, e.x) : 0.f;
  } else {
    for (int k = lane; k < a.k; k += SGH_WAVE)
      if (l.at[k] >= 0) l.p[k] = share(l.p[k], l.x[k]);
  }
  return LOSS ? wave_sum(kl) : 0.f;
}

// Running maximum, and sums of exponentials relative to it: of d / tau where `t`, of d where `one` (tau = 1 makes one of both)
struct Running {
  float m, st, s1;
};
struct Sums {
  bool t, one;
};
// While a thread goes through its logits, its sums are relative to `ref`, which follows the maximum only when that is 2^8 above it: the sums
// stay small enough, and they are rescaled next to never (after every vector that raised the maximum of one of 64 lanes it was a tenth
// of the instructions)
struct Lane {
  float m, ref, far, st, s1;   // far: how far the maximum may be above ref
  __device__ __forceinline__ void start(float ct, Sums want) {
    m = ref = -__builtin_inff();
    st = s1 = 0.f;
    far = 8.f / (want.one ? fmaxf(ct, kLog2e) : ct);
  }
  template <int N>
  __device__ __forceinline__ void take(const float *v, float ct, Sums want) {
    if constexpr (N == 1) {
      m = fmaxf(m, v[0]);
    } else {
#pragma unroll
      for (int j = 0; j < N; j += 2) m = fmaxf(fmaxf(m, v[j]), v[j + 1]);
    }
    if (m - ref > far) {   // (at first: -inf; where all are -inf still, no)
      const float d = ref - m;
      st *= exp2_(d * ct);
      s1 *= exp2_(d * kLog2e);
      ref = m;
    }
    const float r = ref == -__builtin_inff() ? 0.f : ref;
#pragma unroll
    for (int j = 0; j < N; ++j) {
      const float d = v[j] - r;
      if (want.t) st += exp2_(d * ct);
      if (want.one) s1 += exp2_(d * kLog2e);
    }
  }
};

// The sums relative to the maximum of all; `of` is -inf where there was nothing but -inf
__device__ __forceinline__ float rebased(float sum, float of, float m, float c) { return of == m ? sum : sum * exp2_((of - m) * c); }
__device__ __forceinline__ Running wave_sums(const Lane &l, float ct) {
  const float m = wave_max(l.m);
  return {m, wave_sum(rebased(l.st, l.ref, m, ct)), wave_sum(rebased(l.s1, l.ref, m, kLog2e))};
}

// The gradient's factors of a row: dx = ft exp((x - m) / tau) + f1 exp(x - m), less the shares in the list's columns
struct Slope {
  float m, ct, ft, f1, share_t, share_1;
  bool t, one;
  __device__ __forceinline__ float operator()(float v) const {
    const float d = v - m;
    float o = 0.f;
    if (t) o = ft * exp2_(d * ct);
    if (one) o += f1 * exp2_(d * kLog2e);
    return o;
  }
};
template <class T>
__device__ __forceinline__ Slope slope_of(const Rows<T> &a, float w, const Running &r, bool soft, bool hard) {
  Slope s;
  s.m = r.m, s.ct = kLog2e * a.inv_tau;
  s.share_t = soft ? a.scale * w * a.soft * a.tau : 0.f, s.share_1 = hard ? a.scale * w * a.hard : 0.f;
  s.ft = soft ? s.share_t / r.st : 0.f, s.f1 = hard ? s.share_1 / r.s1 : 0.f;
  s.t = soft, s.one = hard;
  if (a.tau == 1.f && soft) s.f1 += s.ft, s.t = false, s.one = true;
  return s;
}

// The columns of the list once more, behind a sync: a column that is there several times is its first entry's
template <int NT, class S>
__device__ __forceinline__ void list_columns(const Rows<typename S::elem> &a, size_t row, size_t from, size_t to, const Slope &s,
                                             const List &l, const Entry<typename S::elem> &e) {
  typename S::elem *dx = a.dx + row * a.dim;
  auto mine = [&](int at) { return at >= 0 && size_t(at) >= from && size_t(at) < to; };
  if (short_list(a.k)) {
    if (Team<NT>::tid() >= SGH_WAVE) return;
    unsigned long long same = __ballot(e.at >= 0);   // lanes with this one's column
    for (unsigned rest = unsigned(a.dim - 1), b = 0; rest >> b; ++b) {
      const unsigned bit = 0u - ((unsigned(e.at) >> b) & 1u);
      const unsigned long long set = __ballot(bit != 0);
      same &= ~(set ^ ((static_cast<unsigned long long>(bit) << 32) | bit));
    }
    const int first = __builtin_amdgcn_mbcnt_hi(unsigned(same >> 32), __builtin_amdgcn_mbcnt_lo(unsigned(same), 0)) == 0;
    float p = e.p;
    if (__ballot(e.at >= 0 && __popcll(same) > 1)) {
      p = 0.f;
      for (int j = 0; j < SGH_WAVE; ++j) {
        const float of = lane_value(e.p, j);
        if (same >> j & 1) p += of;
      }
    }
    const bool labelled = e.at >= 0 && e.at == e.label;
    if (first && mine(e.at)) S::st(dx + e.at, s(e.x) - s.share_t * p - (labelled ? s.share_1 : 0.f));
    if (!__ballot(labelled) && Team<NT>::tid() == 0 && mine(e.label)) S::st(dx + e.label, s(e.label_x) - s.share_1);
    return;
  }
  for (int k = Team<NT>::tid(); k <= a.k; k += Team<NT>::size()) {
    const int at = l.at[k];
    float p = 0.f;
    bool first = true;
#pragma unroll 8
    for (int j = 0; j < a.k; ++j) {
      const bool same = l.at[j] == at;
      p += same ? l.p[j] : 0.f;
      first = first && !(same && j < k);
    }
    float o = s(l.x[k]) - s.share_t * p;
    if (l.at[a.k] == at) o -= s.share_1;
    if (first && mine(at)) S::st(dx + at, o);
  }
}

// A row's vectors through a buffer descriptor: what is behind the last of them reads as zero and is not stored, so that a load or a store needs no
// branch around it, and waiting for one of them leaves the younger ones in flight.  (The offset is all in the lane's register: the
// descriptor's limit is compared with that.)
constexpr unsigned kOutside = 0x07ffffffu;   // (times 16: 2 GB behind the row's beginning; a row has 1 GB at the most)
struct RowBuffer {
  __amdgpu_buffer_rsrc_t r;
  __device__ __forceinline__ RowBuffer(const void *p, unsigned bytes)
      : r(__builtin_amdgcn_make_buffer_rsrc(same(p), 0, __builtin_amdgcn_readfirstlane(int(bytes)), 0x00020000)) {}
  // The same for all lanes, and known to be (each access is a loop over the lanes' descriptors else)
  static __device__ __forceinline__ void *same(const void *p) {
    const uintptr_t v = reinterpret_cast<uintptr_t>(p);
    const unsigned lo = __builtin_amdgcn_readfirstlane(unsigned(v)), hi = __builtin_amdgcn_readfirstlane(unsigned(v >> 32));
    return reinterpret_cast<void *>(uintptr_t(hi) << 32 | lo);
  }
  // of `vecs` vectors behind `pad` places without one, which are asked for at kOutside instead
  static __device__ __forceinline__ RowBuffer padded(const void *first, unsigned vecs, unsigned pad) {
    return RowBuffer(static_cast<const char *>(first) - pad * 16, vecs ? (pad + vecs) * 16 : 0);
  }
  // (STREAM: past the caches, the "nt" bit)
  template <bool STREAM>
  __device__ __forceinline__ sgh_v4u load(unsigned vec) const {
    return __builtin_amdgcn_raw_buffer_load_b128(r, int(vec * 16), 0, STREAM ? 2 : 0);
  }
  template <bool STREAM>
  __device__ __forceinline__ void store(sgh_v4u v, unsigned vec) const {
    __builtin_amdgcn_raw_buffer_store_b128(v, r, int(vec * 16), 0, STREAM ? 2 : 0);
  }
};

// How a row lies: `head` elements up to the first 16-byte boundary, `vecs` vectors, and what is left.  (Vectors that begin between boundaries
// cost a sixth of the rate: 83 -> 97 us for 4096 rows of 50000 and 50001 binary16 values.)  The elements around the vectors are a thread's each:
// `odd` is this one's, or none.  `pad` vectors are missing between a 128-byte line's beginning and the first: where a gradient is stored, the
// first `pad` places of the row are no vectors, so that no line is stored in two
// parts (4096 rows of 65001 bfloat16 values: the gradient 222 -> 194 us, both in one call 243 -> 232).
struct Lie {
  unsigned head, vecs, odd, pad;
};
constexpr unsigned kNone = 0xffffffffu;
constexpr unsigned kLine = 128;
template <class S>
__device__ __forceinline__ Lie lie_of(const typename S::elem *x, unsigned dim, unsigned tid) {
  constexpr unsigned V = S::VEC, e = sizeof(typename S::elem);
  const unsigned off = unsigned(reinterpret_cast<uintptr_t>(x)) & 15u;
  Lie l;
  l.head = ((16u - off) & 15u) / e;
  if (l.head > dim) l.head = dim;
  l.vecs = (dim - l.head) / V;
  const unsigned behind = l.head + l.vecs * V, left = dim - behind;
  l.odd = tid < l.head ? tid : tid >= V && tid - V < left ? behind + tid - V : kNone;
  l.pad = unsigned(reinterpret_cast<uintptr_t>(x + l.head)) % kLine / 16;
  return l;
}
template <class S>
__device__ __forceinline__ void unpack(const sgh_v4u &raw, float *v) {
  sgh_load_any<S, S::VEC>(reinterpret_cast<const typename S::elem *>(&raw), v);
}
template <class S>
__device__ __forceinline__ sgh_v4u packed(const float *v) {
  sgh_v4u o;
  sgh_store_any<S, S::VEC>(reinterpret_cast<typename S::elem *>(&o), v);
  return o;
}

// A row's vectors, U of a thread at a time and the next U in flight: f(vector, its number, whether every thread of the team has one)
constexpr int kAhead = 4;
template <int NT, bool STREAM>
__device__ __forceinline__ void ask_vectors(const RowBuffer &x, unsigned from, sgh_v4u *v, unsigned pad = 0) {
#pragma unroll
  for (int u = 0; u < kAhead; ++u) {
    const unsigned i = from + u * NT + Team<NT>::tid();
    v[u] = x.load<STREAM>(u == 0 && i < pad ? kOutside : i);
  }
}
template <int NT, bool STREAM, class F>
__device__ __forceinline__ void stream_row(const RowBuffer &x, unsigned vecs, sgh_v4u *v, F f) {
  for (unsigned c = 0; c < vecs; c += kAhead * NT) {
    sgh_v4u then[kAhead];
    ask_vectors<NT, STREAM>(x, c + kAhead * NT, then);
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (c + u * NT < vecs) f(v[u], c + u * NT + Team<NT>::tid(), c + (u + 1) * NT <= vecs);
#pragma unroll
    for (int u = 0; u < kAhead; ++u) v[u] = then[u];
  }
}

// A vector into a thread's sums; `all`: every thread of the team has one
template <class S>
__device__ __forceinline__ void take_vector(Lane &sum, const sgh_v4u &raw, unsigned vec, unsigned vecs, bool all, float ct, Sums want) {
  float v[S::VEC];
  unpack<S>(raw, v);
  if (!all) {
#pragma unroll
    for (int j = 0; j < S::VEC; ++j) v[j] = vec < vecs ? v[j] : -__builtin_inff();
  }
  sum.take<S::VEC>(v, ct, want);
}
template <class S>
__device__ __forceinline__ sgh_v4u slope_vector(const Slope &s, const sgh_v4u &raw) {
  float v[S::VEC];
  unpack<S>(raw, v);
#pragma unroll
  for (int j = 0; j < S::VEC; ++j) v[j] = s(v[j]);
  return packed<S>(v);
}

// dx of a row's vectors [from, from + vecs) but for the list's columns, from memory (dx may be x: a thread stores what it has read); `none`: zeros
template <int NT, class S, bool STREAM>
__device__ __forceinline__ void slope_row(const typename S::elem *x, typename S::elem *dx, unsigned vecs, unsigned pad, bool none,
                                          const Slope &s) {
  const RowBuffer from = RowBuffer::padded(x, none ? 0 : vecs, pad), to = RowBuffer::padded(dx, vecs, pad);
  sgh_v4u v[kAhead];
  ask_vectors<NT, STREAM>(from, 0, v, pad);
  stream_row<NT, STREAM>(from, vecs ? pad + vecs : 0, v,
                         [&](const sgh_v4u &raw, unsigned i, bool) { to.store<STREAM>(slope_vector<S>(s, raw), i < pad ? kOutside : i); });
}

// The statistics of a whole row
template <class T>
__device__ __forceinline__ Running of_row(const Rows<T> &a, Running r) {
  if (r.m == -__builtin_inff()) r.st = r.s1 = __builtin_nanf("");   // (no column with a probability)
  if (a.tau == 1.f) r.st = r.s1;
  return r;
}
// The team's statistics from its threads'; `red`: one of each wavefront
template <int NT>
__device__ __forceinline__ Running team_sums(const Lane &lane, float ct, Running *red) {
  Running r = wave_sums(lane, ct);
  constexpr int W = Team<NT>::kWaves;
  static_assert(W <= 16, "a lane of sixteen takes a wavefront's");
  if constexpr (W > 1) {
    if ((threadIdx.x & (SGH_WAVE - 1)) == 0) red[threadIdx.x >> 6] = r;
    __syncthreads();
    const unsigned of = threadIdx.x & 15;
    r = of < Team<NT>::size() / SGH_WAVE ? red[of] : Running{-__builtin_inff(), 0.f, 0.f};
    const float m = max16(r.m);
    r = {m, sum16(rebased(r.st, r.m, m, ct)), sum16(rebased(r.s1, r.m, m, kLog2e))};
  }
  return r;
}

// Loss and statistics of a row, by the wavefront that sees to its list; the teacher's shares are in the list then
template <class T>
__device__ __forceinline__ void store_loss(const Rows<T> &a, size_t row, float w, const Running &r, bool soft, bool hard,
                                           const Teacher &teach, const List &list, Entry<T> &entry) {
  float loss = 0.f;
  if (soft) loss = a.soft * a.tau * a.tau * teacher_shares<true>(a, teach, r.m, logf(r.st), list, entry);
  if ((threadIdx.x & (SGH_WAVE - 1)) != 0) return;
  if (hard) loss += a.hard * (logf(r.s1) - (entry.label_x - r.m));
  a.loss[row] = soft || hard ? w * loss : 0.f;
  if (a.stats) {
    a.stats[row * 3] = soft || hard ? r.m : 0.f;
    a.stats[row * 3 + 1] = soft ? r.st : 0.f;
    a.stats[row * 3 + 2] = hard ? r.s1 : 0.f;
  }
}

// What a row asks for, known before its logits
struct Row {
  float w;
  int label;
  bool may_soft, hard;   // (whether the list has an entry is seen later)
  __device__ __forceinline__ bool any() const { return may_soft || hard; }
};
template <class T>
__device__ __forceinline__ Row row_at(const Rows<T> &a, size_t row, bool count) {
  Row r;
  r.w = a.weights ? a.weights[row] : 1.f;
  r.label = a.labels && a.hard != 0.f ? checked_label(a, a.labels[row], count) : -1;
  r.hard = r.label >= 0 && r.w != 0.f;
  r.may_soft = a.k && a.soft != 0.f && r.w != 0.f;
  return r;
}

// The loss and statistics of a row; GRAD: and its gradient, for which the row is read again, mostly from the last-level cache.  Bound by memory: the
// loss of 4096 rows of 50001 binary16 values 83 us, 4.9 TB/s; with the gradient, 8192 rows of 131072 bfloat16 values 900 us: 4.2 GB that have to move,
// 6.1 that do, 6.2 to 6.8 TB/s.  16 rows of 10007 are a launch and a row's chain of loads, 5.2 us.
template <int NT, class S, bool GRAD, bool STREAM>
__global__ __launch_bounds__(Team<NT>::kThreads) void k_distill_fwd(Rows<typename S::elem> a) {
  typedef Team<NT> G;
  typedef typename S::elem T;
  extern __shared__ char lds[];
  __shared__ Running red[G::kWaves];
  __shared__ int listed;
  const int tid = G::tid();
  const bool lister = tid < SGH_WAVE;
  const float ct = kLog2e * a.inv_tau;
  const size_t step = size_t(gridDim.x) * G::kPerBlock;
  int turn = 0;
  for (size_t row = size_t(blockIdx.x) * G::kPerBlock + G::id(); row < a.batch; row += step) {
    const T *x = a.x + row * a.dim;
    const Lie lie = lie_of<S>(x, unsigned(a.dim), tid);
    const unsigned vecs = lie.vecs;
    // everything is asked for at once, the first vectors of a row that turns out to want nothing as well
    Entry<T> entry;
    if (lister) ask_list(a, row, entry);
    T end = 0;
    if (lie.odd != kNone) end = x[lie.odd];
    const RowBuffer from(x + lie.head, vecs * 16);
    sgh_v4u v[kAhead];
    const Row q = row_at(a, row, tid == 0);
    ask_vectors<NT, STREAM && !GRAD>(from, 0, v);
    const List list = list_at(lds + (G::id() * G::kLists + turn) * list_bytes(a.k), a.k);
    bool any = false;
    if (lister) {   // (entries out of range are counted whatever the weight)
      any = gather_list<S>(a, row, q.hard ? q.label : -1, true, list, entry);
      if (NT != SGH_WAVE && tid == 0) listed = any;
    }
    const Sums want = {q.may_soft && a.tau != 1.f, q.hard || (q.may_soft && a.tau == 1.f)};
    Running r = {0.f, 0.f, 0.f};
    bool soft = false;
    if (q.any()) {
      Lane sum;
      sum.start(ct, want);
      stream_row<NT, STREAM && !GRAD>(
          from, vecs, v, [&](const sgh_v4u &raw, unsigned vec, bool all) { take_vector<S>(sum, raw, vec, vecs, all, ct, want); });
      const float tail = S::ld(&end);
      if (lie.odd != kNone) sum.take<1>(&tail, ct, want);
      r = of_row(a, team_sums<NT>(sum, ct, red));
      soft = q.may_soft && (NT == SGH_WAVE ? any : listed != 0);
    }
    if (lister) {
      const Teacher teach = finish_list<S>(a, any, list, entry);
      store_loss(a, row, q.w, r, soft, q.hard, teach, list, entry);
    }
    if constexpr (GRAD) {
      const Slope s = slope_of(a, q.w, r, soft, q.hard);
      const bool none = !(soft || q.hard);
      if (NT != SGH_WAVE) G::sync();   // (the list's logits are read: dx may be x)
      slope_row<NT, S, STREAM>(x + lie.head, a.dx + row * a.dim + lie.head, vecs, lie.pad, none, s);
      if (lie.odd != kNone) S::st(a.dx + row * a.dim + lie.odd, s(S::ld(&end)));
      G::sync();
      if (!none) list_columns<NT, S>(a, row, 0, a.dim, s, list, entry);
    } else {
      G::sync();   // (`red` and `listed` are read)
    }
    turn = (turn + 1) % G::kLists;
  }
}

// Few long rows are cut in `per_row` parts, a workgroup each, whose statistics go to memory, and the next launch joins them.  What the list and
// the label give to the loss is known but for those statistics: with `top` the largest of the student's logits there,
//   sum_k p_k (log p_k - log q_k) = kl - (top - m) / tau + log S_tau,   kl = sum_k p_k (log p_k - (x_k - top) / tau)
// so that the record of a row is {whether there is an entry, kl, top, x_label}.
template <class T>
__device__ __forceinline__ float4 row_record(const Rows<T> &a, const Teacher &t, const List &l, const Entry<T> &e) {
  const int lane = threadIdx.x & (SGH_WAVE - 1);
  const float log_sum = logf(t.sum), inv = 1.f / t.sum;
  auto share = [&](float v) { return exp2_((v - t.most) * (kLog2e * a.inv_tau)) * inv; };
  auto each = [&](auto f) {   // f(the teacher's logit, the student's) for every entry with a share
    if (short_list(a.k)) {
      if (e.at >= 0 && share(e.v) != 0.f) f(e.v, e.x);
    } else {
      for (int k = lane; k < a.k; k += SGH_WAVE)
        if (l.at[k] >= 0 && share(l.p[k]) != 0.f) f(l.p[k], l.x[k]);
    }
  };
  float top = -__builtin_inff(), kl = 0.f;
  each([&](float, float x) { top = fmaxf(top, x); });
  top = wave_max(top);
  each([&](float v, float x) { kl += share(v) * ((v - t.most) * a.inv_tau - log_sum - (x - top) * a.inv_tau); });
  kl = wave_sum(kl);
  if (top == -__builtin_inff()) kl = __builtin_inff(), top = 0.f;   // (the student gives none of them a probability)
  return {t.any ? 1.f : 0.f, kl, top, e.label_x};
}
template <class S>
__global__ __launch_bounds__(kBlock) void k_distill_part(Rows<typename S::elem> a, unsigned each) {
  typedef typename S::elem T;
  constexpr int NT = kBlock;
  extern __shared__ char lds[];
  __shared__ Running red[NT / SGH_WAVE];
  const unsigned part = blockIdx.y;
  const bool lister = part == 0 && threadIdx.x < SGH_WAVE, begins = part == 0, ends = part + 1 == gridDim.y;
  const float ct = kLog2e * a.inv_tau;
  const size_t row = blockIdx.x;
  const T *x = a.x + row * a.dim;
  const Lie lie = lie_of<S>(x, unsigned(a.dim), threadIdx.x);
  const unsigned first = part * each < lie.vecs ? part * each : lie.vecs, vecs = lie.vecs - first < each ? lie.vecs - first : each;
  const bool odd = lie.odd != kNone && (lie.odd < lie.head ? begins : ends);
  Entry<T> entry;
  if (lister) ask_list(a, row, entry);
  T end = 0;
  if (odd) end = x[lie.odd];
  const RowBuffer from(x + lie.head + size_t(first) * S::VEC, vecs * 16);
  sgh_v4u v[kAhead];
  const Row q = row_at(a, row, begins && threadIdx.x == 0);
  ask_vectors<NT, false>(from, 0, v);
  const List list = list_at(lds, a.k);
  bool any = false;
  if (lister) any = gather_list<S>(a, row, q.hard ? q.label : -1, true, list, entry);
  float4 *out = a.parts + row * (a.per_row + 1);
  if (q.any()) {
    const Sums want = {q.may_soft && a.tau != 1.f, q.hard || (q.may_soft && a.tau == 1.f)};
    Lane sum;
    sum.start(ct, want);
    stream_row<NT, false>(
        from, vecs, v, [&](const sgh_v4u &raw, unsigned vec, bool all) { take_vector<S>(sum, raw, vec, vecs, all, ct, want); });
    const float tail = S::ld(&end);
    if (odd) sum.take<1>(&tail, ct, want);
    const Running r = team_sums<NT>(sum, ct, red);
    if (threadIdx.x == 0) out[1 + part] = {r.m, r.st, r.s1, 0.f};
  }
  if (lister) {
    const Teacher teach = finish_list<S>(a, any, list, entry);
    float4 rec = {0.f, 0.f, 0.f, entry.label_x};
    if (any) rec = row_record(a, teach, list, entry);
    if (threadIdx.x == 0) out[0] = rec;
  }
}
// A row's statistics from its parts', by every wavefront that asks
template <class T>
__device__ __forceinline__ Running joined(const Rows<T> &a, size_t row, float4 *record) {
  const int lane = threadIdx.x & (SGH_WAVE - 1);
  const float4 *p = a.parts + row * (a.per_row + 1);
  *record = p[0];
  const float4 of = lane < a.per_row ? p[1 + lane] : float4{-__builtin_inff(), 0.f, 0.f, 0.f};
  const float m = wave_max(of.x);
  return of_row(a, {m, wave_sum(rebased(of.y, of.x, m, kLog2e * a.inv_tau)), wave_sum(rebased(of.z, of.x, m, kLog2e))});
}
template <class T>
__device__ __forceinline__ void store_joined(const Rows<T> &a, size_t row, float w, const Running &r, bool soft, bool hard, const float4 &record) {
  float loss = 0.f;
  if (soft) loss = a.soft * a.tau * a.tau * (record.y - (record.z - r.m) * a.inv_tau + logf(r.st));
  if (hard) loss += a.hard * (logf(r.s1) - (record.w - r.m));
  a.loss[row] = soft || hard ? w * loss : 0.f;
  if (a.stats) {
    a.stats[row * 3] = soft || hard ? r.m : 0.f;
    a.stats[row * 3 + 1] = soft ? r.st : 0.f;
    a.stats[row * 3 + 2] = hard ? r.s1 : 0.f;
  }
}
// The loss of rows in parts, a wavefront each
template <class T>
__global__ __launch_bounds__(SGH_WAVE) void k_distill_join(Rows<T> a) {
  const size_t row = blockIdx.x;
  const Row q = row_at(a, row, false);
  float4 record;
  const Running r = joined(a, row, &record);
  if (threadIdx.x == 0) store_joined(a, row, q.w, r, q.may_soft && record.x != 0.f, q.hard, record);
}

// Both for rows of at most U * NT vectors, in registers: what bounds it is the logits' way in and the gradient's out.  A workgroup for each row (a
// wavefront, of short ones), so that one's loads are in flight beside another's sums and stores.  (Going from row to row instead, with the
// next row's loads behind this one's stores, these waited for the stores: 530 and 450 us for 16384 rows of 20001 fp32 values, 207 and 186
// for 4096 of 50304 bfloat16.)  2048 rows of 65001 bfloat16 values, labels alone: 106 us; 4096 of 32000, with lists: 106 us, 4.9 TB/s.
template <int NT, int U, int PER_SIMD, class S, bool STREAM>
__global__ __launch_bounds__(Team<NT>::kThreads, PER_SIMD) void k_distill_held(Rows<typename S::elem> a) {
  typedef Team<NT> G;
  typedef typename S::elem T;
  extern __shared__ char lds[];
  __shared__ Running red[G::kWaves];
  __shared__ int listed;
  const int tid = G::tid();
  const unsigned nt = G::size();
  const bool lister = tid < SGH_WAVE;   // the wavefront that sees to the list
  const float ct = kLog2e * a.inv_tau;
  const size_t row = size_t(blockIdx.x) * G::kPerBlock + G::id();
  if (row >= a.batch) return;
  const T *x = a.x + row * a.dim;
  T *dx = a.dx + row * a.dim;
  const Lie lie = lie_of<S>(x, unsigned(a.dim), tid);
  const unsigned first = unsigned(tid) < lie.pad ? kOutside : unsigned(tid), places = lie.pad + lie.vecs;
  // what is small is asked for in front of the row's vectors: loads come back in order
  Entry<T> entry;
  if (lister) ask_list(a, row, entry);
  const Row q = row_at(a, row, tid == 0);
  const RowBuffer from = RowBuffer::padded(x + lie.head, q.any() ? lie.vecs : 0, lie.pad), to = RowBuffer::padded(dx + lie.head, lie.vecs, lie.pad);
  sgh_v4u held[U];
#pragma unroll
  for (int u = 0; u < U; ++u) held[u] = from.load<STREAM>(u == 0 ? first : u * nt + tid);
  T end = 0;
  if (lie.odd != kNone) end = x[lie.odd];
  const List list = list_at(lds + G::id() * list_bytes(a.k), a.k);
  bool any = false;
  if (lister) {   // (entries out of range are counted whatever the weight)
    any = gather_list<S>(a, row, q.hard ? q.label : -1, true, list, entry);
    if (NT != SGH_WAVE && tid == 0) listed = any;
  }
  const Sums want = {q.may_soft && a.tau != 1.f, q.hard || (q.may_soft && a.tau == 1.f)};
  Running r = {0.f, 0.f, 0.f};
  bool soft = false;
  if (q.any()) {
    Lane sum;
    sum.start(ct, want);
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (u * nt < places) {
        const bool all = (u != 0 || lie.pad == 0) && (u + 1) * nt <= places;
        take_vector<S>(sum, held[u], u == 0 ? first : u * nt + tid, places, all, ct, want);
      }
    const float tail = S::ld(&end);
    if (lie.odd != kNone) sum.take<1>(&tail, ct, want);
    r = of_row(a, team_sums<NT>(sum, ct, red));
    soft = q.may_soft && (NT == SGH_WAVE ? any : listed != 0);
  }
  if (lister) {
    const Teacher teach = finish_list<S>(a, any, list, entry);
    store_loss(a, row, q.w, r, soft, q.hard, teach, list, entry);
  }
  const Slope s = slope_of(a, q.w, r, soft, q.hard);
  if (a.in_place && NT != SGH_WAVE) G::sync();   // (the list's logits are read)
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (u * nt < places) held[u] = slope_vector<S>(s, held[u]);   // (nothing but arithmetic in the branch)
    to.store<STREAM>(held[u], u == 0 ? first : u * nt + tid);
  }
  if (lie.odd != kNone) S::st(dx + lie.odd, s(S::ld(&end)));
  G::sync();
  if (soft || q.hard) list_columns<NT, S>(a, row, 0, a.dim, s, list, entry);
}

// The gradient from the statistics, or (PARTS) from a row's parts, whose loss it stores then; a row may be several workgroups', `each` vectors of it
// Bound by memory: 8192 rows of 65536 bfloat16 values 364 us, 5.7 TB/s.  (Registers for 7 wavefronts of a SIMD where teams are small: 16384 rows of
// 5000 bfloat16 values 98.8 -> 83.1 us.  Rows in parts are few: no such limit, which the joining would not fit.)
template <int NT, class S, bool STREAM, bool PARTS>
__global__ __launch_bounds__(Team<NT>::kThreads, NT <= kBlock && !PARTS ? 7 : 4) void k_distill_bwd(Rows<typename S::elem> a, unsigned each) {
  typedef Team<NT> G;
  typedef typename S::elem T;
  extern __shared__ char lds[];
  const int tid = G::tid();
  const bool lister = tid < SGH_WAVE;
  const size_t step = size_t(gridDim.x) * G::kPerBlock;
  int turn = 0;
  for (size_t row = size_t(blockIdx.x) * G::kPerBlock + G::id(); row < a.batch; row += step) {
    const T *x = a.x + row * a.dim;
    T *dx = a.dx + row * a.dim;
    // this workgroup's vectors, the first one's with the elements in front, the last one's with those behind
    const Lie lie = lie_of<S>(x, unsigned(a.dim), tid);
    const unsigned first = blockIdx.y * each < lie.vecs ? blockIdx.y * each : lie.vecs, vecs = lie.vecs - first < each ? lie.vecs - first : each;
    const bool begins = blockIdx.y == 0, ends = blockIdx.y + 1 == gridDim.y;
    const size_t start = lie.head + size_t(first) * S::VEC, from = begins ? 0 : start, to = ends ? a.dim : start + size_t(vecs) * S::VEC;
    const bool odd = lie.odd != kNone && (lie.odd < lie.head ? begins : ends);
    Entry<T> entry;
    if (lister) ask_list(a, row, entry);
    T end = 0;
    if (odd) end = x[lie.odd];
    const Row q = row_at(a, row, false);
    Running r;
    bool soft = q.may_soft, hard = q.hard;
    if constexpr (PARTS) {
      float4 record;
      r = joined(a, row, &record);
      soft = soft && record.x != 0.f;
      if (begins && tid == 0) store_joined(a, row, q.w, r, soft, hard, record);
    } else {   // (a sum of 0: the forward pass found no term)
      r = {a.stats[row * 3], a.stats[row * 3 + 1], a.stats[row * 3 + 2]};
      soft = soft && r.st != 0.f, hard = hard && r.s1 != 0.f;
    }
    const bool none = !(soft || hard);
    const Slope s = slope_of(a, q.w, r, soft, hard);
    const List list = list_at(lds + (G::id() * G::kLists + turn) * list_bytes(a.k), a.k);
    bool any = false;
    if (lister && !none) any = gather_list<S>(a, row, hard ? q.label : -1, false, list, entry);
    auto shares = [&]() {
      if (!lister || none) return;
      const Teacher t = finish_list<S>(a, any, list, entry);
      if (soft) teacher_shares<false>(a, t, 0.f, 0.f, list, entry);
    };
    if (a.in_place) {   // (the list's logits are read before any is stored over)
      shares();
      if (NT != SGH_WAVE) G::sync();
    }
    slope_row<NT, S, STREAM>(x + start, dx + start, vecs, begins ? lie.pad : 0, none, s);
    if (odd) S::st(dx + lie.odd, s(S::ld(&end)));
    if (!a.in_place) shares();
    G::sync();
    if (!none) list_columns<NT, S>(a, row, from, to, s, list, entry);
    turn = (turn + 1) % G::kLists;
  }
}

template <int NT>
size_t lds_for(int k) {
  return short_list(k) ? 0 : size_t(Team<NT>::kPerBlock) * Team<NT>::kLists * (k + 1) * 12;
}
template <int NT>
unsigned blocks_for(size_t batch, size_t most) {
  const size_t n = (batch + Team<NT>::kPerBlock - 1) / Team<NT>::kPerBlock;
  return unsigned(n < most ? n : most);
}
template <class T>
bool streams(const Rows<T> &a) { return a.batch * a.dim * sizeof(T) >= kStreamBytes; }
template <int NT, class S, bool GRAD>
int launch_fwd(const Rows<typename S::elem> &a, hipStream_t s) {
  const dim3 grid{blocks_for<NT>(a.batch, size_t(1) << 20)}, block{unsigned(Team<NT>::kThreads)};
  constexpr bool small = NT == 512 && !GRAD;   // (the loss: at most half as many rows as CUs, of 40000 columns)
  if (!small && streams(a)) SGH_LAUNCH_TIMED((k_distill_fwd<NT, S, GRAD, !small>), grid, block, lds_for<NT>(a.k), s, a);
  else SGH_LAUNCH_TIMED((k_distill_fwd<NT, S, GRAD, false>), grid, block, lds_for<NT>(a.k), s, a);
  SGH_LAUNCH_CHECK();
  return SGH_OK;
}
constexpr size_t kRowsOfLaunch = size_t(1) << 20;   // (a launch has less than 2^32 threads)
template <int NT, int U, int PER_SIMD, class S>
int launch_held(Rows<typename S::elem> a, unsigned threads, hipStream_t s) {
  constexpr bool small = NT == kAny && U == 4;   // (at most 24 wavefronts' rows for each CU, 4 KB a wavefront)
  const bool stream = !small && streams(a);
  const size_t batch = a.batch, most = kRowsOfLaunch;
  for (size_t row = 0; row < batch; row += most) {
    a.batch = batch - row < most ? batch - row : most;
    const dim3 grid{blocks_for<NT>(a.batch, a.batch)}, block{threads};
    if (stream) SGH_LAUNCH_TIMED((k_distill_held<NT, U, PER_SIMD, S, !small>), grid, block, lds_for<NT>(a.k), s, a);
    else SGH_LAUNCH_TIMED((k_distill_held<NT, U, PER_SIMD, S, false>), grid, block, lds_for<NT>(a.k), s, a);
    SGH_LAUNCH_CHECK();
    a.x += a.batch * a.dim, a.dx += a.batch * a.dim, a.loss += a.batch;
    if (a.k) a.top += a.batch * a.k, a.teacher += a.batch * a.k;
    if (a.labels) a.labels += a.batch;
    if (a.weights) a.weights += a.batch;
  }
  return SGH_OK;
}
template <class S>
int launch_parts(const Rows<typename S::elem> &a, hipStream_t s) {
  const unsigned vecs = unsigned(a.dim / S::VEC), each = (vecs + a.per_row - 1) / a.per_row;
  const dim3 grid{unsigned(a.batch), unsigned(a.per_row)};
  hipLaunchKernelGGL((k_distill_part<S>), grid, dim3(kBlock), lds_for<kBlock>(a.k), s, a, each);
  SGH_LAUNCH_CHECK();
  return SGH_OK;
}
template <int NT, class S>
int launch_bwd(const Rows<typename S::elem> &a, unsigned each, hipStream_t s) {
  const unsigned vecs = unsigned(a.dim / S::VEC), ny = vecs > each ? (vecs + each - 1) / each : 1;
  const dim3 grid{blocks_for<NT>(a.batch, size_t(1) << 20), ny}, block{unsigned(Team<NT>::kThreads)};
  constexpr bool parts = NT != SGH_WAVE;   // (rows in parts are long)
  if (parts && a.per_row) SGH_LAUNCH_TIMED((k_distill_bwd<NT, S, false, parts>), grid, block, lds_for<NT>(a.k), s, a, each);   // (past no cache: read again)
  else if (streams(a)) SGH_LAUNCH_TIMED((k_distill_bwd<NT, S, true, false>), grid, block, lds_for<NT>(a.k), s, a, each);
  else SGH_LAUNCH_TIMED((k_distill_bwd<NT, S, false, false>), grid, block, lds_for<NT>(a.k), s, a, each);
  SGH_LAUNCH_CHECK();
  return SGH_OK;
}

// Parts that a row is cut in for the loss, 0: none.  Two launches that have the whole chip for few rows, against one that has a CU for each: a
// row of 262144 bfloat16 values 26 -> 7 us, with its gradient 54 -> 10, 64 rows 27 -> 14 and 56 -> 28; 128 rows of 131072 15.9 -> 13.5 and 32.0 ->
// 28.8.  Short rows have one launch.  The border counts elements, not bytes: a workgroup waits for its row's exponentials as much as for the row.
// One launch and parts, us, 16 rows: the loss of 28000 fp32 values 7.2 and 7.4, of 40000 8.4 and 7.4; of 40000 bfloat16 values 7.2 and 7.3, of 56000 8.6
// and 7.3; with the gradient, 20001 fp32 values 8.9 and 10.1, 28000 10.5 and 10.0, 40000 13.6 and 10.2; 28000 bfloat16 values 9.9 and 10.6, 40000 12.8
// and 11.1.  128 rows gain less (56000 bfloat16 values with the gradient 17.4 and 16.4) and some lose: 48000 fp32 values with it 16.3 and 20.1.
int parts_of(size_t batch, size_t dim, size_t elem, bool grad) {
  const size_t vecs = dim * elem / 16, cus = size_t(sgh_num_cus());
  if (batch * 2 > cus || dim <= (grad ? 28000 : 40000)) return 0;
  size_t n = (4 * cus + batch - 1) / batch;
  const size_t most = vecs / (kBlock * kAhead);   // a turn of every thread at the least (3 parts and more)
  if (n > most) n = most;
  return int(n < size_t(kMostParts) ? n : size_t(kMostParts));
}
size_t parts_bytes(size_t batch, int per_row) { return per_row ? batch * size_t(per_row + 1) * sizeof(float4) : 0; }

// The checks that the three entry points share; SGH_OK with `empty` set where there is nothing to do
template <class T>
int check(const Rows<T> &a, size_t k, bool fwd, bool grad, bool *empty) {
  *empty = false;
  if (a.batch > 0x7fffffffu || a.dim > kMostDim) return SGH_EINVAL;
  if (!(a.tau > 0.f) || !__builtin_isfinite(a.tau * a.tau) || !__builtin_isfinite(kLog2e / a.tau)) return SGH_EINVAL;
  if (k > SGH_DISTILL_MAX_TOP) return SGH_ELIMIT;
  if (a.batch == 0) return *empty = true, SGH_OK;
  if (a.dim == 0) return SGH_EINVAL;   // (a row of no logits has no softmax)
  if (!a.x || (k != 0 && (!a.top || !a.teacher))) return SGH_EINVAL;
  if (fwd && !a.loss) return SGH_EINVAL;
  if ((!fwd || !grad) && !a.stats) return SGH_EINVAL;
  if (grad && !a.dx) return SGH_EINVAL;
  // no result lies over an argument or another result, but for dx over the whole of x
  const size_t bytes = a.batch * a.dim * sizeof(T), lists = a.batch * k * 4, each = a.batch * 4;
  struct {
    const void *p;
    size_t bytes;
  } const of[] = {{a.dx, grad ? bytes : 0}, {a.loss, fwd ? each : 0}, {a.stats, a.stats ? 3 * each : 0}, {a.x, bytes}, {a.top, lists},
                  {a.teacher, lists}, {a.labels, a.labels ? each : 0}, {a.weights, a.weights ? each : 0}};
  const int results = fwd ? 3 : 1;   // (the gradient alone reads stats)
  for (int i = 0; i < results; ++i)
    for (int j = i + 1; j < int(sizeof(of) / sizeof(of[0])); ++j)
      if (sgh_ranges_meet(of[i].p, of[i].bytes, of[j].p, of[j].bytes) && !(i == 0 && of[j].p == a.x && a.dx == a.x))
        return SGH_EINVAL;
  return SGH_OK;
}

template <class S>
int distill(Rows<typename S::elem> a, size_t k, bool fwd, bool grad, void *workspace, size_t ws_bytes, void *stream) {
  bool empty;
  const int rc = check(a, k, fwd, grad, &empty);
  if (rc != SGH_OK || empty) return rc;
  a.k = int(k);
  a.per_row = fwd ? parts_of(a.batch, a.dim, sizeof(typename S::elem), grad) : 0;
  if (a.per_row) {
    if (!workspace || ws_bytes < parts_bytes(a.batch, a.per_row)) return SGH_EWORKSPACE;
    if (reinterpret_cast<uintptr_t>(workspace) % alignof(float4) != 0) return SGH_EINVAL;
    a.parts = static_cast<float4 *>(workspace);
  }
  a.in_place = grad && a.dx == a.x;
  a.inv_tau = 1.f / a.tau;
  hipStream_t s = sgh_stream_of(stream);
  const double bytes = double(a.batch) * a.dim * sizeof(typename S::elem);
  if (grad) sgh_note_write(a.dx, a.batch * a.dim * sizeof(typename S::elem));
  sgh_prof_kernel_scope prof(fwd && grad ? "distill/k_distill_fwd" : fwd ? "distill_fwd/k_distill_fwd" : "distill_bwd/k_distill_bwd",
                             bytes * (grad ? 2 : 1), s);
  const size_t vecs = a.dim / S::VEC, cus = size_t(sgh_num_cus());
  if (a.per_row) {
    prof.span();
    const int failed = launch_parts<S>(a, s);
    if (failed != SGH_OK) return failed;
    if (!grad) {
      hipLaunchKernelGGL((k_distill_join<typename S::elem>), dim3(unsigned(a.batch)), dim3(SGH_WAVE), 0, s, a);
      SGH_LAUNCH_CHECK();
      return SGH_OK;
    }
  } else if (fwd && grad) {
    // places of a row's vectors
    const bool lines = (reinterpret_cast<uintptr_t>(a.x) | a.dim * sizeof(typename S::elem)) % kLine == 0;
    const size_t places = lines ? vecs : vecs + kLine / 16 - 1;
    if (a.batch > kRowsOfLaunch) prof.span();
    if (places <= size_t(kMostThreads) * kHeld) {
      // Vectors of a thread.  4, the shortest way through a row, while the wavefronts find room at once (1 row of 20001 bfloat16 values: 8.1 us, with
      // 16 10.9; 1024 rows with 4, 8, 16: 31.8, 25.3, 27.7).  Then 8, 12 or 16, the fewest that leave a SIMD two of the workgroup's wavefronts, so
      // that two workgroups and more fit a CU (4096 rows of 32000 with 8: 106 us, with 4 145; of 40000 with 8, 12: 161, 145; of 45000 with 12, 16:
      // 145, 200).  A wavefront for rows of up to 256 vectors: a workgroup's sum costs a microsecond.  Rows that leave no room for two
      // workgroups are read twice, from cache the second time, by workgroups that hold nothing (2048 rows of 70001: 135 us, in registers 178; of
      // 65001, which do leave room, 126 and 107), unless there are few.
      auto waves = [&](size_t held) { return unsigned((places + SGH_WAVE * held - 1) / (SGH_WAVE * held)); };
      if (places <= 64 * 4) return launch_held<64, 4, 6, S>(a, kBlock, s);
      if (waves(4) <= 16 && a.batch * waves(4) <= cus * 24) return launch_held<kAny, 4, 6, S>(a, waves(4) * SGH_WAVE, s);
      if (waves(8) <= 8) return launch_held<kAny, 8, 5, S>(a, waves(8) * SGH_WAVE, s);
      if (waves(12) <= 8) return launch_held<kAny, 12, 5, S>(a, waves(12) * SGH_WAVE, s);
      if (waves(kHeld) <= 8 || a.batch <= cus) return launch_held<kAny, kHeld, 4, S>(a, waves(kHeld) * SGH_WAVE, s);
    }
    return launch_fwd<512, S, true>(a, s);
  }
  // Few rows have wide teams, many have teams that are not long at a row.  (The loss of 512 rows of 4096 bfloat16 values with 64, 256 threads
  // each: 5.5, 4.7 us, of 4096 rows of 2000: 8.8, 12.0; 1024 rows of 20001 with 128, 256: 12.4, 13.3, 4096 of 50304: 84.8, 77.9; 64 of 20001 with
  // 256, 512: 5.9, 5.5, 300: 7.5, 7.7.  The gradient of 512 rows of 4096 with 64, 256: 8.3, 6.9, of 4096 rows of 2000: 13.9, 20.0; 1024 rows of 20001
  // with 256, 512: 17.5, 19.8, 512 of 50304: 20.6, 23.4, 64 of those: 7.7, 7.3,
  // 4096: 158.6, 149.1.)
  const bool few = a.batch <= 2 * cus;
  if (vecs <= 128 || (vecs <= 512 && !few)) return grad ? launch_bwd<64, S>(a, unsigned(vecs), s) : launch_fwd<64, S, false>(a, s);
  if (!grad) {
    if (few) return a.batch * 2 <= cus && vecs > 1024 ? launch_fwd<512, S, false>(a, s) : launch_fwd<256, S, false>(a, s);
    return vecs <= 2560 ? launch_fwd<128, S, false>(a, s) : launch_fwd<256, S, false>(a, s);
  }
  // few rows: several workgroups to each, with a turn of every thread's vectors at least
  auto each = [&](size_t threads) {
    const size_t turns = (vecs + threads * kAhead - 1) / (threads * kAhead), want = (4 * cus + a.batch - 1) / a.batch;
    const size_t n = turns < want ? turns : want;
    return unsigned((vecs + n - 1) / n);
  };
  return vecs <= 4096 || (few && a.batch * 4 > cus && vecs <= 8192) ? launch_bwd<256, S>(a, each(256), s) : launch_bwd<512, S>(a, each(512), s);
}

}  // namespace

extern "C" {

#define SGH_DISTILL(SFX, S, T)                                                                                                     \
  int sgh_distill_fwd_##SFX(const T *x, const int32_t *top, const float *teacher, const int32_t *labels, const float *weights,     \
                            size_t batch, size_t dim, size_t k, float temperature, float soft, float hard, float *loss,            \
                            float *stats, void *workspace, size_t ws_bytes, void *stream) {                                        \
    return distill<S>({x, nullptr, top, teacher, labels, weights, loss, stats, batch, dim, 0, temperature, soft, hard, 0.f}, k,    \
                      true, false, workspace, ws_bytes, stream);                                                                   \
  }                                                                                                                                \
  int sgh_distill_bwd_##SFX(const T *x, const float *stats, const int32_t *top, const float *teacher, const int32_t *labels,       \
                            const float *weights, size_t batch, size_t dim, size_t k, float temperature, float soft, float hard,   \
                            float scale, T *dx, void *stream) {                                                                    \
    return distill<S>({x, dx, top, teacher, labels, weights, nullptr, const_cast<float *>(stats), batch, dim, 0, temperature,      \
                       soft, hard, scale}, k, false, true, nullptr, 0, stream);                                                    \
  }                                                                                                                                \
  int sgh_distill_fwd_bwd_##SFX(const T *x, const int32_t *top, const float *teacher, const int32_t *labels,                       \
                                const float *weights, size_t batch, size_t dim, size_t k, float temperature, float soft,           \
                                float hard, float scale, float *loss, T *dx, void *workspace, size_t ws_bytes,                     \
                                void *stream) {                                                                                    \
    return distill<S>({x, dx, top, teacher, labels, weights, loss, nullptr, batch, dim, 0, temperature, soft, hard, scale}, k,     \
                      true, true, workspace, ws_bytes, stream);                                                                    \
  }
SGH_DISTILL(f32, StF32, float)
SGH_DISTILL(f16, StF16, uint16_t)
SGH_DISTILL(bf16, StBF16, uint16_t)
#undef SGH_DISTILL

size_t sgh_distill_workspace_bytes(size_t batch, size_t dim, size_t elem_bytes, int gradient) {
  if (batch == 0 || batch > 0x7fffffffu || dim == 0 || dim > kMostDim || (elem_bytes != 2 && elem_bytes != 4)) return 0;
  return parts_bytes(batch, parts_of(batch, dim, elem_bytes, gradient != 0));
}

int sgh_distill_index_errors(void *stream, int *count) {
  if (!count) return SGH_EINVAL;
  void *counter;
  SGH_HIP_TRY(hipGetSymbolAddress(&counter, HIP_SYMBOL(g_list_errors)));
  return sgh_take_count(static_cast<int *>(counter), sgh_stream_of(stream), count);
}

}  // extern "C"
