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
};

__device__ __forceinline__ float exp2_(float v) { return __builtin_amdgcn_exp2f(v); }

// NT threads share a row: a wavefront (a workgroup then has several rows), or the workgroup
template <int NT>
struct Team {
  static constexpr int kPerBlock = NT == SGH_WAVE ? kBlock / SGH_WAVE : 1;
  static constexpr int kThreads = NT == SGH_WAVE ? kBlock : NT;
  static __device__ __forceinline__ int id() { return NT == SGH_WAVE ? threadIdx.x >> 6 : 0; }
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
  static __device__ __forceinline__ float max(float v, float *red) {
    v = sgh_wave_max(v);
    if constexpr (NT != SGH_WAVE) {
      __syncthreads();
      if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
      __syncthreads();
      v = red[0];
#pragma unroll
      for (int i = 1; i < NT / 64; ++i) v = fmaxf(v, red[i]);
    }
    return v;
  }
  static __device__ __forceinline__ float sum(float v, float *red) {
    v = sgh_wave_sum(v);
    if constexpr (NT != SGH_WAVE) {
      __syncthreads();
      if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
      __syncthreads();
      v = red[0];
#pragma unroll
      for (int i = 1; i < NT / 64; ++i) v += red[i];
    }
    return v;
  }
};

// A list entry as the gradient needs it: its column, the student's logit there, and its share of -dx
struct Entry {
  int at;    // -1: none
  float x, p;
};

// What a row asks for, and its list in LDS (entry k is the label)
struct RowTerms {
  float w;
  bool soft, hard;
  float most, log_sum;   // the teacher's largest logit, the log of the sum of its exponentials relative to that one
};

template <int NT, class S>
__device__ __forceinline__ RowTerms row_terms(const Rows<typename S::elem> &a, size_t row, Entry *list, float *red, bool count) {
  typedef Team<NT> G;
  const int tid = G::tid();
  const typename S::elem *x = a.x + row * a.dim;
  RowTerms t;
  t.w = a.weights ? a.weights[row] : 1.f;
  t.hard = t.soft = false;
  t.most = t.log_sum = 0.f;
  int label = -1;
  if (a.labels && a.hard != 0.f) {
    label = a.labels[row];
    if (label < -1 || (label >= 0 && size_t(label) >= a.dim)) {
      if (count && tid == 0) atomicAdd(&g_list_errors, 1);
      label = -1;
    }
    t.hard = label >= 0 && t.w != 0.f;
  }
  G::sync();   // (the list of the row before is done with)
  if (tid == 0) list[a.k] = Entry{t.hard ? label : -1, t.hard ? S::ld(x + label) : 0.f, 1.f};
  if (a.k && a.soft != 0.f) {
    float most = -__builtin_inff(), present = 0.f;
    for (int k = tid; k < a.k; k += NT) {
      int at = a.top[row * a.k + k];
      const float v = a.teacher[row * a.k + k];
      if (at < -1 || (at >= 0 && size_t(at) >= a.dim)) {
        if (count) atomicAdd(&g_list_errors, 1);
        at = -1;
      }
      if (v == -__builtin_inff()) at = -1;   // (no share)
      list[k] = Entry{at, at >= 0 && t.w != 0.f ? S::ld(x + at) : 0.f, v};
      if (at >= 0) most = fmaxf(most, v), present = 1.f;
    }
    t.soft = G::max(present, red) != 0.f && t.w != 0.f;
    most = G::max(most, red);
    float sum = 0.f;
    const float c = kLog2e / a.tau;
    for (int k = tid; k < a.k; k += NT)
      if (list[k].at >= 0) sum += exp2_((list[k].p - most) * c);
    sum = G::sum(sum, red);
    t.most = most;
    t.log_sum = logf(sum);
    for (int k = tid; k < a.k; k += NT) {
      if (!t.soft) list[k].at = -1;
      if (list[k].at >= 0) list[k].p = exp2_((list[k].p - most) * c) / sum;
    }
  } else {
    for (int k = tid; k < a.k; k += NT) list[k].at = -1;
  }
  G::sync();
  return t;
}

// Running maximum and sums of exponentials relative to it.  tau = 1: both sums are one.
struct Running {
  float m, st, s1;
};
template <int EPL>
__device__ __forceinline__ void take(Running &r, const float *v, float ct, bool soft, bool hard) {
  float most = v[0];
#pragma unroll
  for (int j = 1; j < EPL; ++j) most = fmaxf(most, v[j]);
  if (most > r.m) {
    const float d = r.m - most;   // (-inf at first: the sums are 0)
    r.st *= exp2_(d * ct);
    r.s1 *= exp2_(d * kLog2e);
    r.m = most;
  }
  const float m = r.m == -__builtin_inff() ? 0.f : r.m;
  if (soft) {
#pragma unroll
    for (int j = 0; j < EPL; ++j) r.st += exp2_((v[j] - m) * ct);
  }
  if (hard) {
#pragma unroll
    for (int j = 0; j < EPL; ++j) r.s1 += exp2_((v[j] - m) * kLog2e);
  }
}

template <int NT, class S>
__device__ __forceinline__ Running row_statistics(const typename S::elem *x, size_t dim, float ct, bool soft, bool hard, float *red) {
  typedef Team<NT> G;
  constexpr int V = S::VEC, U = 4;
  const int tid = G::tid();
  Running r = {-__builtin_inff(), 0.f, 0.f};
  const size_t vecs = dim / V;
  size_t i = tid;
  for (; i + (U - 1) * NT < vecs; i += U * NT) {
    float v[U][V];
#pragma unroll
    for (int u = 0; u < U; ++u) sgh_load_any<S, V>(x + (i + u * NT) * V, v[u]);
#pragma unroll
    for (int u = 0; u < U; ++u) take<V>(r, v[u], ct, soft, hard);
  }
  for (; i < vecs; i += NT) {
    float v[V];
    sgh_load_any<S, V>(x + i * V, v);
    take<V>(r, v, ct, soft, hard);
  }
  const size_t last = vecs * V + tid;
  if (last < dim) {
    float v = S::ld(x + last);
    take<1>(r, &v, ct, soft, hard);
  }
  const float m = G::max(r.m, red), d = r.m - m;
  r.st = soft ? G::sum(r.st * exp2_(d * ct), red) : 0.f;
  r.s1 = hard ? G::sum(r.s1 * exp2_(d * kLog2e), red) : 0.f;
  r.m = m;
  return r;
}

// dx of columns [from, to) of a row
template <int NT, class S>
__device__ __forceinline__ void row_gradient(const Rows<typename S::elem> &a, size_t row, size_t from, size_t to, const Running &r,
                                             const RowTerms &t, const Entry *list) {
  typedef Team<NT> G;
  constexpr int V = S::VEC, U = 4;
  const int tid = G::tid();
  const typename S::elem *x = a.x + row * a.dim;
  typename S::elem *dx = a.dx + row * a.dim;
  const bool any = t.soft || t.hard;
  const float ct = kLog2e / a.tau, g = a.scale * t.w;
  const float share_t = t.soft ? g * a.soft * a.tau : 0.f, share_1 = t.hard ? g * a.hard : 0.f;
  const float ft = t.soft ? share_t / r.st : 0.f, f1 = t.hard ? share_1 / r.s1 : 0.f;
  auto value = [&](float v) {
    const float d = v - r.m;
    float o = 0.f;
    if (t.soft) o = ft * exp2_(d * ct);
    if (t.hard) o += f1 * exp2_(d * kLog2e);
    return o;
  };
  const size_t vecs = (to - from) / V;
  size_t i = tid;
  for (; i + (U - 1) * NT < vecs; i += U * NT) {
    float v[U][V];
    if (any) {
#pragma unroll
      for (int u = 0; u < U; ++u) sgh_load_any<S, V>(x + from + (i + u * NT) * V, v[u]);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int j = 0; j < V; ++j) v[u][j] = any ? value(v[u][j]) : 0.f;
      sgh_store_any<S, V>(dx + from + (i + u * NT) * V, v[u]);
    }
  }
  for (; i < vecs; i += NT) {
    float v[V];
    if (any) sgh_load_any<S, V>(x + from + i * V, v);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = any ? value(v[j]) : 0.f;
    sgh_store_any<S, V>(dx + from + i * V, v);
  }
  const size_t last = from + vecs * V + tid;
  if (last < to) S::st(dx + last, any ? value(S::ld(x + last)) : 0.f);
  if (!any) return;   // (the same for the whole team)
  G::sync();   // the columns of the list again, now that the others are stored
  for (int k = tid; k <= a.k; k += NT) {
    const int at = list[k].at;
    if (at < 0 || size_t(at) < from || size_t(at) >= to) continue;
    bool first = true;
    for (int j = 0; j < k; ++j) first &= list[j].at != at;
    if (!first) continue;   // a column that is there twice is its first entry's
    float o = value(list[k].x);
    for (int j = k; j <= a.k; ++j)
      if (list[j].at == at) o -= (j < a.k ? share_t : share_1) * list[j].p;
    S::st(dx + at, o);
  }
}

// The loss and statistics of a row; GRAD: and its gradient
template <int NT, class S, bool GRAD>
__global__ __launch_bounds__(Team<NT>::kThreads) void k_distill_fwd(Rows<typename S::elem> a) {
  typedef Team<NT> G;
  extern __shared__ char lds[];
  __shared__ float red[16];
  Entry *list = reinterpret_cast<Entry *>(lds) + G::id() * (a.k + 1);
  for (size_t row = size_t(blockIdx.x) * G::kPerBlock + G::id(); row < a.batch; row += size_t(gridDim.x) * G::kPerBlock) {
    const RowTerms t = row_terms<NT, S>(a, row, list, red, true);
    Running r = {0.f, 0.f, 0.f};
    if (t.soft || t.hard) r = row_statistics<NT, S>(a.x + row * a.dim, a.dim, kLog2e / a.tau, t.soft, t.hard, red);
    float kl = 0.f;
    if (t.soft) {
      const float log_st = logf(r.st);
      for (int k = G::tid(); k < a.k; k += NT)
        if (list[k].at >= 0 && list[k].p != 0.f) {
          const float log_p = (a.teacher[row * a.k + k] - t.most) / a.tau - t.log_sum;
          kl += list[k].p * (log_p - ((list[k].x - r.m) / a.tau - log_st));
        }
      kl = G::sum(kl, red);
    }
    if (G::tid() == 0) {
      float loss = 0.f;
      if (t.soft) loss += a.soft * a.tau * a.tau * kl;
      if (t.hard) loss += a.hard * (logf(r.s1) - (list[a.k].x - r.m));
      a.loss[row] = t.w == 0.f ? 0.f : t.w * loss;
      if (a.stats) {
        a.stats[row * 3] = r.m;
        a.stats[row * 3 + 1] = r.st;
        a.stats[row * 3 + 2] = r.s1;
      }
    }
    if constexpr (GRAD) row_gradient<NT, S>(a, row, 0, a.dim, r, t, list);
  }
}

// The gradient from the statistics; a row may be several workgroups', `cols` columns each
template <int NT, class S>
__global__ __launch_bounds__(Team<NT>::kThreads) void k_distill_bwd(Rows<typename S::elem> a, size_t cols) {
  typedef Team<NT> G;
  extern __shared__ char lds[];
  __shared__ float red[16];
  Entry *list = reinterpret_cast<Entry *>(lds) + G::id() * (a.k + 1);
  const size_t from = size_t(blockIdx.y) * cols, to = from + cols < a.dim ? from + cols : a.dim;
  for (size_t row = size_t(blockIdx.x) * G::kPerBlock + G::id(); row < a.batch; row += size_t(gridDim.x) * G::kPerBlock) {
    const RowTerms t = row_terms<NT, S>(a, row, list, red, false);
    const Running r = {a.stats[row * 3], a.stats[row * 3 + 1], a.stats[row * 3 + 2]};
    row_gradient<NT, S>(a, row, from, to, r, t, list);
  }
}

template <int NT, class S>
int launch(const Rows<typename S::elem> &a, bool fwd, bool grad, hipStream_t s) {
  typedef Team<NT> G;
  size_t blocks = (a.batch + G::kPerBlock - 1) / G::kPerBlock;
  if (blocks > (1u << 20)) blocks = 1u << 20;
  const size_t lds = size_t(G::kPerBlock) * (a.k + 1) * sizeof(Entry);
  const dim3 grid{unsigned(blocks)}, block{unsigned(G::kThreads)};
  if (fwd && grad)
    SGH_LAUNCH_TIMED((k_distill_fwd<NT, S, true>), grid, block, lds, s, a);
  else if (fwd)
    SGH_LAUNCH_TIMED((k_distill_fwd<NT, S, false>), grid, block, lds, s, a);
  else
    SGH_LAUNCH_TIMED((k_distill_bwd<NT, S>), grid, block, lds, s, a, a.dim);
  SGH_LAUNCH_CHECK();
  return SGH_OK;
}

// The checks that the three entry points share; SGH_OK with `empty` set where there is nothing to do
template <class T>
int check(const Rows<T> &a, size_t k, bool fwd, bool grad, bool *empty) {
  *empty = false;
  if (a.batch > 0x7fffffffu || a.dim > 0x7fffffffu) return SGH_EINVAL;
  if (!(a.tau > 0.f) || !__builtin_isfinite(a.tau) || !__builtin_isfinite(kLog2e / a.tau)) return SGH_EINVAL;
  if (k > SGH_DISTILL_MAX_TOP) return SGH_ELIMIT;
  if (a.batch == 0) return *empty = true, SGH_OK;
  if (a.dim == 0) return SGH_EINVAL;   // (a row of no logits has no softmax)
  if (!a.x || (k != 0 && (!a.top || !a.teacher))) return SGH_EINVAL;
  if (fwd && !a.loss) return SGH_EINVAL;
  if ((!fwd || !grad) && !a.stats) return SGH_EINVAL;
  const size_t bytes = a.batch * a.dim * sizeof(T);
  if (grad) {
    if (!a.dx) return SGH_EINVAL;
    if (a.dx != a.x && sgh_ranges_meet(a.dx, bytes, a.x, bytes)) return SGH_EINVAL;
    if (sgh_ranges_meet(a.dx, bytes, a.top, a.batch * k * 4) || sgh_ranges_meet(a.dx, bytes, a.teacher, a.batch * k * 4) ||
        sgh_ranges_meet(a.dx, bytes, a.labels, a.labels ? a.batch * 4 : 0) ||
        sgh_ranges_meet(a.dx, bytes, a.weights, a.weights ? a.batch * 4 : 0) ||
        sgh_ranges_meet(a.dx, bytes, a.stats, a.stats ? a.batch * 12 : 0))
      return SGH_EINVAL;
  }
  return SGH_OK;
}

template <class S>
int distill(Rows<typename S::elem> a, size_t k, bool fwd, bool grad, void *stream) {
  bool empty;
  const int rc = check(a, k, fwd, grad, &empty);
  if (rc != SGH_OK || empty) return rc;
  a.k = int(k);
  hipStream_t s = sgh_stream_of(stream);
  const double bytes = double(a.batch) * a.dim * sizeof(typename S::elem);
  if (grad) sgh_note_write(a.dx, a.batch * a.dim * sizeof(typename S::elem));
  sgh_prof_kernel_scope prof(fwd && grad ? "distill/k_distill_fwd" : fwd ? "distill_fwd/k_distill_fwd" : "distill_bwd/k_distill_bwd",
                             bytes * (grad ? 2 : 1), s);
  if (a.dim <= 2048) return launch<SGH_WAVE, S>(a, fwd, grad, s);
  return launch<kBlock, S>(a, fwd, grad, s);
}

}  // namespace

extern "C" {

#define SGH_DISTILL(SFX, S, T)                                                                                                     \
  int sgh_distill_fwd_##SFX(const T *x, const int32_t *top, const float *teacher, const int32_t *labels, const float *weights,     \
                            size_t batch, size_t dim, size_t k, float temperature, float soft, float hard, float *loss,            \
                            float *stats, void *stream) {                                                                          \
    return distill<S>({x, nullptr, top, teacher, labels, weights, loss, stats, batch, dim, 0, temperature, soft, hard, 0.f}, k,    \
                      true, false, stream);                                                                                        \
  }                                                                                                                                \
  int sgh_distill_bwd_##SFX(const T *x, const float *stats, const int32_t *top, const float *teacher, const int32_t *labels,       \
                            const float *weights, size_t batch, size_t dim, size_t k, float temperature, float soft, float hard,   \
                            float scale, T *dx, void *stream) {                                                                    \
    return distill<S>({x, dx, top, teacher, labels, weights, nullptr, const_cast<float *>(stats), batch, dim, 0, temperature,      \
                       soft, hard, scale}, k, false, true, stream);                                                                \
  }                                                                                                                                \
  int sgh_distill_fwd_bwd_##SFX(const T *x, const int32_t *top, const float *teacher, const int32_t *labels,                       \
                                const float *weights, size_t batch, size_t dim, size_t k, float temperature, float soft,           \
                                float hard, float scale, float *loss, T *dx, void *stream) {                                       \
    return distill<S>({x, dx, top, teacher, labels, weights, loss, nullptr, batch, dim, 0, temperature, soft, hard, scale}, k,     \
                      true, true, stream);                                                                                         \
  }
SGH_DISTILL(f32, StF32, float)
SGH_DISTILL(f16, StF16, uint16_t)
SGH_DISTILL(bf16, StBF16, uint16_t)
#undef SGH_DISTILL

int sgh_distill_index_errors(void *stream, int *count) {
  if (!count) return SGH_EINVAL;
  SGH_HIP_TRY(hipStreamSynchronize(sgh_stream_of(stream)));
  int v = 0;
  SGH_HIP_TRY(hipMemcpyFromSymbol(&v, HIP_SYMBOL(g_list_errors), sizeof(int), 0, hipMemcpyDeviceToHost));
  const int zero = 0;
  SGH_HIP_TRY(hipMemcpyToSymbol(HIP_SYMBOL(g_list_errors), &zero, sizeof(int), 0, hipMemcpyHostToDevice));
  *count = v;
  return SGH_OK;
}

}  // extern "C"
