// The norms around a block of a token model, with the block's gate, scale and sum, in one pass over the rows:
//   u = h rsqrt(mean h^2 + eps) post,  y = x + scale gate u,  n = y rsqrt(mean y^2 + eps) pre
// and backwards, with t the whole gradient of y, r_h and r the roots that the forward pass kept, unit = h r_h and a = dn pre:
//   t = dy + r a - y r^3 mean(a y),  dx = t,  dgate = scale t u,  dh = r_h b - h r_h^3 mean(b h) with b = scale gate t post,
//   dpost = sum scale gate t unit,  dpre = sum dn y r
//
// A row is a team's: 8 to 1024 threads that hold it in registers, so that every tensor is read once and written once.  Memory is what bounds it.  A
// workgroup goes over its rows with the next row's loads under way before this row's stores are issued: loads and stores are counted by one counter,
// in order, and a load behind a store would wait for it.  The weights stay in registers, and so do the sums over the rows that are the weights'
// gradients.  These are then joined over the workgroups in their order by a second launch: the same bits every time.
//
// Measured: 32768 rows of 4096 bfloat16 values, 16 gates, all weights: forward 206 us (5.2 TB/s), backward 335 to 390 with the clock, its join
// 9 (4.1 to 4.8 TB/s); 8192 fp32 rows of 768 backward 22 us and the join 5; 16 rows of 1000 forward 4 us, the launch and two sums one behind the other.
#include "common.h"
#include "rows.h"

namespace {

struct Args {
  const void *x, *h, *gate, *dy, *dn, *y;
  const float *post, *pre;
  float *stats;
  void *out_y, *out_n, *dx, *dh, *dgate;
  float *part;        // [groups][2][dim]: sums of dpre, dpost; behind them [gates][chunks][dim] of dgate where a gate has several workgroups
  float *gate_part;
  size_t dim;
  unsigned rows, gates, per_gate;   // rows of a gate, 0: no gate
  unsigned each, chunks;            // rows of a team of the grid; workgroups to a gate (backwards; 0: a team has whole gates)
  float scale, eps;
};

template <int TEAM>
__device__ __forceinline__ float team_sum(float x, float *lds) {
#pragma unroll
  for (int m = 1; m < (TEAM < SGH_WAVE ? TEAM : SGH_WAVE); m *= 2) x += __shfl_xor(x, m);
  if constexpr (TEAM > SGH_WAVE) {
    constexpr int W = TEAM / SGH_WAVE;
    if (threadIdx.x % SGH_WAVE == 0) lds[threadIdx.x / SGH_WAVE] = x;
    __syncthreads();
    x = 0.f;
    const float *mine = lds + threadIdx.x / TEAM * W;
#pragma unroll
    for (int w = 0; w < W; ++w) x += mine[w];
  }
  return x;
}

// Where a thread's vectors of a row lie
template <int EPL, int TEAM, int NV>
struct Place {
  unsigned at[NV];
  int dup[NV];    // elements at a vector's front that the vector before it has as well, EPL: no vector
  __device__ __forceinline__ Place(unsigned dim) {
    const unsigned vecs = (dim + EPL - 1) / EPL;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const unsigned v = j * TEAM + threadIdx.x % TEAM;
      at[j] = v * EPL, dup[j] = 0;
      if (v >= vecs) dup[j] = EPL, at[j] = 0;
      else if (at[j] + EPL > dim) dup[j] = int(at[j] + EPL - dim), at[j] = dim - EPL;
    }
  }
  __device__ __forceinline__ bool has(int j) const { return dup[j] != EPL; }
};

// A row's vectors as they are stored
template <class S, int EPL, int NV>
struct Raw {
  typename S::elem e[NV][EPL];
  // STREAM: past the caches; not `there`: zeros
  template <bool STREAM = false, class P>
  __device__ __forceinline__ void load(const void *t, size_t row, size_t dim, const P &p, bool there = true) {
    const typename S::elem *r = static_cast<const typename S::elem *>(t) + row * dim;
#pragma unroll
    for (int j = 0; j < NV; ++j)
      if (p.has(j) && there) {
        if constexpr (STREAM) {
          typedef sgh_v4u anywhere __attribute__((aligned(2)));
          const sgh_v4u v = __builtin_nontemporal_load(reinterpret_cast<const anywhere *>(r + p.at[j]));
          __builtin_memcpy(e[j], &v, 16);
        } else {
          __builtin_memcpy(e[j], r + p.at[j], EPL * sizeof(typename S::elem));
        }
      } else __builtin_memset(e[j], 0, EPL * sizeof(typename S::elem));
  }
  __device__ __forceinline__ float operator()(int j, int i) const { return S::ld(&e[j][i]); }
  __device__ __forceinline__ void get(float (&f)[NV][EPL]) const {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < EPL; ++i) f[j][i] = S::ld(&e[j][i]);
  }
};
template <class S, bool STREAM = false, int EPL, int NV, class P>
__device__ __forceinline__ void store_row(void *t, size_t row, size_t dim, const P &p, const float (&f)[NV][EPL]) {
  typename S::elem *r = static_cast<typename S::elem *>(t) + row * dim;
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (p.has(j)) sgh_store_any<S, EPL, STREAM>(r + p.at[j], f[j]);
}
template <int EPL, int NV, class P>
__device__ __forceinline__ void load_floats(const float *t, const P &p, float (&f)[NV][EPL]) {
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (p.has(j)) __builtin_memcpy(f[j], t + p.at[j], EPL * sizeof(float));
    else __builtin_memset(f[j], 0, EPL * sizeof(float));
}
template <int EPL, int NV, class P>
__device__ __forceinline__ void store_floats(float *t, const P &p, const float (&f)[NV][EPL]) {
#pragma unroll
  for (int j = 0; j < NV; ++j)
    if (p.has(j)) __builtin_memcpy(t + p.at[j], f[j], EPL * sizeof(float));
}
// sum of a[j][i] b[j][i] over the thread's own elements
template <int EPL, int NV, class P>
__device__ __forceinline__ float dot(const float (&a)[NV][EPL], const float (&b)[NV][EPL], const P &p) {
  float x = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < EPL; ++i) x += i < p.dup[j] ? 0.f : a[j][i] * b[j][i];
  return x;
}

template <int TEAM>
constexpr int kThreads = TEAM < 256 ? 256 : TEAM;

// The weights in LDS: post, then pre
template <int THREADS>
__device__ __forceinline__ void keep_weights(const Args &a, float *weights) {
  for (size_t c = threadIdx.x; c < a.dim; c += THREADS) {
    if (a.post) weights[c] = a.post[c];
    if (a.pre) weights[a.dim + c] = a.pre[c];
  }
  __syncthreads();
}

template <class S, int EPL, int TEAM, int NV, bool HOLD, bool STREAM>
__global__ __launch_bounds__(kThreads<TEAM>) void k_norm_fwd(Args a) {
  constexpr int PER = kThreads<TEAM> / TEAM;
  __shared__ float lds[2][16];
  const size_t dim = a.dim;
  const Place<EPL, TEAM, NV> p{unsigned(dim)};
  const bool block = a.h != nullptr;
  // (a team behind the last row goes through the last row's motions: all of a workgroup meet at the sums)
  size_t row = (size_t(blockIdx.x) * PER + threadIdx.x / TEAM) * a.each;
  const size_t last = a.rows - 1;
  float post[NV][EPL], pre[NV][EPL], gate[NV][EPL];
  if (HOLD && a.post) load_floats(a.post, p, post);
  if (HOLD && a.pre) load_floats(a.pre, p, pre);
  Raw<S, EPL, NV> rx, rh, rg;
  const bool token_gate = a.per_gate == 1;
  size_t at = row < last ? row : last, group = ~size_t(0);
  rx.template load<STREAM>(a.x, at, dim, p);
  if (block) rh.template load<STREAM>(a.h, at, dim, p);
  if (token_gate) rg.template load<STREAM>(a.gate, at, dim, p);
  const float inv_dim = 1.f / float(dim);
  for (unsigned i = 0; i < a.each; ++i, ++row) {
    float y[NV][EPL], h[NV][EPL];
    if (!HOLD && i) {
      rx.template load<STREAM>(a.x, at, dim, p);
      if (block) rh.template load<STREAM>(a.h, at, dim, p);
      if (token_gate) rg.template load<STREAM>(a.gate, at, dim, p);
    }
    rx.get(y);
    if (block) rh.get(h);
    if (token_gate) rg.get(gate);
    const size_t next = row + 1 < last ? row + 1 : last;
    if (HOLD && i + 1 < a.each) {
      rx.template load<STREAM>(a.x, next, dim, p);
      if (block) rh.template load<STREAM>(a.h, next, dim, p);
      if (token_gate) rg.template load<STREAM>(a.gate, next, dim, p);
    }
    if (a.per_gate > 1) {
      const size_t g = at / a.per_gate;
      if (!HOLD || g != group) {
        Raw<S, EPL, NV> r;
        r.load(a.gate, g, dim, p);
        r.get(gate);
        group = g;
      }
    }
    float rh_root = 0.f, ry_root = 0.f;
    if (block) {
      if (a.post) {
        if (!HOLD) load_floats(a.post, p, post);
        rh_root = __frsqrt_rn(team_sum<TEAM>(dot(h, h, p), lds[0]) * inv_dim + a.eps);
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int e = 0; e < EPL; ++e) h[j][e] *= rh_root * post[j][e];
      }
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < EPL; ++e) {
          const float u = a.per_gate ? gate[j][e] * h[j][e] : h[j][e];
          y[j][e] = __builtin_fmaf(a.scale, u, y[j][e]);
        }
    }
    const bool mine = row < a.rows;
    if (block && mine) store_row<S, STREAM>(a.out_y, row, dim, p, y);
    if (a.pre) {
      if (!HOLD) load_floats(a.pre, p, pre);
      ry_root = __frsqrt_rn(team_sum<TEAM>(dot(y, y, p), lds[1]) * inv_dim + a.eps);
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < EPL; ++e) y[j][e] *= ry_root * pre[j][e];
      if (mine) store_row<S, STREAM>(a.out_n, row, dim, p, y);
    }
    if (mine && threadIdx.x % TEAM == 0) a.stats[2 * row] = rh_root, a.stats[2 * row + 1] = ry_root;
    at = next;
    if (TEAM > SGH_WAVE && !(a.pre && a.post && block)) __syncthreads();   // (one sum's words are not written again before all have read them)
  }
}

template <class S, int TEAM>
constexpr int kPerSimd = S::VEC == 8 || TEAM == 1024 ? 4 : 2;

template <class S, int EPL, int TEAM, int NV, bool STREAM>
__global__ __launch_bounds__(kThreads<TEAM>, (kPerSimd<S, TEAM>)) void k_norm_bwd(Args a) {
  constexpr int PER = kThreads<TEAM> / TEAM;
  __shared__ float lds[2][16];
  extern __shared__ __align__(16) float kept[];   // the weights, and in the end the teams' sums
  keep_weights<kThreads<TEAM>>(a, kept);
  const float *const post_at = kept, *const pre_at = kept + a.dim;
  const size_t dim = a.dim;
  const Place<EPL, TEAM, NV> p{unsigned(dim)};
  const bool block = a.h != nullptr, token_gate = a.per_gate == 1, shared_gate = a.per_gate > 1;
  // A team's rows: `each` of them one behind the other; of one gate's, where workgroups share it
  const unsigned mine_of = threadIdx.x / TEAM;
  size_t row = (size_t(blockIdx.x) * PER + mine_of) * a.each, end = row + a.each;
  if (a.chunks) {
    const size_t g = blockIdx.x / a.chunks, stop = (g + 1) * a.per_gate;
    row = g * a.per_gate + (size_t(blockIdx.x % a.chunks) * PER + mine_of) * a.each, end = row + a.each;
    if (end > stop) end = stop;
  }
  if (end > a.rows) end = a.rows;
  const unsigned count = row < end ? unsigned(end - row) : 0;
  // Sums over the rows: of dn y r, and of scale t unit, times the gate unless rows share it (a shared gate's sums go into sum_post when its rows are
  // done)
  float gate[NV][EPL], sum_pre[NV][EPL], sum_unit[NV][EPL], sum_post[NV][EPL];
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < EPL; ++e) gate[j][e] = 1.f, sum_pre[j][e] = sum_unit[j][e] = sum_post[j][e] = 0.f;
  auto load_gate = [&](size_t g) {
    Raw<S, EPL, NV> r;
    r.load(a.gate, g, dim, p);
    r.get(gate);
  };
  // (rows that a team does not have are zeros, and add nothing)
  Raw<S, EPL, NV> rt, rn, ry, rh, rg;
  auto request = [&](size_t r, bool there) {
    rt.load(a.dy, r, dim, p, there && a.dy);
    if (a.pre) rn.load(a.dn, r, dim, p, there), ry.load(a.y, r, dim, p, there);
    if (block) rh.load(a.h, r, dim, p, there);
    if (token_gate) rg.load(a.gate, r, dim, p, there);
  };
  size_t group = ~size_t(0), group_end = 0;
  // a shared gate's sums are complete, or those of this team's part: d gets its gradient
  auto leave_gate = [&](float (&d)[NV][EPL]) {
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < EPL; ++e) d[j][e] = 1.f;
    if (a.post) load_floats(post_at, p, d);
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        d[j][e] *= sum_unit[j][e];
        sum_post[j][e] = __builtin_fmaf(gate[j][e], sum_unit[j][e], sum_post[j][e]);
        sum_unit[j][e] = 0.f;
      }
  };
  request(row, count != 0);
  const float inv_dim = 1.f / float(dim);
  for (unsigned i = 0; i < a.each; ++i, ++row) {
    const bool mine = i < count;
    // (as stored until they are used: 16-bit rows then take half of the registers)
    const Raw<S, EPL, NV> ct = rt, cn = rn, cy = ry, ch = rh;
    if (token_gate) rg.get(gate);
    const float rh_root = mine && a.post ? a.stats[2 * row] : 1.f, ry_root = mine ? a.stats[2 * row + 1] : 0.f;
    if (i + 1 < a.each) request(row + 1, i + 1 < count);
    if (shared_gate && mine && row >= group_end) {
      if (group != ~size_t(0)) {
        float d[NV][EPL];
        leave_gate(d);
        store_row<S>(a.dgate, group, dim, p, d);
      }
      group = row / a.per_gate, group_end = (group + 1) * a.per_gate;
      load_gate(group);
    }
    float t[NV][EPL], w[NV][EPL];
    if (a.pre) {
      float c = 0.f;
      load_floats(pre_at, p, w);
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < EPL; ++e) {
          w[j][e] *= cn(j, e);
          c += e < p.dup[j] ? 0.f : w[j][e] * cy(j, e);
        }
      c = team_sum<TEAM>(c, lds[0]) * inv_dim * ry_root * ry_root;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < EPL; ++e) {
          t[j][e] = __builtin_fmaf(ry_root, __builtin_fmaf(-c, cy(j, e), w[j][e]), ct(j, e));
          sum_pre[j][e] = __builtin_fmaf(cn(j, e), cy(j, e) * ry_root, sum_pre[j][e]);
        }
    } else {
      ct.get(t);
    }
    if (mine) store_row<S, STREAM>(a.dx, row, dim, p, t);
    if (block) {
      float c = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < EPL; ++e) w[j][e] = 1.f;
      if (a.post) load_floats(post_at, p, w);
      // (w becomes the gradient by the normalised result, t the gate's)
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < EPL; ++e) {
          const float st = a.scale * t[j][e], each = st * (ch(j, e) * rh_root);
          t[j][e] = each * w[j][e];
          sum_unit[j][e] += shared_gate ? each : each * gate[j][e];
          w[j][e] *= st * gate[j][e];
          c += e < p.dup[j] ? 0.f : w[j][e] * ch(j, e);
        }
      if (token_gate && mine) store_row<S, STREAM>(a.dgate, row, dim, p, t);
      if (a.post) {
        c = team_sum<TEAM>(c, lds[1]) * inv_dim * rh_root * rh_root;
#pragma unroll
        for (int j = 0; j < NV; ++j)
#pragma unroll
          for (int e = 0; e < EPL; ++e) w[j][e] = rh_root * __builtin_fmaf(-c, ch(j, e), w[j][e]);
      }
      if (mine) store_row<S, STREAM>(a.dh, row, dim, p, w);
    }
    if (TEAM > SGH_WAVE && !(a.pre && a.post && block)) __syncthreads();
  }
  // the teams of a workgroup, joined in their order
  float *const sums = kept, *const out = a.part + size_t(blockIdx.x) * 2 * dim;   // sums: [PER][dim]
  auto join = [&](const float (&f)[NV][EPL], auto put) {
    __syncthreads();
    store_floats(sums + mine_of * dim, p, f);
    __syncthreads();
    for (size_t c = threadIdx.x; c < dim; c += kThreads<TEAM>) {
      float x = 0.f;
      for (int k = 0; k < PER; ++k) x += sums[k * dim + c];
      put(c, x);
    }
  };
  float d[NV][EPL];
  if (shared_gate) {
    __builtin_memset(d, 0, sizeof(d));
    if (group != ~size_t(0)) leave_gate(d);
    float *const part = a.gate_part + size_t(blockIdx.x) * dim;
    if (!a.chunks) {
      if (group != ~size_t(0)) store_row<S>(a.dgate, group, dim, p, d);
    } else if constexpr (PER == 1) {
      if (a.chunks > 1) store_floats(part, p, d);
      else store_row<S>(a.dgate, blockIdx.x, dim, p, d);
    } else {
      typename S::elem *whole = static_cast<typename S::elem *>(a.dgate) + size_t(blockIdx.x) * dim;
      join(d, [&](size_t c, float x) {
        if (a.chunks > 1) part[c] = x;
        else S::st(whole + c, x);
      });
    }
  }
  if (a.pre) {
    if constexpr (PER == 1) store_floats(out, p, sum_pre);
    else join(sum_pre, [&](size_t c, float x) { out[c] = x; });
  }
  if (a.post) {
    if (!shared_gate)
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int e = 0; e < EPL; ++e) sum_post[j][e] = sum_unit[j][e];
    if constexpr (PER == 1) store_floats(out + dim, p, sum_post);
    else join(sum_post, [&](size_t c, float x) { out[dim + c] = x; });
  }
}

// Rows of more than 8192 values: a workgroup of 1024 threads has no registers for 16 values of each of four tensors and the sums (kept in scratch
// memory, every load was waited for before the next: 4000 rows of 16384 bfloat16 values 490 us).  It goes over a row three times, the second and
// third time out of the caches, and has the sums in LDS, at places of each thread's own.
constexpr int kWide = 1024;
template <class S, int NV>
__global__ __launch_bounds__(kWide, 4) void k_norm_bwd_wide(Args a) {
  constexpr int EPL = S::VEC;
  typedef typename S::elem elem;
  __shared__ float lds[2][16];
  extern __shared__ __align__(16) float kept[];   // [2][NV][EPL][kWide]
  const size_t dim = a.dim;
  const Place<EPL, kWide, NV> p{unsigned(dim)};
  const bool block = a.h != nullptr, token_gate = a.per_gate == 1, shared_gate = a.per_gate > 1;
  size_t row = size_t(blockIdx.x) * a.each, end = row + a.each;
  if (a.chunks) {
    const size_t g = blockIdx.x / a.chunks, stop = (g + 1) * a.per_gate;
    row = g * a.per_gate + size_t(blockIdx.x % a.chunks) * a.each, end = row + a.each;
    if (end > stop) end = stop;
  }
  if (end > a.rows) end = a.rows;
  float *const out = a.part + size_t(blockIdx.x) * 2 * dim;
  auto sum_pre = [&](int j, int e) -> float & { return kept[(j * EPL + e) * kWide + threadIdx.x]; };
  auto sum_unit = [&](int j, int e) -> float & { return kept[((NV + j) * EPL + e) * kWide + threadIdx.x]; };
  auto vec = [&](const void *t, size_t r, int j, float *f) { sgh_load_any<S, EPL>(static_cast<const elem *>(t) + r * dim + p.at[j], f); };
  auto put = [&](void *t, size_t r, int j, const float *f) { sgh_store_any<S, EPL>(static_cast<elem *>(t) + r * dim + p.at[j], f); };
  auto weight = [&](const float *t, int j, float *f) { __builtin_memcpy(f, t + p.at[j], EPL * sizeof(float)); };
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int e = 0; e < EPL; ++e) sum_pre(j, e) = sum_unit(j, e) = 0.f;
  bool left = false;
  // the part of the gradient of post: an element that two vectors have is the first one's, which the sum so far is read by alone
  auto keep = [&](int j, const float *f) {
    if (p.dup[j] == 0) __builtin_memcpy(out + dim + p.at[j], f, EPL * sizeof(float));
    else
#pragma unroll
      for (int e = 0; e < EPL; ++e)
        if (e >= p.dup[j]) out[dim + p.at[j] + e] = f[e];
  };
  // a shared gate's sums are complete, or this workgroup's part of them
  auto leave_gate = [&](size_t g) {
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!p.has(j)) continue;
      float d[EPL], gate[EPL], sum[EPL];
#pragma unroll
      for (int e = 0; e < EPL; ++e) d[e] = 1.f, sum[e] = 0.f;
      if (a.post) weight(a.post, j, d);
      vec(a.gate, g, j, gate);
      if (a.post && left) weight(out + dim, j, sum);
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        const float x = sum_unit(j, e);
        sum_unit(j, e) = 0.f;
        d[e] *= x;
        sum[e] = __builtin_fmaf(gate[e], x, sum[e]);
      }
      if (a.post) keep(j, sum);
      if (a.chunks > 1) __builtin_memcpy(a.gate_part + size_t(blockIdx.x) * dim + p.at[j], d, sizeof(d));
      else put(a.dgate, g, j, d);
    }
    left = true;
  };
  size_t group = ~size_t(0), group_end = 0;
  const float inv_dim = 1.f / float(dim);
  for (; row < end; ++row) {
    const float rh_root = a.post ? a.stats[2 * row] : 1.f, ry_root = a.stats[2 * row + 1];
    if (shared_gate && row >= group_end) {
      if (group != ~size_t(0)) leave_gate(group);
      group = row / a.per_gate, group_end = (group + 1) * a.per_gate;
    }
    float t[NV][EPL], c = 0.f;
    if (a.pre) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (!p.has(j)) continue;
        float dn[EPL], y[EPL], w[EPL];
        vec(a.dn, row, j, dn), vec(a.y, row, j, y), weight(a.pre, j, w);
#pragma unroll
        for (int e = 0; e < EPL; ++e) c += e < p.dup[j] ? 0.f : w[e] * dn[e] * y[e];
      }
      c = team_sum<kWide>(c, lds[0]) * inv_dim * ry_root * ry_root;
    }
    float d = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (!p.has(j)) continue;
#pragma unroll
      for (int e = 0; e < EPL; ++e) t[j][e] = 0.f;
      if (a.dy) vec(a.dy, row, j, t[j]);
      if (a.pre) {
        float dn[EPL], y[EPL], w[EPL];
        vec(a.dn, row, j, dn), vec(a.y, row, j, y), weight(a.pre, j, w);
#pragma unroll
        for (int e = 0; e < EPL; ++e) {
          t[j][e] = __builtin_fmaf(ry_root, __builtin_fmaf(-c, y[e], w[e] * dn[e]), t[j][e]);
          sum_pre(j, e) += dn[e] * (y[e] * ry_root);
        }
      }
      put(a.dx, row, j, t[j]);
      if (!block) continue;
      float h[EPL], w[EPL], gate[EPL];
#pragma unroll
      for (int e = 0; e < EPL; ++e) w[e] = gate[e] = 1.f;
      vec(a.h, row, j, h);
      if (a.post) weight(a.post, j, w);
      if (a.per_gate) vec(a.gate, token_gate ? row : group, j, gate);
#pragma unroll
      for (int e = 0; e < EPL; ++e) {
        const float st = a.scale * t[j][e], each = st * (h[e] * rh_root);
        sum_unit(j, e) += shared_gate ? each : each * gate[e];
        t[j][e] = w[e] * (st * gate[e]);
        d += e < p.dup[j] ? 0.f : t[j][e] * h[e];
        w[e] *= each;
      }
      if (token_gate) put(a.dgate, row, j, w);
      __builtin_amdgcn_sched_barrier(0);   // (one vector of each tensor at a time: more would not leave the registers)
    }
    if (block) {
      if (a.post) d = team_sum<kWide>(d, lds[1]) * inv_dim * rh_root * rh_root;
      else d = 0.f;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (!p.has(j)) continue;
        float h[EPL];
        vec(a.h, row, j, h);
#pragma unroll
        for (int e = 0; e < EPL; ++e) h[e] = rh_root * __builtin_fmaf(-d, h[e], t[j][e]);
        put(a.dh, row, j, h);
      }
    }
    if (!(a.pre && a.post && block)) __syncthreads();
  }
  if (group != ~size_t(0)) leave_gate(group);
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    if (!p.has(j)) continue;
    float f[EPL], g[EPL];
#pragma unroll
    for (int e = 0; e < EPL; ++e) f[e] = sum_pre(j, e), g[e] = sum_unit(j, e);
    if (a.pre) __builtin_memcpy(out + p.at[j], f, sizeof(f));
    if (a.post && (!shared_gate || !left)) keep(j, g);   // (a workgroup without a row: zeros)
  }
}

// Joins the workgroups' sums: columns of dpre, dpost and (from z = 2 on) of every gate that has several parts
constexpr int kStrips = 32, kColumns = 32;
template <class S>
__global__ __launch_bounds__(kStrips *kColumns) void k_norm_join(Args a, float *dpre, float *dpost, unsigned blocks) {
  __shared__ float lds[kStrips][kColumns];
  const size_t c = size_t(blockIdx.x) * kColumns + threadIdx.x % kColumns;
  const unsigned strip = threadIdx.x / kColumns;
  const bool weights = blockIdx.y < 2;
  if (weights && !(blockIdx.y ? dpost : dpre)) return;
  const unsigned n = weights ? blocks : a.chunks;
  const size_t g = weights ? 0 : blockIdx.y - 2 + size_t(blockIdx.z) * 32768;
  if (!weights && g >= a.gates) return;
  if (weights && blockIdx.z) return;
  const size_t step = weights ? 2 * a.dim : a.dim;
  const float *p = weights ? a.part + blockIdx.y * a.dim + c : a.gate_part + g * a.chunks * a.dim + c;
  float x = 0.f;
  if (c < a.dim) {
    unsigned i = strip;
    for (; i + 3 * kStrips < n; i += 4 * kStrips) {
      float v[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = p[(i + k * kStrips) * step];
      x += (v[0] + v[1]) + (v[2] + v[3]);
    }
    for (; i < n; i += kStrips) x += p[i * step];
  }
  lds[strip][threadIdx.x % kColumns] = x;
  __syncthreads();
  if (strip == 0 && c < a.dim) {
#pragma unroll
    for (int k = 1; k < kStrips; ++k) x += lds[k][threadIdx.x];
    if (weights) (blockIdx.y ? dpost : dpre)[c] = x;
    else S::st(static_cast<typename S::elem *>(a.dgate) + g * a.dim + c, x);
  }
}

// ------------------------------------------------------------------------------------ host

constexpr size_t kMostDim = 16384, kMostRows = 0x7fffffff;

// Threads to a row, eight values each (16 of rows of more than 8192, which leave no registers for the next row), and a workgroup's teams
struct Form {
  int team, per;
  bool wide;
};
Form form_of(size_t dim) {
  for (int team : {8, 32, 64, 128, 256, 512, 1024})
    if (dim <= size_t(team) * 8) return {team, team < 256 ? 256 / team : 1, false};
  return {1024, 1, true};
}
// How a backward pass is cut
struct Plan {
  Form form;
  unsigned each, chunks, blocks;
  size_t part, gate_part;   // floats
  size_t bytes() const { return (part + gate_part) * sizeof(float); }
};
Plan plan_of(size_t rows, size_t dim, size_t gates) {
  Plan p{form_of(dim), 1, 1, 1, 0, 0};
  const size_t teams = size_t(sgh_num_cus()) * (p.form.team <= 256 ? 1024 / kThreads<256> : p.form.team == 512 ? 2 : 1) * p.form.per;
  const size_t per_gate = gates ? rows / gates : 0, per = p.form.per;
  size_t each = (rows + teams - 1) / teams, n;
  if (each < 2) each = 2;   // (a workgroup's sums are as much to write and read as a row of fp32 values)
  p.chunks = 0;
  if (per_gate > each && per_gate * 2 >= per) {   // (a gate has work for half of a workgroup's teams)
    p.chunks = unsigned((per_gate + each * per - 1) / (each * per));
    each = (per_gate + p.chunks * per - 1) / (p.chunks * per);
    n = gates * p.chunks * per;
  } else {
    if (per_gate > 1) each = each > per_gate ? each / per_gate * per_gate : per_gate;
    n = (rows + each - 1) / each;
  }
  p.each = unsigned(each);
  p.blocks = unsigned((n + per - 1) / per);
  p.part = size_t(p.blocks) * 2 * dim;
  p.gate_part = p.chunks > 1 ? gates * p.chunks * dim : 0;
  return p;
}

#define SGH_NORM_FORMS(RUN, S)                                                                                       \
  constexpr int V = S::VEC, N = 8 / V;                                                                               \
  if (a.dim < size_t(V)) { RUN(S, 1, 8, 1, true, false); }                                                           \
  else if (f.wide) { RUN(S, V, 1024, 2 * N, false, false); }                                                         \
  else switch (f.team) {                                                                                             \
    case 8: if (stream) { RUN(S, V, 8, N, true, true); } else { RUN(S, V, 8, N, true, false); } break;               \
    case 32: if (stream) { RUN(S, V, 32, N, true, true); } else { RUN(S, V, 32, N, true, false); } break;            \
    case 64: if (stream) { RUN(S, V, 64, N, true, true); } else { RUN(S, V, 64, N, true, false); } break;            \
    case 128: if (stream) { RUN(S, V, 128, N, true, true); } else { RUN(S, V, 128, N, true, false); } break;         \
    case 256: if (stream) { RUN(S, V, 256, N, true, true); } else { RUN(S, V, 256, N, true, false); } break;         \
    case 512: if (stream) { RUN(S, V, 512, N, true, true); } else { RUN(S, V, 512, N, true, false); } break;         \
    default: if (stream) { RUN(S, V, 1024, N, true, true); } else { RUN(S, V, 1024, N, true, false); } break;        \
  }

// Past the caches from kStreamBytes for a tensor on, the results in both directions and forwards what is read as well (32768 rows of 4096 bfloat16
// values: forward 237 -> 212 us, backward 378 -> 363, with its loads 403)
template <class S>
bool streams(const Args &a) { return a.rows * a.dim * sizeof(typename S::elem) >= kStreamBytes; }

template <class S>
int run_fwd(const Args &a, const Form &f, unsigned blocks, hipStream_t s) {
  const bool stream = streams<S>(a);
#define RUN(S, EPL, TEAM, NV, HOLD, STREAM) \
  SGH_LAUNCH_TIMED((k_norm_fwd<S, EPL, TEAM, NV, HOLD, STREAM>), dim3(blocks), dim3(kThreads<TEAM>), 0, s, a)
  SGH_NORM_FORMS(RUN, S)
#undef RUN
  SGH_LAUNCH_CHECK();
  return SGH_OK;
}
template <class S>
int run_bwd(const Args &a, const Plan &p, float *dpre, float *dpost, hipStream_t s) {
  const Form &f = p.form;
  const bool stream = streams<S>(a);
#define LAUNCH(kern, threads, bytes)                                                                     \
  do {                                                                                                   \
    static std::atomic<unsigned long long> asked{0};                                                     \
    SGH_HIP_TRY(sgh_allow_lds(reinterpret_cast<const void *>(kern), asked));                             \
    hipLaunchKernelGGL(kern, dim3(p.blocks), dim3(threads), bytes, s, a);                                \
  } while (0)
#define RUN(S, EPL, TEAM, NV, HOLD, STREAM)                                                              \
  if constexpr (HOLD) LAUNCH((k_norm_bwd<S, EPL, TEAM, NV, STREAM>), kThreads<TEAM>, (f.per > 2 ? f.per : 2) * a.dim * sizeof(float)); \
  else LAUNCH((k_norm_bwd_wide<S, NV>), kWide, 2 * sizeof(float) * kWide * NV * EPL)
  SGH_NORM_FORMS(RUN, S)
#undef LAUNCH
#undef RUN
  SGH_LAUNCH_CHECK();
  const unsigned gates = p.chunks > 1 ? a.gates : 0, y = 2 + (gates < 32768 ? gates : 32768), z = gates ? (gates + 32767) / 32768 : 1;
  if (dpre || dpost || gates) {
    hipLaunchKernelGGL((k_norm_join<S>), dim3(unsigned((a.dim + kColumns - 1) / kColumns), y, z), dim3(kStrips * kColumns), 0, s, a, dpre, dpost,
                       p.blocks);
    SGH_LAUNCH_CHECK();
  }
  return SGH_OK;
}

int check_sizes(size_t rows, size_t dim, size_t gates) {
  if (rows > kMostRows || (gates != 0 && rows % gates != 0)) return SGH_EINVAL;   // (no rows are divided by any number)
  return dim > kMostDim ? SGH_ELIMIT : SGH_OK;
}

template <class S>
int clear(void *p, size_t n, void *stream) {   // (the bits of 0 are the same in both 16-bit types)
  if constexpr (sizeof(typename S::elem) == 4) return sgh_memset_f32(static_cast<float *>(p), 0.f, n, stream);
  else return sgh_memset_f16(static_cast<uint16_t *>(p), 0.f, n, stream);
}

template <class S>
int forward(const void *x, const void *h, const float *post, const void *gate, const float *pre, size_t rows, size_t dim, size_t gates,
            float scale, float eps, void *y, void *n, float *stats, void *stream) {
  if (rows == 0 || dim == 0) return SGH_OK;
  const int rc = check_sizes(rows, dim, gate ? gates : 0);
  if (rc != SGH_OK) return rc;
  if (!x || !stats || (h && !y) || (pre && !n) || (!h && (post || gate)) || (!h && !pre) || (gate && gates == 0)) return SGH_EINVAL;
  if (!(eps >= 0.f) || !__builtin_isfinite(eps)) return SGH_EINVAL;
  const size_t bytes = rows * dim * sizeof(typename S::elem), weights = dim * sizeof(float);
  const sgh_extent results[] = {{y, h ? bytes : 0}, {n, pre ? bytes : 0}, {stats, rows * 8}};
  const sgh_extent arguments[] = {{x, bytes}, {h, h ? bytes : 0}, {post, post ? weights : 0}, {pre, pre ? weights : 0},
                              {gate, gate ? gates * dim * sizeof(typename S::elem) : 0}};
  if (sgh_any_overlap(results, arguments)) return SGH_EINVAL;
  Args a = {};
  a.x = x, a.h = h, a.gate = gate, a.post = post, a.pre = pre, a.stats = stats, a.out_y = y, a.out_n = n;
  a.dim = dim, a.rows = unsigned(rows), a.gates = unsigned(gates), a.per_gate = gate ? unsigned(rows / gates) : 0, a.scale = scale, a.eps = eps;
  const Form f = form_of(dim);
  const size_t most = size_t(sgh_num_cus()) * (f.team <= 256 ? 8 : f.team == 512 ? 4 : 2) * f.per;
  a.each = unsigned((rows + most - 1) / most);
  const size_t teams = (rows + a.each - 1) / a.each;
  hipStream_t s = sgh_stream_of(stream);
  if (h) sgh_note_write(y, bytes);
  if (pre) sgh_note_write(n, bytes);
  sgh_prof_kernel_scope prof("norm_fwd/k_norm_fwd", double(bytes) * ((h ? 3 : 1) + (pre ? 1 : 0)), s);
  return run_fwd<S>(a, f, unsigned((teams + f.per - 1) / f.per), s);
}

template <class S>
int backward(const void *dy, const void *dn, const void *y, const float *stats, const void *h, const float *post, const void *gate,
             const float *pre, size_t rows, size_t dim, size_t gates, float scale, void *dx, void *dh, float *dpost, void *dgate, float *dpre,
             void *workspace, size_t ws_bytes, void *stream) {
  const int rc = check_sizes(rows, dim, gate ? gates : 0);
  if (rc != SGH_OK) return rc;
  if ((!h && (post || gate)) || (!h && !pre) || (gate && gates == 0 && rows != 0)) return SGH_EINVAL;
  if (dim == 0) return SGH_OK;
  if ((post && !dpost) || (pre && !dpre) || (gate && gates != 0 && !dgate)) return SGH_EINVAL;
  if (rows == 0) {   // (sums over no rows)
    int r = pre ? sgh_memset_f32(dpre, 0.f, dim, stream) : SGH_OK;
    if (r == SGH_OK && post) r = sgh_memset_f32(dpost, 0.f, dim, stream);
    if (r == SGH_OK && gate) r = clear<S>(dgate, gates * dim, stream);
    return r;
  }
  if ((!dy && !dn) || !stats || !dx || (pre && (!dn || !y)) || (h && !dh)) return SGH_EINVAL;
  const Plan p = plan_of(rows, dim, gate ? gates : 0);
  if (!workspace || ws_bytes < p.bytes()) return SGH_EWORKSPACE;
  if (!sgh_aligned16(workspace)) return SGH_EINVAL;
  const size_t bytes = rows * dim * sizeof(typename S::elem), weights = dim * sizeof(float);
  const size_t gate_bytes = gate ? gates * dim * sizeof(typename S::elem) : 0;
  const sgh_extent results[] = {{dx, bytes}, {dh, h ? bytes : 0}, {dpost, post ? weights : 0}, {dgate, gate_bytes}, {dpre, pre ? weights : 0},
                            {workspace, p.bytes()}};
  const sgh_extent arguments[] = {{dy, dy ? bytes : 0}, {dn, pre ? bytes : 0}, {y, pre ? bytes : 0}, {stats, rows * 8}, {h, h ? bytes : 0},
                              {post, post ? weights : 0}, {gate, gate_bytes}, {pre, pre ? weights : 0}};
  if (sgh_any_overlap(results, arguments)) return SGH_EINVAL;
  Args a = {};
  a.dy = dy, a.dn = dn, a.y = y, a.stats = const_cast<float *>(stats), a.h = h, a.post = post, a.gate = gate, a.pre = pre;
  a.dx = dx, a.dh = dh, a.dgate = dgate, a.part = static_cast<float *>(workspace), a.gate_part = a.part + p.part;
  a.dim = dim, a.rows = unsigned(rows), a.gates = unsigned(gates), a.per_gate = gate ? unsigned(rows / gates) : 0, a.scale = scale;
  a.each = p.each, a.chunks = p.chunks;
  hipStream_t s = sgh_stream_of(stream);
  sgh_note_write(dx, bytes);
  if (h) sgh_note_write(dh, bytes);
  if (gate) sgh_note_write(dgate, gate_bytes);
  if (post) sgh_note_write(dpost, weights);
  if (pre) sgh_note_write(dpre, weights);
  sgh_prof_kernel_scope prof("norm_bwd/k_norm_bwd", double(bytes) * ((dy ? 1 : 0) + 1 + (pre ? 2 : 0) + (h ? 2 : 0)), s);
  prof.span();
  return run_bwd<S>(a, p, pre ? dpre : nullptr, post ? dpost : nullptr, s);
}

}  // namespace

extern "C" {

size_t sgh_residual_norm_bwd_workspace_bytes(size_t rows, size_t dim, size_t gates, size_t elem_bytes) {
  if (rows == 0 || dim == 0 || check_sizes(rows, dim, gates) != SGH_OK || (elem_bytes != 2 && elem_bytes != 4)) return 0;
  return plan_of(rows, dim, gates).bytes();
}

#define SGH_RESIDUAL_NORM(SFX, S, T)                                                                                                  \
  int sgh_residual_norm_fwd_##SFX(const T *x, const T *h, const float *post, const T *gate, const float *pre, size_t rows,            \
                                  size_t dim, size_t gates, float scale, float eps, T *y, T *n, float *stats, void *stream) {         \
    return forward<S>(x, h, post, gate, pre, rows, dim, gates, scale, eps, y, n, stats, stream);                                      \
  }                                                                                                                                   \
  int sgh_residual_norm_bwd_##SFX(const T *dy, const T *dn, const T *y, const float *stats, const T *h, const float *post,            \
                                  const T *gate, const float *pre, size_t rows, size_t dim, size_t gates, float scale, T *dx, T *dh,  \
                                  float *dpost, T *dgate, float *dpre, void *workspace, size_t ws_bytes, void *stream) {              \
    return backward<S>(dy, dn, y, stats, h, post, gate, pre, rows, dim, gates, scale, dx, dh, dpost, dgate, dpre, workspace,          \
                       ws_bytes, stream);                                                                                             \
  }
SGH_RESIDUAL_NORM(f32, StF32, float)
SGH_RESIDUAL_NORM(f16, StF16, uint16_t)
SGH_RESIDUAL_NORM(bf16, StBF16, uint16_t)
#undef SGH_RESIDUAL_NORM

}  // extern "C"
