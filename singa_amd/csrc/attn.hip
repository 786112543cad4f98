// Sizes of an attention and the borders of its position buckets.
#include "attn_run.h"

namespace {

// A whole number of up to 96 * 32 bits: products of up to 128 factors of at most 11 bits
struct Big {
  static constexpr int N = 96;
  uint32_t d[N] = {1};
  void times(uint32_t f) {
    uint64_t carry = 0;
    for (int i = 0; i < N; ++i) {
      carry += uint64_t(d[i]) * f;
      d[i] = uint32_t(carry);
      carry >>= 32;
    }
  }
  Big(int a, int na, int b, int nb) {
    for (int i = 0; i < na; ++i) times(uint32_t(a));
    for (int i = 0; i < nb; ++i) times(uint32_t(b));
  }
  bool less_than(const Big &o) const {
    for (int i = N - 1; i >= 0; --i)
      if (d[i] != o.d[i]) return d[i] < o.d[i];
    return false;
  }
};

constexpr int kMostDistance = 1024, kMostLength = 1 << 28, kMostRow = 1 << 20;
constexpr unsigned long long kMostBlocks = 1ull << 22;

}  // namespace

namespace attn {

int check_geom(const sgh_attn_geom *g) {
  if (!g || g->batch < 0 || g->q_len < 0 || g->k_len < 0 || g->heads < 1 || g->kv_heads < 1 || g->heads % g->kv_heads != 0 || g->dim < 1)
    return SGH_EINVAL;
  if (!(g->scale > -__builtin_inff() && g->scale < __builtin_inff())) return SGH_EINVAL;
  if (g->dim > SGH_ATTN_MAX_DIM || g->q_len > kMostLength || g->k_len > kMostLength || (long long)g->heads * g->dim > kMostRow) return SGH_ELIMIT;
  // (the product of all three sizes may pass 64 bits)
  const unsigned long long most = g->batch ? kMostBlocks / unsigned(g->batch) : ~0ull, tiles = g->q_len / 32 + 1, kv_tiles = g->k_len / 32 + 1;
  if (g->heads * tiles > most || g->kv_heads * kv_tiles > most) return SGH_ELIMIT;
  if (g->buckets == 0) return SGH_OK;
  const int n = g->bidirectional ? g->buckets / 2 : g->buckets;
  if (g->buckets < 0 || (g->bidirectional && g->buckets % 2 != 0) || n < 2 || g->max_distance <= n / 2) return SGH_EINVAL;
  if (n > SGH_ATTN_MAX_BUCKETS || g->max_distance > kMostDistance) return SGH_ELIMIT;
  if (g->bounds != n - 1) return SGH_EINVAL;   // (not from sgh_attn_geom_init)
  return SGH_OK;
}

void bounds_of(const sgh_attn_geom *g, Bounds *bounds) {
  bounds->n = g->buckets ? g->bounds : 0;
  for (int i = 0; i < bounds->n; ++i) bounds->at[i] = g->bound[i];
}

}  // namespace attn

hipError_t sgh_allow_lds(const void *kernel, std::atomic<unsigned long long> &asked) {
  int device;
  const hipError_t e = hipGetDevice(&device);
  if (e != hipSuccess) return e;
  const unsigned long long bit = 1ull << (device & 63);
  if (asked.load(std::memory_order_relaxed) & bit) return hipSuccess;
  const hipError_t f = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, 156 * 1024);
  if (f == hipSuccess) asked.fetch_or(bit, std::memory_order_relaxed);
  return f;
}

extern "C" int sgh_attn_geom_init(sgh_attn_geom *g, int batch, int q_len, int k_len, int heads, int kv_heads, int dim, int causal, float scale,
                                  int buckets, int max_distance, int bidirectional) {
  if (!g) return SGH_EINVAL;
  *g = sgh_attn_geom{};
  g->batch = batch, g->q_len = q_len, g->k_len = k_len, g->heads = heads, g->kv_heads = kv_heads, g->dim = dim;
  g->causal = causal != 0, g->scale = scale;
  if (buckets != 0) {
    g->buckets = buckets, g->max_distance = max_distance, g->bidirectional = bidirectional != 0;
    const int n = g->bidirectional ? buckets / 2 : buckets, exact = n / 2;
    g->bounds = n - 1;
    if (buckets > 0 && n >= 2 && n <= SGH_ATTN_MAX_BUCKETS && max_distance > exact && max_distance <= kMostDistance) {
      // distances below `exact` have a bucket each; behind them bucket exact + t begins at the first m with
      // (m / exact)^(n - exact) >= (max_distance / exact)^t, in whole numbers
      for (int i = 0; i < exact; ++i) g->bound[i] = i + 1;
      int m = exact;
      for (int t = 1; t < n - exact; ++t) {
        while (Big(m, n - exact, exact, t).less_than(Big(max_distance, t, exact, n - exact))) ++m;
        g->bound[exact + t - 1] = m;
      }
    }
  }
  return attn::check_geom(g);
}
