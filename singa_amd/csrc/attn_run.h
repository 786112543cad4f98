// Host side that the attention's entry points share: checks of a geometry and of what may overlap, arguments of the kernels.
#ifndef SINGA_AMD_CSRC_ATTN_RUN_H_
#define SINGA_AMD_CSRC_ATTN_RUN_H_

#include <atomic>

#include "attn.h"

namespace attn {

// bytes of LDS that a position bias may take beside the tiles
constexpr size_t kMostBand = 24 << 10;

int check_geom(const sgh_attn_geom *g);                   // (attn.hip)
void bounds_of(const sgh_attn_geom *g, Bounds *bounds);   // (attn.hip)
// (attn.hip) more than 64 KB of LDS have to be asked for, once for each kernel and device; `asked` is the kernel's own
hipError_t allow_lds(const void *kernel, std::atomic<unsigned long long> &asked);

static inline size_t band_bytes(const sgh_attn_geom *g) { return g->buckets ? (2 * size_t(g->max_distance) + 1) * sizeof(float) : 0; }

static inline Shape shape_of(const sgh_attn_geom *g, const float *table, const int32_t *q_lengths, const int32_t *k_lengths,
                             const int32_t *q_starts) {
  return {g->q_len,  g->k_len,  g->heads, g->kv_heads,     g->dim,          g->causal, g->scale, q_lengths, k_lengths,
          q_starts,  g->buckets, g->bidirectional, g->buckets ? g->max_distance : 0, g->buckets ? table : nullptr};
}

struct Extent {
  const void *p;
  size_t bytes;
};
// a result meets an argument or another result
template <int R, int A>
static inline bool any_overlap(const Extent (&results)[R], const Extent (&arguments)[A]) {
  for (int i = 0; i < R; ++i) {
    for (int j = i + 1; j < R; ++j)
      if (sgh_ranges_meet(results[i].p, results[i].bytes, results[j].p, results[j].bytes)) return true;
    for (int j = 0; j < A; ++j)
      if (sgh_ranges_meet(results[i].p, results[i].bytes, arguments[j].p, arguments[j].bytes)) return true;
  }
  return false;
}

}  // namespace attn

#endif  // SINGA_AMD_CSRC_ATTN_RUN_H_
