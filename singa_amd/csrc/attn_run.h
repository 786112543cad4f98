// Host side that the attention's entry points share: checks of a geometry, arguments of the kernels.
#ifndef SINGA_AMD_CSRC_ATTN_RUN_H_
#define SINGA_AMD_CSRC_ATTN_RUN_H_

#include "attn.h"

namespace attn {

// bytes of LDS that a position bias may take beside the tiles
constexpr size_t kMostBand = 24 << 10;

int check_geom(const sgh_attn_geom *g);                   // (attn.hip)
void bounds_of(const sgh_attn_geom *g, Bounds *bounds);   // (attn.hip)

static inline size_t band_bytes(const sgh_attn_geom *g) { return g->buckets ? (2 * size_t(g->max_distance) + 1) * sizeof(float) : 0; }

static inline Shape shape_of(const sgh_attn_geom *g, const float *table, const int32_t *q_lengths, const int32_t *k_lengths,
                             const int32_t *q_starts) {
  return {g->q_len,  g->k_len,  g->heads, g->kv_heads,     g->dim,          g->causal, g->scale, q_lengths, k_lengths,
          q_starts,  g->buckets, g->bidirectional, g->buckets ? g->max_distance : 0, g->buckets ? table : nullptr};
}

// Rows whose length is no multiple of 16 bytes are padded (k_attn_pad): to how many values of elem_bytes bytes, 0 where they are not
static inline int wide_of(int dim, size_t elem_bytes) {
  const int vec = int(16 / elem_bytes);
  return dim % vec == 0 ? 0 : (dim + vec - 1) / vec * vec;
}
// room for `rows` of them, whatever the tensors' type
static inline size_t wide_bytes(int dim, size_t rows) {
  const size_t a = size_t(wide_of(dim, 4)) * 4, b = size_t(wide_of(dim, 2)) * 2;
  return rows * (a > b ? a : b);
}
template <class T>
static inline int pad_rows(const PadArgs &a, int tensors, hipStream_t s) {
  size_t most = 0;
  for (int i = 0; i < tensors; ++i) most = a.rows[i] > most ? a.rows[i] : most;
  const size_t blocks = (most * (a.wide / T::VEC) + kBlock - 1) / kBlock, limit = 8 * size_t(sgh_num_cus());
  if (blocks == 0) return SGH_OK;
  hipLaunchKernelGGL((k_attn_pad<T>), dim3(unsigned(blocks < limit ? blocks : limit), unsigned(tensors)), dim3(kBlock), 0, s, a);
  SGH_LAUNCH_CHECK();
  return SGH_OK;
}

}  // namespace attn

#endif  // SINGA_AMD_CSRC_ATTN_RUN_H_
