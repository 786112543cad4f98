// What the two halves of attention's backward pass share (attn_dq.hip, attn_dkv.hip).
#ifndef SINGA_AMD_CSRC_ATTN_BWD_H_
#define SINGA_AMD_CSRC_ATTN_BWD_H_

#include "attn_run.h"

namespace attn {

struct BwdArgs {
  Shape s;
  const void *q, *k, *v, *o, *dout;
  const float *lse;
  void *dq, *dk, *dv;
  // [2][batch][heads][q_len], from the first half: the logarithms to the base 2 of the row sums, less term_bits() (+inf where a row sees
  // nothing, so that its probabilities are 0), and -delta
  float *stats;
  float *q_part;      // [q_splits][q_units][rows][DP]
  float *bias_part;   // [heads][bias_blocks][buckets]
  float *k_part;      // [k_splits][2][k_units][k_len][DP]
  size_t bias_blocks;
  unsigned q_tiles, q_units, q_splits, k_tiles, k_units, k_splits;
  int pack, keys_each, turns_each;
  bool direct;     // of q, k, v and do, rows of s.dim
  int io_dim;      // o and the results have rows of io_dim
  bool io_direct;
};
constexpr int kRows = 128;   // queries (keys) of a block of the first (second) half

// binary16: the probabilities of the second half are stored times 2^14, so that small ones keep their bits (they are at most 1)
template <class T>
constexpr float term_bits() { return std::is_same<T, F16>::value ? 14.f : 0.f; }

template <class T>
int run_dq(const BwdArgs &a, const Bounds &bounds, float *dtable, hipStream_t s);   // (attn_dq.hip)

// The gradients of the scores in binary16 would leave its range on either side: they are as small as the result's gradient times a probability.
// Each column (a lane and its partner) has a power of two of its own, by which its terms are multiplied and its sums divided in the end; where
// terms grow out of the range the sums are brought down.  bfloat16 and fp32 have the range.
template <class T>
struct Range {
  template <int ND>
  __device__ __forceinline__ void fit(f32x16 &, f32x16 (&)[ND]) {}
  __device__ __forceinline__ float inverse() const { return 1.f; }
};
template <>
struct Range<F16> {
  float f = 0x1p100f;
  template <int ND>
  __device__ __forceinline__ void fit(f32x16 &x, f32x16 (&acc)[ND]) {
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, __builtin_fabsf(x[i]));
    top = max_of_pair(top);
    const bool high = top * f > 0x1p15f;
    if (__ballot(high)) {   // to [2^10, 2^11), for those that need it
      const float now = high ? __builtin_ldexpf(1.f, 11 - __builtin_amdgcn_frexp_expf(top)) : f, down = now / f;
      f = now;
#pragma unroll
      for (int n = 0; n < ND; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[n][i] *= down;
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] *= f;
  }
  __device__ __forceinline__ float inverse() const { return 1.f / f; }
};

}  // namespace attn

#endif  // SINGA_AMD_CSRC_ATTN_BWD_H_
