// Rows of a matrix whose length and start need not be multiples of 16 bytes, moved 16 bytes at a time: global memory takes vector
// accesses at any element, so a row is cut into whole vectors from its own start and the last vector is moved back to end with the row
// (a few elements are then handled twice) rather than taken apart.
#ifndef SINGA_AMD_CSRC_ROWS_H_
#define SINGA_AMD_CSRC_ROWS_H_

#include <stddef.h>

#include "storage.h"

// EPL elements (a vector's worth or one) at any element of a tensor of storage type S, as floats
template <class S, int EPL>
__device__ __forceinline__ void sgh_load_any(const typename S::elem *p, float *out) {
  if constexpr (EPL == 1) {
    out[0] = S::ld(p);
  } else {
    static_assert(EPL == S::VEC, "one 16-byte vector");
    alignas(16) typename S::elem e[EPL];
    __builtin_memcpy(e, p, 16);
    S::template load16<false>(e, out);
  }
}
// The same; STREAM: past the caches
template <class S, int EPL, bool STREAM>
__device__ __forceinline__ void sgh_load_any(const typename S::elem *p, float *out) {
  if constexpr (STREAM && EPL != 1) {
    typedef sgh_v4u anywhere __attribute__((aligned(2)));
    const sgh_v4u v = __builtin_nontemporal_load(reinterpret_cast<const anywhere *>(p));
    sgh_load_any<S, EPL>(reinterpret_cast<const typename S::elem *>(&v), out);
  } else {
    sgh_load_any<S, EPL>(p, out);
  }
}
template <class S, int EPL>
__device__ __forceinline__ void sgh_store_any(typename S::elem *p, const float *in) {
  if constexpr (EPL == 1) {
    S::st(p, in[0]);
  } else {
    static_assert(EPL == S::VEC, "one 16-byte vector");
    alignas(16) typename S::elem e[EPL];
    S::store16(e, in);
    __builtin_memcpy(p, e, 16);
  }
}
template <class S, int EPL, bool STREAM>
__device__ __forceinline__ void sgh_store_any(typename S::elem *p, const float *in) {
  if constexpr (STREAM && EPL != 1) {
    alignas(16) typename S::elem e[EPL];
    S::store16(e, in);
    sgh_v4u v;
    __builtin_memcpy(&v, e, 16);
    typedef sgh_v4u anywhere __attribute__((aligned(2)));
    __builtin_nontemporal_store(v, reinterpret_cast<anywhere *>(p));
  } else {
    sgh_store_any<S, EPL>(p, in);
  }
}

// Tensors of at least this many bytes go past the caches: they would not stay in the 256 MB of the last one until they are read again
constexpr size_t kStreamBytes = size_t(96) << 20;

// [a, a + a_bytes) and [b, b + b_bytes) have a byte in common
static inline bool sgh_ranges_meet(const void *a, size_t a_bytes, const void *b, size_t b_bytes) {
  const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
  return a_bytes != 0 && b_bytes != 0 && x < y + b_bytes && y < x + a_bytes;
}

#endif  // SINGA_AMD_CSRC_ROWS_H_
