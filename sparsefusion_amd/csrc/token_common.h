// Shared pieces of the token operators (layer_norm.hip, linear*.hip): the three storage types and
// their 16-byte chunks.  Arithmetic is fp32 everywhere; a value is rounded once, when it is stored.
#pragma once
#include "sf_common.h"

typedef float sf_f32x4 __attribute__((ext_vector_type(4)));
typedef float sf_f32x16 __attribute__((ext_vector_type(16)));

// One 16-byte chunk of T: V elements.  Rows of odd length start at any multiple of the element
// size; gfx950 serves 16-byte global accesses at such addresses, so the chunk type only promises
// the element's alignment and ragged rows keep the wide loads.
template <typename T>
struct SfChunk {
  static constexpr int V = 16 / sizeof(T);
  typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};

// V values at p + i0 of a row of n elements as fp32; zeros behind its end.  NT: a load that leaves the
// caches to others, for tensors that do not fit them anyway.
template <typename T, bool NT = false>
__device__ __forceinline__ void sf_load_chunk(const T *__restrict__ p, long long i0, long long n,
                                              float *v) {
  constexpr int V = SfChunk<T>::V;
  if (i0 + V <= n) {
    const auto *at = reinterpret_cast<const typename SfChunk<T>::type *>(p + i0);
    typename SfChunk<T>::type c;
    if constexpr (NT) c = __builtin_nontemporal_load(at);
    else c = *at;
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = (float)c[j];
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = i0 + j < n ? (float)p[i0 + j] : 0.0f;
  }
}

template <typename T>
__device__ __forceinline__ void sf_store_chunk(T *__restrict__ p, long long i0, long long n,
                                               const float *v) {
  constexpr int V = SfChunk<T>::V;
  if (i0 + V <= n) {
    typename SfChunk<T>::type c;
#pragma unroll
    for (int j = 0; j < V; ++j) c[j] = (T)v[j];
    *reinterpret_cast<typename SfChunk<T>::type *>(p + i0) = c;
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (i0 + j < n) p[i0 + j] = (T)v[j];
  }
}

// Streams of at least this size are read with NT loads (the last-level cache holds 256 MB, a pass has
// four such).  Add and norm of 259200 x 256 bf16 (133 MB each): 103.7 us without, 87.4 with; its
// gradients 104.7 and 99.6; of 5003 x 333 fp32 (7 MB each, cached): 9.2 and 10.3, gradients 15.1 and 17.3.
constexpr size_t kSfStreamBytes = (size_t)64 << 20;

static inline size_t sf_dtype_size(int dtype) { return dtype == SF_DTYPE_F32 ? 4 : 2; }
