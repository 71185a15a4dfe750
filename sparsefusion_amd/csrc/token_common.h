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

// V values at p + i0 of a row of n elements as fp32; zeros behind its end.
template <typename T>
__device__ __forceinline__ void sf_load_chunk(const T *__restrict__ p, long long i0, long long n,
                                              float *v) {
  constexpr int V = SfChunk<T>::V;
  if (i0 + V <= n) {
    const typename SfChunk<T>::type c = *reinterpret_cast<const typename SfChunk<T>::type *>(p + i0);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = (float)c[j];
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = i0 + j < n ? (float)p[i0 + j] : 0.0f;
  }
}

template <typename T, bool NT = false>
__device__ __forceinline__ void sf_store_chunk(T *__restrict__ p, long long i0, long long n,
                                               const float *v) {
  constexpr int V = SfChunk<T>::V;
  if (i0 + V <= n) {
    typename SfChunk<T>::type c;
#pragma unroll
    for (int j = 0; j < V; ++j) c[j] = (T)v[j];
    auto *at = reinterpret_cast<typename SfChunk<T>::type *>(p + i0);
    if constexpr (NT) __builtin_nontemporal_store(c, at);
    else *at = c;
  } else {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (i0 + j < n) p[i0 + j] = (T)v[j];
  }
}

static inline size_t sf_dtype_size(int dtype) { return dtype == SF_DTYPE_F32 ? 4 : 2; }

// How a kernel's rows lie: RAGGED, some chunk is cut by the row's end; WHOLE, none is; STREAM, none is and
// they go around the caches.
enum { SF_RAGGED, SF_WHOLE, SF_STREAM };

// V values at p + i0 of a row of n elements as they are, zeros behind its end.  Nothing waits for them
// here: converting inside the branch would, a load at a time.
template <typename T, int MODE>
__device__ __forceinline__ typename SfChunk<T>::type sf_load_raw(const T *__restrict__ p, int i0, int n) {
  constexpr int V = SfChunk<T>::V;
  typename SfChunk<T>::type c;
#pragma unroll
  for (int j = 0; j < V; ++j) c[j] = (T)0.0f;
  if (MODE == SF_RAGGED ? i0 + V <= n : i0 < n) {
    const auto *at = reinterpret_cast<const typename SfChunk<T>::type *>(p + i0);
    if constexpr (MODE == SF_STREAM) c = __builtin_nontemporal_load(at);
    else c = *at;
  } else if (MODE == SF_RAGGED && i0 < n) {
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (i0 + j < n) c[j] = p[i0 + j];
  }
  return c;
}

// Whether m rows of `row_bytes` go around the caches, NT: tensors of 64 MB (the last-level cache holds
// 256 MB, a pass has four such) whose rows are whole lines.  In us without and with, inputs and outputs in other
// places each time: add and norm of 259200 x 256 bf16 97 and 91, of 60000 x 512 fp32 90 and 86, their gradients 105
// and 94, 96 and 87; the pass for dz of 32400 x 2048 bf16 and the products that read it 139 and 129.  At 32 MB the
// norms still gain (65536 x 256 bf16 29.2 and 27.3), a dz that is read again loses (52.3 and 53.6).  Rows that share
// lines: gradients of norms of 130000 x 200 fp32 79 and 73, but of 17000 x 2056 142 and 157.
static inline bool sf_streamed(long long m, size_t row_bytes) {
  return row_bytes % 128 == 0 && (size_t)m * row_bytes >= ((size_t)64 << 20);
}
