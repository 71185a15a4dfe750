// Layer norm over the last dimension with the residual add in front of it, forward and backward.
//
//   s = x + r;  mu = mean(s);  rstd = 1 / sqrt(mean((s - mu)^2) + eps);  y = (s - mu) rstd w + b
//   xh = (s - mu) rstd;  g = dy w;  ds = rstd (g - mean(g) - xh mean(g xh)) + dsum
//   dw = sum_rows dy xh;  db = sum_rows dy
//
// Both directions are bound by memory: every tensor is read or written once, the row lives in
// registers between its loads (all in flight at once) and its stores, and all sums are fp32.  The mean is
// summed from s / d, so rows whose sum passes fp32's range keep theirs; it is off by some steps of a large
// common offset.  A second pass over the registers sums what is left of the row, c = s - mu (exact for values
// near mu), and its squares: mean(c) corrects the mean, mean(c^2) - mean(c)^2 is the variance, and the offset
// costs no digits (a row of 1000 times 1000.7 gave up to 0.04 without, 0 with).  259200 x 256 bf16, 531 MB each
// way: add and norm 92 us (5.8 TB/s), gradients 91 us and 5 for the join; a copy of that size moves
// 4.9 TB/s.
//
// A row belongs to a group of LANES lanes, each holding NV 16-byte chunks of it: 8 to 64 lanes of a
// wave for short rows, so that no lane idles at 128 channels, up to a whole workgroup of 1024 lanes
// for long ones.  Rows longer than that (16384 16-bit or 8192 fp32 elements) are walked chunk by
// chunk, re-read for each pass.
//
// The gradient of the weight is a sum over all rows: each group keeps its columns' partial sums in
// registers while it walks its rows, the groups of a workgroup join through LDS, and a second kernel
// adds the workgroups' partials in a fixed order.  No atomics: the same inputs give the same bits.
#include "token_common.h"

namespace {

constexpr int kThreads = 256;

// Sum over the LANES lanes of a group; every lane receives it.  Groups wider than a wave go through
// `red` (16 floats), which is free again after the next call's first barrier.
template <int LANES, int THREADS>
__device__ __forceinline__ float group_sum(float v, float *red) {
#pragma unroll
  for (int d = (LANES < 64 ? LANES : 64) / 2; d > 0; d >>= 1) v += __shfl_xor(v, d, 64);
  if constexpr (LANES > 64) {
    static_assert(LANES == THREADS, "a wide group is the whole workgroup");
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    float t = 0.0f;
#pragma unroll
    for (int i = 0; i < THREADS / 64; ++i) t += red[i];
    v = t;
  }
  return v;
}

// The same for two sums at once.
template <int LANES, int THREADS>
__device__ __forceinline__ void group_sums(float &a, float &b, float (*red)[2]) {
#pragma unroll
  for (int d = (LANES < 64 ? LANES : 64) / 2; d > 0; d >>= 1) {
    const float u = __shfl_xor(a, d, 64), v = __shfl_xor(b, d, 64);
    a += u, b += v;
  }
  if constexpr (LANES > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6][0] = a, red[threadIdx.x >> 6][1] = b;
    __syncthreads();
    a = b = 0.0f;
#pragma unroll
    for (int i = 0; i < THREADS / 64; ++i) a += red[i][0], b += red[i][1];
  }
}

// mean(c^2) - mean(c)^2, which rounding may carry below 0; NaN stays.
__device__ __forceinline__ float variance(float mean_square, float mean) {
  return __builtin_elementwise_maximum(fmaf(-mean, mean, mean_square), 0.0f);
}

template <typename P, int V>
__device__ __forceinline__ void load_param(const void *p, int i0, int n, float fallback, float *v) {
  // parameters may be fp32 beside 16-bit rows, so their chunk is V elements of their own type
  const P *q = static_cast<const P *>(p);
#pragma unroll
  for (int j = 0; j < V; ++j) v[j] = (q && i0 + j < n) ? (float)q[i0 + j] : fallback;
}

template <typename T, typename P, int LANES, int NV, int THREADS, int MODE>
__global__ void __launch_bounds__(THREADS)
norm_fwd_kernel(const T *__restrict__ x, const T *__restrict__ res, const void *w, const void *b,
                T *__restrict__ y, T *__restrict__ sum, float *__restrict__ mean,
                float *__restrict__ rstd, long long m, int d, float eps) {
  constexpr int V = SfChunk<T>::V, GROUPS = THREADS / LANES;
  __shared__ float red[16], red2[16][2];
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const float inv_d = 1.0f / (float)d;
  float wv[NV][V], bv[NV][V];
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    load_param<P, V>(w, (c * LANES + lane) * V, d, 1.0f, wv[c]);
    load_param<P, V>(b, (c * LANES + lane) * V, d, 0.0f, bv[c]);
  }
  for (long long r0 = (long long)blockIdx.x * GROUPS; r0 < m; r0 += (long long)gridDim.x * GROUPS) {
    const long long row = r0 + group;
    const bool live = row < m;      // whole groups only: the shuffles of a group stay inside it
    const long long at = (live ? row : 0) * d;
    float v[NV][V];
    float s = 0.0f;
    typename SfChunk<T>::type rx[NV], rr[NV];      // the row's loads, all in flight
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      rx[c] = sf_load_raw<T, MODE>(x + at, (c * LANES + lane) * V, d);
      if (res) rr[c] = sf_load_raw<T, MODE>(res + at, (c * LANES + lane) * V, d);
    }
#pragma unroll
    for (int c = 0; c < NV; ++c) {
#pragma unroll
      for (int j = 0; j < V; ++j) v[c][j] = (float)rx[c][j];
      if (res) {
#pragma unroll
        for (int j = 0; j < V; ++j) v[c][j] += (float)rr[c][j];
      }
      if (sum && live) sf_store_chunk<T, MODE == SF_STREAM>(sum + at, (c * LANES + lane) * V, d, v[c]);
#pragma unroll
      for (int j = 0; j < V; ++j) s = fmaf(v[c][j], inv_d, s);   // zeros behind the row's end
    }
    const float mu = group_sum<LANES, THREADS>(s, red);
    float q = 0.0f, e = 0.0f;
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int j = 0; j < V; ++j) {
        v[c][j] -= mu;
        if ((c * LANES + lane) * V + j < d) q += v[c][j] * v[c][j], e += v[c][j];
      }
    group_sums<LANES, THREADS>(q, e, red2);
    e *= inv_d;
    const float rs = 1.0f / sqrtf(variance(q * inv_d, e) + eps);
    if (!live) continue;
#pragma unroll
    for (int c = 0; c < NV; ++c) {
#pragma unroll
      for (int j = 0; j < V; ++j) v[c][j] = (v[c][j] - e) * rs * wv[c][j] + bv[c][j];
      sf_store_chunk<T, MODE == SF_STREAM>(y + at, (c * LANES + lane) * V, d, v[c]);
    }
    if (lane == 0) {
      if (mean) mean[row] = mu + e;
      if (rstd) rstd[row] = rs;
    }
  }
}

// Rows too long for registers: three passes over the row, one workgroup each.
template <typename T, typename P>
__global__ void __launch_bounds__(1024)
norm_fwd_long_kernel(const T *__restrict__ x, const T *__restrict__ res, const void *w, const void *b,
                     T *__restrict__ y, T *__restrict__ sum, float *__restrict__ mean,
                     float *__restrict__ rstd, long long m, int d, float eps) {
  constexpr int V = SfChunk<T>::V;
  __shared__ float red[16], red2[16][2];
  const float inv_d = 1.0f / (float)d;
  for (long long row = blockIdx.x; row < m; row += gridDim.x) {
    const long long at = row * d;
    auto load = [&](int i0, float *v) {
      sf_load_chunk<T>(x + at, i0, d, v);
      if (res) {
        float u[V];
        sf_load_chunk<T>(res + at, i0, d, u);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] += u[j];
      }
    };
    float s = 0.0f, q = 0.0f, e = 0.0f, v[V];
    for (long long i0 = threadIdx.x * V; i0 < d; i0 += 1024 * V) {
      load((int)i0, v);
      if (sum) sf_store_chunk<T>(sum + at, i0, d, v);
#pragma unroll
      for (int j = 0; j < V; ++j) s = fmaf(v[j], inv_d, s);
    }
    const float mu = group_sum<1024, 1024>(s, red);
    for (long long i0 = threadIdx.x * V; i0 < d; i0 += 1024 * V) {
      load((int)i0, v);
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (i0 + j < d) q += (v[j] - mu) * (v[j] - mu), e += v[j] - mu;
    }
    group_sums<1024, 1024>(q, e, red2);
    e *= inv_d;
    const float rs = 1.0f / sqrtf(variance(q * inv_d, e) + eps);
    for (long long i0 = threadIdx.x * V; i0 < d; i0 += 1024 * V) {
      float wv[V], bv[V];
      load_param<P, V>(w, (int)i0, d, 1.0f, wv);
      load_param<P, V>(b, (int)i0, d, 0.0f, bv);
      load((int)i0, v);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = (v[j] - mu - e) * rs * wv[j] + bv[j];
      sf_store_chunk<T>(y + at, i0, d, v);
    }
    if (threadIdx.x == 0) {
      if (mean) mean[row] = mu + e;
      if (rstd) rstd[row] = rs;
    }
  }
}

// dx of every row and, in part[block][2][d] (fp32), the workgroup's share of dw and db.
template <typename T, typename P, int LANES, int NV, int THREADS, int MODE>
__global__ void __launch_bounds__(THREADS)
norm_bwd_kernel(const T *__restrict__ dy, const T *__restrict__ x, const float *__restrict__ mean,
                const float *__restrict__ rstd, const void *w, const T *__restrict__ dsum,
                T *__restrict__ dx, float *__restrict__ part, long long m, int d) {
  constexpr int V = SfChunk<T>::V, GROUPS = THREADS / LANES;
  __shared__ float red[16];
  extern __shared__ float cols[];      // [GROUPS][LANES * NV * V], one of dw / db at a time
  const int lane = threadIdx.x % LANES, group = threadIdx.x / LANES;
  const float inv_d = 1.0f / (float)d;
  float wv[NV][V], aw[NV][V], ab[NV][V];
#pragma unroll
  for (int c = 0; c < NV; ++c) {
    load_param<P, V>(w, (c * LANES + lane) * V, d, 1.0f, wv[c]);
#pragma unroll
    for (int j = 0; j < V; ++j) aw[c][j] = ab[c][j] = 0.0f;
  }
  for (long long r0 = (long long)blockIdx.x * GROUPS; r0 < m; r0 += (long long)gridDim.x * GROUPS) {
    const long long row = r0 + group;
    const bool live = row < m;
    const long long at = (live ? row : 0) * d;
    const float mu = mean[live ? row : 0], rs = rstd[live ? row : 0];
    float g[NV][V], xh[NV][V];
    float s1 = 0.0f, s2 = 0.0f;
    typename SfChunk<T>::type ry[NV], rx[NV], rd[NV];      // the row's loads, all in flight
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      ry[c] = sf_load_raw<T, MODE>(dy + at, (c * LANES + lane) * V, d);
      rx[c] = sf_load_raw<T, MODE>(x + at, (c * LANES + lane) * V, d);
      if (dsum) rd[c] = sf_load_raw<T, MODE>(dsum + at, (c * LANES + lane) * V, d);
    }
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      const int i0 = (c * LANES + lane) * V;
#pragma unroll
      for (int j = 0; j < V; ++j) {
        g[c][j] = (float)ry[c][j];
        xh[c][j] = (float)rx[c][j];
        // g is zero behind the row's end, so xh there (a product of nothing but the mean) is harmless
        // unless it is not finite: it is cleared as well
        xh[c][j] = i0 + j < d ? (xh[c][j] - mu) * rs : 0.0f;
        if (live) {
          aw[c][j] += g[c][j] * xh[c][j];
          ab[c][j] += g[c][j];
        }
        g[c][j] *= wv[c][j];
        s1 += g[c][j];
        s2 += g[c][j] * xh[c][j];
      }
    }
    s1 = group_sum<LANES, THREADS>(s1, red) * inv_d;
    s2 = group_sum<LANES, THREADS>(s2, red) * inv_d;
    if (!live) continue;
#pragma unroll
    for (int c = 0; c < NV; ++c) {
      const int i0 = (c * LANES + lane) * V;
      float u[V];
#pragma unroll
      for (int j = 0; j < V; ++j) {
        u[j] = (g[c][j] - s1 - xh[c][j] * s2) * rs;
        if (dsum) u[j] += (float)rd[c][j];
      }
      sf_store_chunk<T, MODE == SF_STREAM>(dx + at, i0, d, u);
    }
  }
  if (!part) return;
  float *out = part + (size_t)blockIdx.x * 2 * d;
  if constexpr (GROUPS == 1) {
#pragma unroll
    for (int c = 0; c < NV; ++c)
#pragma unroll
      for (int j = 0; j < V; j += 4) {
        const int i = (c * LANES + lane) * V + j;
        if (i < d) {
          sf_store_chunk<float>(out, i, d, &aw[c][j]);
          sf_store_chunk<float>(out + d, i, d, &ab[c][j]);
        }
      }
  } else {
    constexpr int W = LANES * NV * V;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      __syncthreads();
#pragma unroll
      for (int c = 0; c < NV; ++c)
#pragma unroll
        for (int j = 0; j < V; ++j)
          cols[group * W + (c * LANES + lane) * V + j] = half ? ab[c][j] : aw[c][j];
      __syncthreads();
      for (int i = threadIdx.x; i < d; i += THREADS) {
        float t = 0.0f;
        for (int k = 0; k < GROUPS; ++k) t += cols[k * W + i];
        out[half * d + i] = t;
      }
    }
  }
}

// Long rows: dx in two passes over the row; the column sums by norm_cols_long_kernel.
template <typename T, typename P>
__global__ void __launch_bounds__(1024)
norm_bwd_long_kernel(const T *__restrict__ dy, const T *__restrict__ x, const float *__restrict__ mean,
                     const float *__restrict__ rstd, const void *w, const T *__restrict__ dsum,
                     T *__restrict__ dx, long long m, int d) {
  constexpr int V = SfChunk<T>::V;
  __shared__ float red[16];
  const float inv_d = 1.0f / (float)d;
  for (long long row = blockIdx.x; row < m; row += gridDim.x) {
    const long long at = row * d;
    const float mu = mean[row], rs = rstd[row];
    float s1 = 0.0f, s2 = 0.0f, g[V], xv[V], wv[V];
    for (long long i0 = threadIdx.x * V; i0 < d; i0 += 1024 * V) {
      sf_load_chunk<T>(dy + at, i0, d, g);
      sf_load_chunk<T>(x + at, i0, d, xv);
      load_param<P, V>(w, (int)i0, d, 1.0f, wv);
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (i0 + j < d) {
          s1 += g[j] * wv[j];
          s2 += g[j] * wv[j] * ((xv[j] - mu) * rs);
        }
    }
    s1 = group_sum<1024, 1024>(s1, red) * inv_d;
    s2 = group_sum<1024, 1024>(s2, red) * inv_d;
    for (long long i0 = threadIdx.x * V; i0 < d; i0 += 1024 * V) {
      float u[V];
      sf_load_chunk<T>(dy + at, i0, d, g);
      sf_load_chunk<T>(x + at, i0, d, xv);
      load_param<P, V>(w, (int)i0, d, 1.0f, wv);
      if (dsum) {
        sf_load_chunk<T>(dsum + at, i0, d, u);
      } else {
#pragma unroll
        for (int j = 0; j < V; ++j) u[j] = 0.0f;
      }
#pragma unroll
      for (int j = 0; j < V; ++j)
        u[j] += (g[j] * wv[j] - s1 - (xv[j] - mu) * rs * s2) * rs;
      sf_store_chunk<T>(dx + at, i0, d, u);
    }
  }
}

// part[blockIdx.y][2][d]: sums of a workgroup's rows, one lane per column.
template <typename T>
__global__ void __launch_bounds__(kThreads)
norm_cols_long_kernel(const T *__restrict__ dy, const T *__restrict__ x,
                      const float *__restrict__ mean, const float *__restrict__ rstd,
                      float *__restrict__ part, long long m, int d) {
  const int i = blockIdx.x * kThreads + threadIdx.x;
  if (i >= d) return;
  float a = 0.0f, s = 0.0f;
  for (long long row = blockIdx.y; row < m; row += gridDim.y) {
    const float g = (float)dy[row * d + i];
    a += g * (((float)x[row * d + i] - mean[row]) * rstd[row]);
    s += g;
  }
  part[((size_t)blockIdx.y * 2) * d + i] = a;
  part[((size_t)blockIdx.y * 2 + 1) * d + i] = s;
}

// Adds the workgroups' partial column sums: 32 columns by 32 strided runs of partials a workgroup.
template <typename P>
__global__ void __launch_bounds__(1024)
norm_join_kernel(const float *__restrict__ part, int blocks, int d, P *__restrict__ dw,
                 P *__restrict__ db) {
  __shared__ float red[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int i = blockIdx.x * 32 + tx;      // of the 2 d sums
  float t = 0.0f;
  if (i < 2 * d) {
    // 16 loads in flight: this kernel is nothing but their latency
    for (int b0 = ty; b0 < blocks; b0 += 16 * 32) {
      float u[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) u[k] = b0 + 32 * k < blocks ? part[(size_t)(b0 + 32 * k) * 2 * d + i] : 0.0f;
#pragma unroll
      for (int k = 0; k < 16; ++k) t += u[k];
    }
  }
  red[ty][tx] = t;
  __syncthreads();
  if (ty == 0 && i < 2 * d) {
    float a = 0.0f;
#pragma unroll
    for (int k = 0; k < 32; ++k) a += red[k][tx];
    if (i < d) {
      if (dw) dw[i] = (P)a;
    } else if (db) {
      db[i - d] = (P)a;
    }
  }
}

struct NormArgs {
  const void *dy, *x, *res, *w, *b;
  void *y, *sum;
  float *mean, *rstd, *part;
  long long m;
  int d, blocks;
  float eps;
  hipStream_t st;
};

// Lanes and chunks per lane of a row of `chunks` 16-byte chunks (see the head of the file); 0 lanes:
// the row does not fit registers.
struct NormShape {
  int lanes, nv, threads;
};
NormShape norm_shape(long long chunks) {
  for (int lanes = 8; lanes <= 64; lanes *= 2)
    if (chunks <= lanes) return {lanes, 1, kThreads};
  if (chunks <= 128) return {64, 2, kThreads};
  if (chunks <= 256) return {256, 1, 256};
  if (chunks <= 512) return {256, 2, 256};
  if (chunks <= 1024) return {1024, 1, 1024};
  if (chunks <= 2048) return {1024, 2, 1024};
  return {0, 0, 1024};
}

long long chunk_count(int d, int dtype) {
  const int v = (int)(16 / sf_dtype_size(dtype));
  return ((long long)d + v - 1) / v;
}

// Most workgroups of a kernel: a CU with more of them in flight than it needs moves less (259200 x 256
// bf16, gradients of 1024, 768 and 512 workgroups 98, 93 and 102 us, add and norm 93, 93 and 109, of 2048
// 105; 40000 x 1024 bf16 gradients 72, 65 and 62); rows that share lines want one more a CU (110000 x 333
// fp32 124 and 139 us of 1024 and 768).
long long most_blocks(const NormShape &s, int d, int dtype) {
  if (s.threads == 1024) return 256;
  return d % (int)(16 / sf_dtype_size(dtype)) ? 1024 : 768;
}

// Workgroups of the backward pass.
int bwd_blocks(long long m, int d, int dtype) {
  const NormShape s = norm_shape(chunk_count(d, dtype));
  const int groups = s.lanes ? s.threads / s.lanes : 1;
  long long b = (m + groups - 1) / groups;
  const long long most = s.lanes ? most_blocks(s, d, dtype) : 512;
  if (s.lanes == 0) b = (m + 63) / 64;      // norm_cols_long_kernel: 64 rows or more each
  return (int)(b < 1 ? 1 : b > most ? most : b);
}

#define SF_NORM_SHAPES(GO)                                                             \
  do {                                                                                 \
    if (s.lanes == 8) { GO(8, 1, 256); }                                               \
    else if (s.lanes == 16) { GO(16, 1, 256); }                                        \
    else if (s.lanes == 32) { GO(32, 1, 256); }                                        \
    else if (s.lanes == 64 && s.nv == 1) { GO(64, 1, 256); }                           \
    else if (s.lanes == 64) { GO(64, 2, 256); }                                        \
    else if (s.lanes == 256 && s.nv == 1) { GO(256, 1, 256); }                         \
    else if (s.lanes == 256) { GO(256, 2, 256); }                                      \
    else if (s.nv == 1) { GO(1024, 1, 1024); }                                         \
    else { GO(1024, 2, 1024); }                                                        \
  } while (0)

template <typename T, typename P>
void launch_fwd(const NormArgs &a) {
  const NormShape s = norm_shape(((long long)a.d + SfChunk<T>::V - 1) / SfChunk<T>::V);
  if (s.lanes == 0) {
    const int grid = (int)(a.m < 1024 ? a.m : 1024);
    hipLaunchKernelGGL((norm_fwd_long_kernel<T, P>), dim3(grid), dim3(1024), 0, a.st, (const T *)a.x,
                       (const T *)a.res, a.w, a.b, (T *)a.y, (T *)a.sum, a.mean, a.rstd, a.m, a.d,
                       a.eps);
    return;
  }
  const int groups = s.threads / s.lanes;
  long long g = (a.m + groups - 1) / groups;
  const long long most = most_blocks(s, a.d, sizeof(T) == 4 ? SF_DTYPE_F32 : SF_DTYPE_F16);
  const int grid = (int)(g < most ? g : most);
  const int mode = a.d % SfChunk<T>::V ? SF_RAGGED : sf_streamed(a.m, (size_t)a.d * sizeof(T)) ? SF_STREAM : SF_WHOLE;
#define SF_GO1(L, N, TH, MODE)                                                                 \
  hipLaunchKernelGGL((norm_fwd_kernel<T, P, L, N, TH, MODE>), dim3(grid), dim3(TH), 0, a.st,     \
                     (const T *)a.x, (const T *)a.res, a.w, a.b, (T *)a.y, (T *)a.sum, a.mean, \
                     a.rstd, a.m, a.d, a.eps)
#define SF_GO(L, N, TH)                                   \
  if (mode == SF_RAGGED) SF_GO1(L, N, TH, SF_RAGGED);     \
  else if (mode == SF_WHOLE) SF_GO1(L, N, TH, SF_WHOLE);  \
  else SF_GO1(L, N, TH, SF_STREAM)
  SF_NORM_SHAPES(SF_GO);
#undef SF_GO
#undef SF_GO1
}

template <typename T, typename P>
void launch_bwd(const NormArgs &a) {
  const NormShape s = norm_shape(((long long)a.d + SfChunk<T>::V - 1) / SfChunk<T>::V);
  if (s.lanes == 0) {
    const int grid = (int)(a.m < 1024 ? a.m : 1024);
    hipLaunchKernelGGL((norm_bwd_long_kernel<T, P>), dim3(grid), dim3(1024), 0, a.st,
                       (const T *)a.dy, (const T *)a.x, a.mean, a.rstd, a.w, (const T *)a.sum,
                       (T *)a.y, a.m, a.d);
    if (a.part)
      hipLaunchKernelGGL((norm_cols_long_kernel<T>), dim3(sf_div_up(a.d, kThreads), a.blocks),
                         dim3(kThreads), 0, a.st, (const T *)a.dy, (const T *)a.x, a.mean, a.rstd,
                         a.part, a.m, a.d);
    return;
  }
  const int mode = a.d % SfChunk<T>::V ? SF_RAGGED : sf_streamed(a.m, (size_t)a.d * sizeof(T)) ? SF_STREAM : SF_WHOLE;
#define SF_GO1(L, N, TH, MODE)                                                                     \
  hipLaunchKernelGGL((norm_bwd_kernel<T, P, L, N, TH, MODE>), dim3(a.blocks), dim3(TH),              \
                     TH == L ? 0 : (size_t)TH * N * SfChunk<T>::V * sizeof(float), a.st,           \
                     (const T *)a.dy, (const T *)a.x, a.mean, a.rstd, a.w, (const T *)a.sum,       \
                     (T *)a.y, a.part, a.m, a.d)
#define SF_GO(L, N, TH)                                   \
  if (mode == SF_RAGGED) SF_GO1(L, N, TH, SF_RAGGED);     \
  else if (mode == SF_WHOLE) SF_GO1(L, N, TH, SF_WHOLE);  \
  else SF_GO1(L, N, TH, SF_STREAM)
  SF_NORM_SHAPES(SF_GO);
#undef SF_GO
#undef SF_GO1
}

template <typename T>
void launch(const NormArgs &a, bool params_f32, bool backward) {
  if (params_f32)
    backward ? launch_bwd<T, float>(a) : launch_fwd<T, float>(a);
  else
    backward ? launch_bwd<T, T>(a) : launch_fwd<T, T>(a);
}

void dispatch(const NormArgs &a, int dtype, bool params_f32, bool backward) {
  if (dtype == SF_DTYPE_F32) launch<float>(a, true, backward);
  else if (dtype == SF_DTYPE_F16) launch<_Float16>(a, params_f32, backward);
  else launch<__bf16>(a, params_f32, backward);
}

#define SF_NORM_CHECK_SIZES()                                                                 \
  SF_CHECK_ARG(m >= 0 && d >= 1 && d <= SF_LAYER_NORM_MOST_FEATURES,                          \
               "layer norm of %lld rows of %d elements", m, d);                               \
  SF_CHECK_ARG(dtype >= SF_DTYPE_F32 && dtype <= SF_DTYPE_BF16, "unknown dtype %d", dtype);   \
  SF_CHECK_ARG(param_dtype == dtype || param_dtype == SF_DTYPE_F32,                           \
               "parameters must have the rows' type or be fp32 (dtype %d)", param_dtype)

}  // namespace

extern "C" int sf_layer_norm(const void *x, const void *residual, const void *weight,
                             const void *bias, void *y, void *sum, float *mean, float *rstd,
                             long long m, int d, float eps, int dtype, int param_dtype,
                             void *stream) {
  SF_NORM_CHECK_SIZES();
  if (m == 0) return SF_OK;
  SF_CHECK_ARG(x && y, "NULL tensor pointer");
  const NormArgs a{nullptr, x, residual, weight, bias, y, sum, mean, rstd, nullptr, m, d, 0, eps,
                   (hipStream_t)stream};
  dispatch(a, dtype, param_dtype == SF_DTYPE_F32, false);
  SF_CHECK_LAUNCH();
  return SF_OK;
}

extern "C" size_t sf_layer_norm_backward_workspace(long long m, int d, int dtype) {
  if (m < 1 || d < 1 || dtype < SF_DTYPE_F32 || dtype > SF_DTYPE_BF16) return 0;
  return (size_t)bwd_blocks(m, d, dtype) * 2 * d * sizeof(float);
}

extern "C" int sf_layer_norm_backward(const void *dy, const void *x, const float *mean,
                                      const float *rstd, const void *weight, const void *dsum,
                                      void *dx, void *dw, void *db, long long m, int d, int dtype,
                                      int param_dtype, void *ws, size_t ws_bytes, void *stream) {
  SF_NORM_CHECK_SIZES();
  const hipStream_t st = (hipStream_t)stream;
  if (m == 0) {      // a sum over no rows
    const size_t words = (size_t)d * sf_dtype_size(param_dtype) / 2;
    for (void *p : {dw, db})
      if (p) {
        hipLaunchKernelGGL(sf_fill_u16_kernel, dim3(sf_grid((long long)words, 256)), dim3(256), 0, st,
                           (uint16_t *)p, words, (uint16_t)0);
        SF_CHECK_LAUNCH();
      }
    return SF_OK;
  }
  SF_CHECK_ARG(dy && x && mean && rstd && dx, "NULL tensor pointer");
  NormArgs a{dy, x, nullptr, weight, nullptr, dx, const_cast<void *>(dsum),
             const_cast<float *>(mean), const_cast<float *>(rstd), nullptr, m, d,
             bwd_blocks(m, d, dtype), 0.0f, st};
  const bool cols = dw || db;
  if (cols) {
    const size_t need = sf_layer_norm_backward_workspace(m, d, dtype);
    if (!ws || ws_bytes < need) {
      sf_set_error("sf_layer_norm_backward needs %zu bytes of workspace, got %zu", need, ws_bytes);
      return SF_ERR_WORKSPACE;
    }
    a.part = (float *)ws;
  }
  dispatch(a, dtype, param_dtype == SF_DTYPE_F32, true);
  SF_CHECK_LAUNCH();
  if (cols) {
    const dim3 grid(sf_div_up(2LL * d, 32));
    if (param_dtype == SF_DTYPE_F32)
      hipLaunchKernelGGL((norm_join_kernel<float>), grid, dim3(1024), 0, st, a.part, a.blocks, d,
                         (float *)dw, (float *)db);
    else if (param_dtype == SF_DTYPE_F16)
      hipLaunchKernelGGL((norm_join_kernel<_Float16>), grid, dim3(1024), 0, st, a.part, a.blocks, d,
                         (_Float16 *)dw, (_Float16 *)db);
    else
      hipLaunchKernelGGL((norm_join_kernel<__bf16>), grid, dim3(1024), 0, st, a.part, a.blocks, d,
                         (__bf16 *)dw, (__bf16 *)db);
    SF_CHECK_LAUNCH();
  }
  return SF_OK;
}
