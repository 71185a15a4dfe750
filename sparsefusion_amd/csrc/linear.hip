// Linear layer y = act(x w^T + b) + r and its gradients: argument checks, the choice of tile and
// splits, and the pass over the output gradient.  The products are gemm_tile.h.
//
//   dz = dy act'(z);  dx = dz w;  dw = dz^T x;  db = sum_rows dz       (dr = dy)
#include "gemm_tile.h"

namespace {

struct Plan {
  int tile, splits;
  long long k_split;
};

// Tile and splits of a np x nq product over nk: the cheapest of the three tiles, each with the splits
// of a long contraction that would fill the chip, by a model of the busiest CU.
Plan make_plan(long long np, long long nq, long long nk, int dtype) {
  const long long bk = 128 / (long long)sf_dtype_size(dtype);
  const long long steps = (nk + bk - 1) / bk;
  Plan best{128, 1, steps * bk};
  if (np < 1 || nq < 1 || nk < 1) return best;      // no product
  double least = 1e30;
  for (int tile : {256, 128, 64}) {
    const long long t = ((np + tile - 1) / tile) * ((nq + tile - 1) / tile);
    for (int full = 0; full < 2; ++full) {
      const int slots = 256 * (tile == 256 ? 1 : tile == 128 ? 2 : 3);
      long long s = full ? slots / t : 1;
      if (s > steps / 4) s = steps / 4;
      if (s < 1 || (full && s == 1)) continue;
      const long long per = (steps + s - 1) / s;
      s = (steps + per - 1) / per;
      const double n = (double)((t * s + 255) / 256);
      double c = dtype == SF_DTYPE_F32
                     ? n * (tile == 256 ? 8 + 7.9 * per : tile == 128 ? 2 + 2.05 * per : 0.7 + 0.55 * per)
                     : n * (tile == 256 ? 8 + 1.5 * per : tile == 128 ? 2 + 0.48 * per : 0.8 + 0.21 * per);
      if (s > 1) c += 3 + 8e-6 * (double)(np * nq * s) / 4.5;
      if (c < least) least = c, best = Plan{tile, (int)s, per * bk};
    }
  }
  return best;
}

size_t partial_bytes(const Plan &pl, long long np, long long nq) {
  return pl.splits > 1 ? (size_t)pl.splits * np * nq * sizeof(float) : 0;
}
size_t align16(size_t v) { return (v + 255) & ~(size_t)255; }

// Whole aligned chunks along the contiguous axis: the operand can go straight to LDS.  A tile's rows
// also have to stay in reach of a 31-bit offset.
bool direct(const void *p, long long ld, long long extent, int dtype) {
  const long long s = (long long)sf_dtype_size(dtype), v = 16 / s;
  return (uintptr_t)p % 16 == 0 && ld % v == 0 && extent % v == 0 && ld * s * 256 < 0x7FFFFFFFLL;
}

int product(SfGemmArgs &a, int layout, int dtype, const Plan &pl, hipStream_t st) {
  a.splits = pl.splits;
  a.k_split = pl.k_split;
  if (a.nk == 0) {      // nothing to sum: the epilogue alone
    a.splits = 0;
    if (dtype == SF_DTYPE_F32) sf_gemm_join<float>(a, st);
    else if (dtype == SF_DTYPE_F16) sf_gemm_join<_Float16>(a, st);
    else sf_gemm_join<__bf16>(a, st);
    SF_CHECK_LAUNCH();
    return SF_OK;
  }
  const bool dma = direct(a.p, a.ldp, layout == 2 ? a.np : a.nk, dtype) &&
                   direct(a.q, a.ldq, layout == 0 ? a.nk : a.nq, dtype);
  const int tile = !dma && pl.tile > 128 ? 128 : pl.tile;      // no 256 tile through registers
  const long long tp = (a.np + tile - 1) / tile, tq = (a.nq + tile - 1) / tile;
  SF_CHECK_ARG(tp * tq * pl.splits < SF_INT_MAX, "linear: %lld x %lld outputs are too many for one launch",
               a.np, a.nq);
  a.tiles_p = (int)tp;
  a.tiles_q = (int)tq;
  int rc;
  if (dtype == SF_DTYPE_F32) rc = sf_gemm_f32(a, layout, tile, dma, st);
  else if (dtype == SF_DTYPE_F16) rc = sf_gemm_f16(a, layout, tile, dma, st);
  else rc = sf_gemm_bf16(a, layout, tile, dma, st);
  if (rc) return rc;
  SF_CHECK_LAUNCH();
  return SF_OK;
}

// ---- dz and the bias gradient -------------------------------------------------------------------
// A workgroup owns 32 chunks of columns and a run of rows, 8 row lanes deep; dz goes out as it is
// computed, the column sums stay in registers, join through LDS and leave as part[run][n].  The sums
// are of the fp32 products, not of the rounded dz.
template <typename T>
__global__ void __launch_bounds__(256)
dz_kernel(const T *__restrict__ dy, const T *__restrict__ pre, int act, T *__restrict__ dz,
          float *__restrict__ part, long long m, long long n, long long run) {
  constexpr int V = 16 / sizeof(T);
  __shared__ float red[8][32 * V + 4];
  const int cl = threadIdx.x & 31, rl = threadIdx.x >> 5;
  const long long col = ((long long)blockIdx.x * 32 + cl) * V;
  const long long r0 = blockIdx.y * run, r1 = r0 + run < m ? r0 + run : m;
  float sum[V];
#pragma unroll
  for (int j = 0; j < V; ++j) sum[j] = 0.0f;
  if (col < n)
    for (long long r = r0 + rl; r < r1; r += 8) {
      float g[V], z[V];
      sf_load_chunk<T>(dy + r * n, col, n, g);
      if (act != SF_ACT_NONE) {
        sf_load_chunk<T>(pre + r * n, col, n, z);
#pragma unroll
        for (int j = 0; j < V; ++j) g[j] *= sf_act_slope<T>(z[j], act);
        if (dz) sf_store_chunk<T>(dz + r * n, col, n, g);
      }
#pragma unroll
      for (int j = 0; j < V; ++j) sum[j] += g[j];
    }
  if (!part) return;
#pragma unroll
  for (int j = 0; j < V; ++j) red[rl][cl * V + j] = sum[j];
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * V; i += 256) {
    const long long c = (long long)blockIdx.x * 32 * V + i;
    if (c >= n) break;
    float t = 0.0f;
#pragma unroll
    for (int k = 0; k < 8; ++k) t += red[k][i];
    part[(long long)blockIdx.y * n + c] = t;
  }
}

template <typename T>
__global__ void __launch_bounds__(1024)
db_join_kernel(const float *__restrict__ part, int runs, long long n, T *__restrict__ db) {
  __shared__ float red[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const long long i = (long long)blockIdx.x * 32 + tx;
  float t = 0.0f;
  if (i < n) {
#pragma unroll 8
    for (int b = ty; b < runs; b += 32) t += part[b * n + i];
  }
  red[ty][tx] = t;
  __syncthreads();
  if (ty == 0 && i < n) {
    float a = 0.0f;
#pragma unroll
    for (int k = 0; k < 32; ++k) a += red[k][tx];
    db[i] = (T)a;
  }
}

// Runs of rows of dz_kernel: about 2048 workgroups in all, at least 32 rows each.
int dz_runs(long long m, long long n, int dtype) {
  const long long v = 16 / (long long)sf_dtype_size(dtype);
  const long long strips = (n + 32 * v - 1) / (32 * v);
  long long runs = (2048 + strips - 1) / strips;
  if (runs > (m + 31) / 32) runs = (m + 31) / 32;
  return (int)(runs < 1 ? 1 : runs);
}

template <typename T>
int run_dz(const void *dy, const void *pre, int act, void *dz, float *part, void *db, long long m,
           long long n, int dtype, hipStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const int want = dz_runs(m, n, dtype);
  const long long run = (m + want - 1) / want;
  const int runs = (int)((m + run - 1) / run);
  const dim3 grid((unsigned)((n + 32 * V - 1) / (32 * V)), runs);
  hipLaunchKernelGGL((dz_kernel<T>), grid, dim3(256), 0, st, (const T *)dy, (const T *)pre, act,
                     (T *)dz, db ? part : nullptr, m, n, run);
  SF_CHECK_LAUNCH();
  if (db) {
    hipLaunchKernelGGL((db_join_kernel<T>), dim3(sf_div_up(n, 32)), dim3(1024), 0, st, part, runs, n,
                       (T *)db);
    SF_CHECK_LAUNCH();
  }
  return SF_OK;
}

int zero_out(void *p, long long elements, int dtype, hipStream_t st) {
  const size_t words = (size_t)elements * sf_dtype_size(dtype) / 2;
  if (!p || !words) return SF_OK;
  hipLaunchKernelGGL(sf_fill_u16_kernel, dim3(sf_grid((long long)words, 256)), dim3(256), 0, st,
                     (uint16_t *)p, words, (uint16_t)0);
  SF_CHECK_LAUNCH();
  return SF_OK;
}

// Where the pieces of the backward pass's workspace start.
struct BackwardPlan {
  Plan dx, dw;
  size_t dz, part, split, bytes;
};
BackwardPlan backward_plan(long long m, long long k, long long n, int dtype, int act) {
  BackwardPlan b;
  b.dx = make_plan(m, k, n, dtype);
  b.dw = make_plan(n, k, m, dtype);
  b.dz = 0;
  b.part = act == SF_ACT_NONE ? 0 : align16((size_t)m * n * sf_dtype_size(dtype));
  b.split = b.part + align16((size_t)dz_runs(m, n, dtype) * n * sizeof(float));
  const size_t s1 = partial_bytes(b.dx, m, k), s2 = partial_bytes(b.dw, n, k);
  b.bytes = b.split + (s1 > s2 ? s1 : s2);      // the two products run one after the other
  return b;
}

bool good_sizes(long long m, long long k, long long n, int dtype) {
  return m >= 0 && k >= 0 && n >= 0 && dtype >= SF_DTYPE_F32 && dtype <= SF_DTYPE_BF16 &&
         m < (1LL << 40) && k <= SF_LINEAR_MOST_FEATURES && n <= SF_LINEAR_MOST_FEATURES;
}

#define SF_LINEAR_CHECK()                                                                          \
  SF_CHECK_ARG(good_sizes(m, k, n, dtype), "linear: bad sizes %lld x %lld x %lld or dtype %d", m, \
               k, n, dtype);                                                                       \
  SF_CHECK_ARG(act >= SF_ACT_NONE && act <= SF_ACT_GELU, "linear: unknown activation %d", act);    \
  SF_CHECK_ARG(ldx >= k, "linear: rows of %lld elements are %lld apart", k, ldx)

}  // namespace

extern "C" size_t sf_linear_workspace(long long m, long long k, long long n, int dtype) {
  if (!good_sizes(m, k, n, dtype) || !m || !n) return 0;
  return partial_bytes(make_plan(m, n, k, dtype), m, n);
}

extern "C" int sf_linear(const void *x, long long ldx, const void *weight, const void *bias,
                         const void *residual, void *y, void *pre, long long m, long long k,
                         long long n, int dtype, int act, void *ws, size_t ws_bytes, void *stream) {
  SF_LINEAR_CHECK();
  if (m == 0 || n == 0) return SF_OK;
  SF_CHECK_ARG(y && ((x && weight) || k == 0), "NULL tensor pointer");
  const Plan pl = make_plan(m, n, k, dtype);
  const size_t need = partial_bytes(pl, m, n);
  if (need && (!ws || ws_bytes < need)) {
    sf_set_error("sf_linear needs %zu bytes of workspace, got %zu", need, ws_bytes);
    return SF_ERR_WORKSPACE;
  }
  SfGemmArgs a{};
  a.p = x, a.q = weight, a.ldp = ldx, a.ldq = k;
  a.np = m, a.nq = n, a.nk = k;
  a.bias = bias, a.residual = residual, a.out = y, a.pre = pre;
  a.partial = (float *)ws;
  a.act = act;
  return product(a, 0, dtype, pl, (hipStream_t)stream);
}

extern "C" size_t sf_linear_backward_workspace(long long m, long long k, long long n, int dtype,
                                               int act) {
  if (!good_sizes(m, k, n, dtype) || !m || !n) return 0;
  return backward_plan(m, k, n, dtype, act).bytes;
}

extern "C" int sf_linear_backward(const void *dy, const void *x, long long ldx, const void *weight,
                                  const void *pre, void *dx, void *dw, void *db, long long m,
                                  long long k, long long n, int dtype, int act, void *ws,
                                  size_t ws_bytes, void *stream) {
  SF_LINEAR_CHECK();
  const hipStream_t st = (hipStream_t)stream;
  int rc;
  if (m == 0 || n == 0) {      // sums over nothing
    if ((rc = zero_out(dx, m * k, dtype, st)) || (rc = zero_out(dw, n * k, dtype, st))) return rc;
    return zero_out(db, n, dtype, st);
  }
  SF_CHECK_ARG(dy && (pre || act == SF_ACT_NONE) && (weight || !dx || !k) && (x || !dw || !k),
               "NULL tensor pointer");
  const BackwardPlan b = backward_plan(m, k, n, dtype, act);
  if (b.bytes && (!ws || ws_bytes < b.bytes)) {
    sf_set_error("sf_linear_backward needs %zu bytes of workspace, got %zu", b.bytes, ws_bytes);
    return SF_ERR_WORKSPACE;
  }
  unsigned char *base = (unsigned char *)ws;
  const void *dz = dy;
  const bool products = (dx || dw) && k > 0;
  if (db || (act != SF_ACT_NONE && products)) {
    void *out = act != SF_ACT_NONE && products ? base + b.dz : nullptr;
    float *part = (float *)(base + b.part);
    if (dtype == SF_DTYPE_F32) rc = run_dz<float>(dy, pre, act, out, part, db, m, n, dtype, st);
    else if (dtype == SF_DTYPE_F16) rc = run_dz<_Float16>(dy, pre, act, out, part, db, m, n, dtype, st);
    else rc = run_dz<__bf16>(dy, pre, act, out, part, db, m, n, dtype, st);
    if (rc) return rc;
    if (out) dz = out;
  }
  if (k == 0) return SF_OK;
  if (dx) {
    SfGemmArgs a{};
    a.p = dz, a.q = weight, a.ldp = n, a.ldq = k;
    a.np = m, a.nq = k, a.nk = n;
    a.out = dx;
    a.partial = (float *)(base + b.split);
    if ((rc = product(a, 1, dtype, b.dx, st))) return rc;
  }
  if (dw) {
    SfGemmArgs a{};
    a.p = dz, a.q = x, a.ldp = n, a.ldq = ldx;
    a.np = n, a.nq = k, a.nk = m;
    a.out = dw;
    a.partial = (float *)(base + b.split);
    if ((rc = product(a, 2, dtype, b.dw, st))) return rc;
  }
  return SF_OK;
}
