// Linear layer y = act(x w^T + b) + r and its gradients: argument checks, the choice of tile and
// splits, and the pass over the output gradient.  The products are gemm_tile.h.
//
//   dz = dy act'(z);  dx = dz w;  dw = dz^T x;  db = sum_rows dz       (dr = dy)
#include "gemm_tile.h"

namespace {

struct Plan {
  int tile, splits;
  long long k_split;
  double cost;
};

// Time (us, without the launch) of t workgroups of a tile's kernel, each `per` steps of 128 bytes of k,
// on the busiest CU; fitted to timings of each tile at 41 sizes from 64 x 64 x 64 to 8192^3, where the tile of
// least cost comes within 10 % (or half a us) of the fastest, but for two sizes of 64 and 128 columns (13 %):
// profiles/token_ops_tile_costs.csv.  Two 16-bit 128 x 128 tiles share a
// CU and take 1.3 times as long as one alone; a 256 x 256 tile reads its residual with nothing under it.
double tile_cost(int tile, long long t, long long per, int dtype, bool residual) {
  const double n = (double)((t + 255) / 256), k = (double)per;
  if (dtype == SF_DTYPE_F32)
    return tile == 256   ? n * ((residual ? 34 : 8) + 7.5 * k)
           : tile == 128 ? n * (2 + 2.05 * k)
           : tile == 64  ? n * (0.7 + (n < 2 ? 0.7 : 0.57) * k)
                         : n * (0.3 + 0.24 * k);
  return tile == 256   ? residual ? n * (11 + 1.75 * k) : n * (8 + 1.65 * k)
         : tile == 128 ? ((double)(t / 512) + (t % 512 == 0 ? 0 : t % 512 > 256 ? 1 : 0.75)) * (4 + k)
         : tile == 64  ? n * (0.8 + 0.3 * k)
                       : n * (0.3 + 0.165 * k);
}

// 32 x 32 tiles only as long as all of them are resident, two to a CU: a workgroup there walks one tile,
// and its start and first loads show in every further round (100000 x 64 -> 32 bf16: 22.6 us, with
// 64 x 64 tiles 11.4; 5000 x 256 -> 64 fp32, 314 tiles: 7.6 and 8.9).
constexpr long long kMostSmallTiles = 512;

// Tile and splits of a np x nq product over nk: the cheapest of the four tiles, each whole or with the
// contraction cut into as many parts as fill the chip.
Plan make_plan(long long np, long long nq, long long nk, int dtype, bool residual, bool tail) {
  const long long bk = 128 / (long long)sf_dtype_size(dtype);
  const long long steps = (nk + bk - 1) / bk;
  Plan best{128, 1, steps * bk, 1e30};
  if (np < 1 || nq < 1 || nk < 1) return best;      // no product
  for (int tile : {256, 128, 64, 32}) {
    if (tile == 256 && tail) continue;      // has no registers left to clear what is behind cut rows
    const long long t = ((np + tile - 1) / tile) * ((nq + tile - 1) / tile);
    for (int full = 0; full < 2; ++full) {
      const int slots = 256 * (tile == 256 ? 1 : tile == 64 ? 3 : 2);
      long long s = 1;
      if (full) {
        s = slots / t < steps / 4 ? slots / t : steps / 4;
        if (s < 2) continue;
      }
      const long long per = (steps + s - 1) / s;
      s = (steps + per - 1) / per;
      if (tile == 32 && t * s > kMostSmallTiles) continue;
      double c = tile_cost(tile, t * s, per, dtype, residual && s == 1);
      if (s > 1) c += 4.5 + 8e-6 * (double)(np * nq * s) / 4.5;      // the parts' round trip and a launch
      if (c < best.cost) best = Plan{tile, (int)s, per * bk, c};
    }
  }
  return best;
}

size_t partial_bytes(const Plan &pl, long long np, long long nq) {
  return pl.splits > 1 ? (size_t)pl.splits * np * nq * sizeof(float) : 0;
}
size_t align256(size_t v) { return (v + 255) & ~(size_t)255; }

// ---- operands of odd shapes -----------------------------------------------------------------------
// The tiles load chunks from any multiple of 4 bytes.  An operand whose rows start elsewhere (an odd number
// of 16-bit elements) is copied first, rows padded with zeros to whole chunks.  (Loading them through
// registers was built and timed: 3001 x 451 -> 333 fp16 13.4 us, 32401 x 255 -> 1023 bf16 87 us, both bound
// by the waits for loads that cannot run ahead.)
bool direct(const void *p, long long ld, int dtype) {
  return (uintptr_t)p % 4 == 0 && ld * (long long)sf_dtype_size(dtype) % 4 == 0 &&
         ld <= 2 * SF_LINEAR_MOST_FEATURES;
}
long long padded(long long cols, int dtype) {
  const long long v = 16 / (long long)sf_dtype_size(dtype);
  return (cols + v - 1) / v * v;
}
size_t padded_bytes(long long rows, long long cols, int dtype) {
  return align256((size_t)rows * padded(cols, dtype) * sf_dtype_size(dtype));
}

struct Repack {
  const void *src;
  void *dst;
  long long ld, rows, cols;
};

template <typename T>
__global__ void __launch_bounds__(256) repack_kernel(Repack x, Repack y) {
  constexpr int V = 16 / sizeof(T);
  const long long cx = (x.cols + V - 1) / V, cy = (y.cols + V - 1) / V;
  const long long nx = x.rows * cx, n = nx + y.rows * cy;
  for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const Repack &r = i < nx ? x : y;
    const long long at = i < nx ? i : i - nx, cols = i < nx ? cx : cy, row = at / cols, c = at - row * cols;
    const T *src = static_cast<const T *>(r.src) + row * r.ld;
    sf_u32x4 v;
    if (c * V + V <= r.cols) {
      v = *reinterpret_cast<const sf_u32x4_any *>(src + c * V);
    } else {
      typename SfMfma<T>::frag e;
#pragma unroll
      for (int j = 0; j < V; ++j) e[j] = c * V + j < r.cols ? src[c * V + j] : (T)0.0f;
      v = __builtin_bit_cast(sf_u32x4, e);
    }
    static_cast<sf_u32x4 *>(r.dst)[at] = v;
  }
}

// Copies x and y (src NULL: not that one) into their padded form.
int repack(const Repack &x, const Repack &y, int dtype, hipStream_t st) {
  const long long chunks = (x.src ? x.rows * padded(x.cols, dtype) : 0) +
                           (y.src ? y.rows * padded(y.cols, dtype) : 0);
  if (!chunks) return SF_OK;
  Repack a = x, b = y;
  if (!a.src) a.rows = a.cols = 0;
  if (!b.src) b.rows = b.cols = 0;
  const dim3 grid(sf_grid(chunks / 4, 256));
  if (dtype == SF_DTYPE_F32) hipLaunchKernelGGL((repack_kernel<float>), grid, dim3(256), 0, st, a, b);
  else if (dtype == SF_DTYPE_F16) hipLaunchKernelGGL((repack_kernel<_Float16>), grid, dim3(256), 0, st, a, b);
  else hipLaunchKernelGGL((repack_kernel<__bf16>), grid, dim3(256), 0, st, a, b);
  SF_CHECK_LAUNCH();
  return SF_OK;
}

int launch(const SfGemmArgs &a, int layout, int dtype, int tile, hipStream_t st) {
  const int rc = dtype == SF_DTYPE_F32   ? sf_gemm_f32(a, layout, tile, st)
                 : dtype == SF_DTYPE_F16 ? sf_gemm_f16(a, layout, tile, st)
                                         : sf_gemm_bf16(a, layout, tile, st);
  if (rc) return rc;
  SF_CHECK_LAUNCH();
  return SF_OK;
}

// The plan into the arguments; false if it has too many tiles.
bool prepare(SfGemmArgs &a, const Plan &pl) {
  const long long tp = (a.np + pl.tile - 1) / pl.tile, tq = (a.nq + pl.tile - 1) / pl.tile;
  a.tiles_p = (int)tp, a.tiles_q = (int)tq;
  a.splits = pl.splits;
  a.k_split = pl.k_split;
  return tp * tq * pl.splits < SF_INT_MAX;
}

int product(SfGemmArgs &a, int layout, int dtype, const Plan &pl, hipStream_t st) {
  if (a.nk == 0) {      // nothing to sum: the epilogue alone
    a.splits = 0;
    if (dtype == SF_DTYPE_F32) sf_gemm_join<float>(a, st);
    else if (dtype == SF_DTYPE_F16) sf_gemm_join<_Float16>(a, st);
    else sf_gemm_join<__bf16>(a, st);
    SF_CHECK_LAUNCH();
    return SF_OK;
  }
  SF_CHECK_ARG(prepare(a, pl), "linear: %lld x %lld outputs are too many for one launch", a.np, a.nq);
  return launch(a, layout, dtype, pl.tile, st);
}

// ---- dz and the bias gradient -------------------------------------------------------------------
// A workgroup owns CL chunks of columns (32, fewer for narrow layers) and a run of rows, 256 / CL at a
// time; dz goes out as it is computed, the column sums stay in registers, join through LDS and leave as
// part[run][n].  The sums are of the fp32 products, not of the rounded dz.  Bound by memory:
// 32400 x 2048 bf16 with GELU 75 us, 398 MB at 5.3 TB/s (four rows in flight instead of two 73, ragged and
// fp32 rows slower; converting where they are loaded, one at a time, 87).
template <typename T, int CL, int MODE>
__global__ void __launch_bounds__(256)
dz_kernel(const T *__restrict__ dy, const T *__restrict__ pre, int act, T *__restrict__ dz, long long ldz,
          float *__restrict__ part, long long m, long long n, long long run) {
  constexpr int V = 16 / sizeof(T), DEEP = 2, RL = 256 / CL;
  __shared__ float red[RL][CL * V + 4];
  const int cl = threadIdx.x % CL, rl = threadIdx.x / CL;
  const long long col = ((long long)blockIdx.x * CL + cl) * V;
  const long long r0 = blockIdx.y * run, r1 = r0 + run < m ? r0 + run : m;
  float sum[V];
#pragma unroll
  for (int j = 0; j < V; ++j) sum[j] = 0.0f;
  if (col < n)
    for (long long r = r0 + rl; r < r1; r += RL * DEEP) {
      // DEEP rows' loads in flight; rows past the run are read again and count for nothing
      typename SfChunk<T>::type gr[DEEP], zr[DEEP];
#pragma unroll
      for (int i = 0; i < DEEP; ++i) {
        const long long row = r + RL * i < r1 ? r + RL * i : r;
        gr[i] = sf_load_raw<T, MODE>(dy + row * n, (int)col, (int)n);
        if (act != SF_ACT_NONE) zr[i] = sf_load_raw<T, MODE>(pre + row * n, (int)col, (int)n);
      }
#pragma unroll
      for (int i = 0; i < DEEP; ++i) {
        if (r + RL * i >= r1) break;
        float g[V];
#pragma unroll
        for (int j = 0; j < V; ++j) g[j] = (float)gr[i][j];
        if (act != SF_ACT_NONE) {
#pragma unroll
          for (int j = 0; j < V; ++j) g[j] = sf_act_gradient<T>(g[j], (float)zr[i][j], act);
        }
        // rows of dz are whole chunks; behind the n-th column dy and pre were read as zeros, and a
        // ReLU's or GELU's gradient of zero is zero
        if (dz) sf_store_chunk<T>(dz + (r + RL * i) * ldz, col, ldz, g);
#pragma unroll
        for (int j = 0; j < V; ++j) sum[j] += g[j];
      }
    }
  if (!part) return;
#pragma unroll
  for (int j = 0; j < V; ++j) red[rl][cl * V + j] = sum[j];
  __syncthreads();
  for (int i = threadIdx.x; i < CL * V; i += 256) {
    const long long c = (long long)blockIdx.x * CL * V + i;
    if (c >= n) break;
    float t = 0.0f;
#pragma unroll
    for (int k = 0; k < RL; ++k) t += red[k][i];
    part[(long long)blockIdx.y * n + c] = t;
  }
}

template <typename T, int TY>
__global__ void __launch_bounds__(32 * TY) db_join_kernel(SfColumnSums c) {
  __shared__ float red[TY * 33];
  sf_join_columns<T, TY>(c, blockIdx.x, red);
}

// Chunks of columns to a workgroup of dz_kernel, and its runs of rows: about 2048 workgroups in all, at
// least four turns of rows each.  (259200 x 64 bf16: 19 us with 8 chunks, 66 with 32.)
int dz_chunks(long long n, int dtype) {
  const long long v = 16 / (long long)sf_dtype_size(dtype), chunks = (n + v - 1) / v;
  return chunks <= 8 ? 8 : chunks <= 16 ? 16 : 32;
}
int dz_runs(long long m, long long n, int dtype) {
  const long long v = 16 / (long long)sf_dtype_size(dtype), cl = dz_chunks(n, dtype);
  const long long strips = (n + cl * v - 1) / (cl * v), least = 4 * 256 / cl;
  long long runs = (2048 + strips - 1) / strips;
  if (runs > (m + least - 1) / least) runs = (m + least - 1) / least;
  return (int)(runs < 1 ? 1 : runs);
}

// dz (or NULL) and the partial sums for db (or NULL).
template <typename T>
void run_dz(const void *dy, const void *pre, int act, void *dz, SfColumnSums &db, float *part, long long m,
            long long n, int dtype, hipStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const int want = dz_runs(m, n, dtype), cl = dz_chunks(n, dtype);
  const long long run = (m + want - 1) / want;
  db.part = part, db.n = n, db.runs = (int)((m + run - 1) / run);
  const dim3 grid((unsigned)((n + cl * V - 1) / (cl * V)), db.runs);
  // dz itself is read again at once
  const int mode = n % V ? SF_RAGGED : sf_streamed(m, (size_t)n * sizeof(T)) ? SF_STREAM : SF_WHOLE;
  auto pick = [&](auto ragged, auto whole, auto stream) {
    return mode == SF_RAGGED ? ragged : mode == SF_WHOLE ? whole : stream;
  };
  auto kern = cl == 8    ? pick(dz_kernel<T, 8, SF_RAGGED>, dz_kernel<T, 8, SF_WHOLE>, dz_kernel<T, 8, SF_STREAM>)
              : cl == 16 ? pick(dz_kernel<T, 16, SF_RAGGED>, dz_kernel<T, 16, SF_WHOLE>, dz_kernel<T, 16, SF_STREAM>)
                         : pick(dz_kernel<T, 32, SF_RAGGED>, dz_kernel<T, 32, SF_WHOLE>, dz_kernel<T, 32, SF_STREAM>);
  hipLaunchKernelGGL(kern, grid, dim3(256), 0, st, (const T *)dy, (const T *)pre, act, (T *)dz,
                     padded(n, dtype), db.out ? part : nullptr, m, n, run);
}
// The sum that the products' launch would have made (`pair`: in the same order), or a deeper one.
template <typename T>
void join_db(const SfColumnSums &db, bool pair, hipStream_t st) {
  const dim3 grid(sf_div_up(db.n, 32));
  if (pair) hipLaunchKernelGGL((db_join_kernel<T, 8>), grid, dim3(256), 0, st, db);
  else hipLaunchKernelGGL((db_join_kernel<T, 32>), grid, dim3(1024), 0, st, db);
}

int zero_out(void *p, long long elements, int dtype, hipStream_t st) {
  const size_t words = (size_t)elements * sf_dtype_size(dtype) / 2;
  if (!p || !words) return SF_OK;
  hipLaunchKernelGGL(sf_fill_u16_kernel, dim3(sf_grid((long long)words, 256)), dim3(256), 0, st,
                     (uint16_t *)p, words, (uint16_t)0);
  SF_CHECK_LAUNCH();
  return SF_OK;
}

// Where the pieces of the backward pass's workspace start, and what is copied first.
struct BackwardPlan {
  Plan dx, dw;
  bool tiny;      // everything in one launch and without workspace
  bool pair;      // both products in one launch
  bool write_dz, pack_x, pack_w, tail;
  size_t dz, x, w, part, split, bytes;
};
BackwardPlan backward_plan(const void *dy, const void *x, long long ldx, const void *w, long long m,
                           long long k, long long n, int dtype, int act) {
  BackwardPlan b;
  b.write_dz = act != SF_ACT_NONE || !direct(dy, n, dtype);
  b.tail = n * (long long)sf_dtype_size(dtype) % 16 != 0 && !b.write_dz;      // a written dz has zeros there
  b.dx = make_plan(m, k, n, dtype, false, b.tail);
  b.dw = make_plan(n, k, m, dtype, false, false);
  auto small = [&](long long np, long long nq, long long nk) {
    const long long bk = 128 / (long long)sf_dtype_size(dtype), steps = (nk + bk - 1) / bk;
    const long long t = ((np + 31) / 32) * ((nq + 31) / 32);
    // workgroups that are not resident from the start cost theirs
    return Plan{32, 1, steps * bk, tile_cost(32, t, steps, dtype, false) + (t > kMostSmallTiles ? t / 512.0 : 0)};
  };
  // Three ways, by cost (us, each launch 3): dz (and db's parts) by a pass of its own, then the two products
  // in one launch each; or both in one launch of 32 x 32 tiles, the one in the other's idle CUs; or these
  // tiles alone, making dz as they read dy.  That is work for each tile again (us a step below), worth it
  // while the steps are few: 400 x 256 -> 128 fp32 ReLU 8.4 us (pass and pair 10.2), bf16 GELU 7.6 (10.1),
  // 200 x 512 -> 512 bf16 ReLU 7.3 (10.0), but 1000 x 256 -> 256 bf16 GELU 13.2 (12.4), 1500 x 128 -> 128 fp32 GELU
  // 28 (18.5).  In between ReLU and no activation take the pass too early, a full chip's steps being charged as
  // much as a lone workgroup's: 500 x 512 -> 512 bf16 ReLU 11.4, and 7.8 in tiles.  With one
  // of the gradients asked for the tiles stay the same, so that its values do.
  const Plan x32 = small(m, k, n), w32 = small(n, k, m);
  const bool copy = !direct(x, ldx, dtype) || !direct(w, k, dtype), all = !copy && direct(dy, n, dtype);
  const double pass = (act == SF_ACT_NONE ? 5 : 6.5) + (copy ? 4 : 0);
  const double two = pass + 9 + b.dx.cost + b.dw.cost, pair = pass + 0.8 * (x32.cost + w32.cost);
  b.pair = k > 0 && m < (1 << 20) && x32.cost + w32.cost < b.dx.cost + b.dw.cost + 4;
  const long long bk = 128 / (long long)sf_dtype_size(dtype), tq = (k + 31) / 32;
  const double sx = (double)((n + bk - 1) / bk), sw = (double)((m + bk - 1) / bk);
  const double tx = (double)((m + 31) / 32 * tq), tw = (double)((n + 31) / 32 * tq);
  const double work = (tx * sx + tw * sw) / 256;
  const double longest = sx > sw ? sx : sw;
  const double step = dtype == SF_DTYPE_F32
                          ? !all ? 0.85 : act == SF_ACT_NONE ? 0.38 : act == SF_ACT_RELU ? 0.45 : 0.52
                          : !all ? 1.4 : act == SF_ACT_NONE ? 0.25 : act == SF_ACT_RELU ? 0.42 : 0.7;
  const double filled = step * work + (tx + tw > kMostSmallTiles ? (tx + tw - kMostSmallTiles) / 256 : 0);
  const double tiny = 3 + (filled > step * longest ? filled : step * longest);
  b.tiny = k > 0 && work < 1000 && longest < 1000 && tiny < (b.pair ? pair : two);
  if (b.tiny) {
    b.bytes = 0;
    return b;
  }
  if (b.pair) b.dx = x32, b.dw = w32;
  b.pack_x = !direct(x, ldx, dtype);
  b.pack_w = !direct(w, k, dtype);
  b.dz = 0;
  b.x = b.write_dz ? padded_bytes(m, n, dtype) : 0;
  b.w = b.x + (b.pack_x ? padded_bytes(m, k, dtype) : 0);
  b.part = b.w + (b.pack_w ? padded_bytes(n, k, dtype) : 0);
  b.split = b.part + align256((size_t)dz_runs(m, n, dtype) * n * sizeof(float));
  const size_t s1 = partial_bytes(b.dx, m, k), s2 = partial_bytes(b.dw, n, k);
  b.bytes = b.split + (s1 > s2 ? s1 : s2);      // the two products run one after the other
  return b;
}

// Whether up to 16 rows go without tiles, by the turns a wave takes at k (us each) and the weight's bytes.
// In us, without and with tiles: 1 x 1024 -> 4096 bf16 4.2 and 6.1, 4096 -> 4096 10.0 and 13.3; the turns
// of a long k for few columns are better spread over workgroups (fp32 4096 -> 64 14 and 6.3), and 16-bit
// rows that start anywhere take long turns (4095 -> 65 bf16 17 and 10, the copy included).
bool few_rows(long long m, long long k, long long n, int dtype, bool copy, double tiles) {
  const double bytes = (double)n * k * sf_dtype_size(dtype), memory = bytes / 4.9e6;
  const double turn = dtype == SF_DTYPE_F32 ? (m > 4 ? 1.8 : 1.4)
                      : copy                ? (m > 4 ? 6 : 3.6)
                                            : (m > 4 ? 1.7 : 1.1);
  const double turns = turn * (double)k * sf_dtype_size(dtype) / 2048;
  if (copy) tiles += 4 + 2 * memory;
  return 1.8 + (turns > memory ? turns : memory) < 2.7 + (tiles > memory ? tiles : memory);
}

// The same for the forward pass.
struct ForwardPlan {
  Plan y;
  bool few, pack_x, pack_w, tail;
  size_t x, w, bytes;
};
ForwardPlan forward_plan(const void *x, long long ldx, const void *w, long long m, long long k, long long n,
                         int dtype, bool residual) {
  ForwardPlan f;
  f.pack_x = !direct(x, ldx, dtype);
  f.pack_w = !direct(w, k, dtype);
  f.tail = k * (long long)sf_dtype_size(dtype) % 16 != 0 && !(f.pack_x && f.pack_w);
  f.y = make_plan(m, n, k, dtype, residual, f.tail);
  f.few = m <= 16 && few_rows(m, k, n, dtype, f.pack_x || f.pack_w, f.y.cost);
  if (f.few) f.y.splits = 1, f.pack_x = f.pack_w = false;
  f.x = align256(partial_bytes(f.y, m, n));
  f.w = f.x + (f.pack_x ? padded_bytes(m, k, dtype) : 0);
  f.bytes = f.w + (f.pack_w ? padded_bytes(n, k, dtype) : 0);
  return f;
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

#define SF_LINEAR_CHECK_WORKSPACE(name, need)                                                      \
  do {                                                                                             \
    if ((need) && (!ws || ws_bytes < (need))) {                                                    \
      sf_set_error("%s needs %zu bytes of workspace, got %zu", name, (size_t)(need), ws_bytes);    \
      return SF_ERR_WORKSPACE;                                                                     \
    }                                                                                              \
    SF_CHECK_ARG(!(need) || (uintptr_t)ws % 16 == 0, "%s: workspace is not 16-byte aligned", name); \
  } while (0)

extern "C" size_t sf_linear_workspace(const void *x, long long ldx, const void *weight, long long m,
                                      long long k, long long n, int dtype, int has_residual) {
  if (!good_sizes(m, k, n, dtype) || !m || !n || !k) return 0;
  return forward_plan(x, ldx, weight, m, k, n, dtype, has_residual != 0).bytes;
}

extern "C" int sf_linear(const void *x, long long ldx, const void *weight, const void *bias,
                         const void *residual, void *y, void *pre, long long m, long long k,
                         long long n, int dtype, int act, void *ws, size_t ws_bytes, void *stream) {
  SF_LINEAR_CHECK();
  if (m == 0 || n == 0) return SF_OK;
  SF_CHECK_ARG(y && ((x && weight) || k == 0), "NULL tensor pointer");
  const hipStream_t st = (hipStream_t)stream;
  SfGemmArgs a{};
  a.p = x, a.q = weight, a.ldp = ldx, a.ldq = k;
  a.np = m, a.nq = n, a.nk = k;
  a.bias = bias, a.residual = residual, a.out = y, a.pre = pre;
  a.act = act;
  if (k == 0) return product(a, 0, dtype, Plan{128, 1, 0, 0}, st);
  const ForwardPlan f = forward_plan(x, ldx, weight, m, k, n, dtype, residual != nullptr);
  if (f.few) return launch(a, 0, dtype, SF_FEW_ROWS, st);
  SF_LINEAR_CHECK_WORKSPACE("sf_linear", f.bytes);
  unsigned char *base = (unsigned char *)ws;
  a.partial = (float *)base;
  const Repack px{f.pack_x ? x : nullptr, base + f.x, ldx, m, k};
  const Repack pw{f.pack_w ? weight : nullptr, base + f.w, k, n, k};
  const int rc = repack(px, pw, dtype, st);
  if (rc) return rc;
  a.tail = f.tail;
  if (f.pack_x) a.p = px.dst, a.ldp = padded(k, dtype);
  if (f.pack_w) a.q = pw.dst, a.ldq = padded(k, dtype);
  return product(a, 0, dtype, f.y, st);
}

extern "C" size_t sf_linear_backward_workspace(const void *dy, const void *x, long long ldx,
                                               const void *weight, long long m, long long k,
                                               long long n, int dtype, int act) {
  if (!good_sizes(m, k, n, dtype) || !m || !n) return 0;
  return backward_plan(dy, x, ldx, weight, m, k, n, dtype, act).bytes;
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
  if (k == 0) dx = dw = nullptr;
  SF_CHECK_ARG(dy && (pre || act == SF_ACT_NONE) && (weight || !dx) && (x || !dw), "NULL tensor pointer");
  const BackwardPlan b = backward_plan(dy, x, ldx, weight, m, k, n, dtype, act);
  SF_LINEAR_CHECK_WORKSPACE("sf_linear_backward", b.bytes);
  if (b.tiny) {
    const SfGradients g{dy, pre, x, weight, dx, dw, db, ldx, m, k, n, act};
    const bool all = direct(dy, n, dtype) && direct(pre, n, dtype) && direct(x, ldx, dtype) &&
                     direct(weight, k, dtype);
    rc = dtype == SF_DTYPE_F32   ? sf_tiny_gradients_f32(g, all, st)
         : dtype == SF_DTYPE_F16 ? sf_tiny_gradients_f16(g, all, st)
                                 : sf_tiny_gradients_bf16(g, all, st);
    SF_CHECK_LAUNCH();
    return rc;
  }
  unsigned char *base = (unsigned char *)ws;
  const void *dz = dy;
  long long ldz = n;
  const bool write_dz = b.write_dz && (dx || dw);
  SfColumnSums sums{};
  sums.out = db;
  if (db || write_dz) {
    void *out = write_dz ? base + b.dz : nullptr;
    float *part = (float *)(base + b.part);
    if (dtype == SF_DTYPE_F32) run_dz<float>(dy, pre, act, out, sums, part, m, n, dtype, st);
    else if (dtype == SF_DTYPE_F16) run_dz<_Float16>(dy, pre, act, out, sums, part, m, n, dtype, st);
    else run_dz<__bf16>(dy, pre, act, out, sums, part, m, n, dtype, st);
    SF_CHECK_LAUNCH();
    if (out) dz = out, ldz = padded(n, dtype);
  }
  const Repack px{b.pack_x && dw ? x : nullptr, base + b.x, ldx, m, k};
  const Repack pw{b.pack_w && dx ? weight : nullptr, base + b.w, k, n, k};
  if ((rc = repack(px, pw, dtype, st))) return rc;
  SfGemmArgs gx{}, gw{};
  gx.p = dz, gx.q = pw.src ? pw.dst : weight, gx.ldp = ldz, gx.ldq = pw.src ? padded(k, dtype) : k;
  gx.np = m, gx.nq = k, gx.nk = n;
  gx.out = dx;
  gx.tail = b.tail;
  gw.p = dz, gw.q = px.src ? px.dst : x, gw.ldp = ldz, gw.ldq = px.src ? padded(k, dtype) : ldx;
  gw.np = n, gw.nq = k, gw.nk = m;
  gw.out = dw;
  gx.partial = gw.partial = (float *)(base + b.split);
  if (dx && dw && b.pair) {
    SF_CHECK_ARG(prepare(gx, b.dx) && prepare(gw, b.dw), "linear: %lld x %lld outputs are too many", m, k);
    rc = dtype == SF_DTYPE_F32   ? sf_gradients_f32(gx, gw, sums, st)
         : dtype == SF_DTYPE_F16 ? sf_gradients_f16(gx, gw, sums, st)
                                 : sf_gradients_bf16(gx, gw, sums, st);
    if (rc) return rc;
    SF_CHECK_LAUNCH();
    return SF_OK;
  }
  if (db) {
    if (dtype == SF_DTYPE_F32) join_db<float>(sums, b.pair, st);
    else if (dtype == SF_DTYPE_F16) join_db<_Float16>(sums, b.pair, st);
    else join_db<__bf16>(sums, b.pair, st);
    SF_CHECK_LAUNCH();
  }
  if (dx && (rc = product(gx, 1, dtype, b.dx, st))) return rc;
  if (dw && (rc = product(gw, 2, dtype, b.dw, st))) return rc;
  return SF_OK;
}
