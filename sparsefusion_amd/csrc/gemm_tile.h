// Matrix product of two row-major operands for the linear layer and its gradients (gfx950).
//
//   out[p][q] = sum_k P(p, k) Q(q, k)
//
// An operand is K-major (rows p, contiguous along k: activations and weights as the forward pass
// has them) or K-minor (rows k, contiguous along p: what a gradient contracts over).  All three
// pairings the linear layer needs run from the same tile, without transposed copies in memory:
//
//   forward  y  = x w^T     P = x  K-major   Q = w K-major
//   backward dx = dz w      P = dz K-major   Q = w K-minor
//   backward dw = dz^T x    P = dz K-minor   Q = x K-minor
//
// A workgroup owns a BP x BQ tile and walks k in steps of 128 bytes (64 16-bit or 32 fp32 elements).
// Both operands' tiles go to LDS in 16-byte chunks, straight from memory (buffer_load ... lds) when
// every chunk is aligned and whole, through registers otherwise; two buffers, the next step's loads
// in flight while this one multiplies.  v_mfma_f32_32x32x16 (32x32x2 for fp32) accumulates in fp32;
// Q is the instruction's first operand, so a lane ends up with four consecutive q of one row p.
// Rows and k outside the operands read as zeros (the buffer descriptor's range check), columns
// outside are never stored.
//
// Chunk swizzles (position = chunk ^ swz(row), applied to the source address because the LDS side
// of a direct load is linear): K-major, swz = (row ^ row >> 3) & 7 gives the 8 rows of a quarter-wave
// b128 read 8 different positions, and 16 rows 16 different 16-byte places of 256 bytes.  K-minor,
// 16-bit: ds_read_b64_tr_b16 hands a lane four k of its column; four rows of 64 bytes are spread over
// the 256 bytes of the banks.  K-minor, fp32: plain b32 reads, the lane halves (k and k + 4) 128
// bytes apart.
#pragma once
#include "token_common.h"

typedef short sf_s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned sf_u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned sf_u32x4_any __attribute__((ext_vector_type(4), aligned(2)));

__device__ __forceinline__ float sf_act(float z, int act) {
  if (act == SF_ACT_RELU) return z > 0.0f ? z : (z != z ? z : 0.0f);
  if (act == SF_ACT_GELU) return 0.5f * z * (1.0f + erff(z * 0.70710678118654752f));
  return z;
}
__device__ __forceinline__ float sf_act_slope(float z, int act) {
  if (act == SF_ACT_RELU) return z > 0.0f ? 1.0f : 0.0f;
  if (act == SF_ACT_GELU)
    return 0.5f * (1.0f + erff(z * 0.70710678118654752f)) +
           z * (__expf(-0.5f * z * z) * 0.39894228040143268f);
  return 1.0f;
}

struct SfGemmArgs {
  const void *p, *q;              // operands
  long long ldp, ldq;             // elements between their rows
  long long np, nq, nk;           // output rows, output columns, contraction
  long long k_split;              // contraction of one split (a multiple of the k step)
  int tiles_p, tiles_q, splits;
  const void *bias, *residual;    // (nq), (np, nq) of T or NULL
  void *out, *pre;                // (np, nq) of T; pre: the values before the activation, or NULL
  float *partial;                 // (splits, np, nq): the sums alone, when splits > 1
  int act;
};

template <typename T> struct SfMfma;
template <> struct SfMfma<float> {
  typedef float frag __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ sf_f32x16 run(frag a, frag b, sf_f32x16 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
};
template <> struct SfMfma<_Float16> {
  typedef _Float16 frag __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ sf_f32x16 run(frag a, frag b, sf_f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
  }
};
template <> struct SfMfma<__bf16> {
  typedef __bf16 frag __attribute__((ext_vector_type(8)));
  static __device__ __forceinline__ sf_f32x16 run(frag a, frag b, sf_f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
};

// One operand's side of the tile: B rows of the output, KMINOR as above.
template <typename T, bool KMINOR, int B, int WAVES, bool DMA>
struct SfOperand {
  static constexpr int S = sizeof(T), V = 16 / S, BK = 128 / S;
  static constexpr int CPR = KMINOR ? B * S / 16 : 8;     // chunks of one LDS row
  static constexpr int ROWB = CPR * 16;
  static constexpr int RPI = 64 / CPR;                    // LDS rows one wave-instruction fills
  static constexpr int NI = B * 128 / 1024 / WAVES;       // instructions of a wave a k step
  static_assert(CPR <= 64 && NI >= 1 && NI * WAVES * 1024 == B * 128, "tile shape");
  typedef typename SfMfma<T>::frag frag;

  static __device__ __forceinline__ int swz(int row) {
    if constexpr (!KMINOR) return (row ^ (row >> 3)) & 7;
    else if constexpr (S == 4) return ((row >> 2) & 1) << 3;
    else if constexpr (CPR == 8) return ((row >> 1) & 1) << 2;
    else return (row & 3) << 2;
  }

  const T *base;            // start of this workgroup's rows / columns, at k = 0
  long long ld, nk;
  long long rows;           // output rows this operand has from `base` on
  unsigned voff[NI];        // byte offset of this lane's chunk from the step's start
  short along[NI];          // K-major: the chunk's k; K-minor: its first output row
  sf_u32x4 reg[DMA ? 1 : NI];

  __device__ __forceinline__ void init(const void *ptr, long long ld_, long long first,
                                       long long total, long long nk_, int wave, int lane) {
    ld = ld_, nk = nk_, rows = total - first;
    base = static_cast<const T *>(ptr) + (KMINOR ? first : first * ld_);
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int row = (j * WAVES + wave) * RPI + lane / CPR;
      const int c = (lane % CPR) ^ swz(row);
      along[j] = (short)(c * V);
      voff[j] = DMA ? (unsigned)((long long)row * ld * S) + c * 16u : (unsigned)row;
    }
  }

  // Bring the step at k0 towards `lds`: the whole way when DMA, into registers otherwise.
  __device__ __forceinline__ void load(long long k0, unsigned char *lds, int wave) {
    const long long left_k = nk - k0;
    if constexpr (DMA) {
#if defined(__HIP_DEVICE_COMPILE__)
      // the range ends with the last element in use, so every row past it reads as zeros; a chunk
      // past the contiguous extent is sent out of range by hand (0x80000000 exceeds any range here)
      const T *at = base + (KMINOR ? k0 * ld : k0);
      long long n = KMINOR ? (left_k < BK ? left_k : BK) : (rows < B ? rows : B);
      const long long last = KMINOR ? rows : left_k;
      const long long bytes = ((n - 1) * ld + last) * S;
      const unsigned range = bytes < 0x7FFFFFFF ? (unsigned)bytes : 0x7FFFFFFFu;
      const __amdgpu_buffer_rsrc_t rs =
          __builtin_amdgcn_make_buffer_rsrc(const_cast<T *>(at), 0, range, 0x00020000);
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const unsigned off = along[j] < last ? voff[j] : 0x80000000u;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rs, (__attribute__((address_space(3))) void *)(lds + (j * WAVES + wave) * 1024), 16, off,
            0, 0, 0);
      }
#endif
    } else {
#pragma unroll
      for (int j = 0; j < NI; ++j) {
        const int row = (int)voff[j], c = along[j];
        const long long n = KMINOR ? left_k : rows;                     // rows there are
        const long long m = (KMINOR ? rows : left_k) - c;               // elements from the chunk on
        const T *at = base + (KMINOR ? (k0 + row) * ld : row * ld + k0) + c;
        sf_u32x4 v = {0, 0, 0, 0};
        if (row < n && m > 0) {
          if (m >= V) {
            v = *reinterpret_cast<const sf_u32x4_any *>(at);
          } else {
            typename SfMfma<T>::frag e;
#pragma unroll
            for (int i = 0; i < V; ++i) e[i] = i < m ? at[i] : (T)0.0f;
            v = __builtin_bit_cast(sf_u32x4, e);
          }
        }
        reg[j] = v;
      }
    }
  }
  // Registers to LDS (nothing to do when the load went there itself).
  __device__ __forceinline__ void store(unsigned char *lds, int wave, int lane) {
    if constexpr (!DMA) {
#pragma unroll
      for (int j = 0; j < NI; ++j)
        *reinterpret_cast<sf_u32x4 *>(lds + (j * WAVES + wave) * 1024 + lane * 16) = reg[j];
    }
  }

  // Fragment of the 32 output rows at row0 for quarter s of the step: this lane's row is
  // row0 + lane % 32, its k are chunk 2 s + lane / 32 of a K-major row.
  static __device__ __forceinline__ frag fragment(const unsigned char *lds, int row0, int s, int lane) {
    const int h = lane >> 5;
    if constexpr (!KMINOR) {
      const int row = row0 + (lane & 31);
      return *reinterpret_cast<const frag *>(lds + row * 128 + (((2 * s + h) ^ swz(row)) << 4));
    } else if constexpr (S == 4) {
      frag f;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int k = 8 * s + 4 * h + i, b = (row0 + (lane & 31)) * 4;
        f[i] = *reinterpret_cast<const float *>(lds + k * ROWB + (((b >> 4) ^ swz(k)) << 4) + (b & 15));
      }
      return f;
    } else {
      frag f = {};
#if defined(__HIP_DEVICE_COMPILE__)
      typedef __attribute__((address_space(3))) sf_s16x4 lds_s16x4;
      sf_s16x4 v[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int k = 16 * s + 8 * h + 4 * i + ((lane & 15) >> 2);
        const int b = (row0 + ((lane >> 4) & 1) * 16 + (lane & 3) * 4) * 2;
        v[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (lds_s16x4 *)(lds + k * ROWB + (((b >> 4) ^ swz(k)) << 4) + (b & 15)));
      }
      f = __builtin_bit_cast(frag, __builtin_shufflevector(v[0], v[1], 0, 1, 2, 3, 4, 5, 6, 7));
#endif
      return f;
    }
  }
};

// The tile's place in a launch of tiles_p x tiles_q x splits workgroups.  Workgroups go to the 8
// XCDs in turn: each XCD gets one contiguous run of the tiles, so that the operand rows its tiles
// share stay in its own L2; within a run, 8 tiles along p by all tiles along q.
__device__ __forceinline__ void sf_tile_of(int b, const SfGemmArgs &a, int *tp, int *tq, int *split) {
  const int nb = gridDim.x, per = nb >> 3, more = nb & 7, x = b & 7, i = b >> 3;
  int t = x * per + (x < more ? x : more) + i;
  const int tiles = a.tiles_p * a.tiles_q;
  *split = t / tiles;
  t -= *split * tiles;
  const int band = t / (8 * a.tiles_q), first = band * 8;
  const int high = a.tiles_p - first < 8 ? a.tiles_p - first : 8;
  t -= band * 8 * a.tiles_q;
  *tp = first + t % high;
  *tq = t / high;
}

template <typename T, bool PMINOR, bool QMINOR, int BP, int BQ, int WP, int WQ, bool DMA, int MINB>
__global__ void __launch_bounds__(WP *WQ * 64, MINB) sf_gemm_kernel(SfGemmArgs a) {
  constexpr int WAVES = WP * WQ, V = 16 / sizeof(T), BK = 128 / sizeof(T);
  constexpr int TP = BP / WP / 32, TQ = BQ / WQ / 32, WTQ = BQ / WQ;
  constexpr bool kReadFirst = sizeof(T) == 2 && (PMINOR || QMINOR);
  typedef SfOperand<T, PMINOR, BP, WAVES, DMA> OP;
  typedef SfOperand<T, QMINOR, BQ, WAVES, DMA> OQ;
  typedef typename SfMfma<T>::frag frag;
  static_assert(WAVES * 32 * WTQ * 4 <= (BP + BQ) * 128, "the epilogue's stage fits one buffer");
  __shared__ __attribute__((aligned(1024))) unsigned char s0[(BP + BQ) * 128];
  __shared__ __attribute__((aligned(1024))) unsigned char s1[(BP + BQ) * 128];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wp = wave / WQ, wq = wave % WQ;
  int tp, tq, split;
  sf_tile_of(blockIdx.x, a, &tp, &tq, &split);
  const long long p0 = (long long)tp * BP, q0 = (long long)tq * BQ;
  const long long k_first = split * a.k_split;
  const long long k_end = k_first + a.k_split < a.nk ? k_first + a.k_split : a.nk;
  const int steps = (int)((k_end - k_first + BK - 1) / BK);

  OP op;
  OQ oq;
  op.init(a.p, a.ldp, p0, a.np, a.nk, wave, lane);
  oq.init(a.q, a.ldq, q0, a.nq, a.nk, wave, lane);
  sf_f32x16 acc[TP][TQ];
#pragma unroll
  for (int i = 0; i < TP; ++i)
#pragma unroll
    for (int j = 0; j < TQ; ++j)
#pragma unroll
      for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;

  // One step: every wave's loads into `cur` have landed and every wave is done with `nxt` (the
  // barrier), the next step's loads start, this step multiplies.
  auto step = [&](unsigned char *cur, unsigned char *nxt, int i) {
    __builtin_amdgcn_s_waitcnt(0x0070);   // vmcnt(0) lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    const bool more = i + 1 < steps;
    frag fp[4][TP], fq[4][TQ];
    auto read = [&](int s) {
#pragma unroll
      for (int t = 0; t < TP; ++t) fp[s][t] = OP::fragment(cur, (wp * TP + t) * 32, s, lane);
#pragma unroll
      for (int t = 0; t < TQ; ++t) fq[s][t] = OQ::fragment(cur + BP * 128, (wq * TQ + t) * 32, s, lane);
    };
    // the transposing reads are opaque to the compiler's alias analysis: behind the loads they would
    // wait for them, so they all go first
    if constexpr (kReadFirst) {
#pragma unroll
      for (int s = 0; s < 4; ++s) read(s);
    }
    if (more) {
      op.load(k_first + (long long)(i + 1) * BK, nxt, wave);
      oq.load(k_first + (long long)(i + 1) * BK, nxt + BP * 128, wave);
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      if constexpr (!kReadFirst) read(s);
#pragma unroll
      for (int t = 0; t < TP; ++t)
#pragma unroll
        for (int u = 0; u < TQ; ++u) acc[t][u] = SfMfma<T>::run(fq[s][u], fp[s][t], acc[t][u]);
    }
    if (more) {
      op.store(nxt, wave, lane);
      oq.store(nxt + BP * 128, wave, lane);
    }
    asm volatile("" ::: "memory");
  };
  if (steps > 0) {
    op.load(k_first, s0, wave);
    oq.load(k_first, s0 + BP * 128, wave);
    op.store(s0, wave, lane);
    oq.store(s0 + BP * 128, wave, lane);
  }
  int i = 0;
  for (; i + 1 < steps; i += 2) {
    step(s0, s1, i);
    step(s1, s0, i + 1);
  }
  if (i < steps) step(s0, s1, i);

  // Epilogue, 32 rows of the wave's tile at a time: the accumulators go through LDS (quads swizzled
  // by the row) so that residual and output move in whole 16-byte chunks of a row.
  __syncthreads();
  constexpr int QUADS = WTQ / 4, CPL = WTQ / V, RPT = 64 / CPL;
  float *stage = reinterpret_cast<float *>(s0) + wave * 32 * WTQ;
  const int cl = lane % CPL, rl = lane / CPL;
  const long long col = q0 + wq * WTQ + cl * V;
  const T *bias = static_cast<const T *>(a.bias), *res = static_cast<const T *>(a.residual);
  T *out = static_cast<T *>(a.out), *pre = static_cast<T *>(a.pre);
  float bv[V];
#pragma unroll
  for (int j = 0; j < V; ++j) bv[j] = 0.0f;
  if (bias && a.splits == 1 && col < a.nq) sf_load_chunk<T>(bias, col, a.nq, bv);
#pragma unroll
  for (int t = 0; t < TP; ++t) {
    const int row = lane & 31, h = lane >> 5;
#pragma unroll
    for (int u = 0; u < TQ; ++u)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int quad = (u * 8 + 2 * g + h) ^ (row & (QUADS - 1));
        *reinterpret_cast<sf_f32x4 *>(stage + row * WTQ + quad * 4) =
            (sf_f32x4){acc[t][u][4 * g], acc[t][u][4 * g + 1], acc[t][u][4 * g + 2],
                       acc[t][u][4 * g + 3]};
      }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int r = 0; r < 32; r += RPT) {
      float v[V];
#pragma unroll
      for (int j = 0; j < V; j += 4) {
        const int quad = ((cl * V + j) / 4) ^ ((r + rl) & (QUADS - 1));
        const sf_f32x4 f = *reinterpret_cast<const sf_f32x4 *>(stage + (r + rl) * WTQ + quad * 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) v[j + e] = f[e];
      }
      const long long prow = p0 + (wp * TP + t) * 32 + r + rl;
      if (prow >= a.np || col >= a.nq) continue;
      const long long at = prow * a.nq;
      if (a.splits > 1) {
        float *part = a.partial + ((long long)split * a.np + prow) * a.nq;
#pragma unroll
        for (int j = 0; j < V; j += 4) sf_store_chunk<float>(part, col + j, a.nq, v + j);
        continue;
      }
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] += bv[j];
      if (pre) sf_store_chunk<T>(pre + at, col, a.nq, v);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] = sf_act(v[j], a.act);
      if (res) {
        float u[V];
        sf_load_chunk<T>(res + at, col, a.nq, u);
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] += u[j];
      }
      sf_store_chunk<T>(out + at, col, a.nq, v);
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
}

// Adds the splits' partial sums in order and applies the epilogue; rows of one chunk a lane.
template <typename T>
__global__ void __launch_bounds__(256) sf_gemm_join_kernel(SfGemmArgs a) {
  constexpr int V = 16 / sizeof(T);
  const long long cpr = (a.nq + V - 1) / V, chunks = a.np * cpr;
  for (long long c = (long long)blockIdx.x * 256 + threadIdx.x; c < chunks;
       c += (long long)gridDim.x * 256) {
    const long long row = c / cpr, col = (c - row * cpr) * V, at = row * a.nq;
    float v[V], u[V];
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = 0.0f;
    for (int s = 0; s < a.splits; ++s) {
      const float *part = a.partial + (long long)s * a.np * a.nq + at;
#pragma unroll
      for (int j = 0; j < V; j += 4) sf_load_chunk<float>(part, col + j, a.nq, u + j);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] += u[j];
    }
    if (a.bias) {
      sf_load_chunk<T>(static_cast<const T *>(a.bias), col, a.nq, u);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] += u[j];
    }
    if (a.pre) sf_store_chunk<T>(static_cast<T *>(a.pre) + at, col, a.nq, v);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = sf_act(v[j], a.act);
    if (a.residual) {
      sf_load_chunk<T>(static_cast<const T *>(a.residual) + at, col, a.nq, u);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] += u[j];
    }
    sf_store_chunk<T>(static_cast<T *>(a.out) + at, col, a.nq, v);
  }
}

// The launches of one storage type (linear_f32.hip, linear_f16.hip, linear_bf16.hip).
// layout 0: P, Q K-major; 1: Q K-minor; 2: both K-minor.
void sf_gemm_f32(const SfGemmArgs &a, int layout, int tile, bool dma, hipStream_t st);
void sf_gemm_f16(const SfGemmArgs &a, int layout, int tile, bool dma, hipStream_t st);
void sf_gemm_bf16(const SfGemmArgs &a, int layout, int tile, bool dma, hipStream_t st);

template <typename T, bool PMINOR, bool QMINOR>
static void sf_gemm_launch(const SfGemmArgs &a, int tile, bool dma, hipStream_t st) {
  const dim3 grid((unsigned)(a.tiles_p * a.tiles_q * a.splits));
#define SF_GO(B, D, MINB)                                                                          \
  hipLaunchKernelGGL((sf_gemm_kernel<T, PMINOR, QMINOR, B, B, 2, 2, D, MINB>), grid, dim3(256), 0, \
                     st, a)
  if (tile == 128) {
    if (dma) SF_GO(128, true, 2);
    else SF_GO(128, false, 2);
  } else {
    if (dma) SF_GO(64, true, 4);
    else SF_GO(64, false, 4);
  }
#undef SF_GO
  if (a.splits > 1) {
    const long long cpr = (a.nq + 16 / (int)sizeof(T) - 1) / (16 / (int)sizeof(T));
    hipLaunchKernelGGL((sf_gemm_join_kernel<T>), dim3(sf_grid(a.np * cpr, 256)), dim3(256), 0, st, a);
  }
}

template <typename T>
static void sf_gemm_any(const SfGemmArgs &a, int layout, int tile, bool dma, hipStream_t st) {
  if (layout == 0) sf_gemm_launch<T, false, false>(a, tile, dma, st);
  else if (layout == 1) sf_gemm_launch<T, false, true>(a, tile, dma, st);
  else sf_gemm_launch<T, true, true>(a, tile, dma, st);
}
