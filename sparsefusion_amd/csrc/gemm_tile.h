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
// Both operands' tiles go to LDS in 16-byte chunks straight from memory (buffer_load ... lds), into a
// ring of buffers up to three steps ahead.  v_mfma_f32_32x32x16 (32x32x2 for fp32) accumulates in fp32;
// Q is the instruction's first operand, so a lane ends up with four consecutive q of one row p.
// Workgroups stay and walk the tiles: the loads of the next tile's first steps run under the epilogue of
// the last.
//
// What bounds it: a 256 x 256 tile's products of 128 bytes of k keep the matrix units busy for as long as
// LDS takes to write the chunks and read the fragments; half of both is reached (16384 x 2048 -> 2048
// bf16 1170 TFLOP/s; fp32 8192 x 2048 -> 2048 142 TFLOP/s, 90 % of the peak).  Short contractions are bound by the epilogue, long outputs by memory:
// 259200 x 1024 -> 256 bf16 with its residual moves 797 MB in 193 us.
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

// GELU, z Phi(z), from the side where Phi is small: with a = |z|, gelu(z) = max(z, 0) - a Phi(-a) keeps its digits
// for negative z too, where it is far smaller than z.  Phi(-a) is fitted for the least maximal error relative to
// itself.  16 bits: 2^P(a), P the polynomial of degree 9 nearest to log2(Phi(-a)) up to 13, off by at most 8e-7,
// 5e-5 of itself up to a = 4 (a fifth of half an fp16 step) and 3.5e-4 farther out, where fp16 has no digits left (a
// sixth of half a bf16 step).  fp32, where P's terms would round to more: exp(-a^2 / 2) M(a), M (Mills' ratio over
// sqrt(2 pi)) = t Q(t) of t = 1 / (1 + 0.34 a) with seven coefficients, off by 5.2e-8 of itself up to a = 1 and
// 5.2e-8 (1 + (a - 1)^3) beyond, where the exponent's rounding, 2.5 a^2 times 2^-24, is as much.
// a stops at 14, where both come out as 0 (v_exp_f32 flushes what is below the smallest normal number): an infinite
// z gives infinity or 0, and NaN stays (minimum and maximum hand it on).  32400 x 256 -> 1024 bf16, 24.4 us without an
// activation: 34.8 us, with a quotient of degrees 4 and 2 for P 36.5, with fmaxf, which takes two instructions, 2.3
// more, with a logistic form, whose error is absolute (4.5 % of gelu(-4)), 34.3.
__device__ __forceinline__ float sf_gauss(float a) {      // exp(-a^2 / 2)
  const float b = a * 0.84932180028801905f;
  return __builtin_amdgcn_exp2f(-(b * b));
}
template <typename T>
__device__ __forceinline__ float sf_phi_below(float a) {      // Phi(-a)
  float q;
  if constexpr (sizeof(T) == 4) {
    const float t = __builtin_amdgcn_rcpf(fmaf(a, 0.34f, 1.0f));
    q = 4.56890270e-02f;
    q = fmaf(q, t, -2.04008249e-01f);
    q = fmaf(q, t, 2.69765421e-01f);
    q = fmaf(q, t, -3.55146202e-02f);
    q = fmaf(q, t, 1.58752532e-01f);
    q = fmaf(q, t, 1.29248573e-01f);
    q = fmaf(q, t, 1.36067344e-01f);
    return sf_gauss(a) * (q * t);
  } else {
    q = -6.95180746e-10f;
    q = fmaf(q, a, 7.87926524e-08f);
    q = fmaf(q, a, -3.26799250e-06f);
    q = fmaf(q, a, 7.15041460e-05f);
    q = fmaf(q, a, -9.55835043e-04f);
    q = fmaf(q, a, 8.49724654e-03f);
    q = fmaf(q, a, -5.38178124e-02f);
    q = fmaf(q, a, -4.58641291e-01f);
    q = fmaf(q, a, -1.15119171e+00f);
    q = fmaf(q, a, -9.99997973e-01f);
    return __builtin_amdgcn_exp2f(q);
  }
}
__device__ __forceinline__ float sf_below(float z) { return __builtin_elementwise_minimum(__builtin_fabsf(z), 14.0f); }
template <typename T>
__device__ __forceinline__ float sf_gelu(float z) {
  const float a = sf_below(z);
  return fmaf(-a, sf_phi_below<T>(a), __builtin_elementwise_maximum(z, 0.0f));
}
// Phi(z) + z phi(z): 1 - s for s of -z
template <typename T>
__device__ __forceinline__ float sf_gelu_slope(float z) {
  const float a = sf_below(z), s = fmaf(a * -0.39894228040143268f, sf_gauss(a), sf_phi_below<T>(a));
  return z < 0.0f ? s : 1.0f - s;
}
template <typename T>
__device__ __forceinline__ float sf_act(float z, int act) {
  if (act == SF_ACT_RELU) return z > 0.0f ? z : (z != z ? z : 0.0f);
  if (act == SF_ACT_GELU) return sf_gelu<T>(z);
  return z;
}
template <typename T>
__device__ __forceinline__ float sf_act_gradient(float g, float z, int act) {
  if (act == SF_ACT_RELU) return z <= 0.0f ? 0.0f : g;      // whatever g is
  if (act == SF_ACT_GELU) return g * sf_gelu_slope<T>(z);
  return g;
}

struct SfGemmArgs {
  const void *p, *q;              // operands
  long long ldp, ldq;             // elements between their rows
  long long np, nq, nk;           // output rows, output columns, contraction
  long long k_split;              // contraction of one split (a multiple of the k step)
  int tiles_p, tiles_q, splits;
  int tail;                       // whether what is behind a K-major operand's rows has to be cleared
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

// 16 bytes per lane straight into LDS, lane L's to lds + 16 L (wave-uniform), zeros for an offset out
// of rs's range.  Written as assembly because the compiler makes every LDS read that it cannot tell
// from the destination wait for the builtin form, all of it, and these loads are meant to stay in
// flight under such reads.  Nothing comes back in registers; who reads the destination waits for
// vmcnt(0) by hand and meets the other waves at a barrier.  (The compiler's own counted waits only
// become stricter: vmcnt retires in order.)
// `lds` + OFFSET goes to m0; the wait states cover an SGPR that a vector instruction wrote just before.
template <int OFFSET>
__device__ __forceinline__ void sf_lds_load16(const sf_u32x4 &rs, unsigned lds, unsigned off) {
#if defined(__HIP_DEVICE_COMPILE__)
  asm volatile("s_add_u32 m0, %0, %3\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
               :
               : "s"((unsigned)__builtin_amdgcn_readfirstlane((int)lds)), "v"(off), "s"(rs), "i"(OFFSET)
               : "m0", "scc", "memory");
#endif
}

// One operand's side of the tile: B rows of the output, KMINOR as above, STEP bytes of a row's k (128
// or 64) brought at a time.
template <typename T, bool KMINOR, int B, int WAVES, int STEP>
struct SfOperand {
  static constexpr int S = sizeof(T), V = 16 / S, BK = STEP / S;
  static constexpr int CPR = KMINOR ? B * S / 16 : STEP / 16;     // chunks of one LDS row
  static constexpr int ROWB = CPR * 16;
  static constexpr int RPI = 64 / CPR;                    // LDS rows one wave-instruction fills
  static constexpr int NI = B * STEP / 1024 / WAVES;      // instructions of a wave a step
  static_assert(CPR <= 64 && NI >= 1 && NI * WAVES * 1024 == B * STEP, "tile shape");
  typedef typename SfMfma<T>::frag frag;

  static __device__ __forceinline__ int swz(int row) {
    if constexpr (!KMINOR && STEP == 128) return (row ^ (row >> 3)) & 7;
    else if constexpr (!KMINOR) return (row >> 3) & 3;
    else if constexpr (S == 4) return CPR == 8 ? 0 : ((row >> 2) & 1) << 3;
    else if constexpr (CPR == 4) return 0;
    else if constexpr (CPR == 8) return ((row >> 1) & 1) << 2;
    else return (row & 3) << 2;
  }

  const T *at;              // the step being loaded: the tile's first row / column at its k
  long long rows;           // output rows this operand has from the tile's first on
  long long ld;
  int steps, last_k;        // steps to go in this tile, k of its last one
  unsigned range, range_last;       // bytes from `at` to the last element of a step in use
  unsigned voff[NI];        // byte offset of this lane's chunk from `at`
  int along[NI];            // K-major: the chunk's k; K-minor: its first output row

  __device__ __forceinline__ void init(long long ld_, int wave, int lane) {
    ld = ld_;
#pragma unroll
    for (int j = 0; j < NI; ++j) {
      const int row = (j * WAVES + wave) * RPI + lane / CPR;
      const int c = (lane % CPR) ^ swz(row);
      along[j] = c * V;
      voff[j] = (unsigned)((long long)row * ld * S) + c * 16u;
    }
  }
  // A tile: output rows `first` on (of `total`), k from k0 on in `steps` steps, the last of last_k.  Rows
  // start at multiples of 4 bytes; rows past the range read as zeros, a dword at a time (all of it fits 31
  // bits: the host sees to both).  A chunk that a row's end cuts brings what is behind it: other columns'
  // outputs, which nobody stores, or for a K-major operand k that clear() makes zeros.
  __device__ __forceinline__ void open(const void *ptr, long long first, long long total, long long k0,
                                       int steps_, int last_k_) {
    steps = steps_;
    at = static_cast<const T *>(ptr) + (KMINOR ? first + k0 * ld : first * ld + k0);
    if constexpr (KMINOR) {
      rows = total - first, last_k = last_k_;
      range = (unsigned)(((BK - 1) * ld + rows) * S + 3) & ~3u;
      range_last = (unsigned)(((last_k - 1) * ld + rows) * S + 3) & ~3u;
    } else {
      rows = total - first, last_k = last_k_;
      const int n = rows < B ? (int)rows : B;
      range = (unsigned)(((n - 1) * ld + BK) * S + 3) & ~3u;
      range_last = (unsigned)(((n - 1) * ld + last_k) * S + 3) & ~3u;
    }
  }
  // Zeros behind the first `k` of a step's rows (inside a chunk) at `tile`, by the whole workgroup.
  static __device__ __forceinline__ void clear(unsigned char *tile, int k) {
    if constexpr (!KMINOR)
      for (int row = threadIdx.x; row < B; row += WAVES * 64) {
        T *chunk = reinterpret_cast<T *>(tile + row * STEP + ((k / V ^ swz(row)) << 4));
#pragma unroll
        for (int j = 1; j < V; ++j)
          if (j >= k % V) chunk[j] = (T)0.0f;
      }
  }
  __device__ __forceinline__ void close() {      // nothing left to load: zeros from here on
    range = range_last = 0;
    steps = 0x7FFFFFFF;
  }

  // DMA of instruction J of the step towards LDS address `lds`; next() goes on to the following step.
  // A chunk past the contiguous extent is sent out of range by hand (the others are past a row's end).
  template <int J>
  __device__ __forceinline__ void issue(unsigned lds_wave) const {
    const unsigned long long addr = (unsigned long long)at;
    const sf_u32x4 rs = {(unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)addr),
                         (unsigned)__builtin_amdgcn_readfirstlane((int)(unsigned)(addr >> 32)) & 0xFFFFu,
                         (unsigned)__builtin_amdgcn_readfirstlane((int)(steps == 1 ? range_last : range)),
                         0x00020000u};
    const int end = KMINOR ? (rows < B ? (int)rows : B) : (steps == 1 ? last_k : BK);
    sf_lds_load16<J * WAVES * 1024>(rs, lds_wave, along[J] < end ? voff[J] : 0x80000000u);
  }
  __device__ __forceinline__ void next() {
    at += KMINOR ? BK * ld : BK;
    --steps;
  }

  // Fragment of the 32 output rows at row0 for the step's s-th 32 bytes of k: this lane's row is
  // row0 + lane % 32, its k are chunk 2 s + lane / 32 of a K-major row.
  static __device__ __forceinline__ frag fragment(const unsigned char *lds, int row0, int s, int lane) {
    const int h = lane >> 5;
    if constexpr (!KMINOR) {
      const int row = row0 + (lane & 31);
      return *reinterpret_cast<const frag *>(lds + row * STEP + (((2 * s + h) ^ swz(row)) << 4));
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

// Place of work item b of nb = tiles_p x tiles_q x splits.  Workgroups go to the 8 XCDs in turn (and
// walk the items in strides of a multiple of 8): each XCD gets one contiguous run of the tiles, so
// that the operand rows its tiles share stay in its own L2; within a run, 8 tiles along p by all
// tiles along q.
__device__ __forceinline__ void sf_tile_of(int b, int nb, const SfGemmArgs &a, int *tp, int *tq,
                                           int *split) {
  const int per = nb >> 3, more = nb & 7, x = b & 7, i = b >> 3;
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

// Steps of a tile's contraction.
template <int BK>
__device__ __forceinline__ int sf_steps(const SfGemmArgs &a, int split) {
  const long long first = split * a.k_split;
  const long long n = first + a.k_split < a.nk ? a.k_split : a.nk - first;
  return (int)((n + BK - 1) / BK);
}

// Epilogue of a wave's TP x TQ blocks of 32 x 32 at (p0, q0).  A block goes through the wave's own
// 4 KB of LDS (quads of columns swizzled by the row) so that bias, pre, residual and output move in
// whole 16-byte chunks of a row; the plain sums when the contraction is split.  Tiles whose rows and columns all
// exist are straight-line code over all blocks (whole, sums), so that the next block's work runs under a
// block's loads and stores; cut ones a loop over the blocks (ragged).
template <typename T, int TP, int TQ>
struct SfEpilogue {
  static constexpr int V = 16 / sizeof(T), CPL = 32 / V, RPT = 64 / CPL, ITS = 32 / RPT;
  const SfGemmArgs &a;
  float *stage;
  long long p0, q0;
  int split, lane;

  __device__ __forceinline__ void put(const sf_f32x16 &c) const {
    const int h = lane >> 5, row = lane & 31;
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<sf_f32x4 *>(stage + row * 32 + (((2 * g + h) ^ row ^ (row >> 3)) & 7) * 4) =
          (sf_f32x4){c[4 * g], c[4 * g + 1], c[4 * g + 2], c[4 * g + 3]};
  }
  static __device__ __forceinline__ void meet() {      // the wave's writes before its reads, and back
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  }
  // this lane's chunk of row r (0..31) of the staged block
  __device__ __forceinline__ void get(int r, float *v) const {
    const int cl = lane % CPL;
#pragma unroll
    for (int j = 0; j < V; j += 4) {
      const int quad = ((cl * V + j) / 4 ^ r ^ (r >> 3)) & 7;
      const sf_f32x4 f = *reinterpret_cast<const sf_f32x4 *>(stage + r * 32 + quad * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[j + e] = f[e];
    }
  }
  __device__ __forceinline__ long long row_of(int t, int it) const {
    return p0 + t * 32 + it * RPT + lane / CPL;
  }
  typedef typename SfChunk<T>::type chunk;
  typedef SfChunk<float>::type chunk4;

  // All rows and columns of the wave's blocks exist: straight-line code, so that nothing waits for
  // stores (their vmcnt is shared with the loads) and the residual comes a stripe of 32 rows ahead.
  struct Ahead {
    chunk r[2][TQ][ITS];
  };
  __device__ __forceinline__ void prefetch(Ahead &n, int t) const {
    const T *res = static_cast<const T *>(a.residual) + q0 + (lane % CPL) * V;
#pragma unroll
    for (int it = 0; it < ITS; ++it)
#pragma unroll
      for (int u = 0; u < TQ; ++u)
        n.r[t & 1][u][it] = *reinterpret_cast<const chunk *>(res + row_of(t, it) * a.nq + u * 32);
  }
  __device__ __forceinline__ void sums(const sf_f32x16 (&acc)[TP][TQ]) const {
#pragma unroll
    for (int t = 0; t < TP; ++t)
#pragma unroll
      for (int u = 0; u < TQ; ++u) {
        put(acc[t][u]);
        meet();
#pragma unroll
        for (int it = 0; it < ITS; ++it) {
          float v[V];
          get(it * RPT + lane / CPL, v);
          float *part = a.partial + ((long long)split * a.np + row_of(t, it)) * a.nq + q0 +
                        (lane % CPL) * V + u * 32;
#pragma unroll
          for (int j = 0; j < V; j += 4)
            *reinterpret_cast<chunk4 *>(part + j) = (chunk4){v[j], v[j + 1], v[j + 2], v[j + 3]};
        }
        meet();
      }
  }
  template <bool RES>
  __device__ __forceinline__ void whole(const sf_f32x16 (&acc)[TP][TQ], Ahead &ahead) const {
    const long long col = q0 + (lane % CPL) * V;
    T *out = static_cast<T *>(a.out) + col, *pre = static_cast<T *>(a.pre);
    if (pre) pre += col;
    chunk b[TQ];
#pragma unroll
    for (int u = 0; u < TQ; ++u) {
#pragma unroll
      for (int j = 0; j < V; ++j) b[u][j] = (T)0.0f;
      if (a.bias) b[u] = *reinterpret_cast<const chunk *>(static_cast<const T *>(a.bias) + col + u * 32);
    }
#pragma unroll
    for (int t = 0; t < TP; ++t) {
      if constexpr (RES)
        if (t + 1 < TP) prefetch(ahead, t + 1);
#pragma unroll
      for (int u = 0; u < TQ; ++u) {
        put(acc[t][u]);
        meet();
        float v[ITS][V];
#pragma unroll
        for (int it = 0; it < ITS; ++it) get(it * RPT + lane / CPL, v[it]);
        meet();
#pragma unroll
        for (int it = 0; it < ITS; ++it) {
          const long long at = row_of(t, it) * a.nq + u * 32;
          chunk c;
#pragma unroll
          for (int j = 0; j < V; ++j) v[it][j] += (float)b[u][j];
          if (pre) {
#pragma unroll
            for (int j = 0; j < V; ++j) c[j] = (T)v[it][j];
            *reinterpret_cast<chunk *>(pre + at) = c;
          }
          if (a.act == SF_ACT_GELU) {
#pragma unroll
            for (int j = 0; j < V; ++j) v[it][j] = sf_act<T>(v[it][j], SF_ACT_GELU);
          } else if (a.act == SF_ACT_RELU) {
#pragma unroll
            for (int j = 0; j < V; ++j) v[it][j] = sf_act<T>(v[it][j], SF_ACT_RELU);
          }
          if constexpr (RES) {
#pragma unroll
            for (int j = 0; j < V; ++j) v[it][j] += (float)ahead.r[t & 1][u][it][j];
          }
#pragma unroll
          for (int j = 0; j < V; ++j) c[j] = (T)v[it][j];
          *reinterpret_cast<chunk *>(out + at) = c;
        }
      }
    }
  }

  // Some rows or columns are past the end: element by element where a chunk is cut.  Blocks are a real
  // loop; the accumulators cannot be indexed by it, so each is picked by comparison.
  __device__ __forceinline__ void ragged(const sf_f32x16 (&acc)[TP][TQ]) const {
    const T *bias = static_cast<const T *>(a.bias), *res = static_cast<const T *>(a.residual);
    T *out = static_cast<T *>(a.out), *pre = static_cast<T *>(a.pre);
#pragma unroll 1
    for (int tu = 0; tu < TP * TQ; ++tu) {
      const int t = tu / TQ, u = tu % TQ;
      if (p0 + t * 32 >= a.np || q0 + u * 32 >= a.nq) continue;
      const long long col = q0 + u * 32 + (lane % CPL) * V;
      float w[ITS][V], b[V];
#pragma unroll
      for (int j = 0; j < V; ++j) b[j] = 0.0f;
      if (bias && a.splits == 1 && col < a.nq) sf_load_chunk<T>(bias, col, a.nq, b);
#pragma unroll
      for (int it = 0; it < ITS; ++it) {
        const long long row = row_of(t, it);
#pragma unroll
        for (int j = 0; j < V; ++j) w[it][j] = 0.0f;
        if (res && a.splits == 1 && row < a.np && col < a.nq)
          sf_load_chunk<T>(res + row * a.nq, col, a.nq, w[it]);
      }
#pragma unroll
      for (int i = 0; i < TP * TQ; ++i)
        if (tu == i) put(acc[i / TQ][i % TQ]);
      meet();
#pragma unroll
      for (int it = 0; it < ITS; ++it) {
        const long long row = row_of(t, it);
        if (row >= a.np || col >= a.nq) continue;
        float v[V];
        get(it * RPT + lane / CPL, v);
        const long long at = row * a.nq;
        if (a.splits > 1) {
          float *part = a.partial + (long long)split * a.np * a.nq + at;
#pragma unroll
          for (int j = 0; j < V; j += 4) sf_store_chunk<float>(part, col + j, a.nq, v + j);
          continue;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] += b[j];
        if (pre) sf_store_chunk<T>(pre + at, col, a.nq, v);
        if (a.act == SF_ACT_GELU) {
#pragma unroll
          for (int j = 0; j < V; ++j) v[j] = sf_act<T>(v[j], SF_ACT_GELU);
        } else if (a.act == SF_ACT_RELU) {
#pragma unroll
          for (int j = 0; j < V; ++j) v[j] = sf_act<T>(v[j], SF_ACT_RELU);
        }
        if (res) {
#pragma unroll
          for (int j = 0; j < V; ++j) v[j] += w[it][j];
        }
        sf_store_chunk<T>(out + at, col, a.nq, v);
      }
      meet();
    }
  }
};

template <int N> struct SfInt { static constexpr int value = N; };
template <int I, int N, typename F>
__device__ __forceinline__ void sf_unroll(F &&f) {
  if constexpr (I < N) {
    f(SfInt<I>());
    sf_unroll<I + 1, N>(static_cast<F &&>(f));
  }
}

// Shape of a kernel: BP x BQ outputs by WP x WQ waves, steps of STEP bytes of k in a ring of RING
// buffers, WGS workgroups to a CU.  RES: a residual may be added.  TAIL: clears what is behind cut rows.
template <int BP_, int BQ_, int WP_, int WQ_, int STEP_, int RING_, int WGS_, bool RES_ = true, bool TAIL_ = false>
struct SfShape {
  static constexpr bool RES = RES_, TAIL = TAIL_;
  static constexpr int BP = BP_, BQ = BQ_, WP = WP_, WQ = WQ_, STEP = STEP_, RING = RING_, WGS = WGS_;
  static constexpr int WAVES = WP * WQ, BYTES = (BP + BQ) * STEP, LDS = RING * BYTES + WAVES * 4096;
  static_assert(LDS * WGS <= 160 * 1024 && (RING == 2 || RING == 4), "LDS of a CU");
};

// s_waitcnt vmcnt(N) lgkmcnt(0)
template <int N>
__device__ __forceinline__ void sf_wait_loads() {
  static_assert(N < 64, "vmcnt has 6 bits");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0070);
}

// Workgroup `group` of `groups`, which share the tiles of the product.
template <typename T, bool PMINOR, bool QMINOR, typename SH>
__device__ __forceinline__ void sf_gemm(const SfGemmArgs &a, unsigned char *lds, int group, int groups) {
  constexpr int BP = SH::BP, BQ = SH::BQ, WQ = SH::WQ, WAVES = SH::WAVES, STEP = SH::STEP;
  constexpr int RING = SH::RING, BYTES = SH::BYTES, BK = STEP / (int)sizeof(T), NS = STEP / 32;
  constexpr int V = 16 / sizeof(T);
  constexpr int TP = BP / SH::WP / 32, TQ = BQ / WQ / 32;
  typedef SfOperand<T, PMINOR, BP, WAVES, STEP> OP;
  typedef SfOperand<T, QMINOR, BQ, WAVES, STEP> OQ;
  typedef typename SfMfma<T>::frag frag;
  constexpr int NI = OP::NI + OQ::NI;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wp = wave / WQ, wq = wave % WQ;
  float *stage = reinterpret_cast<float *>(lds + RING * BYTES) + wave * 1024;
#if defined(__HIP_DEVICE_COMPILE__)
  const unsigned lds0 = (unsigned)(unsigned long long)(__attribute__((address_space(3))) unsigned char *)lds;
#else
  const unsigned lds0 = 0;
#endif
  const int tiles = a.tiles_p * a.tiles_q * a.splits;

  // The loads run ahead of the products, across the tiles of this workgroup: `lt` is the tile being
  // loaded.  Behind the last one they go on as loads of nothing, so that the counted waits hold.
  OP op;
  OQ oq;
  op.init(a.ldp, wave, lane);
  oq.init(a.ldq, wave, lane);
  int lt = group;
  auto open = [&]() {
    int tp, tq, split;
    sf_tile_of(lt, tiles, a, &tp, &tq, &split);
    const long long k0 = split * a.k_split;
    const int steps = sf_steps<BK>(a, split);
    const long long left = a.nk - k0 - (long long)(steps - 1) * BK;
    const int last = left < BK ? (int)left : BK;
    op.open(a.p, (long long)tp * BP, a.np, k0, steps, last);
    oq.open(a.q, (long long)tq * BQ, a.nq, k0, steps, last);
  };
  auto advance = [&]() {      // behind the last instruction of a step's load
    op.next(), oq.next();
    if (op.steps == 0) {
      lt += groups;
      if (lt < tiles) open();
      else op.close(), oq.close();
    }
  };
  // instructions [FROM, TO) of the load of a step into the buffer at `buf`
  const unsigned lds_wave = lds0 + wave * 1024;
  auto issue = [&](auto from, auto to, int buf) {
    sf_unroll<decltype(from)::value, decltype(to)::value>([&](auto j) {
      constexpr int J = decltype(j)::value;
      if constexpr (J < OP::NI) op.template issue<J>(lds_wave + buf);
      else oq.template issue<J - OP::NI>(lds_wave + buf + BP * STEP);
    });
  };
  auto read_one = [&](frag (&fp)[TP], frag (&fq)[TQ], int buf, int s, int r) {
    // in the order in which the products need them: p0, q0, q1, .., p1, ..
    if (r == 0) fp[0] = OP::fragment(lds + buf, wp * TP * 32, s, lane);
    else if (r <= TQ) fq[r - 1] = OQ::fragment(lds + buf + BP * STEP, (wq * TQ + r - 1) * 32, s, lane);
    else fp[r - TQ] = OP::fragment(lds + buf, (wp * TP + r - TQ) * 32, s, lane);
  };

  sf_f32x16 acc[TP][TQ];
  frag fp[2][TP], fq[2][TQ];
  constexpr int M = TP * TQ, R = TP + TQ, HALF = RING == 2 ? NI : NI / 2;
  // The products of 32 bytes of k, fragments in set `s`; between them the reads of the following 32
  // bytes (part rs of the buffer at rbuf, into the other set) and, evenly, `count` instructions of a
  // load from `from` on.  A wave issues in order and the matrix unit is busy for 32 cycles a product
  // (64 for fp32): what is not spread between the products holds them up.
  auto multiply = [&](auto set, int rbuf, int rs, auto from, auto count, int lbuf) {
    constexpr int SET = decltype(set)::value, FROM = decltype(from)::value, N = decltype(count)::value;
    sf_unroll<0, M>([&](auto mm) {
      constexpr int m = decltype(mm)::value, t = m / TQ, u = m % TQ;
      __builtin_amdgcn_sched_barrier(0);
      acc[t][u] = SfMfma<T>::run(fq[SET][u], fp[SET][t], acc[t][u]);
#pragma unroll
      for (int r = m * R / M; r < (m + 1) * R / M; ++r) read_one(fp[1 - SET], fq[1 - SET], rbuf, rs, r);
      issue(SfInt<FROM + m * N / M>(), SfInt<FROM + (m + 1) * N / M>(), lbuf);
    });
    __builtin_amdgcn_sched_barrier(0);
  };

  // behind the barrier that shows step `step` of tile `t` in `buf`
  auto clear_tail = [&](int t, int step, int buf) {
    int tp, tq, split;
    sf_tile_of(t, tiles, a, &tp, &tq, &split);
    const long long left = a.nk - split * a.k_split - (long long)step * BK;
    if (left >= BK || left % V == 0) return;
    OP::clear(lds + buf, (int)left);
    OQ::clear(lds + buf + BP * STEP, (int)left);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
  };
  int cur = 0, last = (RING - 1) * BYTES;      // last: the buffer whose load is half issued
  open();
#pragma unroll
  for (int i = 0; i + 1 < RING; ++i) {
    issue(SfInt<0>(), SfInt<NI>(), i * BYTES);
    advance();
  }
  issue(SfInt<0>(), SfInt<HALF>(), last);
  sf_wait_loads<(RING - 2) * NI + HALF>();
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  if (SH::TAIL && a.tail && group < tiles) clear_tail(group, 0, 0);
  for (int tile = group; tile < tiles; tile += groups) {
    int tp, tq, split;
    sf_tile_of(tile, tiles, a, &tp, &tq, &split);
    const int steps = sf_steps<BK>(a, split);
#pragma unroll
    for (int i = 0; i < TP; ++i)
#pragma unroll
      for (int j = 0; j < TQ; ++j)
#pragma unroll
        for (int e = 0; e < 16; ++e) acc[i][j][e] = 0.0f;
#pragma unroll
    for (int r = 0; r < R; ++r) read_one(fp[0], fq[0], cur, 0, r);      // visible since the last barrier
    const long long p0 = (long long)tp * BP + wp * TP * 32, q0 = (long long)tq * BQ + wq * TQ * 32;
    // the epilogue's addresses are not worth registers in the main loop: keep them from being hoisted
    int l = lane;
    asm volatile("" : "+v"(l));
    const SfEpilogue<T, TP, TQ> epilogue{a, stage, p0, q0, split, l};
    typename SfEpilogue<T, TP, TQ>::Ahead ahead;
    const bool inside = q0 + TQ * 32 <= a.nq && p0 + TP * 32 <= a.np;
    const bool residual = SH::RES && a.residual && a.splits == 1;
    // A step: the fragments of each 32 bytes of k are read while the 32 before multiply, and the
    // second half of the youngest load is issued.  Ahead of the last products the next step has landed
    // (every wave waits for its own loads, the barrier joins them) and nobody needs this step's buffer
    // any more: the next step's first fragments and the first half of the load into the freed buffer
    // run under them.
    for (int i = 0; i < steps; ++i) {
      const int nxt = cur + BYTES == RING * BYTES ? 0 : cur + BYTES;
      multiply(SfInt<0>(), cur, 1, SfInt<HALF>(), SfInt<NI - HALF>(), last);
#pragma unroll
      for (int s = 1; s + 2 < NS; s += 2) {
        multiply(SfInt<1>(), cur, s + 1, SfInt<0>(), SfInt<0>(), 0);
        multiply(SfInt<0>(), cur, s + 2, SfInt<0>(), SfInt<0>(), 0);
      }
      advance();
      asm volatile("" ::: "memory");
      sf_wait_loads<(RING - 2) * NI>();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (SH::TAIL && a.tail && i + 2 >= steps) {
        if (i + 2 == steps) clear_tail(tile, i + 1, nxt);
        else if (tile + groups < tiles) clear_tail(tile + groups, 0, nxt);
      }
      if (i + 1 == steps && inside && residual) epilogue.prefetch(ahead, 0);
      multiply(SfInt<1>(), nxt, 0, SfInt<0>(), SfInt<HALF>(), cur);
      last = cur;
      cur = nxt;
    }
    if (!inside) epilogue.ragged(acc);
    else if (a.splits > 1) epilogue.sums(acc);
    else if (residual) epilogue.template whole<true>(acc, ahead);
    else epilogue.template whole<false>(acc, ahead);
  }
  sf_wait_loads<0>();      // the loads of nothing still write zeros into this workgroup's LDS
}

template <typename T, bool PMINOR, bool QMINOR, typename SH>
__global__ void __launch_bounds__(SH::WAVES * 64, SH::WGS * SH::WAVES / 4) sf_gemm_kernel(SfGemmArgs a) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[SH::LDS];
  sf_gemm<T, PMINOR, QMINOR, SH>(a, lds, blockIdx.x, gridDim.x);
}

// Adds the splits' partial sums in order and applies the epilogue; a chunk of a row by SL lanes, which
// take turns at the splits and meet in LDS, each with four loads in flight.
template <typename T, int SL>
__global__ void __launch_bounds__(256) sf_gemm_join_kernel(SfGemmArgs a) {
  constexpr int V = 16 / sizeof(T), CL = 256 / SL, DEEP = 4;
  __shared__ float red[SL > 1 ? SL - 1 : 1][SL > 1 ? CL : 1][V + 1];
  const int cl = threadIdx.x % CL, sl = threadIdx.x / CL;
  const long long cpr = (a.nq + V - 1) / V, chunks = a.np * cpr;
  for (long long c0 = (long long)blockIdx.x * CL; c0 < chunks; c0 += (long long)gridDim.x * CL) {
    const bool live = c0 + cl < chunks;
    const long long c = live ? c0 + cl : 0, row = c / cpr, col = (c - row * cpr) * V, at = row * a.nq;
    float v[V], u[DEEP][V];
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = 0.0f;
    for (int s = sl; s < a.splits; s += SL * DEEP) {
#pragma unroll
      for (int i = 0; i < DEEP; ++i) {
        // past the last split the last is read again and counts for nothing
        const long long k = s + i * SL < a.splits ? s + i * SL : a.splits - 1;
        const float *part = a.partial + k * a.np * a.nq + at;
#pragma unroll
        for (int j = 0; j < V; j += 4) sf_load_chunk<float>(part, col + j, a.nq, u[i] + j);
      }
#pragma unroll
      for (int i = 0; i < DEEP; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] += s + i * SL < a.splits ? u[i][j] : 0.0f;
    }
    if constexpr (SL > 1) {
      if (sl) {
#pragma unroll
        for (int j = 0; j < V; ++j) red[sl - 1][cl][j] = v[j];
      }
      __syncthreads();
      if (sl == 0) {
#pragma unroll
        for (int k = 0; k < SL - 1; ++k)
#pragma unroll
          for (int j = 0; j < V; ++j) v[j] += red[k][cl][j];
      }
      __syncthreads();
      if (sl) continue;
    }
    if (!live) continue;
    if (a.bias) {
      sf_load_chunk<T>(static_cast<const T *>(a.bias), col, a.nq, u[0]);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] += u[0][j];
    }
    if (a.pre) sf_store_chunk<T>(static_cast<T *>(a.pre) + at, col, a.nq, v);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = sf_act<T>(v[j], a.act);
    if (a.residual) {
      sf_load_chunk<T>(static_cast<const T *>(a.residual) + at, col, a.nq, u[0]);
#pragma unroll
      for (int j = 0; j < V; ++j) v[j] += u[0][j];
    }
    sf_store_chunk<T>(static_cast<T *>(a.out) + at, col, a.nq, v);
  }
}

// Eight lanes a chunk where there are many splits of few outputs: 64 x 256 outputs in 127 parts 9.1 us,
// with one lane a chunk 72.
template <typename T>
static void sf_gemm_join(const SfGemmArgs &a, hipStream_t st) {
  const long long cpr = (a.nq + 16 / (int)sizeof(T) - 1) / (16 / (int)sizeof(T)), chunks = a.np * cpr;
  if (a.splits >= 8 && chunks < 65536)
    hipLaunchKernelGGL((sf_gemm_join_kernel<T, 8>), dim3(sf_grid(chunks, 32)), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((sf_gemm_join_kernel<T, 1>), dim3(sf_grid(chunks, 256)), dim3(256), 0, st, a);
}

// The launches of one storage type (linear_f32.hip, linear_f16.hip, linear_bf16.hip).
// layout 0: P, Q K-major; 1: Q K-minor; 2: both K-minor.  tile 32, 64, 128 or 256, operands whose rows
// start at multiples of 4 bytes; layout 0 only: SF_FEW_ROWS, any operands.
#define SF_FEW_ROWS 16
int sf_gemm_f32(const SfGemmArgs &a, int layout, int tile, hipStream_t st);
int sf_gemm_f16(const SfGemmArgs &a, int layout, int tile, hipStream_t st);
int sf_gemm_bf16(const SfGemmArgs &a, int layout, int tile, hipStream_t st);
// Both gradients' products, 32 x 32 tiles, and the bias gradient's sum.
struct SfColumnSums;
int sf_gradients_f32(const SfGemmArgs &dx, const SfGemmArgs &dw, const SfColumnSums &db, hipStream_t st);
int sf_gradients_f16(const SfGemmArgs &dx, const SfGemmArgs &dw, const SfColumnSums &db, hipStream_t st);
int sf_gradients_bf16(const SfGemmArgs &dx, const SfGemmArgs &dw, const SfColumnSums &db, hipStream_t st);

// A tiny layer's gradients without a pass ahead; dx, dw or db may be NULL.  direct: rows of all tensors
// start at multiples of 4 bytes.
struct SfGradients {
  const void *dy, *pre, *x, *w;
  void *dx, *dw, *db;
  long long ldx, m, k, n;
  int act;
};
int sf_tiny_gradients_f32(const SfGradients &g, bool direct, hipStream_t st);
int sf_tiny_gradients_f16(const SfGradients &g, bool direct, hipStream_t st);
int sf_tiny_gradients_bf16(const SfGradients &g, bool direct, hipStream_t st);

// ---- small products -------------------------------------------------------------------------------
// Too few 64 x 64 tiles to fill the chip leave each CU with one workgroup that walks a long contraction
// alone.  Here a workgroup owns 32 x 32 outputs and its four waves share each step's 128 bytes of k, 32
// each, so a step takes a quarter of the products' time; a ring of eight buffers keeps seven steps in
// flight.  The waves' sums meet in LDS.  In us, 64 x 64 tiles against these: 200 x 128 -> 256 fp32 5.9 and
// 4.3, 400 x 1024 -> 256 bf16 7.8 and 5.6 (fp32 23 and 10), 1000 x 512 -> 512 fp32 14 and 10.3; twice the
// operand bytes per output loses once the chip is full (2000 x 512 -> 512 fp32 15.0 and 19.6).
struct SfSmall {
  static constexpr int B = 32, STEP = 128, RING = 8, BYTES = 2 * B * STEP, LDS = RING * BYTES;
};

// The sum of the four waves' blocks (in 16 KB of LDS that nobody uses any more): four columns of a row
// for each thread, row threadIdx.x / 8, columns from 4 (threadIdx.x % 8) on.
__device__ __forceinline__ void sf_add_shares(const sf_f32x16 &acc, unsigned char *lds, float *v) {
  // lane (row = lane % 32, h = lane / 32) holds columns 8 g + 4 h + 0..3: the waves' blocks behind each
  // other, quads swizzled by the row
  float *part = reinterpret_cast<float *>(lds);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 31, h = lane >> 5;
#pragma unroll
  for (int g = 0; g < 4; ++g)
    *reinterpret_cast<sf_f32x4 *>(part + wave * 1024 + row * 32 + (((2 * g + h) ^ row ^ (row >> 3)) & 7) * 4) =
        (sf_f32x4){acc[4 * g], acc[4 * g + 1], acc[4 * g + 2], acc[4 * g + 3]};
  __syncthreads();
  const int r = threadIdx.x >> 3, quad = threadIdx.x & 7;
#pragma unroll
  for (int j = 0; j < 4; ++j) v[j] = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const sf_f32x4 f =
        *reinterpret_cast<const sf_f32x4 *>(part + w * 1024 + r * 32 + ((quad ^ r ^ (r >> 3)) & 7) * 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] += f[j];
  }
}

template <typename T, bool PMINOR, bool QMINOR>
__device__ __forceinline__ void sf_small(const SfGemmArgs &a, unsigned char *lds, int group) {
  constexpr int B = SfSmall::B, STEP = SfSmall::STEP, RING = SfSmall::RING, BYTES = SfSmall::BYTES;
  constexpr int V = 16 / sizeof(T), BK = STEP / (int)sizeof(T);
  typedef SfOperand<T, PMINOR, B, 4, STEP> OP;
  typedef SfOperand<T, QMINOR, B, 4, STEP> OQ;
  typedef typename SfMfma<T>::frag frag;
  constexpr int NI = OP::NI + OQ::NI;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
#if defined(__HIP_DEVICE_COMPILE__)
  const unsigned lds0 = (unsigned)(unsigned long long)(__attribute__((address_space(3))) unsigned char *)lds;
#else
  const unsigned lds0 = 0;
#endif
  const int split = group / (a.tiles_p * a.tiles_q), tile = group - split * (a.tiles_p * a.tiles_q);
  const long long p0 = (long long)(tile / a.tiles_q) * B, q0 = (long long)(tile % a.tiles_q) * B;
  const long long k0 = split * a.k_split;
  const int steps = sf_steps<BK>(a, split);
  const long long left = a.nk - k0 - (long long)(steps - 1) * BK;
  const int last_k = left < BK ? (int)left : BK;
  OP op;
  OQ oq;
  op.init(a.ldp, wave, lane);
  oq.init(a.ldq, wave, lane);
  op.open(a.p, p0, a.np, k0, steps, last_k);
  oq.open(a.q, q0, a.nq, k0, steps, last_k);
  auto load = [&](int buf) {      // behind the last step: loads of nothing, so that the counted waits hold
    sf_unroll<0, OP::NI>([&](auto j) { op.template issue<decltype(j)::value>(lds0 + buf + wave * 1024); });
    sf_unroll<0, OQ::NI>([&](auto j) {
      oq.template issue<decltype(j)::value>(lds0 + buf + B * STEP + wave * 1024);
    });
    op.next(), oq.next();
    if (op.steps == 0) op.close(), oq.close();
  };
#pragma unroll
  for (int i = 0; i + 1 < RING; ++i) load(i * BYTES);
  sf_f32x16 acc;
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] = 0.0f;
  int cur = 0, old = (RING - 1) * BYTES;
  for (int i = 0; i < steps; ++i) {
    asm volatile("" ::: "memory");
    sf_wait_loads<(RING - 2) * NI>();
    __builtin_amdgcn_s_barrier();      // step i has landed, everyone has read step i - 1
    asm volatile("" ::: "memory");
    if (a.tail && i + 1 == steps && last_k % V) {
      OP::clear(lds + cur, last_k);
      OQ::clear(lds + cur + B * STEP, last_k);
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    }
    const frag fp = OP::fragment(lds + cur, 0, wave, lane);
    const frag fq = OQ::fragment(lds + cur + B * STEP, 0, wave, lane);
    load(old);
    acc = SfMfma<T>::run(fq, fp, acc);
    old = cur;
    cur = cur + BYTES == RING * BYTES ? 0 : cur + BYTES;
  }
  sf_wait_loads<0>();
  __syncthreads();
  float v[4];
  sf_add_shares(acc, lds, v);
  const int r = threadIdx.x >> 3, quad = threadIdx.x & 7;      // 32 rows by 8 quads
  const long long prow = p0 + r, col = q0 + 4 * quad;
  if (prow < a.np) {
    const T *bias = static_cast<const T *>(a.bias), *res = static_cast<const T *>(a.residual);
    T *out = static_cast<T *>(a.out), *pre = static_cast<T *>(a.pre);
    const long long at = prow * a.nq + col;
    if (a.splits > 1) {
      if (col < a.nq) sf_store_chunk<float>(a.partial + ((long long)split * a.np + prow) * a.nq, col, a.nq, v);
      return;
    }
    float b[4], x[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {      // columns past the end read the last one's
      const long long c = col + j < a.nq ? j : a.nq - 1 - col;
      b[j] = bias ? (float)bias[col + c] : 0.0f;
      x[j] = res ? (float)res[at + c] : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (col + j < a.nq) {
        const float z = v[j] + b[j];
        if (pre) pre[at + j] = (T)z;
        out[at + j] = (T)(sf_act<T>(z, a.act) + x[j]);
      }
  }
}

template <typename T, bool PMINOR, bool QMINOR>
__global__ void __launch_bounds__(256) sf_small_kernel(SfGemmArgs a) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[SfSmall::LDS];
  sf_small<T, PMINOR, QMINOR>(a, lds, blockIdx.x);
}

template <typename T, bool PMINOR, bool QMINOR, typename SH>
static int sf_gemm_go(const SfGemmArgs &a, hipStream_t st) {
  static SfSlotCache cache;
  auto kern = sf_gemm_kernel<T, PMINOR, QMINOR, SH>;
  int slots = sf_resident_slots(cache, kern, SH::WAVES * 64, 0, SH::LDS);
  if (slots < 8) {
    sf_set_error("no occupancy for the matrix product kernel on this device");
    return SF_ERR_HIP;
  }
  slots &= ~7;
  const long long items = (long long)a.tiles_p * a.tiles_q * a.splits;
  hipLaunchKernelGGL(kern, dim3((unsigned)(items < slots ? items : slots)), dim3(SH::WAVES * 64), 0, st,
                     a);
  return SF_OK;
}

// 256 x 256: steps of 128 bytes bring whole lines (those of 64 ask the L2 for each line twice), but leave no
// registers for a residual fetched ahead.  bf16, 64 and 128 bytes: 32400 x 256 -> 1024 GELU 35.2 and
// 33.7 us, 259200 x 1024 -> 256 167 and 160, 16384 x 2048 -> 2048 123 and 117 (1170 TFLOP/s); with a
// residual 259200 x 1024 -> 256 takes 200 and 204, 32400 x 256 -> 1024 56 and 59.
typedef SfShape<256, 256, 2, 4, 64, 4, 1> SfTile256;
typedef SfShape<256, 256, 2, 4, 128, 2, 1, false> SfTile256Plain;
template <bool TAIL> using SfTile128 = SfShape<128, 128, 2, 2, 128, 2, 2, true, TAIL>;
// 64 x 64: deep enough to cover the latency of one workgroup alone (64 x 4096 -> 4096 bf16: 33 us with a
// ring of 2, 21 with 4); fp32's products cover it themselves, three workgroups level the CUs better
// (35344 x 512 -> 512: 164 us against 168).
template <typename T, bool TAIL>
using SfTile64 = SfShape<64, 64, 2, 2, 128, sizeof(T) == 4 ? 2 : 4, sizeof(T) == 4 ? 3 : 2, true, TAIL>;

template <typename T, bool PMINOR, bool QMINOR>
static int sf_gemm_launch(const SfGemmArgs &a, int tile, hipStream_t st) {
  int rc = SF_OK;
  if (tile == 32) {
    hipLaunchKernelGGL((sf_small_kernel<T, PMINOR, QMINOR>), dim3(a.tiles_p * a.tiles_q * a.splits), dim3(256),
                       0, st, a);
  } else if (tile == 256) {
    if constexpr (!PMINOR && !QMINOR)      // gradients have no residual
      if (a.residual && a.splits == 1) return sf_gemm_go<T, PMINOR, QMINOR, SfTile256>(a, st);
    rc = sf_gemm_go<T, PMINOR, QMINOR, SfTile256Plain>(a, st);
  } else if (PMINOR || !a.tail) {
    if (tile == 128) rc = sf_gemm_go<T, PMINOR, QMINOR, SfTile128<false>>(a, st);
    else rc = sf_gemm_go<T, PMINOR, QMINOR, SfTile64<T, false>>(a, st);
  } else if constexpr (!PMINOR) {
    if (tile == 128) rc = sf_gemm_go<T, PMINOR, QMINOR, SfTile128<true>>(a, st);
    else rc = sf_gemm_go<T, PMINOR, QMINOR, SfTile64<T, true>>(a, st);
  }
  if (rc) return rc;
  if (a.splits > 1) sf_gemm_join<T>(a, st);
  return SF_OK;
}

// ---- a small layer's gradients in one launch --------------------------------------------------------
// Sums of `runs` partial rows of n, 32 columns by TY strided runs of rows a workgroup of 32 TY.
struct SfColumnSums {
  const float *part;      // (runs, n)
  void *out;              // (n) of T, or NULL: nothing to do
  long long n;
  int runs;
};
template <typename T, int TY>
__device__ __forceinline__ void sf_join_columns(const SfColumnSums &c, int group, float *red) {
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const long long i = (long long)group * 32 + tx;
  float t = 0.0f;
  if (i < c.n) {
    for (int b0 = ty; b0 < c.runs; b0 += 16 * TY) {      // 16 loads in flight
      float u[16];
#pragma unroll
      for (int k = 0; k < 16; ++k) u[k] = b0 + TY * k < c.runs ? c.part[(b0 + TY * k) * c.n + i] : 0.0f;
#pragma unroll
      for (int k = 0; k < 16; ++k) t += u[k];
    }
  }
  red[ty * 33 + tx] = t;
  __syncthreads();
  if (ty == 0 && i < c.n) {
    float v = 0.0f;
#pragma unroll
    for (int k = 0; k < TY; ++k) v += red[k * 33 + tx];
    static_cast<T *>(c.out)[i] = (T)v;
  }
}

// dx = dz w, dw = dz^T x and db's last sum by different workgroups of one launch, the longest first:
// products of a few tiles each are all latency.  400 x 256 -> 128 with the pass for dz in front: fp32
// 10.0 us, bf16 10.3 (64 x 64 tiles in one launch 16.9, one product behind the other 21);
// 1000 x 512 -> 512 bf16 17.9 (26).
template <typename T>
__global__ void __launch_bounds__(256)
sf_gradients_kernel(SfGemmArgs dx, int dx_groups, SfGemmArgs dw, int dw_groups, SfColumnSums db) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[SfSmall::LDS];
  const int g = blockIdx.x;
  if (g < dw_groups) sf_small<T, true, true>(dw, lds, g);
  else if (g < dx_groups + dw_groups) sf_small<T, false, true>(dx, lds, g - dw_groups);
  else sf_join_columns<T, 8>(db, g - dx_groups - dw_groups, reinterpret_cast<float *>(lds));
}

template <typename T>
static int sf_gradients_go(const SfGemmArgs &dx, const SfGemmArgs &dw, const SfColumnSums &db, hipStream_t st) {
  const int nx = dx.tiles_p * dx.tiles_q, nw = dw.tiles_p * dw.tiles_q;
  const int nb = db.out ? (int)((db.n + 31) / 32) : 0;
  hipLaunchKernelGGL((sf_gradients_kernel<T>), dim3(nx + nw + nb), dim3(256), 0, st, dx, nx, dw, nw, db);
  return SF_OK;
}

// ---- a tiny layer's gradients in one launch, straight from dy ---------------------------------------
// Chunk of row `row` (of n) at element i0 (of nk), zeros outside.
template <typename T>
__device__ __forceinline__ typename SfMfma<T>::frag sf_row_chunk(const T *p, long long ld, long long row,
                                                                 long long n, long long i0, long long nk) {
  constexpr int V = 16 / sizeof(T);
  typename SfMfma<T>::frag e = {};
  if (row < n) {
    const T *at = p + row * ld + i0;
    if (i0 + V <= nk) {
      e = __builtin_bit_cast(typename SfMfma<T>::frag, *reinterpret_cast<const sf_u32x4_any *>(at));
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j)
        if (i0 + j < nk) e[j] = at[j];
    }
  }
  return e;
}

// The 32 x 32 outputs of which four waves hold a share each: added up and stored.
template <typename T>
__device__ __forceinline__ void sf_store_shared(const sf_f32x16 &acc, unsigned char *lds, T *out, long long p0,
                                                long long np, long long q0, long long nq) {
  float v[4];
  sf_add_shares(acc, lds, v);
  const long long row = p0 + (threadIdx.x >> 3), col = q0 + 4 * (threadIdx.x & 7);
  if (row >= np) return;
#pragma unroll
  for (int j = 0; j < 4; ++j)
    if (col + j < nq) out[row * nq + col + j] = (T)v[j];
}

// dx = dz w, dw = dz^T x and db = sum dz of a tiny layer by different workgroups of one launch, the
// longest first.  dz = dy act'(pre) is made where it is used, on the way from registers into LDS, so there
// is no pass ahead and nothing to copy: loads need no alignment, and what is outside reads as zeros.
// 32 x 32 tiles, a step's 128 bytes of k shared by the four waves, DEEP steps' loads in flight.  Bound by
// the step: 0.4 us in fp32, in GELU's slope 0.5 (16 bits 0.7), one wave a SIMD.  400 x 256 -> 128 fp32 ReLU
// 8.3 us, 200 x 256 -> 256 bf16 GELU 5.7; with a pass for dz ahead 10.2 and 9.8, and a launch more.
template <typename T, bool DW, bool DIRECT>
__device__ __forceinline__ void sf_tiny_gradient(const SfGradients &g, unsigned char *lds, int group) {
  constexpr int B = 32, STEP = 128, V = 16 / sizeof(T), BK = STEP / (int)sizeof(T), DEEP = 4;
  typedef SfOperand<T, DW, B, 4, STEP> OP;
  typedef SfOperand<T, true, B, 4, STEP> OQ;
  typedef typename SfMfma<T>::frag frag;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const T *dy = static_cast<const T *>(g.dy), *pre = static_cast<const T *>(g.pre);
  const T *q = static_cast<const T *>(DW ? g.x : g.w);
  const long long np = DW ? g.n : g.m, nk = DW ? g.m : g.n, ldq = DW ? g.ldx : g.k;
  const int tiles_q = (int)((g.k + B - 1) / B), steps = (int)((nk + BK - 1) / BK);
  const long long p0 = (long long)(group / tiles_q) * B, q0 = (long long)(group % tiles_q) * B;
  // this thread's chunk of a step of each operand: its place in LDS is 16 threadIdx.x
  const int prow = wave * OP::RPI + lane / OP::CPR, pc = ((lane % OP::CPR) ^ OP::swz(prow)) * V;
  const int qrow = wave * OQ::RPI + lane / OQ::CPR, qc = ((lane % OQ::CPR) ^ OQ::swz(qrow)) * V;
  frag ry[DEEP], rz[DEEP], rq[DEEP];
  // chunk (row0 + r, col0 + c) of a tensor of rows x cols, row0 and col0 the same for the workgroup
  auto fetch = [&](const T *t, long long ld, long long rows, long long cols, long long row0, int r,
                   long long col0, int c) -> frag {
    if constexpr (DIRECT) {      // no branches: the buffer's range check makes the zeros
      const long long left = ((rows - 1) * ld + cols - row0 * ld - col0) * (long long)sizeof(T);
      const auto rs = __builtin_amdgcn_make_buffer_rsrc(
          const_cast<T *>(t + row0 * ld + col0), 0,
          row0 >= rows || left < 0 ? 0 : left < 0x7FFFFFF0 ? ((int)left + 3) & ~3 : 0x7FFFFFF0, 0x00020000);
      const unsigned off = (unsigned)((r * ld + c) * (long long)sizeof(T));
      return __builtin_bit_cast(frag, __builtin_amdgcn_raw_buffer_load_b128(rs, col0 + c < cols ? off : 0x80000000u, 0, 0));
    } else {
      return sf_row_chunk<T>(t, ld, row0 + r, col0 + c < cols ? rows : 0, col0 + c, cols);
    }
  };
  auto load = [&](auto slot, int step) {
    constexpr int D = decltype(slot)::value;
    const long long k0 = (long long)step * BK, row0 = DW ? k0 : p0, col0 = DW ? p0 : k0;
    ry[D] = fetch(dy, g.n, g.m, g.n, row0, prow, col0, pc);
    if (g.act != SF_ACT_NONE) rz[D] = fetch(pre, g.n, g.m, g.n, row0, prow, col0, pc);
    rq[D] = fetch(q, ldq, nk, g.k, k0, qrow, q0, qc);
  };
  auto put = [&](auto slot, int step, unsigned char *buf) {
    constexpr int D = decltype(slot)::value;
    frag e = ry[D];
    if (g.act == SF_ACT_GELU) {
#pragma unroll
      for (int j = 0; j < V; ++j) e[j] = (T)sf_act_gradient<T>((float)e[j], (float)rz[D][j], SF_ACT_GELU);
    } else if (g.act == SF_ACT_RELU) {
#pragma unroll
      for (int j = 0; j < V; ++j) e[j] = (T)sf_act_gradient<T>((float)e[j], (float)rz[D][j], SF_ACT_RELU);
    }
    if constexpr (!DW && DIRECT)
      if (g.n % V) {      // a chunk that dy's row end cuts brings the next row's first values
#pragma unroll
        for (int j = 0; j < V; ++j) e[j] = (long long)step * BK + pc + j < g.n ? e[j] : (T)0.0f;
      }
    *reinterpret_cast<frag *>(buf + 16 * threadIdx.x) = e;
    *reinterpret_cast<frag *>(buf + B * STEP + 16 * threadIdx.x) = rq[D];
  };
  sf_f32x16 acc;
#pragma unroll
  for (int e = 0; e < 16; ++e) acc[e] = 0.0f;
  sf_unroll<0, DEEP>([&](auto d) { load(d, decltype(d)::value); });
  for (int i0 = 0; i0 < steps; i0 += DEEP)
    sf_unroll<0, DEEP>([&](auto d) {
      const int i = i0 + decltype(d)::value;
      if (i >= steps) return;
      unsigned char *buf = lds + (decltype(d)::value & 1) * (2 * B * STEP);      // DEEP is even
      put(d, i, buf);
      load(d, i + DEEP);
      // LDS only: the loads stay in flight.  The buffer of step i - 1 is free behind this barrier
      asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      const frag fp = OP::fragment(buf, 0, wave, lane);
      const frag fq = OQ::fragment(buf + B * STEP, 0, wave, lane);
      acc = SfMfma<T>::run(fq, fp, acc);
    });
  __syncthreads();
  sf_store_shared<T>(acc, lds, static_cast<T *>(DW ? g.dw : g.dx), p0, np, q0, g.k);
}

// db of 32 columns: the sums of the fp32 products, not of the rounded dz.
template <typename T>
__device__ __forceinline__ void sf_tiny_db(const SfGradients &g, float *red, int group) {
  constexpr int V = 16 / sizeof(T), CL = 32 / V, RL = 256 / CL, DEEP = 4;
  typedef typename SfMfma<T>::frag frag;
  const T *dy = static_cast<const T *>(g.dy), *pre = static_cast<const T *>(g.pre);
  const int cl = threadIdx.x % CL, rl = threadIdx.x / CL;
  const long long col = (long long)group * 32 + cl * V;
  float sum[V];
#pragma unroll
  for (int j = 0; j < V; ++j) sum[j] = 0.0f;
  for (long long r = rl; r < g.m; r += RL * DEEP) {
    frag e[DEEP], z[DEEP] = {};
#pragma unroll
    for (int i = 0; i < DEEP; ++i) {
      e[i] = sf_row_chunk<T>(dy, g.n, r + i * RL, col < g.n ? g.m : 0, col, g.n);
      if (g.act != SF_ACT_NONE) z[i] = sf_row_chunk<T>(pre, g.n, r + i * RL, col < g.n ? g.m : 0, col, g.n);
    }
    auto add = [&](auto act) {      // one branch a turn: with one an element they run one behind the other
#pragma unroll
      for (int i = 0; i < DEEP; ++i)
#pragma unroll
        for (int j = 0; j < V; ++j)
          sum[j] += sf_act_gradient<T>((float)e[i][j], (float)z[i][j], decltype(act)::value);
    };
    if (g.act == SF_ACT_GELU) add(SfInt<SF_ACT_GELU>());
    else if (g.act == SF_ACT_RELU) add(SfInt<SF_ACT_RELU>());
    else add(SfInt<SF_ACT_NONE>());
  }
#pragma unroll
  for (int j = 0; j < V; ++j) red[rl * 33 + cl * V + j] = sum[j];
  __syncthreads();
  if (threadIdx.x < 32 && group * 32 + threadIdx.x < g.n) {
    float t = 0.0f;
    for (int i = 0; i < RL; ++i) t += red[i * 33 + threadIdx.x];
    static_cast<T *>(g.db)[group * 32 + threadIdx.x] = (T)t;
  }
}

template <typename T, bool DIRECT>
__global__ void __launch_bounds__(256) sf_tiny_gradients_kernel(SfGradients g, int dw_groups, int dx_groups) {
  __shared__ __attribute__((aligned(1024))) unsigned char lds[4 * 32 * 128];
  const int b = blockIdx.x;
  if (b < dw_groups) sf_tiny_gradient<T, true, DIRECT>(g, lds, b);
  else if (b < dw_groups + dx_groups) sf_tiny_gradient<T, false, DIRECT>(g, lds, b - dw_groups);
  else sf_tiny_db<T>(g, reinterpret_cast<float *>(lds), b - dw_groups - dx_groups);
}

template <typename T>
static int sf_tiny_gradients_go(const SfGradients &g, bool direct, hipStream_t st) {
  const long long tq = (g.k + 31) / 32;
  const int nw = g.dw ? (int)((g.n + 31) / 32 * tq) : 0, nx = g.dx ? (int)((g.m + 31) / 32 * tq) : 0;
  const int nb = g.db ? (int)((g.n + 31) / 32) : 0;
  if (!(nw + nx + nb)) return SF_OK;
  auto kern = direct ? sf_tiny_gradients_kernel<T, true> : sf_tiny_gradients_kernel<T, false>;
  hipLaunchKernelGGL(kern, dim3(nw + nx + nb), dim3(256), 0, st, g, nw, nx);
  return SF_OK;
}

// ---- few rows -------------------------------------------------------------------------------------
// y of up to 16 rows: bound by the weight's bytes and by latency, so there is no tile in LDS and no
// pipeline.  A workgroup owns 16 columns; its 8 waves share the contraction in turns of 4 x 64 bytes of k
// and each loads its operands' fragments straight from memory, all in flight at once (lane = row % 16,
// 16-byte chunk lane / 16: a row's 64 bytes are one line's half).  The waves' sums meet in LDS.
template <typename T> struct SfMfma16;
template <> struct SfMfma16<float> {
  static __device__ __forceinline__ sf_f32x4 run(SfMfma<float>::frag a, SfMfma<float>::frag b, sf_f32x4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
};
template <> struct SfMfma16<_Float16> {
  static __device__ __forceinline__ sf_f32x4 run(SfMfma<_Float16>::frag a, SfMfma<_Float16>::frag b,
                                                 sf_f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};
template <> struct SfMfma16<__bf16> {
  static __device__ __forceinline__ sf_f32x4 run(SfMfma<__bf16>::frag a, SfMfma<__bf16>::frag b,
                                                 sf_f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};

template <typename T>
__global__ void __launch_bounds__(512) sf_few_rows_kernel(SfGemmArgs a) {
  constexpr int V = 16 / sizeof(T), WAVES = 8, UNROLL = 4;
  __shared__ float part[WAVES][64][4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 15, c = lane >> 4;
  const long long q0 = (long long)blockIdx.x * 16;
  const T *p = static_cast<const T *>(a.p), *q = static_cast<const T *>(a.q);
  sf_f32x4 acc = {0.f, 0.f, 0.f, 0.f};
  constexpr int K = 4 * V;      // k of 64 bytes
  for (long long k0 = wave * K; k0 < a.nk; k0 += UNROLL * WAVES * K) {
    typename SfMfma<T>::frag fq[UNROLL], fp[UNROLL];
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) {
      const long long k = k0 + i * WAVES * K + c * V;
      fq[i] = sf_row_chunk<T>(q, a.ldq, q0 + row, k < a.nk ? a.nq : 0, k, a.nk);
      fp[i] = sf_row_chunk<T>(p, a.ldp, row, k < a.nk ? a.np : 0, k, a.nk);
    }
#pragma unroll
    for (int i = 0; i < UNROLL; ++i) acc = SfMfma16<T>::run(fq[i], fp[i], acc);
  }
  // accumulator: row p = lane % 16, columns q = 4 (lane / 16) + 0..3
  *reinterpret_cast<sf_f32x4 *>(part[wave][lane]) = acc;
  __syncthreads();
  if (wave) return;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int w = 0; w < WAVES; ++w)
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] += part[w][lane][j];
  if (row >= a.np) return;
  const T *bias = static_cast<const T *>(a.bias), *res = static_cast<const T *>(a.residual);
  T *out = static_cast<T *>(a.out), *pre = static_cast<T *>(a.pre);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const long long col = q0 + 4 * c + j, at = row * a.nq + col;
    if (col >= a.nq) break;
    float z = v[j] + (bias ? (float)bias[col] : 0.0f);
    if (pre) pre[at] = (T)z;
    z = sf_act<T>(z, a.act);
    out[at] = (T)(z + (res ? (float)res[at] : 0.0f));
  }
}

template <typename T>
static int sf_few_rows(const SfGemmArgs &a, hipStream_t st) {
  hipLaunchKernelGGL((sf_few_rows_kernel<T>), dim3((unsigned)((a.nq + 15) / 16)), dim3(512), 0, st, a);
  return SF_OK;
}

template <typename T>
static int sf_gemm_any(const SfGemmArgs &a, int layout, int tile, hipStream_t st) {
  if (tile == SF_FEW_ROWS) return sf_few_rows<T>(a, st);
  if (layout == 0) return sf_gemm_launch<T, false, false>(a, tile, st);
  if (layout == 1) return sf_gemm_launch<T, false, true>(a, tile, st);
  return sf_gemm_launch<T, true, true>(a, tile, st);
}
