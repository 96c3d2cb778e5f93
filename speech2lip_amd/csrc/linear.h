// A dense layer of any size with its epilogue, and its gradients:
//
//   z = x W^T + b     y = act(z) + residual                          x [rows, in], W [out, in], y [rows, out]
//   dz = dy * act'(z)     dx = dz W     dW = dz^T x     db = sum over rows of dz     (d residual = dy)
//
// in fp32 (fp32 MFMA), bf16 or f16 (16-bit MFMA), all sums in fp32, one rounding at each store.  What is kept between the passes: for the
// kinked activations one BIT per element, the exact sign of the fp32 z (so that the gradient's side of the kink never depends on how z would
// round), for the smooth ones z in the call's own type (its relative rounding, 2^-8 / 2^-11 at most, moves act' by |z act''| < 0.35
// times that: a third of the rounding of a gradient of that size).
//
// Operands whose rows are whole 16-byte pieces come to LDS by the DMA path (dma_kernel; dx and dW in one launch, both_kernel); all others through
// registers (tile_kernel), which the following describes.  An operand whose contraction index is contiguous in memory (KC: x and W of the forward, dz of
// dx) lies in LDS as [row][128 bytes of k] with its 16-byte pieces XOR-swizzled by the row; one whose contraction index is the row (W of dx,
// both operands of dW) lies as it comes, [k][columns], and is transposed on the way out of LDS (the 16-bit types by the transposing LDS
// read, fp32 by 4-byte reads).  Global memory is read as 16-byte pieces at element alignment into registers one k-tile ahead, so odd widths
// and row strides take the same path; only tiles at an edge check bounds.  The bit gate of a kinked activation is applied between register
// and LDS, which saves the pass that would write dz.  v_mfma_f32_32x32x* throughout, with the operands swapped so that a lane holds four
// consecutive columns of ONE output row.
#pragma once
#include "tile_core.h"

namespace s2l {
namespace lin {

using core::f16v;
using core::mma;
using core::u4;

constexpr int kThreads = 256;
constexpr int kBkBytes = 128;               // bytes of contraction per LDS row and k-tile: 64 16-bit values or 32 floats
constexpr int kSkinnyRows = 8;              // up to this many rows the forward is one pass over W (skinny_kernel)

struct Args {
  const void* a;        // KC: [m][k]; else [k][m]
  const void* b;        // KC: [n][k]; else [k][n]
  const uint8_t* gate;  // sign bits of z, laid over operand a's memory layout: byte (row * gate_ld + column / 8)
  int64_t lda, ldb, gate_ld;
  int64_t m, n, k;
  int64_t k_per_split;  // multiple of the k-tile; grid.y splits
  float slope;          // gate: factor where the bit is 0
  // epilogue
  const void* bias;
  const void* residual;
  void* out;
  uint8_t* bits;        // forward: sign bits out, row stride ceil(n/8)
  void* zsave;          // forward: z out, row stride n
  float* partial;       // != NULL: [split][m][n] fp32 instead of the epilogue
  float* colsum;        // wgrad: [split][m] sums of operand a over k (the bias gradient), written by the first column of tiles
  int64_t ldr, ldo;
  int act;
};

template <typename T> struct Traits;
template <> struct Traits<float> { static constexpr int kChunk = 4; };
template <> struct Traits<_Float16> { static constexpr int kChunk = 8; };
template <> struct Traits<__bf16> { static constexpr int kChunk = 8; };

template <typename T> __device__ __forceinline__ T from_f(float v) { return (T)v; }

// 16 bytes at element alignment: the target's unaligned global access makes this one load
template <typename T> __device__ __forceinline__ u4 load16(const T* p) { u4 v; __builtin_memcpy(&v, p, 16); return v; }

// the first `count` (< a piece) elements, the rest zero
template <typename T> __device__ __forceinline__ u4 load_some(const T* p, int count) {
  union { u4 v; T e[Traits<T>::kChunk]; } r;
  r.v = u4{0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < Traits<T>::kChunk; ++i)
    if (i < count) r.e[i] = p[i];
  return r.v;
}

// Phi(z) = erfc(-z / sqrt 2) / 2, the normal distribution function, and density's exponential exp(-z^2 / 2).  By erfc, which keeps the tail's
// significant bits (1 + erf rounds to steps of 2^-24 there, which is all of Phi below -5.4).  fp32: the library's.  16-bit types: erfc(x) =
// t (c1 + t (c2 + ... t c6)) exp(-x^2) with t = 1 / (1 + 0.413 x), the form of Abramowitz and Stegun 7.1.26 with coefficients fitted here (linear programming on
// x in 0 .. 9.5, the smaller of a relative and an absolute bound): half of it is off by at most 2e-7 and, down to z = -13, by at most 4.8e-5 of itself, a
// tenth of f16's rounding.  In a third of the instructions: 16384 x 1024 x 4096 bf16, a forward that keeps nothing, 160 us without an activation, 176 so
// (294 with the library's erf).
template <typename T> __device__ __forceinline__ float normal_cdf(float z, float* density) {
  if constexpr (std::is_same_v<T, float>) {
    *density = expf(-0.5f * z * z);
    return 0.5f * erfcf(z * -0.70710678118654752f);
  } else {
    const float x = fabsf(z) * 0.70710678118654752f;
    const float e = __builtin_amdgcn_exp2f(-1.4426950408889634f * x * x);
    const float t = __builtin_amdgcn_rcpf(fmaf(0.413f, x, 1.f));
    float q = fmaf(t, -0.17319834f, 0.54030871f);
    q = fmaf(t, q, -0.15108114f);
    q = fmaf(t, q, 0.34107009f);
    q = fmaf(t, q, 0.20799284f);
    q = fmaf(t, q, 0.23490781f) * t * e * 0.5f;      // half of erfc(x)
    *density = e;
    return z > 0.f ? 1.f - q : q;
  }
}
template <typename T> __device__ __forceinline__ float sigmoid(float z) {
  if constexpr (std::is_same_v<T, float>) return 1.f / (1.f + expf(-z));
  else return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * z));
}

// N values at once, one branch for all of them.  (gelu of -infinity: -inf * 0 is NaN, as the formula has it; of large finite z: exactly 0 or z)
template <typename T, int N> __device__ __forceinline__ void activate(float (&z)[N], int act, float slope) {
  if (act == S2L_ACT_RELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] = z[i] > 0.f ? z[i] : z[i] != z[i] ? z[i] : 0.f;
  } else if (act == S2L_ACT_LEAKY_RELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] = z[i] > 0.f ? z[i] : z[i] * slope;
  } else if (act == S2L_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float e;
      z[i] *= normal_cdf<T>(z[i], &e);
    }
  } else if (act == S2L_ACT_SILU) {
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] *= sigmoid<T>(z[i]);
  }
}

template <typename T> __device__ __forceinline__ float act_slope(float z, int act) {
  if (act == S2L_ACT_GELU) {
    float e;
    const float phi = normal_cdf<T>(z, &e);
    return fmaf(z * e, 0.39894228040143268f, phi);
  }
  const float s = sigmoid<T>(z);      // silu; z -> -inf: s = 0 and s (1 + z (1 - s)) = 0 for every finite z
  return s * (1.f + z * (1.f - s));
}

// ---- epilogue of one piece: eight consecutive columns (a byte of sign bits) of one row --------------------------------------------------
constexpr int kFinish = 8;
template <typename T> struct Eight { T e[kFinish]; };
template <typename T> __device__ __forceinline__ Eight<T> load8(const T* p, bool full, int count) {
  Eight<T> v;
  if (full) {
    __builtin_memcpy(&v, p, sizeof(v));
  } else {
#pragma unroll
    for (int i = 0; i < kFinish; ++i) v.e[i] = i < count ? p[i] : (T)0.f;
  }
  return v;
}
template <typename T> __device__ __forceinline__ void store8(T* p, const Eight<T>& v, bool full, int count) {
  if (full) {
    __builtin_memcpy(p, &v, sizeof(v));
  } else {
#pragma unroll
    for (int i = 0; i < kFinish; ++i)
      if (i < count) p[i] = v.e[i];
  }
}

// z as the backward pass reads it: a 16-bit type's largest value in place of an overflow (act' has long settled there, and no inf * 0 comes of it)
template <typename T> __device__ __forceinline__ T saved_z(float z) {
  if constexpr (std::is_same_v<T, _Float16>) z = z > 65504.f ? 65504.f : z < -65504.f ? -65504.f : z;
  if constexpr (std::is_same_v<T, __bf16>) z = z > 3.3895313892515355e38f ? 3.3895313892515355e38f : z < -3.3895313892515355e38f ? -3.3895313892515355e38f : z;
  return from_f<T>(z);
}

// N pieces of a lane: everything that they read is requested before the first is used (one after the other they wait out a memory latency each:
// 36864 x 256 with a residual took 40 us where its bytes take 12).  row[i] < 0: nothing there.
template <typename T, int N> __device__ __forceinline__ void finish_pieces(const Args& g, const int64_t (&row)[N], const int64_t (&col)[N], float (&z)[N * kFinish],
                                                                           const Eight<T> (&res)[N]) {
  const T* bias = static_cast<const T*>(g.bias);
  int count[N];
#pragma unroll
  for (int p = 0; p < N; ++p) count[p] = row[p] < 0 ? 0 : col[p] + kFinish <= g.n ? kFinish : (int)(g.n - col[p]);
  if (bias) {
#pragma unroll
    for (int p = 0; p < N; ++p) {
      const Eight<T> b = load8(bias + col[p], count[p] == kFinish, count[p]);
#pragma unroll
      for (int i = 0; i < kFinish; ++i) z[p * kFinish + i] += (float)b.e[i];
    }
  }
  if (g.bits) {      // the side of the kink, from the fp32 z
#pragma unroll
    for (int p = 0; p < N; ++p) {
      uint32_t m = 0;
#pragma unroll
      for (int i = 0; i < kFinish; ++i) m |= z[p * kFinish + i] > 0.f ? 1u << i : 0u;
      if (count[p]) g.bits[row[p] * ((g.n + 7) >> 3) + (col[p] >> 3)] = (uint8_t)m;
    }
  }
  if (g.zsave) {
#pragma unroll
    for (int p = 0; p < N; ++p) {
      Eight<T> s;
#pragma unroll
      for (int i = 0; i < kFinish; ++i) s.e[i] = saved_z<T>(z[p * kFinish + i]);
      store8(static_cast<T*>(g.zsave) + row[p] * g.n + col[p], s, count[p] == kFinish, count[p]);
    }
  }
  activate<T>(z, g.act, g.slope);
#pragma unroll
  for (int p = 0; p < N; ++p) {
    Eight<T> o;
    if (g.residual) {
#pragma unroll
      for (int i = 0; i < kFinish; ++i) z[p * kFinish + i] += (float)res[p].e[i];
    }
#pragma unroll
    for (int i = 0; i < kFinish; ++i) o.e[i] = from_f<T>(z[p * kFinish + i]);
    store8(static_cast<T*>(g.out) + row[p] * g.ldo + col[p], o, count[p] == kFinish, count[p]);
  }
}
template <typename T> __device__ __forceinline__ Eight<T> residual_at(const Args& g, int64_t row, int64_t col) {
  const bool full = col + kFinish <= g.n;
  return load8(static_cast<const T*>(g.residual) + row * g.ldr + col, full, full ? kFinish : (int)(g.n - col));
}

// ---- one operand's k-tile: global -> registers -> LDS, laid out as core::Tile ------------------------------------------------------------
template <typename T, int ROWS, bool KC, bool GATE> struct Operand {
  using L = core::Tile<T, ROWS, KC, kBkBytes>;
  static constexpr int C = Traits<T>::kChunk;
  static constexpr int BK = L::BK;
  static constexpr int kPieces = ROWS * 8 / kThreads;                     // per thread
  static constexpr int kRowPieces = KC ? 8 : ROWS / C;                    // pieces per LDS row
  static constexpr int kBytes = L::kBytes;
  u4 r[kPieces];
  uint32_t gate[GATE ? kPieces : 1];

  // base: the operand; row0 / k0: origin of the tile; rows / k_end: ends
  __device__ __forceinline__ void load(const T* base, int64_t ld, int64_t row0, int64_t k0, int64_t rows, int64_t k_end, const uint8_t* gates,
                                       int64_t gate_ld) {
    const int64_t line0 = KC ? row0 : k0, col0 = KC ? k0 : row0;
    const int64_t lines = KC ? rows : k_end, cols = KC ? k_end : rows;
    constexpr int kLines = KC ? ROWS : BK;
    const bool inside = line0 + kLines <= lines && col0 + kRowPieces * C <= cols;      // uniform: the whole tile
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int p = threadIdx.x + i * kThreads;
      const int64_t line = line0 + p / kRowPieces, col = col0 + (p % kRowPieces) * C;
      if (inside) {
        r[i] = load16(base + line * ld + col);
        if constexpr (GATE) gate[i] = gates[line * gate_ld + (col >> 3)];
      } else {
        r[i] = u4{0, 0, 0, 0};
        if constexpr (GATE) gate[i] = 0;
        if (line < lines && col < cols) {
          r[i] = col + C <= cols ? load16(base + line * ld + col) : load_some(base + line * ld + col, (int)(cols - col));
          if constexpr (GATE) gate[i] = gates[line * gate_ld + (col >> 3)];
        }
      }
      if constexpr (GATE && C == 4) gate[i] >>= (col & 4);
    }
  }

  __device__ __forceinline__ void commit(char* lds, float slope) {
#pragma unroll
    for (int i = 0; i < kPieces; ++i) {
      const int p = threadIdx.x + i * kThreads;
      u4 v = r[i];
      if constexpr (GATE) {
        union { u4 v; T e[C]; } x;
        x.v = v;
#pragma unroll
        for (int j = 0; j < C; ++j)
          if (!((gate[i] >> j) & 1)) x.e[j] = slope == 0.f ? (T)0.f : from_f<T>((float)x.e[j] * slope);
        v = x.v;
      }
      *reinterpret_cast<u4*>(lds + L::place(p / kRowPieces, p % kRowPieces)) = v;
    }
  }

};

template <typename T> __device__ __forceinline__ u4 ones16() {
  union { u4 v; T e[Traits<T>::kChunk]; } x;
#pragma unroll
  for (int i = 0; i < Traits<T>::kChunk; ++i) x.e[i] = (T)1.f;
  return x.v;
}

// ---- the waves' results, FM x FN blocks of 32 x 32, through LDS in fp32, 32 rows at a time, so that a lane finishes whole pieces of a row and
// neighbouring lanes neighbouring pieces.  rbase / cbase: the wave's first row and column; scratch: 32 * (32 FN + 4) floats of its own.
template <typename T, int FM, int FN> __device__ __forceinline__ void finish(const Args& g, f16v (&acc)[FM][FN], int64_t rbase, int64_t cbase, float* scratch, int lane, int split) {
  constexpr int W = 32 * FN, kLd = W + 4, kPieces = W / kFinish / 2;
#pragma unroll
  for (int i = 0; i < FM; ++i) {
    int64_t row[kPieces], col[kPieces];
    Eight<T> res[kPieces];
#pragma unroll
    for (int p = 0; p < kPieces; ++p) {
      row[p] = rbase + 32 * i + (lane + 64 * p) / (W / kFinish);
      col[p] = cbase + lane % (W / kFinish) * kFinish;
      if (row[p] >= g.m || col[p] >= g.n) row[p] = -1;
      if (g.residual && !g.partial && row[p] >= 0) res[p] = residual_at<T>(g, row[p], col[p]);
    }
#pragma unroll
    for (int j = 0; j < FN; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<f4*>(scratch + (lane & 31) * kLd + 32 * j + 8 * q + 4 * (lane >> 5)) =
            f4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (g.partial) {
      constexpr int kPer = W / 4;
      float* out = g.partial + (int64_t)split * g.m * g.n;
#pragma unroll
      for (int p = lane; p < 32 * kPer; p += 64) {
        const int64_t row = rbase + 32 * i + p / kPer, col = cbase + (p % kPer) * 4;
        const f4 v = *reinterpret_cast<const f4*>(scratch + (p / kPer) * kLd + (p % kPer) * 4);
        if (row < g.m && col < g.n) {
          if (col + 4 <= g.n) __builtin_memcpy(out + row * g.n + col, &v, 16);
          else {
#pragma unroll
            for (int e = 0; e < 3; ++e)
              if (col + e < g.n) out[row * g.n + col + e] = v[e];
          }
        }
      }
    } else {
      constexpr int kPer = W / kFinish, N = 32 * kPer / 64;
      float z[N * kFinish];
#pragma unroll
      for (int p = 0; p < N; ++p) {
        const float* src = scratch + ((lane + 64 * p) / kPer) * kLd + (lane % kPer) * kFinish;
        *reinterpret_cast<f4*>(z + p * kFinish) = *reinterpret_cast<const f4*>(src);
        *reinterpret_cast<f4*>(z + p * kFinish + 4) = *reinterpret_cast<const f4*>(src + 4);
      }
      finish_pieces<T, N>(g, row, col, z, res);
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// dbias: the sums over k of operand a's rows, from products with ones (accs: 32 x 32 blocks of equal columns)
template <int FM> __device__ __forceinline__ void put_sums(const Args& g, const f16v (&accs)[FM], int64_t rbase, int lane, int split) {
  if (lane < 32) {
#pragma unroll
    for (int i = 0; i < FM; ++i) {
      const int64_t row = rbase + 32 * i + lane;
      if (row < g.m) g.colsum[split * g.m + row] = accs[i][0];
    }
  }
}

// TILE x TILE outputs per workgroup, four waves of TILE/2 x TILE/2.
template <typename T, int TILE, bool AKC, bool BKC, bool GATE>
__global__ __launch_bounds__(kThreads, 2) void tile_kernel(Args g) {
  constexpr int W = TILE / 2, F = W / 32;
  using OpA = Operand<T, TILE, AKC, GATE>;
  using OpB = Operand<T, TILE, BKC, false>;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int64_t tiles_n = (g.n + TILE - 1) / TILE;
  const int64_t tile = core::xcd_order(blockIdx.x, gridDim.x);
  const int64_t m0 = tile / tiles_n * TILE, n0 = tile % tiles_n * TILE;
  const int64_t k_begin = (int64_t)blockIdx.y * g.k_per_split;
  const int64_t k_end = k_begin + g.k_per_split < g.k ? k_begin + g.k_per_split : g.k;
  const int wm = (wave >> 1) * W, wn = (wave & 1) * W;
  const bool sums = g.colsum != nullptr && n0 == 0 && wn == 0;

  f16v acc[F][F], accs[F];
#pragma unroll
  for (int i = 0; i < F; ++i) {
#pragma unroll
    for (int r = 0; r < 16; ++r) accs[i][r] = 0.f;
#pragma unroll
    for (int j = 0; j < F; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  }

  OpA oa;
  OpB ob;
  const T* a = static_cast<const T*>(g.a);
  const T* b = static_cast<const T*>(g.b);
  if (k_begin < k_end) {
    oa.load(a, g.lda, m0, k_begin, g.m, k_end, g.gate, g.gate_ld);
    ob.load(b, g.ldb, n0, k_begin, g.n, k_end, nullptr, 0);
  }
  int buf = 0;
  for (int64_t k0 = k_begin; k0 < k_end; k0 += OpA::BK) {
    char* la = smem + buf * (OpA::kBytes + OpB::kBytes);
    char* lb = la + OpA::kBytes;
    oa.commit(la, g.slope);
    ob.commit(lb, 0.f);
    __syncthreads();      // the other buffer's readers passed this barrier before they can be overtaken: one barrier per k-tile
    if (k0 + OpA::BK < k_end) {
      oa.load(a, g.lda, m0, k0 + OpA::BK, g.m, k_end, g.gate, g.gate_ld);
      ob.load(b, g.ldb, n0, k0 + OpA::BK, g.n, k_end, nullptr, 0);
    }
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      u4 fa[F], fb[F];
#pragma unroll
      for (int i = 0; i < F; ++i) fa[i] = OpA::L::fragment(la, wm + 32 * i, s, lane);
#pragma unroll
      for (int j = 0; j < F; ++j) fb[j] = OpB::L::fragment(lb, wn + 32 * j, s, lane);
#pragma unroll
      for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j) acc[i][j] = mma<T>(fb[j], fa[i], acc[i][j]);
      if (!AKC && sums)
#pragma unroll
        for (int i = 0; i < F; ++i) accs[i] = mma<T>(ones16<T>(), fa[i], accs[i]);
    }
    buf ^= 1;
  }

  if (!AKC && sums) put_sums(g, accs, m0 + wm, lane, blockIdx.y);
  __syncthreads();      // the k-tiles are dead: LDS is the waves' own scratch from here
  finish<T, F, F>(g, acc, m0 + wm, n0 + wn, reinterpret_cast<float*>(smem) + wave * 32 * (W + 4), lane, blockIdx.y);
}

// The same product where everything is a multiple of the pieces (rule: dense_pieces below): operands by LDS-DMA, several k-tiles ahead.
// BM x BN outputs, WAVES_M x WAVES_N waves.
template <typename T, int BM, int BN, int WAVES_M, int WAVES_N, bool AKC, bool BKC, int STAGES>
__device__ __forceinline__ void dma_tile(const Args& g, int block, int blocks, int split, char* smem) {
  using P = core::Product<T, BM, BN, WAVES_M, WAVES_N, 1, AKC, BKC, kBkBytes, STAGES>;
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int tiles_n = (int)((g.n + BN - 1) / BN);
  const int tile = core::xcd_order(block, blocks);
  const int64_t m0 = (int64_t)(tile / tiles_n) * BM, n0 = (int64_t)(tile % tiles_n) * BN;
  const int64_t k_begin = (int64_t)split * g.k_per_split;
  const int64_t k_end = k_begin + g.k_per_split < g.k ? k_begin + g.k_per_split : g.k;
  const int wm = wave / WAVES_N * P::WM, wn = wave % WAVES_N * P::WN;
  const bool sums = g.colsum != nullptr && n0 == 0 && wn == 0;
  f16v acc[P::FM][P::FN], accs[P::FM];
#pragma unroll
  for (int i = 0; i < P::FM; ++i) {
#pragma unroll
    for (int r = 0; r < 16; ++r) accs[i][r] = 0.f;
#pragma unroll
    for (int j = 0; j < P::FN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  }
  typename P::SA sa;
  typename P::SB sb;
  sa.setup(static_cast<const T*>(g.a), g.lda, m0, g.m, k_begin, wave, lane);
  sb.setup(static_cast<const T*>(g.b), g.ldb, n0, g.n, k_begin, wave, lane);
  P::run(sa, sb, (int)((k_end - k_begin) / P::BK), smem, acc, wave, lane, [&](auto& fa) {
    if (!AKC && sums)
#pragma unroll
      for (int i = 0; i < P::FM; ++i) accs[i] = mma<T>(ones16<T>(), fa[0][i], accs[i]);
  });
  if (!AKC && sums) put_sums(g, accs, m0 + wm, lane, split);
  finish<T, P::FM, P::FN>(g, acc, m0 + wm, n0 + wn, reinterpret_cast<float*>(smem) + wave * 32 * (P::WN + 4), lane, split);
}

template <typename T, int BM, int BN, int WAVES_M, int WAVES_N, bool AKC, bool BKC, int STAGES>
__global__ __launch_bounds__(64 * WAVES_M * WAVES_N, 2) void dma_kernel(Args g) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  dma_tile<T, BM, BN, WAVES_M, WAVES_N, AKC, BKC, STAGES>(g, blockIdx.x, gridDim.x, blockIdx.y, smem);
}

// dx and dW in one launch, dW's workgroups (the longer contraction) first: a launch less, and neither waits for the other's last workgroups.
constexpr int stages_of(int tile) { return tile == 64 ? 3 : 2; }
template <typename T, int DX, int DW> __global__ __launch_bounds__(kThreads, 2) void both_kernel(Args dx, Args dw, int dw_tiles, int dw_blocks) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int id = blockIdx.x;
  if (id < dw_blocks) dma_tile<T, DW, DW, 2, 2, false, false, stages_of(DW)>(dw, id % dw_tiles, dw_tiles, id / dw_tiles, smem);
  else {
    const int blocks = gridDim.x - dw_blocks;
    dma_tile<T, DX, DX, 2, 2, true, false, stages_of(DX)>(dx, id - dw_blocks, blocks, 0, smem);
  }
}

// ---- the splits of a long contraction joined, in a fixed order: out = finish(sum over s of partial[s]) -----------------------------------
// 64 pieces per workgroup, the splits dealt to its four waves and joined through LDS.
template <typename T> __global__ __launch_bounds__(kThreads) void join_kernel(Args g, int splits, int blocks, int sums, const float* colsum, T* dbias) {
  constexpr int C = kFinish;
  __shared__ float part[4][64][C + 1];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if ((int)blockIdx.x >= blocks) {      // behind the pieces: the bias gradient, sixteen columns to a workgroup
    float* rows = &part[0][0][0];
    const int column = threadIdx.x & 15, first = threadIdx.x >> 4;
    const int64_t i = (int64_t)(blockIdx.x - blocks) * 16 + column;
    float v = 0.f;
    if (i < g.m) {
#pragma unroll 8
      for (int s = first; s < sums; s += 16) v += colsum[(int64_t)s * g.m + i];
    }
    rows[first * 17 + column] = v;
    __syncthreads();
    if (threadIdx.x < 16 && i < g.m) {
      v = 0.f;
#pragma unroll
      for (int s = 0; s < 16; ++s) v += rows[s * 17 + column];
      dbias[i] = from_f<T>(v);
    }
    return;
  }
  const int64_t per = (g.n + C - 1) / C, id = (int64_t)blockIdx.x * 64 + lane;
  const int64_t row = id / per, col = id % per * C;
  float v[C];
#pragma unroll
  for (int e = 0; e < C; ++e) v[e] = 0.f;
  const bool live = row < g.m, full = col + C <= g.n;
  if (live) {
    const float* src = g.partial + row * g.n + col;
    if (full) {
#pragma unroll 4
      for (int s = wave; s < splits; s += 4) {
        float t[C];
        __builtin_memcpy(t, src + (int64_t)s * g.m * g.n, sizeof(t));
#pragma unroll
        for (int e = 0; e < C; ++e) v[e] += t[e];
      }
    } else {
      for (int s = wave; s < splits; s += 4)
#pragma unroll
        for (int e = 0; e < C; ++e)
          if (col + e < g.n) v[e] += src[(int64_t)s * g.m * g.n + e];
    }
  }
#pragma unroll
  for (int e = 0; e < C; ++e) part[wave][lane][e] = v[e];
  __syncthreads();
  if (wave == 0 && live) {
#pragma unroll
    for (int e = 0; e < C; ++e) v[e] = (part[0][lane][e] + part[1][lane][e]) + (part[2][lane][e] + part[3][lane][e]);
    const int64_t rows[1] = {row}, cols[1] = {col};
    Eight<T> res[1];
    if (g.residual) res[0] = residual_at<T>(g, row, col);
    finish_pieces<T, 1>(g, rows, cols, v, res);
  }
}

// ---- few rows: one pass over W, a wave per output column, the contraction over its lanes -------------------------------------------------
template <typename T, int R> __global__ __launch_bounds__(kThreads) void skinny_kernel(Args g) {
  constexpr int C = Traits<T>::kChunk;
  const int lane = threadIdx.x & 63;
  const int64_t col = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (col >= g.n) return;
  const T* x = static_cast<const T*>(g.a);
  const T* w = static_cast<const T*>(g.b) + col * g.ldb;
  float acc[R];
#pragma unroll
  for (int r = 0; r < R; ++r) acc[r] = 0.f;
  union P { u4 v; T e[C]; };
#pragma unroll 2
  for (int64_t k = lane * C; k < g.k; k += 64 * C) {
    const bool full = k + C <= g.k;
    const int count = full ? C : (int)(g.k - k);
    P pw, px;
    pw.v = full ? load16(w + k) : load_some(w + k, count);
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (r < g.m) {
        px.v = full ? load16(x + r * g.lda + k) : load_some(x + r * g.lda + k, count);
#pragma unroll
        for (int e = 0; e < C; ++e) acc[r] = fmaf((float)px.e[e], (float)pw.e[e], acc[r]);
      }
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r)
#pragma unroll
    for (int d = 32; d; d >>= 1) acc[r] += __shfl_xor(acc[r], d);
  // lane r finishes row r
  float z = acc[0];
#pragma unroll
  for (int r = 1; r < R; ++r) z = lane == r ? acc[r] : z;
  if (lane < g.m) {
    const T* bias = static_cast<const T*>(g.bias);
    const T* res = static_cast<const T*>(g.residual);
    if (bias) z += (float)bias[col];
    float y[1] = {z};
    activate<T>(y, g.act, g.slope);
    if (g.zsave) static_cast<T*>(g.zsave)[lane * g.n + col] = saved_z<T>(z);
    if (res) y[0] += (float)res[lane * g.ldr + col];
    static_cast<T*>(g.out)[lane * g.ldo + col] = from_f<T>(y[0]);
  }
}

// dz = dy * act'(z) of the kinked activations, where both products then take the LDS-DMA path (which has no place for the gate); exact but for
// leaky_relu's factor.
template <typename T> __global__ __launch_bounds__(kThreads) void gate_kernel(const T* __restrict__ dy, int64_t lddy, const uint8_t* __restrict__ bits, T* __restrict__ dz,
                                                                               int64_t rows, int64_t n, float slope) {
  const int64_t per = (n + kFinish - 1) / kFinish, id = (int64_t)blockIdx.x * kThreads + threadIdx.x;
  const int64_t row = id / per, col = id % per * kFinish;
  if (row >= rows) return;
  const bool full = col + kFinish <= n;
  const int count = full ? kFinish : (int)(n - col);
  Eight<T> a = load8(dy + row * lddy + col, full, count);
  const uint32_t m = bits[row * per + (col >> 3)];
#pragma unroll
  for (int e = 0; e < kFinish; ++e)
    if (!((m >> e) & 1)) a.e[e] = slope == 0.f ? (T)0.f : from_f<T>((float)a.e[e] * slope);
  store8(dz + row * n + col, a, full, count);
}

// dz = dy * act'(z) of the smooth ones, rounded to the call's type: the products' matrix instructions take no other (2^-8 / 2^-11 relative at
// most; f16 below its smallest normal value, 2^-14, in steps of 2^-24, as any f16 gradient: a loss is scaled so that its gradients lie above).  The bias gradient's sums are taken here, from the values before that rounding: its terms cancel as the result's do, so that their
// roundings would show in it as large as its own (bf16 2.3e-3 of the gradient's norm against 1.7e-3, which is its own rounding).  Memory bound with
// gelu's arithmetic beside it: 16384 x 4096 bf16 122 us, 97 without the sums.  A workgroup: `groups` pieces of eight columns (a power of two, up to
// 32) by 256 / groups rows, `times` times; all workgroups move down the matrix together (each on rows of its own: 130 us).  colsum: [workgroup row][n].
template <typename T, int ACT> __global__ __launch_bounds__(kThreads) void slope_kernel(const T* __restrict__ dy, int64_t lddy, const T* __restrict__ z, T* __restrict__ dz,
                                                                                int64_t rows, int64_t n, int groups, int times, int columns, float* __restrict__ colsum) {
  __shared__ float part[kThreads][kFinish + 1];
  const int lanes = kThreads / groups, lane = threadIdx.x / groups, group = threadIdx.x % groups;
  const int by = blockIdx.x / columns, bx = blockIdx.x - by * columns;
  const int64_t col = ((int64_t)bx * groups + group) * kFinish, row0 = (int64_t)by * lanes + lane, stride = (int64_t)(gridDim.x / columns) * lanes;
  const bool full = col + kFinish <= n;
  const int count = full ? kFinish : (int)(n - col);
  float sum[kFinish];
#pragma unroll
  for (int e = 0; e < kFinish; ++e) sum[e] = 0.f;
  if (count > 0) {
    for (int t = 0; t < times; t += 4) {      // (rows of a step past `times` lie past the last one)
      Eight<T> a[4], v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int64_t row = row0 + (t + u) * stride;
        if (row < rows) {
          a[u] = load8(dy + row * lddy + col, full, count);
          v[u] = load8(z + row * n + col, full, count);
        }
      }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int64_t row = row0 + (t + u) * stride;
        if (row >= rows) break;
#pragma unroll
        for (int e = 0; e < kFinish; ++e) {
          const float d = (float)a[u].e[e] * act_slope<T>((float)v[u].e[e], ACT);
          sum[e] += d;
          a[u].e[e] = from_f<T>(d);
        }
        store8(dz + row * n + col, a[u], full, count);
      }
    }
  }
  if (!colsum) return;
#pragma unroll
  for (int e = 0; e < kFinish; ++e) part[threadIdx.x][e] = sum[e];
  __syncthreads();
  for (int i = threadIdx.x; i < groups * kFinish; i += kThreads) {
    const int64_t at = (int64_t)bx * groups * kFinish + i;
    if (at >= n) break;
    float v = 0.f;
    for (int k = 0; k < lanes; ++k) v += part[k * groups + i / kFinish][i % kFinish];
    colsum[(int64_t)by * n + at] = v;
  }
}

// ---- host --------------------------------------------------------------------------------------------------------------------------------

constexpr int64_t kMaxDim = (int64_t)1 << 31;
inline bool too_many(int64_t blocks, int threads = kThreads) { return blocks * threads >= (int64_t)1 << 32; }      // a launch counts its threads in 32 bits
inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct Plan {
  int tile;        // 256 (LDS-DMA only; else 128), 128 or 64
  int splits;
  int64_t k_per_split;
};

// The workgroups of a product of [m, k] and [k, n]: 128-wide tiles where they alone give every CU one and the contraction is long enough to be
// bound by LDS, or four (short contractions are bound by memory, which more and smaller workgroups keep busier: 36864 x 256 x 256 with a
// residual 25 us against 35), else 64-wide ones; where that is still too few the contraction is split, down to four k-tiles a split.  The CU
// count is the part's (256): a plan must not depend on the device that is current when the workspace is sized.  wide: 256-wide tiles are there
// (not for dW, whose sums for dbias and two transposed operands do not leave the registers for them).
inline Plan plan_of(int64_t m, int64_t n, int64_t k, int size, bool wide = true) {
  constexpr int64_t kCus = 256;
  const int64_t bk = kBkBytes / size, k_tiles = ceil_div(k, bk);
  const auto count = [&](int64_t t) { return ceil_div(m, t) * ceil_div(n, t); };
  Plan p;
  p.tile = wide && size == 2 && count(256) >= kCus ? 256 : count(128) >= 4 * kCus || (count(128) >= kCus && k_tiles >= 16) ? 128 : 64;
  if (p.tile == 64 && count(64) < kCus && k_tiles >= 64 && m >= 128 && n >= 128) p.tile = 128;      // long contraction: wide tiles, split
  const int64_t tiles = count(p.tile);
  const int64_t want = p.tile == 128 && k_tiles >= 128 ? 2 * kCus : kCus;      // two 128-wide ones to a CU hide each other's barriers
  int64_t s = tiles == 0 || tiles >= want ? 1 : ceil_div(want, tiles);      // (no rows: no tiles)
  if (s > k_tiles / 4) s = k_tiles / 4;
  if (s < 1) s = 1;
  p.k_per_split = ceil_div(k_tiles, s) * bk;
  if (p.k_per_split == 0) p.k_per_split = bk;
  p.splits = (int)(k ? ceil_div(k, p.k_per_split) : 1);
  return p;
}

// Whether both operands' k-tiles are whole 16-byte pieces at their own alignment: what LDS-DMA moves.
inline bool dense_pieces(const Args& g, bool akc, bool bkc, int size) {
  const int64_t c = 16 / size, bk = kBkBytes / size;
  const auto fine = [&](const void* p, int64_t ld, bool kc, int64_t rows) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % c == 0 && (kc || rows % c == 0) && ld * size < (1 << 23);      // 256 rows: 32-bit offsets
  };
  return g.k > 0 && g.k % bk == 0 && !g.gate && fine(g.a, g.lda, akc, g.m) && fine(g.b, g.ldb, bkc, g.n);
}

inline int64_t align256(int64_t b) { return (b + 255) & ~(int64_t)255; }
inline int64_t partial_bytes(const Plan& p, int64_t m, int64_t n) { return p.splits > 1 ? align256((int64_t)p.splits * m * n * 4) : 0; }

template <typename T, int TILE, bool AKC, bool BKC, bool GATE> int launch_tile(const Args& g, const Plan& p, hipStream_t st) {
  constexpr int kStage = 2 * TILE * kBkBytes;
  constexpr int kScratch = 4 * 32 * (TILE / 2 + 4) * 4;
  constexpr int kLds = 2 * kStage > kScratch ? 2 * kStage : kScratch;
  static_assert(kLds <= 65536, "above 64 KiB the launch needs an opt-in");
  const int64_t tiles = ceil_div(g.m, TILE) * ceil_div(g.n, TILE);
  if (too_many(tiles)) return S2L_E_SIZE;
  hipLaunchKernelGGL((tile_kernel<T, TILE, AKC, BKC, GATE>), dim3((unsigned)tiles, (unsigned)p.splits), dim3(kThreads), kLds, st, g);
  return (int)hipGetLastError();
}

template <typename T, int BM, int BN, int WAVES_M, int WAVES_N, bool AKC, bool BKC, int STAGES> int launch_dma(const Args& g, const Plan& p, hipStream_t st) {
  using P = core::Product<T, BM, BN, WAVES_M, WAVES_N, 1, AKC, BKC, kBkBytes, STAGES>;
  constexpr int kScratch = P::kWaves * 32 * (P::WN + 4) * 4;
  constexpr int lds = P::kLds > kScratch ? P::kLds : kScratch;
  const auto kernel = dma_kernel<T, BM, BN, WAVES_M, WAVES_N, AKC, BKC, STAGES>;
  if constexpr (lds > 65536) {
    static LdsOptIn opted;
    int dev, cus;
    int rc = current_device_cus(&dev, &cus);
    if (rc) return rc;
    rc = ensure_dynamic_lds(reinterpret_cast<const void*>(kernel), lds, opted, dev);
    if (rc) return rc;
  }
  const int64_t tiles = ceil_div(g.m, BM) * ceil_div(g.n, BN);
  if (too_many(tiles, P::kThreads)) return S2L_E_SIZE;
  hipLaunchKernelGGL(kernel, dim3((unsigned)tiles, (unsigned)p.splits), dim3(P::kThreads), lds, st, g);
  return (int)hipGetLastError();
}

// after a product: its splits' partial sums joined, and the bias gradient's
struct Sums {
  void* dbias;
  int rows;           // of its partial sums
  float* partial;
};
template <typename T> int joined(int rc, const Args& g, const Plan& p, Sums sums, hipStream_t st) {
  if (rc || (p.splits == 1 && !sums.dbias)) return rc;
  const int64_t blocks = p.splits == 1 ? 0 : ceil_div(g.m * ceil_div(g.n, kFinish), 64), more = sums.dbias ? ceil_div(g.m, 16) : 0;
  if (too_many(blocks + more)) return S2L_E_SIZE;
  hipLaunchKernelGGL((join_kernel<T>), dim3((unsigned)(blocks + more)), dim3(kThreads), 0, st, g, p.splits, (int)blocks, sums.rows, sums.partial, static_cast<T*>(sums.dbias));
  return (int)hipGetLastError();
}

// the kernel of a product alone
struct Route {
  bool dma;
  int tile;
};
inline Route route_of(const Args& g, const Plan& p, bool akc, bool bkc, int size) {
  const bool dma = dense_pieces(g, akc, bkc, size);
  return Route{dma, p.tile == 256 && !dma ? 128 : p.tile};
}

template <typename T, bool AKC, bool BKC> int product(Args g, const Plan& p, float* partial, hipStream_t st, Sums sums = {}) {
  g.k_per_split = p.k_per_split;
  g.partial = p.splits > 1 ? partial : nullptr;
  int rc;
  const Route r = route_of(g, p, AKC, BKC, sizeof(T));
  if (r.dma) {
    if (r.tile == 64) return joined<T>(launch_dma<T, 64, 64, 2, 2, AKC, BKC, stages_of(64)>(g, p, st), g, p, sums, st);
    if constexpr (sizeof(T) == 2 && AKC)
      if (r.tile == 256) return joined<T>(launch_dma<T, 256, 256, 2, 4, AKC, BKC, 2>(g, p, st), g, p, sums, st);
    return joined<T>(launch_dma<T, 128, 128, 2, 2, AKC, BKC, stages_of(128)>(g, p, st), g, p, sums, st);
  }
  if (r.tile == 128) {
    if constexpr (AKC && BKC) rc = launch_tile<T, 128, AKC, BKC, false>(g, p, st);
    else rc = g.gate ? launch_tile<T, 128, AKC, BKC, true>(g, p, st) : launch_tile<T, 128, AKC, BKC, false>(g, p, st);
  } else {
    if constexpr (AKC && BKC) rc = launch_tile<T, 64, AKC, BKC, false>(g, p, st);
    else rc = g.gate ? launch_tile<T, 64, AKC, BKC, true>(g, p, st) : launch_tile<T, 64, AKC, BKC, false>(g, p, st);
  }
  return joined<T>(rc, g, p, sums, st);
}

template <typename T, int DX, int DW> int launch_both(const Args& dx, const Args& dw, const Plan& pw, hipStream_t st) {
  using PX = core::Product<T, DX, DX, 2, 2, 1, true, false, kBkBytes, stages_of(DX)>;
  using PW = core::Product<T, DW, DW, 2, 2, 1, false, false, kBkBytes, stages_of(DW)>;
  constexpr int lds = PX::kLds > PW::kLds ? PX::kLds : PW::kLds;
  static_assert(lds <= 65536 && lds >= 4 * 32 * (DX / 2 + 4) * 4 && lds >= 4 * 32 * (DW / 2 + 4) * 4, "");
  const int64_t x = ceil_div(dx.m, DX) * ceil_div(dx.n, DX), w = ceil_div(dw.m, DW) * ceil_div(dw.n, DW);
  if (too_many(x + w * pw.splits)) return S2L_E_SIZE;
  hipLaunchKernelGGL((both_kernel<T, DX, DW>), dim3((unsigned)(x + w * pw.splits)), dim3(kThreads), lds, st, dx, dw, (int)w, (int)(w * pw.splits));
  return (int)hipGetLastError();
}

// few rows, unless sign bits are wanted: a lane there has one column, a byte of them is eight
inline bool skinny(int64_t rows, bool bits) { return rows <= kSkinnyRows && !bits; }

template <typename T> int forward(Args g, float* work, hipStream_t st) {
  if (skinny(g.m, g.bits != nullptr)) {
    if (too_many(ceil_div(g.n, 4))) return S2L_E_SIZE;
    const dim3 grid((unsigned)ceil_div(g.n, 4));
    if (g.m == 1) hipLaunchKernelGGL((skinny_kernel<T, 1>), grid, dim3(kThreads), 0, st, g);
    else if (g.m <= 4) hipLaunchKernelGGL((skinny_kernel<T, 4>), grid, dim3(kThreads), 0, st, g);
    else hipLaunchKernelGGL((skinny_kernel<T, 8>), grid, dim3(kThreads), 0, st, g);
    return (int)hipGetLastError();
  }
  return product<T, true, true>(g, plan_of(g.m, g.n, g.k, sizeof(T)), work, st);
}

// slope_kernel's grid: one row a thread, more of them (up to 32) while two workgroups to a CU remain: 4096 x 256 fp32 13 us with 64 workgroups,
// 7 with 512
struct Slope {
  int groups, times, sums;      // sums: workgroup rows
};
inline Slope slope_plan(int64_t rows, int64_t n) {
  Slope s{1, 1, 0};
  while (s.groups < 32 && s.groups * kFinish < n) s.groups *= 2;
  const int64_t columns = ceil_div(n, (int64_t)s.groups * kFinish), lanes = kThreads / s.groups;
  while (s.times < 32 && ceil_div(rows, 2 * s.times * lanes) * columns >= 512) s.times *= 2;
  s.sums = rows ? (int)ceil_div(rows, s.times * lanes) : 1;
  return s;
}

struct Back {      // the workspace of the backward pass
  Plan dx, dw;
  Slope slope;
  int64_t dz, partial, colsum, total;      // bytes; the partials of dx and of dW take turns
};

inline Back back_plan(int64_t rows, int64_t in, int64_t out, int size, int act) {
  Back b;
  b.dx = plan_of(rows, in, out, size);
  b.dw = plan_of(out, in, rows, size, false);
  const int64_t bk = kBkBytes / size;
  const bool gated = act == S2L_ACT_RELU || act == S2L_ACT_LEAKY_RELU;      // (the rule goes by the sizes alone: the workspace's size does)
  const bool smooth = act == S2L_ACT_GELU || act == S2L_ACT_SILU;
  b.slope = slope_plan(rows, out);
  b.dz = smooth || (gated && rows % bk == 0 && out % bk == 0 && in % (16 / size) == 0) ? align256(rows * out * size) : 0;
  const int64_t p1 = partial_bytes(b.dx, rows, in), p2 = partial_bytes(b.dw, out, in);
  b.partial = p1 > p2 ? p1 : p2;
  b.colsum = align256((int64_t)(smooth ? b.slope.sums : b.dw.splits) * out * 4);
  b.total = b.dz + b.partial + b.colsum;
  return b;
}

// what the two products of the backward pass read and write, dz given
struct Products {
  Args dx, dw;
  bool together;      // one launch for both
};
inline Products products_of(const Back& b, const void* dz, int64_t lddz, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* saved, void* dx, int64_t lddx, void* dw,
                            float* colsum, int64_t rows, int64_t in, int64_t out, int size, int act, float slope) {
  const bool gated = (act == S2L_ACT_RELU || act == S2L_ACT_LEAKY_RELU) && !b.dz;
  Args g{};
  g.a = dz;
  g.lda = lddz;
  g.gate = gated ? static_cast<const uint8_t*>(saved) : nullptr;
  g.gate_ld = (out + 7) >> 3;
  g.slope = act == S2L_ACT_LEAKY_RELU ? slope : 0.f;
  g.act = S2L_ACT_NONE;
  Args d = g;      // dx = dz W
  d.b = w;
  d.ldb = ldw;
  d.m = rows;
  d.n = in;
  d.k = out;
  d.out = dx;
  d.ldo = lddx;
  Args e = g;      // dW = dz^T x
  e.b = x;
  e.ldb = ldx;
  e.m = out;
  e.n = in;
  e.k = rows;
  e.out = dw;
  e.ldo = in;
  e.colsum = colsum;
  return Products{d, e, dx && dw && b.dx.tile <= 128 && b.dx.splits == 1 && dense_pieces(d, true, false, size) && dense_pieces(e, false, false, size)};
}

template <typename T> int backward(const void* dy, int64_t lddy, const void* x, int64_t ldx, const void* w, int64_t ldw, const void* saved, void* dx, int64_t lddx,
                                   void* dw, void* db, char* work, int64_t rows, int64_t in, int64_t out, int act, float slope, hipStream_t st) {
  const Back b = back_plan(rows, in, out, sizeof(T), act);
  const void* dz = dy;
  int64_t lddz = lddy;
  float* sums = db ? reinterpret_cast<float*>(work + b.dz + b.partial) : nullptr;
  const bool summed = (act == S2L_ACT_GELU || act == S2L_ACT_SILU) && rows;      // by slope_kernel; else dW's product does it
  if (b.dz && rows) {
    if (act == S2L_ACT_GELU || act == S2L_ACT_SILU) {
      const int64_t columns = ceil_div(out, (int64_t)b.slope.groups * kFinish);
      if (too_many(columns * b.slope.sums)) return S2L_E_SIZE;
      const auto kernel = act == S2L_ACT_GELU ? slope_kernel<T, S2L_ACT_GELU> : slope_kernel<T, S2L_ACT_SILU>;
      hipLaunchKernelGGL(kernel, dim3((unsigned)(columns * b.slope.sums)), dim3(kThreads), 0, st, static_cast<const T*>(dy), lddy, static_cast<const T*>(saved),
                         reinterpret_cast<T*>(work), rows, out, b.slope.groups, b.slope.times, (int)columns, sums);
    } else {
      const int64_t blocks = ceil_div(rows * ceil_div(out, kFinish), kThreads);
      if (too_many(blocks)) return S2L_E_SIZE;
      hipLaunchKernelGGL((gate_kernel<T>), dim3((unsigned)blocks), dim3(kThreads), 0, st, static_cast<const T*>(dy), lddy, static_cast<const uint8_t*>(saved),
                         reinterpret_cast<T*>(work), rows, out, act == S2L_ACT_LEAKY_RELU ? slope : 0.f);
    }
    const int rc = (int)hipGetLastError();
    if (rc) return rc;
    dz = work;
    lddz = out;
  }
  float* partial = reinterpret_cast<float*>(work + b.dz);
  Products both = products_of(b, dz, lddz, x, ldx, w, ldw, saved, dx, lddx, dw, summed ? nullptr : sums, rows, in, out, sizeof(T), act, slope);
  Args &d = both.dx, &e = both.dw;
  if (both.together) {
    d.k_per_split = b.dx.k_per_split;
    e.k_per_split = b.dw.k_per_split;
    e.partial = b.dw.splits > 1 ? partial : nullptr;
    int rc;
    if (b.dx.tile == 64) rc = b.dw.tile == 64 ? launch_both<T, 64, 64>(d, e, b.dw, st) : launch_both<T, 64, 128>(d, e, b.dw, st);
    else rc = b.dw.tile == 64 ? launch_both<T, 128, 64>(d, e, b.dw, st) : launch_both<T, 128, 128>(d, e, b.dw, st);
    return joined<T>(rc, e, b.dw, Sums{db, summed ? b.slope.sums : b.dw.splits, sums}, st);
  }
  if (dx && rows) {
    const int rc = product<T, true, false>(d, b.dx, partial, st);
    if (rc) return rc;
  }
  if (dw) return product<T, false, false>(e, b.dw, partial, st, Sums{db, summed ? b.slope.sums : b.dw.splits, sums});
  return 0;
}

}  // namespace lin
}  // namespace s2l
