// Newton-Schulz orthogonalisation of a set of matrices, and the optimiser step that is built on it.
//
//   X0 = G / max(||G||_F, eps);   `steps` times:  A = X X^T,  B = a I + b A + c A A,  X <- B X      (X: the shorter side first)
//   Muon:  m <- m + (1 - mu) (g - m),  u = g + mu (m - g)  (or m),  p <- (1 - lr wd) p - lr_p X_steps(u)
//
// Every singular value s of X0 becomes p(p(...s)) with p(s) = a s + b s^3 + c s^5; with the usual (3.4445, -4.7750, 2.0315) and five steps all but
// the smallest end in 0.7 .. 1.2: U V^T but for that band.  p amplifies small singular values by a = 3.44 a step (485 over five), and with them
// whatever rounding put into their directions, so the products' precision goes by the STEP, not by the type alone: X, A and B are held as two
// IEEE halves (hi = f16(x), lo = f16(x - hi): 22 significant bits) and a product is three f16 MFMAs, hi hi + hi lo + lo hi, summed in fp32 --
// fp32's own accuracy at 2.7 times the fp32 MFMA's peak -- in every step for fp32 and f16 input, and in all but the last two steps for bf16 input,
// whose last two run on hi alone (their roundings of 2^-11 are amplified at most 12-fold and stay below the result's own 2^-8; one product in
// every step would leave 2-4 % of error on matrices of fast falling spectrum, and bf16 products 15-30 %).  Measured against 64 bits on 512 and
// 1024 square matrices (gradient-like; singular values 1 / i and 1 / i^2), relative: fp32 0.4 to 1.1 times the error of the same iteration in fp32
// products, f16 its own rounding, bf16 1.8e-3 to 2.2e-3 where its own rounding is 1.66e-3 (four 2048 x 2048 take 2.31 ms with halves in every step, 1.79 so).
// Values are scaled by 2^11: |X| <= ||X||_2 <= 1.2 and the entries of A and B <= 3.5 use the range of the halves from 2^-24 to 7168.
//
// All matrices of a call go through the same 2 + 3 * steps launches (one more a step where a long Gram product is cut along k): one pass for the
// Frobenius norms (with the momentum update), one that scales and splits into X^T, then per step the Gram product (symmetric: tiles on and below the diagonal, written twice), the polynomial (the same, its
// epilogue adds a I + b A), and X <- B X, which leaves X^T or, last, writes the result: the rounded output, or the parameter's update.  X is held
// transposed only: X <- B X reads it with k contiguous, the Gram product along its rows, through the transposing LDS read (X beside it cost
// twice the stores: four 2048 x 2048 206 against 186 us a product, and what a launch leaves in L2 is written back before the next one starts).
// Matrices lie zero-padded to multiples of 64 in the workspace, so that the products' main loop has no edges.
#include <cmath>

#include "tile_core.h"

namespace s2l {
namespace ns {

using core::f16v;
using core::u4;

constexpr int kPad = 64;
constexpr int kMaxMatrices = 56;            // of one set of launches: the table crosses as a kernel argument (below 4 KiB)
constexpr int kMaxPartials = 1024;          // partial sums of squares of a matrix
constexpr float kScale = 2048.f;
constexpr int kThreads = 256;

struct Mat {
  const void* in;       // [rows][cols] dense: the update, or (Muon) the gradient
  void* out;            // the result, or (Muon) the parameter
  float* momentum;      // Muon
  int64_t base;         // byte offset of this matrix's arrays in the workspace
  int rows, cols;
  float step;           // Muon: lr_p
  int stat;             // first partial sum of squares
};

enum { STAT = 0, PACK = 1, SYM = 2, RECT = 3, DEEP = 4, KINDS = 5 };      // the kinds of launches (DEEP: the Gram products where some are cut along k)

struct Table {
  int first[KINDS][kMaxMatrices];      // each matrix's first workgroup; 0x7fffffff behind the last matrix
  Mat mat[kMaxMatrices];
};
static_assert(sizeof(Table) <= 3840, "the table and a few scalars share the 4 KiB of kernel arguments");

__host__ __device__ inline int padded(int v) { return (v + kPad - 1) / kPad * kPad; }
__host__ __device__ inline int64_t tiles(int v, int tile) { return (padded(v) + tile - 1) / tile; }
__host__ __device__ inline int64_t elements_of(const Mat& t) { return (int64_t)t.rows * t.cols; }
__host__ __device__ inline int64_t chunk_of(int64_t elements) {      // elements of one workgroup of the first pass: a multiple of its 2048
  const int64_t c = (elements + kMaxPartials - 1) / kMaxPartials;
  return c <= 4096 ? 4096 : (c + 2047) / 2048 * 2048;
}

// the arrays of one matrix, in halves from its base: each has room for pairs (core::pair_at); in steps on hi alone it holds rows of those
struct Arrays {
  int m, n, mp, np;
  int64_t xt[2], a, b, total;
};
__host__ __device__ inline Arrays arrays_of(int rows, int cols) {
  Arrays r;
  r.m = rows < cols ? rows : cols;
  r.n = rows < cols ? cols : rows;
  r.mp = padded(r.m);
  r.np = padded(r.n);
  const int64_t mn = (int64_t)r.mp * r.np, mm = (int64_t)r.mp * r.mp;
  r.xt[0] = 0;
  r.xt[1] = 2 * mn;
  r.a = 4 * mn;
  r.b = r.a + 2 * mm;
  r.total = r.b + 2 * mm;
  return r;
}

constexpr int kWorthCutting = 1024;      // what a cut has to take off the longest workgroup's k: 20 us, against the join's 8
// A long Gram product (n >> m) is cut along k into pieces of about `chunk`, whose sums join_kernel adds: see chunk_for.  0: none is.
struct Pieces {
  int count, depth;      // depth of each but the last: a multiple of 64
};
__host__ __device__ inline Pieces pieces_of(int np, int chunk) {
  if (!chunk) return Pieces{1, np};
  int count = (np + chunk / 2) / chunk;
  count = count < 1 ? 1 : count > 16 ? 16 : count;
  const int depth = (np / 64 + count - 1) / count * 64;
  return np - depth < kWorthCutting ? Pieces{1, np} : Pieces{(np + depth - 1) / depth, depth};
}
__host__ __device__ inline int64_t sums_bytes(int count, int tiles) { return count > 1 ? (int64_t)count * tiles * 128 * 128 * 4 : 0; }

constexpr int64_t kTableBytes = 4096;
constexpr int64_t partial_bytes(int stat_blocks) { return ((int64_t)stat_blocks * 8 + 255) / 256 * 256; }

// which matrix workgroup `id` of a launch belongs to: every lane compares one first workgroup
__device__ __forceinline__ int owner(const int* first, int id) {
  const int lane = threadIdx.x & 63;
  const int mine = lane < kMaxMatrices ? first[lane] : 0x7fffffff;
  return __builtin_amdgcn_readfirstlane(__popcll(__ballot(mine <= id)) - 1);
}

// How a workgroup finds its matrix.  Each memory round trip of it is 0.45 us of launches of 3 .. 6 us where the matrices are small, so: matrices
// of one size, their inputs and outputs at equal distances (one matrix; a batch), from the kernel's arguments alone; others from a record per
// workgroup, which the first pass writes (one round trip; looking through the table took two).
struct Record {
  int64_t base;
  int rows, cols, index, id, piece, pad;
};
struct Alike {
  Mat mat;
  int per[KINDS];      // workgroups of one matrix; 0: not alike, look into the records
  int stride;          // bytes from one input / output to the next (at most 56 of them: below 2^31 checked)
  int64_t bytes;       // of one matrix's arrays
  int64_t records[3];  // byte offset of the records of SYM, RECT and DEEP launches in the workspace
};
struct Place {
  Mat mat;        // (in, out, momentum, step: where alike; else look at Table::mat[index] for them)
  int index;      // of the matrix
  int id;         // workgroup within the matrix (DEEP: within the piece)
  int piece;
};
__device__ __forceinline__ Place alike_place(const Alike& alike, int kind, int id) {
  const int k = id / alike.per[kind];
  Mat m = alike.mat;
  m.in = static_cast<const char*>(m.in) + (int64_t)k * alike.stride;
  m.out = static_cast<char*>(m.out) + (int64_t)k * alike.stride;
  m.base += k * alike.bytes;
  m.stat += k * alike.per[STAT];
  return Place{m, k, id - k * alike.per[kind], 0};
}
// What every workgroup of a product needs first: plain scalars at the front of the kernel's arguments, which the hardware puts into scalar registers
// with the wave (the build asks for 16 dwords of it), so that matrices alike need no load at all before their first operand request.
#define S2L_FRONT char *work, int per, int rows, int cols, int64_t base, int64_t bytes_or_records, int from, int parts_out, float coef_a, float coef_b, float coef_c, int blocks
#define S2L_FRONT_PASS work, per, rows, cols, base, bytes_or_records
__device__ __forceinline__ Place place_of(const char* work, int per, int rows, int cols, int64_t base, int64_t bytes_or_records, int id) {
  Place p{};
  if (per) {
    p.index = id / per;
    p.id = id - p.index * per;
    p.mat.rows = rows;
    p.mat.cols = cols;
    p.mat.base = base + p.index * bytes_or_records;
    return p;
  }
  const Record* rec = reinterpret_cast<const Record*>(work + bytes_or_records) + id;
  p.mat.base = core::uniform64(rec->base);
  p.mat.rows = __builtin_amdgcn_readfirstlane(rec->rows);
  p.mat.cols = __builtin_amdgcn_readfirstlane(rec->cols);
  p.index = __builtin_amdgcn_readfirstlane(rec->index);
  p.id = __builtin_amdgcn_readfirstlane(rec->id);
  p.piece = __builtin_amdgcn_readfirstlane(rec->piece);
  return p;
}
// a PACK launch's, from the table (once a call); a result's destination
__device__ __forceinline__ Place pack_place(const char* work, const Alike& alike, int id) {
  if (alike.per[0]) return alike_place(alike, PACK, id);
  const Table* t = reinterpret_cast<const Table*>(work);
  const int k = owner(t->first[PACK], id);
  return Place{t->mat[k], k, id - t->first[PACK][k], 0};
}
__device__ __forceinline__ void destination(const char* work, const Alike& alike, Place& p) {
  if (alike.per[0]) {
    p.mat.out = static_cast<char*>(alike.mat.out) + (int64_t)p.index * alike.stride;
    p.mat.step = alike.mat.step;
    return;
  }
  const Mat& m = reinterpret_cast<const Table*>(work)->mat[p.index];
  p.mat.out = core::uniform64(m.out);
  p.mat.step = m.step;
}

template <typename T> __device__ __forceinline__ void load8(const T* p, int64_t left, float* v) {
  if (left >= 8) {
    T t[8];
    __builtin_memcpy(t, p, sizeof(t));
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = (float)t[i];
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < left ? (float)p[i] : 0.f;
  }
}
__device__ __forceinline__ void store8f(float* p, int64_t left, const float* v) {
  if (left >= 8) {
    __builtin_memcpy(p, v, 32);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < left) p[i] = v[i];
  }
}

// the records' places in the workspace and their numbers: SYM, RECT, DEEP
struct Lists {
  int64_t at[3];
  int count[3];
};

struct Momentum {
  float mu;
  int nesterov;
};

// ---- first pass: the sums of squares in 64 bits (every later product scales with the norm: a sum over millions of squares in 32 bits is off by
// more than all other roundings together), with the momentum update.  Memory bound: reads g, reads and writes m.
template <typename T, bool MUON> __global__ __launch_bounds__(kThreads) void norm_kernel(Table t, char* work, Momentum mo, Lists lists) {
  __shared__ double part[4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (blockIdx.x == 0) {      // the table for the launches that follow
    const uint32_t* src = reinterpret_cast<const uint32_t*>(&t);
    for (int i = threadIdx.x; i < (int)(sizeof(Table) / 4); i += kThreads) reinterpret_cast<uint32_t*>(work)[i] = src[i];
  }
  // ... and the records (none where matrices are alike)
  const int syms = lists.count[0], rects = lists.count[1];
  for (int i = blockIdx.x * kThreads + threadIdx.x; i < syms + rects + lists.count[2]; i += gridDim.x * kThreads) {
    const int list = i < syms ? 0 : i < syms + rects ? 1 : 2, id = i - (list == 0 ? 0 : list == 1 ? syms : syms + rects);
    const int* first = list == 0 ? t.first[SYM] : list == 1 ? t.first[RECT] : t.first[DEEP];
    int k = 0;
    while (k + 1 < kMaxMatrices && first[k + 1] <= id) ++k;
    Record rec{t.mat[k].base, t.mat[k].rows, t.mat[k].cols, k, id - first[k], 0, 0};
    if (list == 2) {      // piece by piece: neighbours read the same rows
      const int side = (int)tiles(rec.rows < rec.cols ? rec.rows : rec.cols, 128), all = side * (side + 1) / 2;
      rec.piece = rec.id / all;
      rec.id -= rec.piece * all;
    }
    reinterpret_cast<Record*>(work + (list == 0 ? lists.at[0] : list == 1 ? lists.at[1] : lists.at[2]))[id] = rec;
  }
  const Mat& mat = t.mat[owner(t.first[STAT], blockIdx.x)];
  const int64_t total = elements_of(mat), chunk = chunk_of(total);
  const int64_t begin = (int64_t)(blockIdx.x - mat.stat) * chunk, end = begin + chunk < total ? begin + chunk : total;
  const T* g = static_cast<const T*>(mat.in);
  double sum = 0.0;
#pragma unroll 2
  for (int64_t i = begin + threadIdx.x * 8; i < end; i += kThreads * 8) {
    float v[8];
    load8(g + i, end - i, v);
    if constexpr (MUON) {
      float m[8];
      load8(mat.momentum + i, end - i, m);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        m[e] = fmaf(1.f - mo.mu, v[e] - m[e], m[e]);
        v[e] = mo.nesterov ? fmaf(mo.mu, m[e] - v[e], v[e]) : m[e];
      }
      store8f(mat.momentum + i, end - i, m);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) sum = fma((double)v[e], (double)v[e], sum);
  }
#pragma unroll
  for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
  if (lane == 0) part[wave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) reinterpret_cast<double*>(work + kTableBytes)[blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
}

__device__ __forceinline__ uint32_t halves(float v) {      // hi | lo << 16
  const _Float16 hi = (_Float16)v;
  const _Float16 lo = (_Float16)(v - (float)hi);
  return (uint32_t)__builtin_bit_cast(uint16_t, hi) | (uint32_t)__builtin_bit_cast(uint16_t, lo) << 16;
}

// eight neighbouring values (hi | lo << 16 each) to (row, col) of a matrix of `parts` halves
__device__ __forceinline__ void put8(_Float16* p, int64_t row, int64_t col, int64_t ld, int parts, const uint32_t* w) {
  _Float16* hi = p + (parts == 2 ? core::pair_at<2>(row, col, ld) : core::pair_at<1>(row, col, ld));
  u4 v;
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = (w[2 * e] & 0xffffu) | w[2 * e + 1] << 16;
  *reinterpret_cast<u4*>(hi) = v;
  if (parts == 2) {
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = w[2 * e] >> 16 | (w[2 * e + 1] & 0xffff0000u);
    *reinterpret_cast<u4*>(hi + core::kPairs) = v;
  }
}

// ---- second pass: X and X^T = 2^11 u / max(norm, eps), split into halves, zero-padded.  A workgroup: 64 x 64 of the padded matrix as it lies.
template <typename T, bool MUON> __global__ __launch_bounds__(kThreads) void split_kernel(char* work, Alike alike, Momentum mo, float eps, int parts) {
  __shared__ uint32_t tile[64][65];
  __shared__ double part[4];
  const Place at0 = pack_place(work, alike, blockIdx.x);
  const Mat& mat = at0.mat;
  const Arrays r = arrays_of(mat.rows, mat.cols);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const double* partial = reinterpret_cast<const double*>(work + kTableBytes) + mat.stat;
  const int64_t total = elements_of(mat), chunk = chunk_of(total);
  const int partials = (int)((total + chunk - 1) / chunk);
  double sum = 0.0;
  for (int i = threadIdx.x; i < partials; i += kThreads) sum += partial[i];
#pragma unroll
  for (int d = 32; d; d >>= 1) sum += __shfl_xor(sum, d);
  if (lane == 0) part[wave] = sum;
  __syncthreads();
  const double norm = sqrt((part[0] + part[1]) + (part[2] + part[3]));
  const double scale = (double)kScale / (norm < (double)eps ? (double)eps : norm);      // (a NaN norm stays one)

  const int tiles_c = padded(mat.cols) / 64, id = at0.id;
  const int r0 = id / tiles_c * 64, c0 = id % tiles_c * 64;
  // X^T has the longer side's length in rows: the matrix as it lies where that is tall, else turned through LDS
  const bool tall = mat.rows > mat.cols;
  _Float16* xt = reinterpret_cast<_Float16*>(work + mat.base) + r.xt[0];
#pragma unroll
  for (int p = threadIdx.x; p < 512; p += kThreads) {
    const int row = r0 + (p >> 3), col = c0 + (p & 7) * 8;
    float v[8];
    if (row < mat.rows && col < mat.cols) {
      const int64_t at = (int64_t)row * mat.cols + col;
      load8(static_cast<const T*>(mat.in) + at, mat.cols - col, v);
      if constexpr (MUON) {
        float m[8];
        load8(mat.momentum + at, mat.cols - col, m);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = mo.nesterov ? fmaf(mo.mu, m[e] - v[e], v[e]) : m[e];
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 0.f;
    }
    uint32_t w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = row < mat.rows && col + e < mat.cols ? halves((float)((double)v[e] * scale)) : 0u;
    if (tall) {
      put8(xt, row, col, r.mp, parts, w);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) tile[p >> 3][(p & 7) * 8 + e] = w[e];
    }
  }
  if (tall) return;
  __syncthreads();
#pragma unroll
  for (int p = threadIdx.x; p < 512; p += kThreads) {      // neighbouring lanes: neighbouring pieces of a row of X^T
    const int col = p >> 3, row = (p & 7) * 8;
    uint32_t w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = tile[row + e][col];
    put8(xt, c0 + col, r0 + row, r.mp, parts, w);
  }
}

enum { GRAM = 0, POLY = 1, APPLY = 2, LAST = 3, CUT = 4 };      // CUT: Gram products, some of them in pieces

// from: which of the two X^T arrays holds this step's; parts_out: halves that the next reader wants; coef_*: the step's coefficients
struct Step {
  float shrink;         // LAST, Muon: 1 - lr wd
  int* nan_flags;       // LAST, Muon: one int per matrix, set where the parameter as read holds a NaN
  int chunk;            // CUT: as pieces_of takes it
};

// Tiles: 128 x 128 by four waves of 64 x 64 (two halves: 32 k a stage, two workgroups to a CU), or 64 x 64 by four of 32 x 32.  Else 64 k a stage.
// GROUPS 2: eight waves, each four of them on every other k-step, for launches of one workgroup to a CU at most: see groups_for.
template <int TILE, int PARTS, int STAGES, int KIND, int GROUPS>
using Core = core::Product<_Float16, TILE, TILE, 2, 2, PARTS, KIND != GRAM && KIND != CUT, KIND != GRAM && KIND != CUT, TILE == 128 && PARTS == 2 ? 64 : 128, STAGES, GROUPS>;

// a 32 x 32 block in LDS (rows of 33) to its place at (rb, cb), and mirrored: 32 rows of four pieces, two pieces a lane
template <bool PLAIN> __device__ __forceinline__ void put_block(_Float16* to, const uint32_t* scratch, int rb, int cb, int ld, int parts, bool mirrored, int lane) {
#pragma unroll
  for (int e = 0; PLAIN && e < 2; ++e) {
    const int row = (lane >> 2) + 16 * e, c = lane & 3;
    uint32_t w[8];
#pragma unroll
    for (int x = 0; x < 8; ++x) w[x] = scratch[row * 33 + 8 * c + x];
    put8(to, rb + row, cb + 8 * c, ld, parts, w);
  }
  if (mirrored) {
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int row = (lane >> 2) + 16 * e, c = lane & 3;
      uint32_t w[8];
#pragma unroll
      for (int x = 0; x < 8; ++x) w[x] = scratch[(8 * c + x) * 33 + row];
      put8(to, cb + row, rb + 8 * c, ld, parts, w);
    }
  }
}

// tile id of the lower triangle: id = ti (ti + 1) / 2 + tj
__device__ __forceinline__ void triangle(int id, int& ti, int& tj) {
  ti = (int)((sqrtf(8.f * (float)id + 1.f) - 1.f) * 0.5f);
  while (ti * (ti + 1) / 2 > id) --ti;
  while ((ti + 1) * (ti + 2) / 2 <= id) ++ti;
  tj = id - ti * (ti + 1) / 2;
}

template <int TILE, int PARTS, int STAGES, int KIND, bool MUON, typename T, int GROUPS>
__global__ __launch_bounds__(GROUPS * kThreads, GROUPS == 2 ? 1 : 2) void product_kernel(S2L_FRONT, Alike alike, Step st) {
  using C = Core<TILE, PARTS, STAGES, KIND, GROUPS>;
  constexpr int W = TILE / 2, F = W / 32;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, group = GROUPS == 2 ? __builtin_amdgcn_readfirstlane(threadIdx.x >> 8) : 0;
  const int part = wave & 3;      // of the tile
  constexpr bool kGram = KIND == GRAM || KIND == CUT, kSym = kGram || KIND == POLY;
  Place at0 = place_of(S2L_FRONT_PASS, core::xcd_order(blockIdx.x, blocks));
  if constexpr (KIND == LAST) destination(work, alike, at0);
  const Mat& mat = at0.mat;
  const Arrays r = arrays_of(mat.rows, mat.cols);
  _Float16* arrays = reinterpret_cast<_Float16*>(work + mat.base);
  int ti, tj;
  if constexpr (kSym) {
    triangle(at0.id, ti, tj);
  } else {
    const int id = at0.id, tiles_n = (r.np + TILE - 1) / TILE;
    ti = id / tiles_n;
    tj = id % tiles_n;
  }
  const int m0 = ti * TILE, n0 = tj * TILE;

  int depth = kGram ? r.np : r.mp, k0 = 0;
  [[maybe_unused]] Pieces pieces{1, 0};
  if constexpr (KIND == CUT) {
    pieces = pieces_of(r.np, st.chunk);
    k0 = at0.piece * pieces.depth;
    depth = r.np - k0 < pieces.depth ? r.np - k0 : pieces.depth;
  }
  typename C::SA sa;
  typename C::SB sb;
  const _Float16* xt = arrays + (from ? r.xt[1] : r.xt[0]);
  sa.setup(kGram ? xt : KIND == POLY ? arrays + r.a : arrays + r.b, r.mp, m0, r.mp, k0, wave, lane);
  sb.setup(KIND == POLY ? arrays + r.a : xt, r.mp, n0, kSym ? r.mp : r.np, k0, wave, lane);
  f16v acc[F][F];
#pragma unroll
  for (int i = 0; i < F; ++i)
#pragma unroll
    for (int j = 0; j < F; ++j)
#pragma unroll
      for (int q = 0; q < 16; ++q) acc[i][j][q] = 0.f;
  // POLY's own A, requested ahead of the main loop's stream where there are registers for it (small tiles: their time is latency)
  constexpr bool kAhead = KIND == POLY && F == 1;
  uint64_t own[kAhead ? 4 : 1][PARTS];
  if constexpr (kAhead) {
    const _Float16* a = arrays + r.a + core::pair_at<PARTS>(m0 + (part >> 1) * W + (lane & 31), n0 + (part & 1) * W, r.mp) + 4 * (lane >> 5);
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int p = 0; p < PARTS; ++p) __builtin_memcpy(&own[q][p], a + 8 * q + p * core::kPairs, 8);
  }
  C::run(sa, sb, depth / C::BK, smem, acc, wave, lane, [](auto&) {});
  constexpr int kSums = GROUPS == 2 ? 2 * 4 * F * 4 * 64 * 16 : 0;
  if constexpr (GROUPS == 2) {      // each group hands the other's half of the rows over, in whole pieces, and goes on with its own
    static_assert(F == 2, "a block of rows for each group");
    f4* sums = reinterpret_cast<f4*>(smem);
    const auto at = [&](int reader, int j, int q) { return (((reader * 4 + part) * F + j) * 4 + q) * 64 + lane; };
#pragma unroll
    for (int i = 0; i < F; ++i) {
      if (i == group) continue;
#pragma unroll
      for (int j = 0; j < F; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) sums[at(i, j, q)] = f4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < F; ++i) {
      if (i != group) continue;
#pragma unroll
      for (int j = 0; j < F; ++j)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f4 o = sums[at(i, j, q)];
#pragma unroll
          for (int e = 0; e < 4; ++e) acc[i][j][4 * q + e] += o[e];
        }
    }
  }

  if constexpr (KIND == CUT) {
    if (pieces.count > 1) {      // raw sums, 1 KiB a store, in the order in which join_kernel reads them
      const int side = (int)tiles(r.m, TILE);
      f4* to = reinterpret_cast<f4*>(arrays + r.total) + ((int64_t)at0.piece * (side * (side + 1) / 2) + at0.id) * (TILE * TILE / 4) + lane;
#pragma unroll
      for (int i = 0; i < F; ++i)
#pragma unroll
        for (int j = 0; j < F; ++j)
#pragma unroll
          for (int q = 0; q < 4; ++q) to[(((wave * F + i) * F + j) * 4 + q) * 64] = f4{acc[i][j][4 * q], acc[i][j][4 * q + 1], acc[i][j][4 * q + 2], acc[i][j][4 * q + 3]};
      return;
    }
  }
  // lane: row lane & 31 of a 32 x 32 block, register q: column 8 (q / 4) + 4 (lane / 32) + q % 4.  Through LDS, a block at a time and a wave by
  // itself, so that both orientations leave as whole 16-byte pieces.
  const int wm = m0 + (part >> 1) * W, wn = n0 + (part & 1) * W;
  const int rows_end = r.mp, cols_end = kSym ? r.mp : r.np;
  if (wm >= rows_end || wn >= cols_end) return;      // (a 128-wide tile of an odd number of 64s)
  uint32_t* scratch = reinterpret_cast<uint32_t*>(smem + kSums) + wave * 32 * 33;
  const int li = lane & 31, h = lane >> 5;
#pragma unroll
  for (int i = 0; i < F; ++i) {
    if (GROUPS == 2 && i != group) continue;
#pragma unroll
    for (int j = 0; j < F; ++j) {
      const int rb = wm + 32 * i, cb = wn + 32 * j;
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int row = rb + li, col = cb + 8 * q + 4 * h;
        float v[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] = acc[i][j][4 * q + e];
        if constexpr (KIND == POLY) {
          _Float16 hi[4], lo[4];
          if constexpr (kAhead) {
            __builtin_memcpy(hi, &own[q][0], 8);
            if constexpr (PARTS == 2) __builtin_memcpy(lo, &own[q][1], 8);
          } else {
            const _Float16* a = arrays + r.a + core::pair_at<PARTS>(row, col, r.mp);
            __builtin_memcpy(hi, a, 8);
            if constexpr (PARTS == 2) __builtin_memcpy(lo, a + core::kPairs, 8);
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float x = (float)hi[e];
            if constexpr (PARTS == 2) x += (float)lo[e];
            v[e] = fmaf(coef_c, v[e] * (1.f / kScale), coef_b * x) + (row == col + e ? coef_a * kScale : 0.f);
          }
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] *= KIND == LAST ? 1.f / (kScale * kScale) : 1.f / kScale;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) scratch[li * 33 + 8 * q + 4 * h + e] = KIND == LAST ? __builtin_bit_cast(uint32_t, v[e]) : halves(v[e]);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      if constexpr (KIND == LAST) {
        const bool tall = mat.rows > mat.cols;
        T* out = static_cast<T*>(mat.out);
        // neighbouring lanes: neighbouring columns of the matrix as it lies
        const int row0 = (tall ? cb : rb) + h, col = (tall ? rb : cb) + li;
        T* at = out + (int64_t)row0 * mat.cols + col;
        float p[16];
        if constexpr (MUON) {      // (all sixteen requests before the first use)
#pragma unroll
          for (int e = 0; e < 16; ++e) p[e] = row0 + 2 * e < mat.rows && col < mat.cols ? at[(int64_t)2 * e * mat.cols] : 0.f;
        }
        bool bad = false;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          const int major = 2 * e + h;
          const float o = __builtin_bit_cast(float, tall ? scratch[li * 33 + major] : scratch[major * 33 + li]);
          if (row0 + 2 * e < mat.rows && col < mat.cols) {
            if constexpr (MUON) {
              bad |= p[e] != p[e];
              at[(int64_t)2 * e * mat.cols] = fmaf(p[e], st.shrink, -mat.step * o);
            } else {
              at[(int64_t)2 * e * mat.cols] = (T)o;
            }
          }
        }
        if (MUON && bad && st.nan_flags) st.nan_flags[at0.index] = 1;
      } else {
        put_block<kSym>(arrays + (kGram ? r.a : KIND == POLY ? r.b : from ? r.xt[0] : r.xt[1]), scratch, rb, cb, r.mp, parts_out, !kSym || ti != tj, lane);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  }
}

// A = the sum of its pieces, in their order.  A wave: a 32 x 32 block; memory bound (4 bytes a piece read, 8 or 4 written an element).
__global__ __launch_bounds__(kThreads) void join_kernel(char* work, int64_t records, int parts_out, int chunk) {
  __shared__ uint32_t blocks[4][32 * 33];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const Place at0 = place_of(work, 0, 0, 0, 0, records, blockIdx.x >> 2);
  const Arrays r = arrays_of(at0.mat.rows, at0.mat.cols);
  const Pieces pieces = pieces_of(r.np, chunk);
  if (pieces.count == 1) return;
  _Float16* arrays = reinterpret_cast<_Float16*>(work + at0.mat.base);
  const int side = (int)tiles(r.m, 128), all = side * (side + 1) / 2;
  int ti, tj;
  triangle(at0.id, ti, tj);
  const int block = (blockIdx.x & 3) * 4 + wave;      // (wave of the product, i, j)
  const int rb = ti * 128 + (block >> 3) * 64 + (block >> 1 & 1) * 32, cb = tj * 128 + (block >> 2 & 1) * 64 + (block & 1) * 32;
  if (rb >= r.mp || cb >= r.mp) return;
  const f4* from = reinterpret_cast<const f4*>(arrays + r.total) + (int64_t)at0.id * 4096 + block * 256 + lane;
  f4 sum[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) sum[q] = from[q * 64];
  for (int p = 1; p < pieces.count; ++p) {
    f4 v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) v[q] = from[(int64_t)p * all * 4096 + q * 64];
#pragma unroll
    for (int q = 0; q < 4; ++q)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[q][e] += v[q][e];
  }
  uint32_t* scratch = blocks[wave];
#pragma unroll
  for (int q = 0; q < 4; ++q)
#pragma unroll
    for (int e = 0; e < 4; ++e) scratch[(lane & 31) * 33 + 8 * q + 4 * (lane >> 5) + e] = halves(sum[q][e] * (1.f / kScale));
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
  put_block<true>(arrays + r.a, scratch, rb, cb, r.mp, parts_out, ti != tj, lane);
}

// ---- few and small matrices: 32 x 32 tiles, the k-steps of a stage dealt to the four waves ------------------------------------------------
// Four times the workgroups of the 64-wide tiles, a quarter of the work each: the launches of a few 256 x 256 matrices then use the whole chip
// instead of a quarter of it, and a workgroup's LDS (what the 64-wide tiles wait for: 768 of their 1000 cycles a stage) moves a quarter.  The
// waves' partial sums meet in LDS, in a fixed order; 128 threads then write the tile, 128 its mirror image.
constexpr int kSmallStages = 4;
template <int PARTS, int KIND> struct Small {
  using S = core::Stream<_Float16, 32, KIND != GRAM, 128, PARTS, 4>;
  using L = typename S::L;
  static constexpr int kStage = 2 * PARTS * L::kBytes, kLds = kSmallStages * kStage, kRequests = 2 * PARTS * S::kPer;
  static_assert(kLds >= 4 * 32 * 36 * 4, "the waves' sums");
};

template <int N, int REQUESTS> __device__ __forceinline__ void wait_younger(int younger) {
  if (N == 0 || younger >= N) asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(N * REQUESTS) : "memory");
  else wait_younger<(N > 0 ? N - 1 : 0), REQUESTS>(younger);
}

template <int PARTS, int KIND, bool MUON, typename T>
__global__ __launch_bounds__(kThreads, 2) void small_kernel(S2L_FRONT, Alike alike, Step st) {
  using C = Small<PARTS, KIND>;
  using L = typename C::L;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  constexpr bool kSym = KIND == GRAM || KIND == POLY;
  Place at0 = place_of(S2L_FRONT_PASS, core::xcd_order(blockIdx.x, blocks));
  if constexpr (KIND == LAST) destination(work, alike, at0);
  const Mat& mat = at0.mat;
  const Arrays r = arrays_of(mat.rows, mat.cols);
  _Float16* arrays = reinterpret_cast<_Float16*>(work + mat.base);
  int ti, tj;
  if constexpr (kSym) {
    triangle(at0.id, ti, tj);
  } else {
    ti = at0.id / (r.np / 32);
    tj = at0.id - ti * (r.np / 32);
  }
  const int m0 = ti * 32, n0 = tj * 32;
  typename C::S sa, sb;
  const _Float16* xt = arrays + (from ? r.xt[1] : r.xt[0]);
  sa.setup(KIND == GRAM ? xt : KIND == POLY ? arrays + r.a : arrays + r.b, r.mp, m0, r.mp, 0, wave, lane);
  sb.setup(KIND == POLY ? arrays + r.a : xt, r.mp, n0, kSym ? r.mp : r.np, 0, wave, lane);
  const int stages = __builtin_amdgcn_readfirstlane((KIND == GRAM ? r.np : r.mp) / 64);
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)smem);
  int put = 0, get = 0;
  auto fill = [&]() {
    sa.issue(lds0 + put * C::kStage, wave);
    sb.issue(lds0 + put * C::kStage + PARTS * L::kBytes, wave);
    put = put + 1 == kSmallStages ? 0 : put + 1;
  };
  f16v acc;
#pragma unroll
  for (int q = 0; q < 16; ++q) acc[q] = 0.f;
  asm volatile("s_nop 4" : : : "memory");      // scalar registers that a vector instruction wrote, read by the assembly text's loads
  for (int s = 0; s < kSmallStages - 1 && s < stages; ++s) fill();
  for (int kt = 0; kt < stages; ++kt) {
    wait_younger<kSmallStages - 2, C::kRequests>(stages - 1 - kt);
    __builtin_amdgcn_s_barrier();
    asm volatile("" : : : "memory");
    if (kt + kSmallStages - 1 < stages) fill();
    const char* la = smem + get * C::kStage;
    const char* lb = la + PARTS * L::kBytes;
    get = get + 1 == kSmallStages ? 0 : get + 1;
    u4 fa[PARTS], fb[PARTS];
#pragma unroll
    for (int q = 0; q < PARTS; ++q) {
      fa[q] = L::fragment(la + q * L::kBytes, 0, wave, lane);
      fb[q] = L::fragment(lb + q * L::kBytes, 0, wave, lane);
    }
    if constexpr (PARTS == 2) {
      acc = core::mma<_Float16>(fb[1], fa[0], acc);
      acc = core::mma<_Float16>(fb[0], fa[1], acc);
    }
    acc = core::mma<_Float16>(fb[0], fa[0], acc);
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" : : : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" : : : "memory");
  // sums: [wave][row 32][36]; lane: row lane & 31, register q: column 8 (q / 4) + 4 (lane / 32) + q % 4
  float* sums = reinterpret_cast<float*>(smem);
  {
    float* mine = sums + wave * 32 * 36 + (lane & 31) * 36 + 4 * (lane >> 5);
#pragma unroll
    for (int q = 0; q < 4; ++q) *reinterpret_cast<f4*>(mine + 8 * q) = f4{acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
  }
  __syncthreads();
  const auto total = [&](int row, int col) {
    const float* p = sums + row * 36 + col;
    return (p[0] + p[32 * 36]) + (p[2 * 32 * 36] + p[3 * 32 * 36]);
  };
  if constexpr (KIND == LAST) {
    const bool tall = mat.rows > mat.cols;
    T* out = static_cast<T*>(mat.out);
    const int minor = threadIdx.x & 31, major0 = threadIdx.x >> 5;      // neighbouring lanes: neighbouring columns of the matrix as it lies
    const int row0 = (tall ? n0 : m0) + major0, col = (tall ? m0 : n0) + minor;
    T* at = out + (int64_t)row0 * mat.cols + col;
    float p[4];
    if constexpr (MUON) {
#pragma unroll
      for (int e = 0; e < 4; ++e) p[e] = row0 + 8 * e < mat.rows && col < mat.cols ? at[(int64_t)8 * e * mat.cols] : 0.f;
    }
    bool bad = false;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int major = major0 + 8 * e;
      const float o = (tall ? total(minor, major) : total(major, minor)) * (1.f / (kScale * kScale));
      if (row0 + 8 * e < mat.rows && col < mat.cols) {
        if constexpr (MUON) {
          bad |= p[e] != p[e];
          at[(int64_t)8 * e * mat.cols] = fmaf(p[e], st.shrink, -mat.step * o);
        } else {
          at[(int64_t)8 * e * mat.cols] = (T)o;
        }
      }
    }
    if (MUON && bad && st.nan_flags) st.nan_flags[at0.index] = 1;
  } else {
    const bool mirror = KIND == APPLY || threadIdx.x >= 128;      // X^T is written mirrored only
    if (KIND == APPLY ? threadIdx.x >= 128 : mirror && ti == tj) return;
    const int row = (threadIdx.x & 127) >> 2, c = (threadIdx.x & 3) * 8;      // of the (mirrored) tile: eight columns of one row
    const int grow = (mirror ? n0 : m0) + row, gcol = (mirror ? m0 : n0) + c;
    uint32_t w[8];
    [[maybe_unused]] _Float16 hi[8], lo[8];
    if constexpr (KIND == POLY) {      // A is its own mirror image, to a rounding of its sums
      const _Float16* a = arrays + r.a + core::pair_at<PARTS>(grow, gcol, r.mp);
      __builtin_memcpy(hi, a, 16);
      if constexpr (PARTS == 2) __builtin_memcpy(lo, a + core::kPairs, 16);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float v = mirror ? total(c + e, row) : total(row, c + e);
      if constexpr (KIND == POLY) {
        float x = (float)hi[e];
        if constexpr (PARTS == 2) x += (float)lo[e];
        v = fmaf(coef_c, v * (1.f / kScale), coef_b * x) + (grow == gcol + e ? coef_a * kScale : 0.f);
      } else {
        v *= 1.f / kScale;
      }
      w[e] = halves(v);
    }
    put8(arrays + (KIND == GRAM ? r.a : KIND == POLY ? r.b : from ? r.xt[0] : r.xt[1]), grow, gcol, r.mp, parts_out, w);
  }
}

// ---- host --------------------------------------------------------------------------------------------------------------------------------

constexpr int kMaxSide = 1 << 17;
constexpr int kMaxSteps = 100;
constexpr int64_t kMaxBlocks = ((int64_t)1 << 32) / kThreads - 1;      // a launch counts its threads in 32 bits

struct Layout {
  int tile_sym, tile_rect;
  int blocks[KINDS];
  int64_t records[3];      // byte offsets: SYM, RECT, DEEP
  int chunk;               // of Gram products in pieces; 0: none
  int64_t bytes;
};

// Table and workspace of one set of launches.  128-wide tiles where they alone occupy half of the part's 256 CUs (they read half as much per
// product and their waves twice as little of LDS), else 64-wide ones: four times the workgroups; 32-wide where those are too few as well.
inline int tile_for(int64_t of128, int64_t of64) { return of128 >= 128 ? 128 : of64 >= 128 ? 64 : 32; }

// Two groups of waves where 128-wide tiles give no CU a second workgroup, whose waves would work while the first one's
// wait (a call of one 2048 x 2048 in fp32: 723 against 796 us; of four 1024 x 1024: 414 against 454).
inline int groups_for(int blocks) { return blocks <= 256 ? 2 : 1; }

// How long the pieces are: half of what a CU has to do on average (it runs two workgroups), where the longest product is so much longer that the
// other CUs would wait for it; only in 128-wide tiles (0.02 us per k of a workgroup's).  A Muon step of four 1024 x 1024 with a 4096 x 1024 and its
// transpose: 1060 us uncut, 960 cut (half as long pieces gained less: products that stay whole are then twice as long as the pieces, and whole ones
// fill some XCDs, pieces others); two 2048 x 5504 in bf16: 2167 against 2112.
inline int chunk_for(const s2l_matrix* in, int count) {
  int64_t work = 0;
  int longest = 0;
  for (int i = 0; i < count; ++i) {
    const int m = in[i].rows < in[i].cols ? in[i].rows : in[i].cols, np = padded(in[i].rows < in[i].cols ? in[i].cols : in[i].rows);
    work += tiles(m, 128) * (tiles(m, 128) + 1) / 2 * np;
    longest = np > longest ? np : longest;
  }
  int64_t chunk = work / 512;
  if (chunk < 512) chunk = 512;
  return pieces_of(longest, (int)(chunk < longest ? chunk : longest)).count > 1 ? (int)chunk : 0;
}

inline int lay_out(const s2l_matrix* in, int count, Table* t, Layout* l) {
  int64_t sym[2] = {}, rect[2] = {};
  for (int i = 0; i < count; ++i) {
    const int m = in[i].rows < in[i].cols ? in[i].rows : in[i].cols, n = in[i].rows < in[i].cols ? in[i].cols : in[i].rows;
    for (int k = 0; k < 2; ++k) {
      const int tile = k ? 64 : 128;
      sym[k] += tiles(m, tile) * (tiles(m, tile) + 1) / 2;
      rect[k] += tiles(m, tile) * tiles(n, tile);
    }
  }
  l->tile_sym = tile_for(sym[0], sym[1]);
  l->tile_rect = tile_for(rect[0], rect[1]);
  l->chunk = l->tile_sym == 128 ? chunk_for(in, count) : 0;
  int64_t at[KINDS] = {}, base = 0;
  for (int i = 0; i < kMaxMatrices; ++i)
    for (int k = 0; k < KINDS; ++k) t->first[k][i] = 0x7fffffff;
  for (int i = 0; i < count; ++i) {
    Mat& m = t->mat[i];
    m.in = in[i].in;
    m.out = in[i].out;
    m.momentum = in[i].momentum;
    m.rows = in[i].rows;
    m.cols = in[i].cols;
    m.step = in[i].step;
    const Arrays r = arrays_of(m.rows, m.cols);
    const int64_t total = elements_of(m), chunk = chunk_of(total), ts = tiles(r.m, l->tile_sym);
    for (int k = 0; k < KINDS; ++k) t->first[k][i] = (int)at[k];
    m.stat = (int)at[STAT];
    m.base = base;
    at[STAT] += (total + chunk - 1) / chunk;
    at[PACK] += (int64_t)(r.mp / 64) * (r.np / 64);
    at[SYM] += ts * (ts + 1) / 2;
    at[RECT] += tiles(r.m, l->tile_rect) * tiles(r.n, l->tile_rect);
    const int cut = pieces_of(r.np, l->chunk).count;
    at[DEEP] += l->chunk ? cut * (ts * (ts + 1) / 2) : 0;
    base += r.total * 2 + sums_bytes(cut, (int)(ts * (ts + 1) / 2));
    if (at[PACK] > kMaxBlocks || 4 * at[SYM] > kMaxBlocks || at[RECT] > kMaxBlocks || at[DEEP] > kMaxBlocks) return S2L_E_SIZE;      // (4: join_kernel's)
  }
  for (int k = 0; k < KINDS; ++k) l->blocks[k] = (int)at[k];
  int64_t front = kTableBytes + partial_bytes((int)at[STAT]);
  for (int k = 0; k < 3; ++k) {
    l->records[k] = front;
    front += at[SYM + k] * (int64_t)sizeof(Record);
  }
  front = (front + 255) / 256 * 256;
  for (int i = 0; i < count; ++i) t->mat[i].base += front;
  l->bytes = front + base;
  return 0;
}

inline Alike alike_of(const Table& t, const Layout& l, int count, int size, bool muon) {
  Alike a{};
  for (int k = 0; k < 3; ++k) a.records[k] = l.records[k];
  a.mat = t.mat[0];
  const int64_t stride = count > 1 ? static_cast<const char*>(t.mat[1].in) - static_cast<const char*>(t.mat[0].in) : 0;
  if (l.chunk) return a;
  if (count > 1 && (muon || stride < 0 || stride > 0x7fffffff / count)) return a;
  for (int i = 1; i < count; ++i)
    if (t.mat[i].rows != a.mat.rows || t.mat[i].cols != a.mat.cols || static_cast<const char*>(t.mat[i].in) != static_cast<const char*>(a.mat.in) + i * stride ||
        static_cast<char*>(t.mat[i].out) != static_cast<char*>(a.mat.out) + i * stride)
      return a;
  for (int k = 0; k < KINDS; ++k) a.per[k] = l.blocks[k] / count;
  a.stride = (int)stride;
  a.bytes = arrays_of(a.mat.rows, a.mat.cols).total * 2;
  return a;
}

// Whether the halves hold every X, A and B of `steps` steps with these coefficients: singular values start at most at 1 (the Frobenius norm) and
// p's largest value on the interval so far bounds the next; entries are bounded by the largest singular value.  2^11 * 16 < 65504.
inline bool within_range(double a, double b, double c, int steps) {
  double top = 1.0;
  for (int k = 0; k < steps; ++k) {
    double next = 0.0, poly = 0.0;
    for (int i = 0; i <= 256; ++i) {
      const double s = top * i / 256, q = std::fabs(a + b * s * s + c * s * s * s * s);
      if (!(q <= 16.0)) return false;
      poly = q > poly ? q : poly;
      next = s * q > next ? s * q : next;
    }
    top = next * 1.01;      // between two samples, and the roundings
    if (k + 1 < steps && !(top <= 4.0)) return false;      // A's entries: top^2 <= 16
    if (top < 1e-6) top = 1e-6;
  }
  return true;
}

struct Front {
  int per, rows, cols;
  int64_t base, bytes_or_records;
  int from, parts_out;
  float a, b, c;
};
#define S2L_FRONT_OF(f) (f).per, (f).rows, (f).cols, (f).base, (f).bytes_or_records, (f).from, (f).parts_out, (f).a, (f).b, (f).c, blocks

struct Call {
  Alike alike;
  char* work;
  hipStream_t st;
  int dev;
};

template <int TILE, int PARTS, int STAGES, int KIND, bool MUON, typename T, int GROUPS = 1> int one(int blocks, const Call& c, const Front& f, const Step& s) {
  using C = Core<TILE, PARTS, STAGES, KIND, GROUPS>;
  constexpr int epilogue = GROUPS * 4 * 32 * 33 * 4 + (GROUPS == 2 ? 65536 : 0), lds = C::kLds > epilogue ? C::kLds : epilogue;
  static_assert(lds <= 160 * 1024, "");
  const auto kernel = product_kernel<TILE, PARTS, STAGES, KIND, MUON, T, GROUPS>;
  if constexpr (lds > 65536) {
    static LdsOptIn opted;
    const int rc = ensure_dynamic_lds(reinterpret_cast<const void*>(kernel), lds, opted, c.dev);
    if (rc) return rc;
  }
  hipLaunchKernelGGL(kernel, dim3(blocks), dim3(GROUPS * kThreads), lds, c.st, c.work, S2L_FRONT_OF(f), c.alike, s);
  return (int)hipGetLastError();
}

template <int PARTS, int KIND, bool MUON, typename T> int small(int blocks, const Call& c, const Front& f, const Step& s) {
  constexpr int lds = Small<PARTS, KIND>::kLds;
  static_assert(lds <= 65536, "above 64 KiB the launch needs an opt-in");
  hipLaunchKernelGGL((small_kernel<PARTS, KIND, MUON, T>), dim3(blocks), dim3(kThreads), lds, c.st, c.work, S2L_FRONT_OF(f), c.alike, s);
  return (int)hipGetLastError();
}

template <int PARTS, int KIND, bool MUON, typename T> int sized(int tile, int blocks, const Call& c, const Front& f, const Step& s) {
  if constexpr (KIND == CUT) return one<128, PARTS, 2, KIND, MUON, T>(blocks, c, f, s);
  else if (tile == 32) return small<PARTS, KIND, MUON, T>(blocks, c, f, s);
  else if (tile == 128 && groups_for(blocks) == 2) return one<128, PARTS, 4, KIND, MUON, T, 2>(blocks, c, f, s);
  else if (tile == 128) return one<128, PARTS, 2, KIND, MUON, T>(blocks, c, f, s);
  else return one<64, PARTS, 3, KIND, MUON, T>(blocks, c, f, s);
}

// how many halves step k works on
template <typename T> int parts_of(int k, int steps) { return !std::is_same_v<T, __bf16> || k < steps - 2 ? 2 : 1; }

template <int KIND, bool MUON, typename T> int any(int tile, int parts, int blocks, const Call& c, Front f, const Step& s) {
  constexpr int kind = KIND == CUT ? DEEP : KIND == GRAM || KIND == POLY ? SYM : RECT;
  f.per = c.alike.per[kind];
  f.bytes_or_records = f.per ? c.alike.bytes : c.alike.records[kind - SYM];
  if constexpr (KIND == LAST) return sized<std::is_same_v<T, __bf16> ? 1 : 2, KIND, MUON, T>(tile, blocks, c, f, s);      // (parts_of the last step)
  else return parts == 2 ? sized<2, KIND, MUON, T>(tile, blocks, c, f, s) : sized<1, KIND, MUON, T>(tile, blocks, c, f, s);
}

template <typename T, bool MUON>
int run(const s2l_matrix* in, int count, double a, double b, double c, float eps, int steps, Momentum mo, float shrink, int* nan_flags, char* work, hipStream_t st) {
  int dev, cus;
  int rc = current_device_cus(&dev, &cus);
  if (rc) return rc;
  for (int first = 0; first < count; first += kMaxMatrices) {
    const int n = count - first < kMaxMatrices ? count - first : kMaxMatrices;
    Table t;
    Layout l;
    rc = lay_out(in + first, n, &t, &l);
    if (rc) return rc;
    const Call call{alike_of(t, l, n, sizeof(T), MUON), work, st, dev};
    const auto parts = [&](int k) { return parts_of<T>(k, steps); };
    Lists lists{};
    for (int k = 0; k < 3 && !call.alike.per[0]; ++k) {
      lists.at[k] = l.records[k];
      lists.count[k] = l.blocks[SYM + k];
    }
    hipLaunchKernelGGL((norm_kernel<T, MUON>), dim3(l.blocks[STAT]), dim3(kThreads), 0, st, t, work, mo, lists);
    rc = (int)hipGetLastError();
    if (rc) return rc;
    hipLaunchKernelGGL((split_kernel<T, MUON>), dim3(l.blocks[PACK]), dim3(kThreads), 0, st, work, call.alike, mo, eps, parts(0));
    rc = (int)hipGetLastError();
    if (rc) return rc;
    for (int k = 0; k < steps; ++k) {
      const Step s{shrink, nan_flags ? nan_flags + first : nullptr, l.chunk};
      Front f{0, call.alike.mat.rows, call.alike.mat.cols, call.alike.mat.base, 0, k & 1, parts(k), (float)a, (float)b, (float)c};
      // (GRAM, POLY and APPLY do not depend on the matrices' type: one instance)
      if (l.chunk) {
        rc = any<CUT, false, float>(l.tile_sym, parts(k), l.blocks[DEEP], call, f, s);
        if (rc) return rc;
        hipLaunchKernelGGL(join_kernel, dim3(4 * l.blocks[SYM]), dim3(kThreads), 0, st, work, l.records[0], parts(k), l.chunk);
        rc = (int)hipGetLastError();
      } else {
        rc = any<GRAM, false, float>(l.tile_sym, parts(k), l.blocks[SYM], call, f, s);
      }
      if (rc) return rc;
      rc = any<POLY, false, float>(l.tile_sym, parts(k), l.blocks[SYM], call, f, s);
      if (rc) return rc;
      if (k + 1 < steps) {
        f.parts_out = parts(k + 1);
        rc = any<APPLY, false, float>(l.tile_rect, parts(k), l.blocks[RECT], call, f, s);
      } else {
        rc = any<LAST, MUON, T>(l.tile_rect, parts(k), l.blocks[RECT], call, f, s);
      }
      if (rc) return rc;
    }
  }
  return 0;
}

inline int check(const s2l_matrix* mats, int64_t count, bool muon, int size) {
  if (count < 0 || count > (1 << 20)) return S2L_E_SIZE;
  if (count && !mats) return S2L_E_NULL;
  for (int64_t i = 0; i < count; ++i) {
    if (mats[i].rows < 1 || mats[i].cols < 1 || mats[i].rows > kMaxSide || mats[i].cols > kMaxSide) return S2L_E_SIZE;
    if (!mats[i].in || !mats[i].out || (muon && !mats[i].momentum)) return S2L_E_NULL;
    for (const void* p : {mats[i].in, (const void*)mats[i].out, (const void*)(muon ? mats[i].momentum : nullptr)})
      if (reinterpret_cast<uintptr_t>(p) & (size - 1)) return S2L_E_ALIGN;
  }
  return 0;
}

}  // namespace ns
}  // namespace s2l

extern "C" int64_t s2l_orthogonalize_work_bytes(const s2l_matrix* matrices_host, int64_t count) {
  using namespace s2l::ns;
  if (count <= 0 || !matrices_host || count > (1 << 20)) return 0;
  int64_t most = 0;
  for (int64_t first = 0; first < count; first += kMaxMatrices) {
    const int n = (int)(count - first < kMaxMatrices ? count - first : kMaxMatrices);
    for (int i = 0; i < n; ++i) {
      const s2l_matrix& m = matrices_host[first + i];
      if (m.rows < 1 || m.cols < 1 || m.rows > kMaxSide || m.cols > kMaxSide) return 0;
    }
    Table t;
    Layout l;
    if (lay_out(matrices_host + first, n, &t, &l)) return 0;
    most = l.bytes > most ? l.bytes : most;
  }
  return most;
}

extern "C" int s2l_orthogonalize(int dtype, const s2l_matrix* matrices_host, int64_t count, double a, double b, double c, float eps, int steps, void* work,
                                 s2l_stream_t stream) {
  using namespace s2l::ns;
  const int size = dtype == S2L_DTYPE_F32 ? 4 : dtype == S2L_DTYPE_BF16 || dtype == S2L_DTYPE_F16 ? 2 : 0;
  if (!size) return S2L_E_UNSUPPORTED;
  const int rc = check(matrices_host, count, false, size);
  if (rc) return rc;
  if (steps < 1 || steps > kMaxSteps || !(eps > 0.f) || !within_range(a, b, c, steps)) return S2L_E_SIZE;
  if (count == 0) return S2L_OK;
  if (!work) return S2L_E_NULL;
  if (s2l::misaligned16(work)) return S2L_E_ALIGN;
  hipStream_t st = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(work);
  const int n = (int)count;
  if (dtype == S2L_DTYPE_F32) return run<float, false>(matrices_host, n, a, b, c, eps, steps, Momentum{}, 0.f, nullptr, ws, st);
  if (dtype == S2L_DTYPE_BF16) return run<__bf16, false>(matrices_host, n, a, b, c, eps, steps, Momentum{}, 0.f, nullptr, ws, st);
  return run<_Float16, false>(matrices_host, n, a, b, c, eps, steps, Momentum{}, 0.f, nullptr, ws, st);
}

extern "C" int s2l_muon_step(const s2l_matrix* matrices_host, int64_t count, float momentum, int nesterov, float shrink, double a, double b, double c, float eps,
                             int steps, int* nan_flags, void* work, s2l_stream_t stream) {
  using namespace s2l::ns;
  const int rc = check(matrices_host, count, true, 4);
  if (rc) return rc;
  if (steps < 1 || steps > kMaxSteps || !(eps > 0.f) || !within_range(a, b, c, steps)) return S2L_E_SIZE;
  if (count == 0) return S2L_OK;
  if (!work) return S2L_E_NULL;
  if (s2l::misaligned16(work)) return S2L_E_ALIGN;
  return run<float, true>(matrices_host, (int)count, a, b, c, eps, steps, Momentum{momentum, nesterov}, shrink, nan_flags, static_cast<char*>(work),
                          static_cast<hipStream_t>(stream));
}
