// The main loop of a matrix product on 16-bit or fp32 MFMA, shared by the dense layer (linear.hip) and the orthogonalisation
// (orthogonalize.hip): C[m, n] = sum over k of A(m, k) B(n, k), operand tiles streamed into LDS by LDS-DMA, `STAGES` k-tiles deep.
#pragma once
#include <type_traits>

#include "s2l_common.h"

namespace s2l {
namespace core {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef __bf16 b8 __attribute__((ext_vector_type(8)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef float f16v __attribute__((ext_vector_type(16)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// c += a b over 16 bytes of k per half-wave (32 x 32 outputs; 16 k of a 16-bit type, 8 of fp32).  Lane: A row / B column lane & 31, the
// (lane / 32)-th 16 bytes of k.  Result lane: column lane & 31; register r: row 8 (r / 4) + 4 (lane / 32) + r % 4.  Callers pass the operands
// swapped, mma(B, A), so that a lane holds four consecutive columns of one row of C.
template <typename T> __device__ __forceinline__ f16v mma(u4 a, u4 b, f16v c) {
  if constexpr (std::is_same_v<T, float>) {
    union { u4 v; float f[4]; } x, y;
    x.v = a;
    y.v = b;
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(x.f[j], y.f[j], c, 0, 0, 0);
    return c;
  } else if constexpr (std::is_same_v<T, _Float16>) {
    union { u4 v; h8 h; } x, y;
    x.v = a;
    y.v = b;
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(x.h, y.h, c, 0, 0, 0);
  } else {
    union { u4 v; b8 h; } x, y;
    x.v = a;
    y.v = b;
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x.h, y.h, c, 0, 0, 0);
  }
}

// Workgroups of one XCD (blockIdx mod 8, the hardware's round robin) take neighbouring tiles, whose operand panels then meet in its L2.
__device__ __forceinline__ int xcd_order(int id, int n) {
  const int per = n >> 3, rest = n & 7, x = id & 7, i = id >> 3;
  return x * per + (x < rest ? x : rest) + i;
}

// a wave-uniform 64-bit value, in scalar registers
template <typename P> __device__ __forceinline__ P uniform64(P v) {
  const uint64_t x = (uint64_t)v;
  // (readfirstlane returns an int: without the inner casts the low word's sign would fill the high one)
  return (P)((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)x) | (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(x >> 32)) << 32);
}

// 16 bytes per lane from base + offset (a per-lane byte offset) to LDS at lds + 16 * lane.  Assembly text: the compiler would otherwise drain
// vmcnt before every LDS access that may alias an LDS-DMA it knows of; retired by the counted waits of the loop.
__device__ __forceinline__ void dma16(const void* base, uint32_t offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(lds), "v"(offset), "s"(base) : "memory");
}

// One operand's k-tile in LDS.  KC (k contiguous in memory): [ROWS][ROWB bytes of k], 16-byte piece c of row r at c ^ swizzle(r): 16 neighbouring
// rows at one k then cover all 64 banks once.  Not KC (k is the row): [BK][ROWS elements]; the 32-byte blocks of a k-row of a 16-bit type at
// block ^ ((k & 3) | (k >> 3 & 1) << 2), which spreads the eight k-rows that one transposing read touches over the banks.
template <typename T, int ROWS, bool KC, int ROWB> struct Tile {
  static constexpr int C = 16 / (int)sizeof(T);
  static constexpr int BK = ROWB / (int)sizeof(T);
  static constexpr int kBytes = ROWS * ROWB;
  static constexpr int kLine = KC ? ROWB : ROWS * (int)sizeof(T);        // bytes of an LDS row
  static constexpr int kBlockMask = ROWS * (int)sizeof(T) / 32 - 1;
  static_assert(ROWB == 64 || ROWB == 128, "");

  __device__ __forceinline__ static int swizzle(int line, int piece) {    // its own inverse in `piece`
    if constexpr (KC) return piece ^ (ROWB == 128 ? (line >> 1) & 7 : (line >> 2) & 3);
    else if constexpr (sizeof(T) == 2) return piece ^ ((((line & 3) | ((line >> 1) & 4)) & kBlockMask) << 1);
    else return piece;
  }
  __device__ __forceinline__ static int place(int line, int piece) { return line * kLine + (swizzle(line, piece) << 4); }

  // 16 bytes of fragment for k-step s (32 bytes of k): rows row .. row + 31; half-wave h holds the h-th 16 bytes
  __device__ __forceinline__ static u4 fragment(const char* lds, int row, int s, int lane) {
    const int h = lane >> 5;
    if constexpr (KC) {
      return *reinterpret_cast<const u4*>(lds + place(row + (lane & 31), 2 * s + h));
    } else if constexpr (sizeof(T) == 2) {
      // each 16-lane group reads a [4 k][16 columns] block: lane i passes the address of k-row i / 4, columns 4 (i % 4) .. and receives
      // column i of the four k-rows
      const int i = lane & 15, col = row + (lane & 16) + 4 * (i & 3), k = 16 * s + 8 * h + (i >> 2);
      typedef __attribute__((address_space(3))) s4* lds_s4;
      union { s4 a[2]; u4 v; } x;
      x.a[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(lds + place(k, col >> 3) + ((col & 4) << 1)));
      x.a[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s4)(lds + place(k + 4, col >> 3) + ((col & 4) << 1)));
      return x.v;
    } else {
      union { float f[4]; u4 v; } x;
      const float* p = reinterpret_cast<const float*>(lds) + (8 * s + 4 * h) * ROWS + row + (lane & 31);
#pragma unroll
      for (int j = 0; j < 4; ++j) x.f[j] = p[j * ROWS];
      return x.v;
    }
  }
};

// Where element (row, col) of a matrix of halves pairs lies: 32 hi, then their 32 lo -- one 128-byte line, so that tiles of 32 columns write whole
// lines and a k-tile's two parts are neighbours.  One part: rows of hi alone.
constexpr int kPairs = 32;
template <int PARTS> __host__ __device__ inline int64_t pair_at(int64_t row, int64_t col, int64_t ld) {
  return PARTS == 1 ? row * ld + col : row * 2 * ld + col / kPairs * (2 * kPairs) + col % kPairs;
}

// The LDS-DMA stream of one operand (PARTS 2: halves pairs as pair_at lays them).  WAVES waves share a k-tile; a wave's request moves 1 KiB.  Rows
// (KC) or columns past the end are clamped to valid ones: what they produce is not stored.
template <typename T, int ROWS, bool KC, int ROWB, int PARTS, int WAVES> struct Stream {
  using L = Tile<T, ROWS, KC, ROWB>;
  static constexpr int kPer = L::kBytes / 1024 / WAVES;      // requests of a wave per part and k-tile
  static_assert(kPer * 1024 * WAVES == L::kBytes, "");
  const char* base[PARTS];
  uint32_t off[kPer];
  int64_t step;                                              // bytes from one k-tile to the next

  // ld: row stride in elements (of one part); row0: first row (KC) / column of the tile; rows: how many there are; k0: first k.
  // (PARTS * 128 * ld * sizeof(T) < 2^32: the caller checks)
  __device__ __forceinline__ void setup(const T* p, int64_t ld, int64_t row0, int64_t rows, int64_t k0, int wave, int lane) {
    const T* origin = p + (KC ? pair_at<PARTS>(row0, k0, ld) : pair_at<PARTS>(k0, row0, ld));
    step = uniform64((KC ? (int64_t)L::BK : (int64_t)L::BK * ld) * PARTS * (int64_t)sizeof(T));
#pragma unroll
    for (int q = 0; q < PARTS; ++q) base[q] = uniform64(reinterpret_cast<const char*>(origin + q * kPairs));
    const int64_t left = rows - row0;
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int at = (wave * kPer + j) * 1024 + lane * 16;
      int line = at / L::kLine;
      int piece = L::swizzle(line, at % L::kLine / 16);
      if constexpr (KC) line = line < left ? line : (int)left - 1;
      else piece = (piece + 1) * L::C <= left ? piece : 0;
      off[j] = (uint32_t)(line * ld * PARTS * (int64_t)sizeof(T)) + (PARTS == 2 ? (piece >> 2) * 128 + (piece & 3) * 16 : piece * 16);
    }
  }
  __device__ __forceinline__ void issue(uint32_t lds, int wave) {      // the next k-tile, to LDS at `lds`
#pragma unroll
    for (int q = 0; q < PARTS; ++q) {
#pragma unroll
      for (int j = 0; j < kPer; ++j) dma16(base[q], off[j], lds + q * L::kBytes + (wave * kPer + j) * 1024);
      base[q] += step;
    }
  }
};

// BM x BN outputs per workgroup, WM x WN waves (KGROUPS times: group g of them takes every KGROUPS-th k-step, and the caller adds the groups' sums).
// PARTS 2: hi + lo halves of both operands, three products per pair (lo lo is below fp32's rounding).
template <typename T, int BM, int BN, int WAVES_M, int WAVES_N, int PARTS, bool AKC, bool BKC, int ROWB, int STAGES, int KGROUPS = 1, bool AHEAD = (KGROUPS > 1)> struct Product {
  static constexpr int kWaves = WAVES_M * WAVES_N * KGROUPS, kThreads = 64 * kWaves;
  static constexpr int WM = BM / WAVES_M, WN = BN / WAVES_N, FM = WM / 32, FN = WN / 32;
  using SA = Stream<T, BM, AKC, ROWB, PARTS, kWaves>;
  using SB = Stream<T, BN, BKC, ROWB, PARTS, kWaves>;
  using LA = typename SA::L;
  using LB = typename SB::L;
  static constexpr int BK = LA::BK;
  static constexpr int kStage = PARTS * (LA::kBytes + LB::kBytes);
  static constexpr int kLds = STAGES * kStage;
  static constexpr int kRequests = PARTS * (SA::kPer + SB::kPer);      // a wave's vector-memory operations per k-tile

  template <int N> __device__ __forceinline__ static void wait() {     // at most N requests of this wave outstanding, its LDS reads done
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(N) : "memory");
  }

  // at most N younger k-tiles in flight, fewer at the end
  template <int N> __device__ __forceinline__ static void wait_younger(int younger) {
    static_assert(N * kRequests < 64, "the counter's range");
    if constexpr (N == 0) wait<0>();
    else if (younger >= N) wait<N * kRequests>();
    else wait_younger<N - 1>(younger);
  }

  // acc += over k-tiles [0, tiles).  `each(fa)` sees every k-step's A fragments (PARTS == 1).
  template <typename Each>
  __device__ __forceinline__ static void run(SA& a, SB& b, int count, char* smem, f16v (&acc)[FM][FN], int wave, int lane, Each&& each) {
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)smem);
    const int tiles = __builtin_amdgcn_readfirstlane(count);
    const int uwave = __builtin_amdgcn_readfirstlane(wave);
    [[maybe_unused]] const int group = uwave / (WAVES_M * WAVES_N);
    const int wm = (wave / WAVES_N % WAVES_M) * WM, wn = (wave % WAVES_N) * WN;
    int put = 0, get = 0;      // stage to fill, stage to use
    auto fill = [&]() {
      a.issue(lds0 + put * kStage, uwave);
      b.issue(lds0 + put * kStage + PARTS * LA::kBytes, uwave);
      put = put + 1 == STAGES ? 0 : put + 1;
    };
    asm volatile("s_nop 4" : : : "memory");      // scalar registers that a vector instruction wrote, read by the assembly text's loads
    if constexpr (AHEAD) {
      // One workgroup alone on its CU: its waves run in step, so what they do one after the other the CU does one after the other.  Each k-tile's
      // fragments are therefore read between the products of the tile before.
      constexpr int kSteps = ROWB / 32 / KGROUPS, kReads = kSteps * PARTS * (FM + FN), kProducts = kSteps * (2 * PARTS - 1) * FM * FN;
      static_assert(kReads <= kProducts, "");
      u4 frag[2][kSteps][PARTS][FM + FN];      // A's, then B's
      auto read = [&](int set, const char* lds, int u) __attribute__((always_inline)) {
        const int f = u % (FM + FN), q = u / (FM + FN) % PARTS, s = u / (FM + FN) / PARTS;
        frag[set][s][q][f] = f < FM ? LA::fragment(lds + q * LA::kBytes, wm + 32 * f, s * KGROUPS + group, lane)
                                    : LB::fragment(lds + PARTS * LA::kBytes + q * LB::kBytes, wn + 32 * (f - FM), s * KGROUPS + group, lane);
      };
      auto next = [&]() __attribute__((always_inline)) {
        const char* lds = smem + get * kStage;
        get = get + 1 == STAGES ? 0 : get + 1;
        return lds;
      };
      auto step = [&](int set, int kt) __attribute__((always_inline)) {      // k-tile kt, whose fragments are on their way to `set`
        wait_younger<STAGES - 2>(tiles - 2 - kt > 0 ? tiles - 2 - kt : 0);      // k-tile kt + 1 has landed, and this wave has read k-tile kt
        __builtin_amdgcn_s_barrier();                                          // ... everybody's, everybody has
        asm volatile("" : : : "memory");
        const char* lds = next();      // (behind the last k-tile: what lies there, unused)
#pragma unroll
        for (int t = 0; t < kProducts; ++t) {
          const int j = t % FN, i = t / FN % FM, p = 2 * PARTS - 2 - t / (FN * FM) % (2 * PARTS - 1), s = t / (FN * FM) / (2 * PARTS - 1);
          acc[i][j] = mma<T>(frag[set][s][p == 2][FM + j], frag[set][s][p == 1][i], acc[i][j]);      // lo hi, hi lo, hi hi: the small products first
          __builtin_amdgcn_sched_barrier(0);
          if (t < kReads) read(set ^ 1, lds, t);
          if (t == kReads - 1 && kt + STAGES < tiles) fill();      // into k-tile kt's place
          __builtin_amdgcn_sched_barrier(0);
        }
      };
      for (int s = 0; s < STAGES && s < tiles; ++s) fill();
      wait_younger<STAGES - 1>(tiles - 1);
      __builtin_amdgcn_s_barrier();
      asm volatile("" : : : "memory");
      const char* first = next();
#pragma unroll
      for (int u = 0; u < kReads; ++u) read(0, first, u);
      int kt = 0;
      for (; kt + 1 < tiles; kt += 2) {
        step(0, kt);
        step(1, kt + 1);
      }
      if (kt < tiles) step(0, kt);
      wait<0>();
      __builtin_amdgcn_s_barrier();
      asm volatile("" : : : "memory");
      return;
    }
    for (int s = 0; s < STAGES - 1 && s < tiles; ++s) fill();
    for (int kt = 0; kt < tiles; ++kt) {
      // k-tile kt has landed when at most the younger ones' requests are outstanding (loads retire in order)
      wait_younger<STAGES - 2>(tiles - 1 - kt);
      __builtin_amdgcn_s_barrier();      // everybody's part of k-tile kt is in LDS; everybody has left k-tile kt - 1, whose stage is filled next
      asm volatile("" : : : "memory");
      if (kt + STAGES - 1 < tiles) fill();
      const char* la = smem + get * kStage;
      const char* lb = la + PARTS * LA::kBytes;
      get = get + 1 == STAGES ? 0 : get + 1;
      // the fragments of a k-step are read while the matrix cores work on the step before (left to itself the compiler reads them right
      // before their use, and every step waits out the LDS latency)
      u4 fa[2][PARTS][FM], fb[2][PARTS][FN];
      auto fetch = [&](int s) {
#pragma unroll
        for (int q = PARTS - 1; q >= 0; --q) {
#pragma unroll
          for (int j = 0; j < FN; ++j) fb[s & 1][q][j] = LB::fragment(lb + q * LB::kBytes, wn + 32 * j, s, lane);
#pragma unroll
          for (int i = 0; i < FM; ++i) fa[s & 1][PARTS - 1 - q][i] = LA::fragment(la + (PARTS - 1 - q) * LA::kBytes, wm + 32 * i, s, lane);
        }
      };
      constexpr bool kPin = FM * FN == 1;
      fetch(0);
#pragma unroll
      for (int s = 0; s < ROWB / 32; ++s) {
        if (s + 1 < ROWB / 32) {
          fetch(s + 1);
          if (kPin) __builtin_amdgcn_sched_barrier(0);
        }
        const auto& a0 = fa[s & 1];
        const auto& b0 = fb[s & 1];
        if constexpr (PARTS == 2) {      // the small products first
#pragma unroll
          for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = mma<T>(b0[1][j], a0[0][i], acc[i][j]);
#pragma unroll
          for (int i = 0; i < FM; ++i)
#pragma unroll
            for (int j = 0; j < FN; ++j) acc[i][j] = mma<T>(b0[0][j], a0[1][i], acc[i][j]);
        }
#pragma unroll
        for (int i = 0; i < FM; ++i)
#pragma unroll
          for (int j = 0; j < FN; ++j) acc[i][j] = mma<T>(b0[0][j], a0[0][i], acc[i][j]);
        each(a0);
        if (kPin && s + 1 < ROWB / 32) __builtin_amdgcn_sched_barrier(0);
      }
    }
    wait<0>();
    __builtin_amdgcn_s_barrier();      // the k-tiles are dead: LDS is the caller's
    asm volatile("" : : : "memory");
  }
};

}  // namespace core
}  // namespace s2l
