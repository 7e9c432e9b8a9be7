// Matrix products grouped by expert on the matrix cores: the tiled kernel.
//
// A workgroup computes a BN x BM tile of the output (n = contiguous columns of
// the output, m = its rows) and walks the reduction in slabs of 128 bytes per row
// (64 elements of 16 bits, 128 of 8).  The matrix instruction takes the n side as
// its first operand, so that a lane's accumulators are consecutive columns of one
// output row: stores are vectors and a row's scale is one value per lane.
//
// Each operand is either held with the reduction contiguous ("along") or with its
// own index contiguous ("across"):
//                      n side            m side
//   y  = x W^T  (NK)   w, along          x, along
//   y  = x W    (KN)   w, across         x, along
//   dw = dy^T x        x, across         dy, across
// An "along" tile lies in LDS as rows of 128 bytes whose eight 16-byte chunks are
// exchanged by a function of the row, so that the eight lanes that a 128-bit read
// serves at a time meet eight different chunks.  An "across" tile keeps its rows
// of the reduction and is read with the transposing LDS loads, four rows by 32
// bytes at a time; its 32-byte units are exchanged by a function of the row.
//
// Measured: 8192^3 bf16 1.35 PFLOP/s (matrix cores about half the time busy: the rest is
// what waits and stores cost), e4m3 2.0 to 2.15; 16384 rows of 16 experts, 4096 x 4096
// bf16, 0.52 to 0.55 ms (1.0 PFLOP/s: experts' last tiles and weights from memory); one
// token through 8 of 64 experts, 2048 x 4096, 26 us (5.2 TB/s of weights).
#pragma once
#include "flagcx_amd/fx_model.h"
#include "fx_vec.hpp"

namespace fx {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));

// 8-bit matrix instructions.  Within each run of eight of the reduction they cut every product, towards zero, to 13 bits
// below the largest sum of two factors' exponents (subnormals: -6), and add up exactly; runs are added in fp32.  That
// costs a run less than 8 x 2^-13 = 2^-10 of its largest product.  All 8-bit forms of this chip do so, the narrower ones
// too; sums without the cut are E4m3Exact's (8192^3: 1742 us against 516, warm).
struct E4m3 {};
struct E4m3Exact {};   // widened to bf16 first: sums as in fp32

template <class T>
constexpr int kBytes = 2;
template <>
inline constexpr int kBytes<E4m3> = 1;
template <>
inline constexpr int kBytes<E4m3Exact> = 1;

struct ProductArgs {
  const void *pn, *pm;             // operands of the n side and the m side
  void *y;
  const float *sn, *sm;            // e4m3: scales of the n side (blocks) and of the m side (rows)
  const int32_t *offsets;
  size_t ldn, ldm, ldy;            // elements
  size_t expertN, expertY;         // products: weights' stride; dw: output's stride
  size_t ldsn, ldsm, expertSn;
  uint32_t experts, rows;
  uint32_t n, m, k;                // output columns; dw: output rows; products: length of the reduction
  uint32_t mTiles, nTiles;         // products: upper bound of row tiles over all experts; dw: per expert
  uint32_t group;                  // products: columns of tiles that are taken together
};

// What one workgroup computes.
struct Tile {
  uint32_t expert, m0, mEnd, n0, k0, kLen;   // rows [m0, mEnd) of the m side; reduction [k0, k0 + kLen)
};

__device__ __forceinline__ uint32_t uniform(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }

// Expert boundaries as the kernels use them: never outside [0, rows].
__device__ __forceinline__ uint32_t bound(const ProductArgs &a, uint32_t e) {
  const int32_t o = a.offsets[e];
  return o < 0 ? 0u : ((uint32_t)o > a.rows ? a.rows : (uint32_t)o);
}

__device__ __forceinline__ uint32_t waveScan(uint32_t v) {   // inclusive prefix sum over the wavefront
#pragma unroll
  for (int d = 1; d < 64; d <<= 1) {
    const uint32_t o = (uint32_t)__shfl_up((int)v, d);
    if ((int)(threadIdx.x & 63) >= d) v += o;
  }
  return v;
}

// Rows of expert e.
__device__ __forceinline__ uint32_t rowsOf(const ProductArgs &a, uint32_t e, uint32_t *first) {
  *first = 0;
  if (e >= a.experts) return 0;
  *first = bound(a, e);
  const uint32_t last = bound(a, e + 1);
  return last > *first ? last - *first : 0;
}

// Consecutive tiles of one die (workgroups go to the eight dies in turn) are made
// neighbours: a die's L2 then holds the operands of a block of kPanel row tiles by
// a few column tiles.
constexpr uint32_t kDies = 8, kPanel = 8, kUnits = 256;
constexpr int kKinds = 5;   // whole tiles, and last tiles by quarters
__device__ __forceinline__ uint32_t dieOrder(uint32_t id, uint32_t total) {
  const uint32_t die = id % kDies, at = id / kDies, q = total / kDies, r = total % kDies;
  return die * q + (die < r ? die : r) + at;
}
__device__ __forceinline__ void panelOrder(uint32_t id, uint32_t mTiles, uint32_t nTiles, uint32_t *mt, uint32_t *nt) {
  const uint32_t panel = id / (kPanel * nTiles), rem = id - panel * kPanel * nTiles;
  const uint32_t left = mTiles - panel * kPanel, h = left < kPanel ? left : kPanel;
  *mt = panel * kPanel + rem % h;
  *nt = rem / h;
}

// The row tiles of all experts are counted on the device (the host knows only an
// upper bound, the grid): every wavefront scans the boundaries, 64 experts at a time.
// ORDERED: a.group columns of tiles at a time, first the whole tiles of all experts,
// then the experts' last tiles, by the quarter of their rows that they have: they
// take that much less time, and the shortest fill up the end of the call.  A group's
// weights are used by whole and last tiles while the memory-side cache holds them.  In a
// call of less than two rounds of workgroups the last tiles' order counts for more:
// eight columns at a time (4096 rows of 16 experts, 4096 x 4096: 202 -> 186 us, e4m3 144
// -> 122; eight where there are more rounds: 300 -> 306 us for 8192 rows, e4m3 with 32
// experts 222 -> 234).
// Boundaries that do not ascend may count more tiles than the grid has, up to a whole
// call's for every other expert: the counts end at kMostTiles, far above any grid's,
// so that what they are multiplied with stays below 2^32.
constexpr uint32_t kMostTiles = 1u << 26;
template <int BN, int BM, bool ORDERED>
__device__ __forceinline__ bool findTile(const ProductArgs &a, Tile *t) {
  uint32_t mt, nt, id = blockIdx.x;
  if (!a.offsets) {
    const uint32_t mTiles = (a.rows + BM - 1) / BM;
    if (id >= mTiles * a.nTiles) return false;
    panelOrder(dieOrder(id, mTiles * a.nTiles), mTiles, a.nTiles, &mt, &nt);
    *t = Tile{0, mt * BM, a.rows, nt * BN, 0, a.k};
    return true;
  }
  const uint32_t lane = threadIdx.x & 63;
  uint32_t first = 0, rows = 0, scan = 0, tiles[kKinds] = {};
  // Tiles of kind 0 of this lane's expert; of the others it has one at most.
  auto whole = [&] { return ORDERED ? rows / BM : (rows + BM - 1) / BM; };
  auto isKind = [&](int k) { return ORDERED && rows % BM != 0 && (int)((rows % BM - 1) / (BM / 4)) == 4 - k; };
  for (uint32_t e = 0; e < a.experts; e += 64) {
    rows = rowsOf(a, e + lane, &first);
    scan = waveScan(whole());
    tiles[0] += uniform((uint32_t)__shfl((int)scan, 63));
    if (ORDERED && tiles[0] > kMostTiles) tiles[0] = kMostTiles;
#pragma unroll
    for (int k = 1; k < kKinds; k++) {
      tiles[k] += (uint32_t)__popcll(__ballot(isKind(k)));
      if (tiles[k] > kMostTiles) tiles[k] = kMostTiles;
    }
  }
  uint32_t mTiles = 0;
#pragma unroll
  for (int k = 0; k < kKinds; k++) mTiles += tiles[k];
  if (id >= mTiles * a.nTiles) return false;
  const uint32_t wide = ORDERED ? a.group : a.nTiles, group = id / (mTiles * wide);
  const uint32_t left = a.nTiles - group * wide, w = left < wide ? left : wide;   // columns of tiles in this group
  id -= group * mTiles * wide;
  int kind = 0;
  uint32_t all = tiles[0];
#pragma unroll
  for (int k = 1; k < kKinds; k++)
    if (kind == k - 1 && id >= all * w) {
      id -= all * w;
      kind = k;
      all = tiles[k];
    }
  const uint32_t at = dieOrder(id, all * w);
  mt = at / w;
  nt = group * wide + at % w;
  for (uint32_t e = 0, before = 0; e < a.experts; e += 64) {
    if (a.experts > 64) {
      rows = rowsOf(a, e + lane, &first);
      scan = waveScan(whole());
    }
    const uint64_t set = __ballot(isKind(kind));
    const uint32_t here = kind ? (uint32_t)__popcll(set) : uniform((uint32_t)__shfl((int)scan, 63));
    if (mt < before + here) {
      const uint32_t want = mt - before;             // which of this kind's tiles among the 64 experts
      const uint32_t ahead = kind ? (uint32_t)__builtin_amdgcn_mbcnt_hi((uint32_t)(set >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)set, 0))
                                  : scan - whole();
      const bool mine = kind ? isKind(kind) && ahead == want : ahead <= want && want < scan;
      const uint64_t one = __ballot(mine);
      if (!one) return false;                        // boundaries that changed between two readings
      const uint32_t l = (uint32_t)__builtin_ctzll(one);
      const uint32_t skip = kind ? rows / BM : want - ahead;                // tiles of the same expert in front
      const uint32_t f = uniform((uint32_t)__shfl((int)first, (int)l)), r = uniform((uint32_t)__shfl((int)rows, (int)l));
      const uint32_t m0 = f + uniform((uint32_t)__shfl((int)skip, (int)l)) * BM;
      *t = Tile{e + l, m0, f + r, nt * BN, 0, a.k};
      return m0 < f + r;
    }
    before += here;
  }
  return false;
}

// Experts differ in length, so each one's tiles are dealt to all dies, and the
// longest expert's come first (up to 64 experts; more are taken as they lie).
template <int BN, int BM>
__device__ __forceinline__ bool findTileDw(const ProductArgs &a, Tile *t) {
  const uint32_t per = a.mTiles * a.nTiles, turn = blockIdx.x / per;
  uint32_t mt, nt, e = turn, first = 0, rows = a.rows;
  panelOrder(dieOrder(blockIdx.x - turn * per, per), a.mTiles, a.nTiles, &mt, &nt);
  if (a.offsets) {
    if (a.experts <= 64) {
      const uint32_t lane = threadIdx.x & 63;
      rows = rowsOf(a, lane, &first);
      uint32_t rank = 0;
      for (uint32_t j = 0; j < a.experts; j++) {
        const uint32_t other = (uint32_t)__builtin_amdgcn_readlane((int)rows, (int)j);
        rank += other > rows || (other == rows && j < lane);
      }
      const uint64_t one = __ballot(lane < a.experts && rank == turn);
      e = one ? (uint32_t)__builtin_ctzll(one) : turn;
    }
    rows = uniform(rowsOf(a, e, &first));
    first = uniform(first);
  }
  *t = Tile{e, mt * BM, a.m, nt * BN, first, rows};
  return true;
}

// ------------------------------------------------------- one operand's tile

// Chunk exchange of an "along" tile.  On the m side the sixteen lanes of a
// fragment are rows 16 f + i; on the n side rows 8 (i / 4) + i % 4, + 4 in odd
// fragments, of a block of 32, which gives a lane eight consecutive columns over two
// fragments and the four lane groups a row's 32.
template <bool NSIDE>
__device__ __forceinline__ uint32_t exchange(uint32_t r) {
  return NSIDE ? ((r & 3) | ((r >> 1) & 4)) : (r & 7);
}

// Unit exchange of an "across" tile whose rows span all 64 banks: by the row's two low
// bits, so that the four rows of a transposing load meet different banks, and by its
// fourth, so that two lane groups, eight rows apart, do.
template <int R>
__device__ __forceinline__ uint32_t exchangeUnits(uint32_t row) {
  return (row & 3) | (R >= 128 ? (row >> 1) & 4 : 0);
}

// R = extent of the tile in its own index, NT = threads, ES = bytes per element.
template <int R, int NT, int ES, bool ACROSS, bool NSIDE>
struct Side {
  static constexpr int kLoads = R * 8 / NT;              // 16-byte chunks per thread and slab
  static constexpr int kPerRow = ACROSS ? R / 8 : 8;     // chunks per LDS row
  static constexpr int kStep = NT / kPerRow;             // rows between a thread's chunks
  static constexpr int kElems = 16 / ES;
  static constexpr uint32_t kSlab = 128 / ES;            // reduction elements per slab

  static_assert(kStep % 16 == 0, "a thread's chunks lie in rows that the exchange treats alike");

  // position of this thread's first chunk
  uint32_t row, chunk;
  __device__ __forceinline__ void init() {
    row = threadIdx.x / kPerRow;
    const uint32_t p = threadIdx.x % kPerRow;
    chunk = ACROSS ? ((((p >> 1) ^ exchangeUnits<R>(row)) << 1) | (p & 1)) : (p ^ exchange<NSIDE>(row));
  }

  // One chunk, element by element where it is not whole; `base` = the tile's own
  // index 0 at reduction 0.  own / red: how much of the tile's own index and of the
  // slab's reduction exists.
  __device__ __forceinline__ u32x4 guarded(const char *base, size_t ld, int i, uint32_t own, uint32_t red) const {
    const uint32_t r = row + i * kStep, c = chunk * kElems;
    u32x4 v = {};
    const uint32_t rows = ACROSS ? red : own, cols = ACROSS ? own : red;
    if (r >= rows || c >= cols) return v;
    const char *p = base + ((size_t)r * ld + c) * ES;
    if (c + kElems <= cols) return *reinterpret_cast<const u32x4_anywhere *>(p);
    if constexpr (ES == 2) {
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (c + j < cols) v[j >> 1] |= (uint32_t)reinterpret_cast<const uint16_t *>(p)[j] << (16 * (j & 1));
    } else {
#pragma unroll
      for (int j = 0; j < 16; j++)
        if (c + j < cols) v[j >> 2] |= (uint32_t) reinterpret_cast<const uint8_t *>(p)[j] << (8 * (j & 3));
    }
    return v;
  }
};

// Fragment reads.  lane l: index i = l % 16 of the fragment, reduction group g = l / 16.
template <bool NSIDE>
__device__ __forceinline__ u32x4 readAlong(const char *lds, uint32_t wave0, int f, int half, uint32_t i, uint32_t g) {
  const uint32_t r = NSIDE ? wave0 + 32 * (f >> 1) + 8 * (i >> 2) + 4 * (f & 1) + (i & 3) : wave0 + 16 * f + i;
  return *reinterpret_cast<const u32x4 *>(lds + r * 128 + (((uint32_t)(half * 4) + g) ^ exchange<NSIDE>(r)) * 16);
}
template <int R>
__device__ __forceinline__ u32x4 readAcross(const char *lds, uint32_t wave0, int f, int half, uint32_t i, uint32_t g) {
  typedef __attribute__((address_space(3))) s16x4 *lds64;
  const uint32_t unit = (wave0 + 16 * f) / 16;
  const uint32_t k = 32 * half + 8 * g + (i >> 2);
  const uint32_t at = k * (R * 2) + ((unit ^ exchangeUnits<R>(k)) * 32) + (i & 3) * 8;
  const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds64)(lds + at));
  const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds64)(lds + at + 4 * R * 2));
  const u32x2 x = __builtin_bit_cast(u32x2, a), y = __builtin_bit_cast(u32x2, b);
  return u32x4{x[0], x[1], y[0], y[1]};
}

// eight e4m3 codes (two words) as bf16: exact
__device__ __forceinline__ bf16x8 widen(uint32_t lo, uint32_t hi) {
  typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
  const bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, false), b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.f, true);
  const bf16x2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, false), d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.f, true);
  return bf16x8{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}

template <class T>
__device__ __forceinline__ f32x4 mma(u32x4 n, u32x4 m, f32x4 c) {
  if constexpr (__is_same(T, __bf16))
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, n), __builtin_bit_cast(bf16x8, m), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, n), __builtin_bit_cast(f16x8, m), c, 0, 0, 0);
}

// 128 products of e4m3 values: two chunks per side
template <class T>
__device__ __forceinline__ f32x4 mma8(const u32x4 (&n)[2], const u32x4 (&m)[2]) {
  f32x4 c = {};
  if constexpr (__is_same(T, E4m3)) {
    const i32x8 a = {(int)n[0][0], (int)n[0][1], (int)n[0][2], (int)n[0][3], (int)n[1][0], (int)n[1][1], (int)n[1][2], (int)n[1][3]};
    const i32x8 b = {(int)m[0][0], (int)m[0][1], (int)m[0][2], (int)m[0][3], (int)m[1][0], (int)m[1][1], (int)m[1][2], (int)m[1][3]};
    c = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, c, 0, 0, 0, 0, 0, 0);
  } else {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(n[h][0], n[h][1]), widen(m[h][0], m[h][1]), c, 0, 0, 0);
      c = __builtin_amdgcn_mfma_f32_16x16x32_bf16(widen(n[h][2], n[h][3]), widen(m[h][2], m[h][3]), c, 0, 0, 0);
    }
  }
  return c;
}

// 16 bytes without the first `bytes` of them, moved to the front; zeros behind.
__device__ __forceinline__ u32x4 dropFront(u32x4 v, uint32_t bytes) {
  uint32_t w[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
  for (int b = 1; b < 4; b <<= 1)
#pragma unroll
    for (int j = 0; j < 4; j++) w[j] = (bytes >> 2 & b) ? (j + b < 4 ? w[j + b] : 0u) : w[j];
#pragma unroll
  for (int j = 0; j < 4; j++) v[j] = bytes >= 16 ? 0u : __builtin_amdgcn_alignbyte(j < 3 ? w[j < 3 ? j + 1 : 3] : 0u, w[j], bytes & 3);
  return v;
}

// N consecutive columns of one output row
template <class Out, int N>
__device__ __forceinline__ void storeRun(Out *p, uint32_t c, uint32_t cols, const float (&f)[N]) {
  if (c + N <= cols) {
    if constexpr (sizeof(Out) == 4) {
#pragma unroll
      for (int q = 0; q < N / 4; q++) {
        u32x4 v;
#pragma unroll
        for (int j = 0; j < 4; j++) v[j] = __builtin_bit_cast(uint32_t, f[4 * q + j]);
        *reinterpret_cast<u32x4_anywhere *>(p + c + 4 * q) = v;
      }
    } else {
      typedef uint32_t words __attribute__((ext_vector_type(N / 2 < 4 ? N / 2 : 4), aligned(1)));
      constexpr int W = N / 2 < 4 ? N / 2 : 4;
#pragma unroll
      for (int q = 0; q < N / (2 * W); q++) {
        words v;
#pragma unroll
        for (int j = 0; j < W; j++)
          v[j] = (uint32_t)__builtin_bit_cast(uint16_t, (Out)f[2 * W * q + 2 * j]) |
                 ((uint32_t)__builtin_bit_cast(uint16_t, (Out)f[2 * W * q + 2 * j + 1]) << 16);
        *reinterpret_cast<words *>(p + c + 2 * W * q) = v;
      }
    }
  } else {
#pragma unroll
    for (int j = 0; j < N; j++)
      if (c + j < cols) p[c + j] = (Out)f[j];
  }
}

// Two fragments side by side, of each of which a lane of group g holds columns
// 4 g .. 4 g + 3: exchanged between the lane groups so that group g holds columns
// 8 g .. 8 g + 7 of the 32, the first four in x and the others in y, and a store
// writes a row's columns without gaps.
__device__ __forceinline__ void sideBySide(uint32_t &x, uint32_t &y) {
  const auto halves = __builtin_amdgcn_permlane32_swap(x, y, false, false);            // groups 2, 3 of x against 0, 1 of y
  const auto quarters = __builtin_amdgcn_permlane16_swap(halves[0], halves[1], false, false);   // 1, 3 against 0, 2
  x = quarters[0];
  y = quarters[1];
}
template <class Out>
__device__ __forceinline__ void storeAcross(Out *row, uint32_t c, uint32_t cols, f32x4 a, f32x4 b) {
  if constexpr (sizeof(Out) == 4) {
    float v[8];
#pragma unroll
    for (int j = 0; j < 4; j++) {
      const float fa = a[j], fb = b[j];       // values: __builtin_bit_cast of a vector's element takes the first
      uint32_t x = __builtin_bit_cast(uint32_t, fa), y = __builtin_bit_cast(uint32_t, fb);
      sideBySide(x, y);
      v[j] = __builtin_bit_cast(float, x);
      v[4 + j] = __builtin_bit_cast(float, y);
    }
    storeRun(row, c, cols, v);
  } else {
    u32x4 w;
#pragma unroll
    for (int j = 0; j < 2; j++) {
      uint32_t x = (uint32_t)__builtin_bit_cast(uint16_t, (Out)a[2 * j]) | ((uint32_t)__builtin_bit_cast(uint16_t, (Out)a[2 * j + 1]) << 16);
      uint32_t y = (uint32_t)__builtin_bit_cast(uint16_t, (Out)b[2 * j]) | ((uint32_t)__builtin_bit_cast(uint16_t, (Out)b[2 * j + 1]) << 16);
      sideBySide(x, y);
      w[j] = x;
      w[2 + j] = y;
    }
    if (c + 8 <= cols) {
      *reinterpret_cast<u32x4_anywhere *>(row + c) = w;
    } else {
#pragma unroll
      for (int j = 0; j < 8; j++)
        if (c + j < cols) reinterpret_cast<uint16_t *>(row)[c + j] = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
    }
  }
}

// ---------------------------------------------------------------- the kernel

// WN x WM wavefronts, each with a (BN / WN) x (BM / WM) part of the tile.
template <class T, class Out, int BN, int BM, int WN, int WM, bool NACROSS, bool MACROSS, bool DW>
struct Product {
  static constexpr int kThreads = WN * WM * 64, ES = kBytes<T>;
  static constexpr int TN = BN / WN, TM = BM / WM, FN = TN / 16, FM = TM / 16;
  static constexpr bool kScaled = ES == 1;
  static_assert(TN % 64 == 0 && TM % 16 == 0, "whole fragments");
  using N = Side<BN, kThreads, ES, NACROSS, true>;
  using M = Side<BM, kThreads, ES, MACROSS, false>;
  static constexpr uint32_t kSlab = N::kSlab;
  static constexpr int kLdsN = BN * 128, kLdsM = BM * 128;

  f32x4 acc[FN][FM];
  uint32_t i, g, wn, wm;

  __device__ __forceinline__ void init() {
    const uint32_t wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
    i = lane & 15;
    g = lane >> 4;
    wn = (wave % WN) * TN;
    wm = (wave / WN) * TM;
#pragma unroll
    for (int f = 0; f < FN; f++)
#pragma unroll
      for (int h = 0; h < FM; h++) acc[f][h] = f32x4{};
  }

  __device__ __forceinline__ u32x4 readN(const char *lds, int f, int half) const {
    if constexpr (NACROSS) return readAcross<BN>(lds, wn, f, half, i, g);
    else return readAlong<true>(lds, wn, f, half, i, g);
  }
  __device__ __forceinline__ u32x4 readM(const char *lds, int f, int half) const {
    if constexpr (MACROSS) return readAcross<BM>(lds, wm, f, half, i, g);
    else return readAlong<false>(lds, wm, f, half, i, g);
  }

  // One slab from LDS.  scale: this slab's m-side scale per fragment, times the n side's
  __device__ __forceinline__ void slab(const char *ln, const char *lm, const float (&scale)[FM]) {
    if constexpr (kScaled) {
      u32x4 n[FN][2];
#pragma unroll
      for (int f = 0; f < FN; f++)
#pragma unroll
        for (int h = 0; h < 2; h++) n[f][h] = readN(ln, f, h);
#pragma unroll
      for (int q = 0; q < FM; q++) {
        const u32x4 m[2] = {readM(lm, q, 0), readM(lm, q, 1)};
#pragma unroll
        for (int f = 0; f < FN; f++) {
          const f32x4 p = mma8<T>(n[f], m);
#pragma unroll
          for (int v = 0; v < 4; v++) acc[f][q][v] = __builtin_fmaf(p[v], scale[q], acc[f][q][v]);
        }
      }
    } else {
#pragma unroll
      for (int h = 0; h < 2; h++) {
        u32x4 n[FN];
#pragma unroll
        for (int f = 0; f < FN; f++) n[f] = readN(ln, f, h);
#pragma unroll
        for (int q = 0; q < FM; q++) {
          const u32x4 m = readM(lm, q, h);
#pragma unroll
          for (int f = 0; f < FN; f++) acc[f][q] = mma<T>(n[f], m, acc[f][q]);
        }
      }
    }
  }

  __device__ __forceinline__ void store(const ProductArgs &a, const Tile &t) const {
    Out *y = (Out *)a.y + (DW ? (size_t)t.expert * a.expertY : 0);
#pragma unroll
    for (int q = 0; q < FM; q++) {
      const uint32_t m = t.m0 + wm + 16 * q + i;
      const bool live = m < t.mEnd;
      if (!NACROSS && !live) continue;        // the across form exchanges between lanes first
      Out *row = y + (size_t)m * a.ldy;
#pragma unroll
      for (int b = 0; b < FN / 2; b++) {
        const uint32_t c = t.n0 + wn + 32 * b + 8 * g;
        if constexpr (NACROSS) {
          storeAcross<Out>(row, live ? c : a.n, a.n, acc[2 * b][q], acc[2 * b + 1][q]);
        } else {
          float v[8];
#pragma unroll
          for (int j = 0; j < 8; j++) v[j] = acc[2 * b + (j >> 2)][q][j & 3];
          storeRun(row, c, a.n, v);
        }
      }
    }
  }

  // m-side scales of slab s for this lane's rows, and the n side's block scale.
  // A wavefront's 64 columns lie in one block of 128; columns and rows that do not
  // exist take an existing scale (their products are not stored).
  __device__ __forceinline__ void scales(const ProductArgs &a, const Tile &t, uint32_t s, float (&rows)[FM], float &block) const {
    if constexpr (kScaled) {
      static_assert(TN == 64, "one block scale per wavefront");
      const uint32_t last = (a.n - 1) / FX_SCALE_GROUP, b = (t.n0 + wn) / FX_SCALE_GROUP;
      block = a.sn[(size_t)t.expert * a.expertSn + (size_t)(b < last ? b : last) * a.ldsn + s];
#pragma unroll
      for (int q = 0; q < FM; q++) {
        const uint32_t m = t.m0 + wm + 16 * q + i;
        rows[q] = a.sm[(size_t)(m < t.mEnd ? m : t.mEnd - 1) * a.ldsm + s];
      }
    }
  }
};

// Any alignment and any sizes: chunks go through registers, and the next slab's are on
// their way while this one is multiplied.  No branch stands between the loads: a
// chunk that a row ends in, or that lies behind its end, is loaded from the row's last
// whole chunk and shifted into place on its way to LDS, and rows that do not exist
// are loaded from the last one that does; of these, only what lies behind the end of
// the reduction has to become zeros (the rest meets no result that is stored).
// 16384 rows of 16 experts, n = 4096: k = 4096 538 us (direct), 4100 830, 4101 986; the
// unaligned loads bound it, a second slab on its way gained nothing.  Tiles of 64 where
// the account below puts them ahead (1024 rows of 8 experts, 1029 x 2053: 42 -> 29 us).
template <int R, int NT, int ES, bool ACROSS, bool NSIDE>
struct NearSide : Side<R, NT, ES, ACROSS, NSIDE> {
  using S = Side<R, NT, ES, ACROSS, NSIDE>;
  const char *p[S::kLoads];       // this thread's chunks of the slab to load next
  size_t ld, advance;             // bytes
  uint32_t own, redLast, drop;    // redLast: reduction elements of the last slab; drop: bytes that a chunk starts too early
  __device__ __forceinline__ void start(const char *base, size_t elements, uint32_t ownHere, uint32_t red) {
    S::init();
    ld = elements * ES;
    own = ownHere;
    redLast = red;
    advance = ACROSS ? S::kSlab * ld : 128;
    const int32_t c = (int32_t)(S::chunk * S::kElems), end = (int32_t)(ACROSS ? own : red) - S::kElems;
    drop = c > end ? (uint32_t)(c - end) * ES : 0;
#pragma unroll
    for (int i = 0; i < S::kLoads; i++) {
      const uint32_t r = S::row + i * S::kStep;
      p[i] = base + (size_t)(ACROSS || r < own ? r : own - 1) * ld + S::chunk * 16 - (ACROSS ? drop : 0);
    }
  }
  __device__ __forceinline__ void load(u32x4 (&v)[S::kLoads], bool last) {
    if (last)
#pragma unroll
      for (int i = 0; i < S::kLoads; i++) {
        const uint32_t r = S::row + i * S::kStep;
        if (!ACROSS) p[i] -= drop;
        else if (r >= redLast) p[i] -= (size_t)(r - redLast + 1) * ld;
      }
#pragma unroll
    for (int i = 0; i < S::kLoads; i++) {
      v[i] = *reinterpret_cast<const u32x4_anywhere *>(p[i]);
      p[i] += advance;
    }
  }
  __device__ __forceinline__ void store(char *lds, u32x4 (&v)[S::kLoads], bool last) const {
    if (ACROSS ? own < R : last)
#pragma unroll
      for (int i = 0; i < S::kLoads; i++) v[i] = dropFront(v[i], drop);
    if (ACROSS && last)
#pragma unroll
      for (int i = 0; i < S::kLoads; i++)
        if (S::row + i * S::kStep >= redLast) v[i] = u32x4{};
#pragma unroll
    for (int i = 0; i < S::kLoads; i++) *reinterpret_cast<u32x4 *>(lds + (i * NT + threadIdx.x) * 16) = v[i];
  }
};

template <class T, class Out, int BN, int BM, int WN, int WM, bool NACROSS, bool MACROSS, bool DW>
__global__ void __launch_bounds__(WN *WM * 64, (__is_same(T, E4m3Exact) ? 1 : 2)) productNear(ProductArgs a) {
  using P = Product<T, Out, BN, BM, WN, WM, NACROSS, MACROSS, DW>;
  constexpr int kStage = P::kLdsN + P::kLdsM;
  __shared__ __attribute__((aligned(1024))) char lds[2 * kStage];
  Tile t;
  if (!(DW ? findTileDw<BN, BM>(a, &t) : findTile<BN, BM, true>(a, &t))) return;
  P p;
  p.init();
  const size_t nAt = NACROSS ? (size_t)t.k0 * a.ldn + t.n0 : (size_t)t.n0 * a.ldn + t.k0;
  const size_t mAt = MACROSS ? (size_t)t.k0 * a.ldm + t.m0 : (size_t)t.m0 * a.ldm + t.k0;
  const uint32_t slabs = (t.kLen + P::kSlab - 1) / P::kSlab;
  if (slabs) {
    NearSide<BN, P::kThreads, P::ES, NACROSS, true> sn;
    NearSide<BM, P::kThreads, P::ES, MACROSS, false> sm;
    const uint32_t redLast = t.kLen - (slabs - 1) * P::kSlab;
    sn.start((const char *)a.pn + (nAt + (DW ? 0 : (size_t)t.expert * a.expertN)) * P::ES, a.ldn, a.n - t.n0, redLast);
    sm.start((const char *)a.pm + mAt * P::ES, a.ldm, t.mEnd - t.m0, redLast);
    u32x4 vn[P::N::kLoads], vm[P::M::kLoads];
    float rows[P::FM], block = 0.f;
    sn.load(vn, slabs == 1);
    sm.load(vm, slabs == 1);
    p.scales(a, t, 0, rows, block);
    sn.store(lds, vn, slabs == 1);
    sm.store(lds + P::kLdsN, vm, slabs == 1);
    for (uint32_t s = 0; s < slabs; s++) {
      const char *now = lds + (s & 1) * kStage;
      char *then = lds + (~s & 1) * kStage;
      const bool more = s + 1 < slabs, last = s + 2 == slabs;
      float scale[P::FM];
#pragma unroll
      for (int q = 0; q < P::FM; q++) scale[q] = P::kScaled ? rows[q] * block : 0.f;
      __syncthreads();
      if (more) {
        sn.load(vn, last);
        sm.load(vm, last);
        p.scales(a, t, s + 1, rows, block);
      }
      p.slab(now, now + P::kLdsN, scale);
      if (more) {
        sn.store(then, vn, last);
        sm.store(then + P::kLdsN, vm, last);
      }
    }
  }
  p.store(a, t);
}

// Rows of less than a chunk: element by element.
template <class T, class Out, int BN, int BM, int WN, int WM, bool NACROSS, bool MACROSS, bool DW>
__global__ void __launch_bounds__(WN *WM * 64) productGuarded(ProductArgs a) {
  using P = Product<T, Out, BN, BM, WN, WM, NACROSS, MACROSS, DW>;
  __shared__ __attribute__((aligned(1024))) char lds[P::kLdsN + P::kLdsM];
  char *ln = lds, *lm = lds + P::kLdsN;
  Tile t;
  if (!(DW ? findTileDw<BN, BM>(a, &t) : findTile<BN, BM, true>(a, &t))) return;
  P p;
  p.init();
  typename P::N sn;
  typename P::M sm;
  sn.init();
  sm.init();
  const size_t nAt = NACROSS ? (size_t)t.k0 * a.ldn + t.n0 : (size_t)t.n0 * a.ldn + t.k0;
  const size_t mAt = MACROSS ? (size_t)t.k0 * a.ldm + t.m0 : (size_t)t.m0 * a.ldm + t.k0;
  const char *bn = (const char *)a.pn + (nAt + (DW ? 0 : (size_t)t.expert * a.expertN)) * P::ES;
  const char *bm = (const char *)a.pm + mAt * P::ES;
  const uint32_t ownN = a.n - t.n0, ownM = t.mEnd - t.m0;
  const uint32_t slabs = (t.kLen + P::kSlab - 1) / P::kSlab;
  u32x4 vn[P::N::kLoads], vm[P::M::kLoads];
  auto load = [&](uint32_t s) {
    const uint32_t k = s * P::kSlab, red = t.kLen - k;
    const char *pn = bn + (NACROSS ? (size_t)k * a.ldn : (size_t)k) * P::ES;
    const char *pm = bm + (MACROSS ? (size_t)k * a.ldm : (size_t)k) * P::ES;
#pragma unroll
    for (int q = 0; q < P::N::kLoads; q++) vn[q] = sn.guarded(pn, a.ldn, q, ownN, red);
#pragma unroll
    for (int q = 0; q < P::M::kLoads; q++) vm[q] = sm.guarded(pm, a.ldm, q, ownM, red);
  };
  if (slabs) load(0);
  for (uint32_t s = 0; s < slabs; s++) {
    float scale[P::FM], rows[P::FM], block = 0.f;
    p.scales(a, t, s, rows, block);
#pragma unroll
    for (int q = 0; q < P::FM; q++) scale[q] = P::kScaled ? rows[q] * block : 0.f;
    __syncthreads();
#pragma unroll
    for (int q = 0; q < P::N::kLoads; q++) *reinterpret_cast<u32x4 *>(ln + (q * P::kThreads + threadIdx.x) * 16) = vn[q];
#pragma unroll
    for (int q = 0; q < P::M::kLoads; q++) *reinterpret_cast<u32x4 *>(lm + (q * P::kThreads + threadIdx.x) * 16) = vm[q];
    __syncthreads();
    if (s + 1 < slabs) load(s + 1);
    p.slab(ln, lm, scale);
  }
  p.store(a, t);
}

// Aligned operands: the chunks go from memory to LDS without passing through
// registers (buffer loads with the LDS flag), one slab ahead, into the other of
// two buffers.  A wavefront's 64 chunks land in 1024 consecutive bytes, so the
// exchange of chunks is in the addresses that the lanes load from.  Chunks that
// do not exist are given an offset outside the buffer and arrive as zeros.
//
// The loads are issued from inline assembly (they have no register outputs): the
// compiler does not know that they write LDS, and every read of LDS behind one
// would otherwise wait for it.  The waits are therefore written here: a slab is
// read only behind a wait for all of this wavefront's loads and a barrier.  The LDS
// address is an operand in m0, so the compiler knows what that register holds.
constexpr uint32_t kOutside = 0x80000000u;
__device__ __forceinline__ void loadToLds(uint32_t ldsAt, uint32_t voff, __amdgpu_buffer_rsrc_t rsrc, uint32_t soff) {
  asm volatile("s_nop 0\n\tbuffer_load_dwordx4 %1, %2, %3 offen lds" ::"{m0}"(ldsAt), "v"(voff), "s"(rsrc), "s"(soff));
}
// `left` = loads of this wavefront that may still be on their way.
template <int left>
__device__ __forceinline__ void waitAndMeet() {
  static_assert(left < 64, "six bits of counter");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(left) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

template <int R, int NT, int ES, bool ACROSS, bool NSIDE>
struct DirectSide : Side<R, NT, ES, ACROSS, NSIDE> {
  using S = Side<R, NT, ES, ACROSS, NSIDE>;
  uint32_t voff[S::kLoads];
  uint32_t step;          // bytes between a thread's chunks
  uint64_t at, advance;   // address of the slab to load next; bytes per slab
  __device__ __forceinline__ void start(const char *base, size_t ld, uint32_t own) {
    S::init();
    step = uniform((uint32_t)(S::kStep * ld * ES));
    at = (uint64_t)(uintptr_t)base;
    advance = ACROSS ? S::kSlab * ld * ES : 128;
#pragma unroll
    for (int q = 0; q < S::kLoads; q++)
      voff[q] = (ACROSS ? S::chunk * S::kElems < own : S::row + q * S::kStep < own) ? (uint32_t)((S::row * ld + S::chunk * S::kElems) * ES) : kOutside;
  }
  __device__ __forceinline__ void skip(int64_t slabs) { at += slabs * (int64_t)advance; }
  // red: reduction elements left from this slab on
  __device__ __forceinline__ void issue(uint32_t lds, uint32_t wave, uint32_t red) {
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)(uintptr_t)at, 0, 0x7fffffff, 0x00020000);
#pragma unroll
    for (int q = 0; q < S::kLoads; q++) {
      const bool there = ACROSS ? S::row + q * S::kStep < red : S::chunk * S::kElems < red;
      loadToLds(lds + (q * NT + wave * 64) * 16, there ? voff[q] : kOutside, rsrc, q * step);
    }
    at += advance;
  }
};

// The e4m3 rows' scales of one slab, one float per row of the tile, brought to LDS.
// Every wavefront issues one load, also those without a row, so that all count alike.
template <int BM>
struct DirectScales {
  uint32_t voff;
  uint64_t at;
  __device__ __forceinline__ void start(const float *base, size_t ld, uint32_t own) {
    const uint32_t row = threadIdx.x;
    voff = row < BM && row < own ? (uint32_t)(row * ld * 4) : kOutside;
    at = (uint64_t)(uintptr_t)base;
  }
  __device__ __forceinline__ void issue(uint32_t lds, uint32_t wave, bool there) {
    const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)(uintptr_t)at, 0, 0x7fffffff, 0x00020000);
    asm volatile("s_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"{m0}"(lds + wave * 256),
                 "v"(there ? voff : kOutside), "s"(rsrc));
    at += 4;
  }
};

// TOUCH: the largest e4m3 tile has LDS for two buffers only, and one slab's time is
// less than memory takes under load.  Two wavefronts also touch lines of a slab
// further on, four bytes of each that nobody reads, which brings them into the die's
// cache; neighbouring tiles share a slab's lines out among them.  Loads return in
// order; the wait for a slab leaves the last touch out, so it has two slabs' time.
// (8192^3 from memory 588 -> 543 us; 4096 rows each of 4 experts, 4096 x 4096, 352 ->
// 339; where few tiles share weights it gains nothing.)
constexpr uint32_t kTouchAhead = 4;
constexpr uint32_t kTurn = 37;

// The slabs as a pipeline.  A slab is multiplied in phases; the fragments of
// the next phase are read from LDS while this one's are multiplied.  In front of
// the last phase all of a slab's fragments are in registers: there the wavefronts
// meet, its buffers are handed to the loads of slabs further on, and the next
// slab, whose loads have had SN - 1 and SM - 1 slabs' time, is read from.  (Weights
// come from memory more often than rows do, and have the deeper ring where LDS
// allows.)  Loads past the last slab have no lanes inside the buffer and read nothing.
//
// 16 bits: two halves of the reduction, each with two groups of m fragments.
// e4m3, eight m fragments to a wavefront: a phase is two m fragments and takes the n
// fragments in turn, two products with each, so that in a slab's last phase an n
// fragment's successor is read six products ahead of its use (registers: 128 of
// accumulators, 32 of n, 32 of m fragments; a phase of one m fragment: 362 us against
// 346 for 16384 rows of 16 experts, 4096 x 4096).  A product of 128 goes to registers of
// its own and is scaled into the accumulators three products later, in the shadow of the
// matrix instructions (two later 353 us, one later 384).  Without the scaling 8192^3
// would take 440 us, without reading fragments 408, with neither 406; it takes 508 (warm:
// the same operands call after call; with others in turn all of these are 20 to 40 longer).
#define FX_FENCE() __builtin_amdgcn_sched_barrier(0)

// Two wavefronts to a SIMD, from one workgroup or from two, where LDS holds them.
template <class T, int THREADS, int LDS>
constexpr int kToSimd = THREADS >= 512 || (THREADS == 256 && 2 * LDS <= 160 * 1024 && !__is_same(T, E4m3Exact)) ? 2 : 1;

template <class T, class Out, int BN, int BM, int WN, int WM, int SN, int SM, bool NACROSS, bool MACROSS, bool DW, bool TOUCH>
__global__ void __launch_bounds__(WN *WM * 64, (kToSimd<T, WN * WM * 64, (SN * BN + SM * BM) * 128 + SM * WN * WM * 256>)) productDirect(ProductArgs a) {
  using P = Product<T, Out, BN, BM, WN, WM, NACROSS, MACROSS, DW>;
  constexpr uint32_t kStageM = P::kLdsM + (P::kScaled ? P::kThreads * 4 : 0), kLds = SN * P::kLdsN + SM * kStageM;
  constexpr int kLoadsN = P::N::kLoads + TOUCH, kLoadsM = P::M::kLoads + P::kScaled;   // per thread and slab
  static_assert(BM <= P::kThreads && SN >= SM && SM >= 2, "a thread per row's scale");
  static_assert(!TOUCH || (!NACROSS && !MACROSS && BN == 256 && BM == 256 && SN == 2), "lines as rows");
  __shared__ __attribute__((aligned(1024))) char lds[kLds + (TOUCH ? 256 : 0)];
  typedef __attribute__((address_space(3))) char *ldsPtr;
  const uint32_t lds0 = (uint32_t)(uintptr_t)(ldsPtr)lds;
  Tile t;
  if (!(DW ? findTileDw<BN, BM>(a, &t) : findTile<BN, BM, true>(a, &t))) return;
  P p;
  p.init();
  const uint32_t wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63;
  DirectSide<BN, P::kThreads, P::ES, NACROSS, true> sn;
  DirectSide<BM, P::kThreads, P::ES, MACROSS, false> sm;
  DirectScales<BM> ss;
  const size_t nAt = NACROSS ? (size_t)t.k0 * a.ldn + t.n0 : (size_t)t.n0 * a.ldn + t.k0;
  const size_t mAt = MACROSS ? (size_t)t.k0 * a.ldm + t.m0 : (size_t)t.m0 * a.ldm + t.k0;
  sn.start((const char *)a.pn + (nAt + (DW ? 0 : (size_t)t.expert * a.expertN)) * P::ES, a.ldn, a.n - t.n0);
  sm.start((const char *)a.pm + mAt * P::ES, a.ldm, t.mEnd - t.m0);
  const float *blockScale = nullptr;
  if constexpr (P::kScaled) {
    ss.start(a.sm + (size_t)t.m0 * a.ldsm, a.ldsm, t.mEnd - t.m0);
    const uint32_t last = (a.n - 1) / FX_SCALE_GROUP, b = (t.n0 + p.wn) / FX_SCALE_GROUP;
    blockScale = a.sn + (size_t)t.expert * a.expertSn + (size_t)(b < last ? b : last) * a.ldsn;
  }
  const uint32_t slabs = (t.kLen + P::kSlab - 1) / P::kSlab;
  // The slabs s + SM of the m side and s + SN of the n side, into the buffers of slab s.
  // left: reduction elements from the next slab to the end, 0 when all have been issued.
  // Experts start their walk at different slabs and wrap around: rows lie a power of two
  // apart more often than not, and all workgroups at the same slab meet on the same
  // memory channels, while an expert's own workgroups share what they read (64 rows each
  // of 16 experts, 4096 x 4096: 130 -> 99 us; 16 each of 64 experts: 249 -> 176 us).
  const uint32_t turn = DW || !slabs ? 0 : t.expert * kTurn % slabs;
  uint32_t curN = 0, curM = SN * P::kLdsN, leftN = t.kLen - turn * P::kSlab, leftM = leftN, todoN = slabs, todoM = slabs;
  if constexpr (!DW) {
    sn.skip(turn);
    sm.skip(turn);
  }
  if constexpr (P::kScaled) ss.at += turn * 4;
  auto nextOf = [&](auto &side, uint32_t &left, uint32_t &todo) {
    if constexpr (DW) {
      left = left > P::kSlab ? left - P::kSlab : 0;
      return false;
    } else {
      const bool wrap = left <= P::kSlab;
      todo -= todo != 0;
      if (wrap) side.skip(-(int64_t)slabs);
      left = todo == 0 ? 0 : wrap ? t.kLen : left - P::kSlab;
      return wrap;
    }
  };
  uint32_t touched = kOutside;
  if constexpr (TOUCH) {
    const uint32_t rn = t.m0 / BM % 8 * 32 + lane, rm = t.n0 / BN % 4 * 64 + lane;
    if (wave == 0 && lane < 32 && rn < a.n - t.n0) touched = (uint32_t)(rn * a.ldn * P::ES);
    if (wave == 1 && rm < t.mEnd - t.m0) touched = (uint32_t)(rm * a.ldm * P::ES);
  }
  auto issueN = [&] {
    sn.issue(lds0 + curN, wave, leftN);
    if constexpr (TOUCH) {                    // sn.at is a slab further already, and sm.at too
      const uint64_t from = (wave == 0 ? sn.at : sm.at) + (kTouchAhead - 1) * 128;
      const __amdgpu_buffer_rsrc_t rsrc = __builtin_amdgcn_make_buffer_rsrc((void *)(uintptr_t)from, 0, 0x7fffffff, 0x00020000);
      asm volatile("s_nop 0\n\tbuffer_load_dword %1, %2, 0 offen lds" ::"{m0}"(lds0 + kLds),
                   "v"(leftN > kTouchAhead * P::kSlab ? touched : kOutside), "s"(rsrc));
    }
    nextOf(sn, leftN, todoN);
    curN = curN + P::kLdsN < SN * P::kLdsN ? curN + P::kLdsN : 0;
  };
  auto issueM = [&] {
    sm.issue(lds0 + curM, wave, leftM);
    if constexpr (P::kScaled) ss.issue(lds0 + curM + P::kLdsM, wave, leftM != 0);
    const bool wrapped = nextOf(sm, leftM, todoM);
    if constexpr (P::kScaled)
      if (wrapped) ss.at -= (uint64_t)slabs * 4;
    curM = curM + kStageM < kLds ? curM + kStageM : SN * P::kLdsN;
  };
  // The block's scale of the walk's s-th slab; lane l of `blocks` holds slab 64 * (slab / 64) + l's.
  auto scaleOf = [&](float &blocks, uint32_t s) {
    uint32_t at = s + turn;
    at = at < slabs ? at : at - slabs;
    if (s == 0 || (at & 63) == 0) blocks = (at & ~63u) + lane < slabs ? blockScale[(at & ~63u) + lane] : 0.f;
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, blocks), (int)(at & 63)));
  };
  if (slabs) {
#pragma unroll
    for (int q = 0; q < SN; q++) {
      if (q < SM) issueM();
      issueN();
    }
    waitAndMeet<(SM - 1) * kLoadsM + (SN - 1) * kLoadsN + TOUCH>();
    const char *ln = lds, *lm = lds + SN * P::kLdsN;
    auto nextSlab = [&] {
      FX_FENCE();
      waitAndMeet<(SM - 2) * kLoadsM + (SN - 2) * kLoadsN + TOUCH>();
      issueM();
      issueN();
      ln = lds + curN;
      lm = lds + curM;
    };
    // An expert's last tile may have no row for this wavefront, or rows for half of its
    // fragments at most.
    const bool few = !DW && t.m0 + p.wm + P::TM / 2 >= t.mEnd;
    if (t.m0 + p.wm >= t.mEnd) {
      for (uint32_t s = 0; s < slabs; s++) nextSlab();
    } else if constexpr (P::kScaled && P::FM <= 4) {
      // Small e4m3 tiles: all of a slab's fragments are read a slab ahead.
      struct Slab {
        u32x4 n[P::FN][2], m[P::FM][2];
        float scale[P::FM];
      } even, odd;
      float blocks = 0.f;
      auto read = [&](Slab &b) {
#pragma unroll
        for (int f = 0; f < P::FN; f++)
#pragma unroll
          for (int h = 0; h < 2; h++) b.n[f][h] = p.readN(ln, f, h);
#pragma unroll
        for (int q = 0; q < P::FM; q++) {
#pragma unroll
          for (int h = 0; h < 2; h++) b.m[q][h] = p.readM(lm, q, h);
          b.scale[q] = *reinterpret_cast<const float *>(lm + P::kLdsM + (p.wm + 16 * q + p.i) * 4);
        }
      };
      auto multiply = [&](const Slab &b, uint32_t s) {
        const float sb = scaleOf(blocks, s);
        f32x4 part[3];
        float w[P::FM];
        auto scaled = [&](int at) {
          const int f = at % P::FN, q = at / P::FN;
#pragma unroll
          for (int v = 0; v < 4; v++) p.acc[f][q][v] = __builtin_fmaf(part[at % 3][v], w[q], p.acc[f][q][v]);
          asm volatile("" : "+v"(p.acc[f][q]));   // see below
        };
#pragma unroll
        for (int q = 0; q < P::FM; q++) w[q] = b.scale[q] * sb;
#pragma unroll
        for (int at = 0; at < P::FM * P::FN; at++) {
          part[at % 3] = mma8<T>(b.n[at % P::FN], b.m[at / P::FN]);
          if (at >= 2) scaled(at - 2);
          FX_FENCE();
        }
        scaled(P::FM * P::FN - 2);
        scaled(P::FM * P::FN - 1);
      };
      auto step = [&](uint32_t s, const Slab &now, Slab &then) {
        nextSlab();
        FX_FENCE();
        read(then);
        FX_FENCE();
        multiply(now, s);
      };
      read(even);
      uint32_t s = 0;
      for (; s + 1 < slabs; s += 2) {
        step(s, even, odd);
        step(s + 1, odd, even);
      }
      if (s < slabs) step(s, even, odd);
    } else if constexpr (P::kScaled) {
      u32x4 n[P::FN][2], m[2][2][2];
      constexpr int kBehind = 3;              // products between one and its scaling
      f32x4 part[kBehind + 1];
      float scale[2][2], blocks = 0.f;
      auto readM = [&](int buffer, int pair) {
#pragma unroll
        for (int j = 0; j < 2; j++) {
          m[buffer][j][0] = p.readM(lm, 2 * pair + j, 0);
          m[buffer][j][1] = p.readM(lm, 2 * pair + j, 1);
          scale[buffer][j] = *reinterpret_cast<const float *>(lm + P::kLdsM + (p.wm + 16 * (2 * pair + j) + p.i) * 4);
        }
      };
      auto readN = [&](int f) {
        n[f][0] = p.readN(ln, f, 0);
        n[f][1] = p.readN(ln, f, 1);
      };
      auto walk = [&](auto fragments) {
        constexpr int Q = decltype(fragments)::value, kPhases = Q / 2, kAll = Q * P::FN;
        static_assert(kPhases % 2 == 0, "pair 0 goes to buffer 0");
        float w[Q];
        auto scaled = [&](int at) {           // product `at` into its accumulators
          const int f = at / 2 % P::FN, q = at / (2 * P::FN) * 2 + at % 2;
#pragma unroll
          for (int v = 0; v < 4; v++) p.acc[f][q][v] = __builtin_fmaf(part[at % (kBehind + 1)][v], w[q], p.acc[f][q][v]);
          asm volatile("" : "+v"(p.acc[f][q]));   // here, not sunk behind the slab with all products alive
        };
        readM(0, 0);
#pragma unroll
        for (int f = 0; f < P::FN; f++) readN(f);
        for (uint32_t s = 0; s < slabs; s++) {
          const float sb = scaleOf(blocks, s);
#pragma unroll
          for (int ph = 0; ph < kPhases; ph++) {
            if (ph == kPhases - 1) nextSlab();
            FX_FENCE();
#pragma unroll
            for (int j = 0; j < 2; j++) w[2 * ph + j] = scale[ph & 1][j] * sb;
            readM((ph + 1) & 1, (ph + 1) % kPhases);
            FX_FENCE();
#pragma unroll
            for (int f = 0; f < P::FN; f++)
#pragma unroll
              for (int j = 0; j < 2; j++) {
                const int at = (ph * P::FN + f) * 2 + j;
                part[at % (kBehind + 1)] = mma8<T>(n[f], m[ph & 1][j]);
                if (at >= kBehind) scaled(at - kBehind);
                FX_FENCE();
                if (j == 1 && ph == kPhases - 1) readN(f);
              }
          }
#pragma unroll
          for (int at = kAll - kBehind; at < kAll; at++) scaled(at);
        }
      };
      if (few) walk(std::integral_constant<int, P::FM / 2>());
      else walk(std::integral_constant<int, P::FM>());
    } else {
      constexpr int GQ = P::FM / 2;
      u32x4 n[2][P::FN], m[2][GQ];
      auto readN = [&](int half) {
#pragma unroll
        for (int f = 0; f < P::FN; f++) n[half][f] = p.readN(ln, f, half);
      };
      auto walk = [&](auto groups) {            // of m fragments
        constexpr int G = decltype(groups)::value, kPhases = 2 * G;
        auto readM = [&](int ph) {
#pragma unroll
          for (int j = 0; j < GQ; j++) m[ph & 1][j] = p.readM(lm, ph % G * GQ + j, ph / G);
        };
        readN(0);
        readM(0);
        for (uint32_t s = 0; s < slabs; s++) {
#pragma unroll
          for (int ph = 0; ph < kPhases; ph++) {
            if (ph == kPhases - 1) nextSlab();
            FX_FENCE();
            readM((ph + 1) % kPhases);
            if (ph == 0) readN(1);
            if (ph == kPhases - 1) readN(0);
            FX_FENCE();
#pragma unroll
            for (int j = 0; j < GQ; j++)
#pragma unroll
              for (int f = 0; f < P::FN; f++) {
                const int q = ph % G * GQ + j;
                p.acc[f][q] = mma<T>(n[ph / G][f], m[ph & 1][j], p.acc[f][q]);
              }
            FX_FENCE();
          }
        }
      };
      if (few) walk(std::integral_constant<int, 1>());
      else walk(std::integral_constant<int, 2>());
    }
  }
  // The loads behind the last slab have to have ended before this workgroup's LDS is another's.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  p.store(a, t);
}

// Few rows per expert: the weights are read once, straight into registers, and
// memory bounds the call.  A workgroup owns 16 RN columns of the output and up to
// 16 FM rows; its wavefronts share the reduction, slab by slab in turn (so that
// together they read long runs of each weight row), and their partial sums meet
// in LDS in a fixed order.  U slabs are loaded while U are multiplied, without a
// branch: lanes without a row, a column or a slab load from outside the buffer,
// which touches no memory and gives zeros.  Each tile starts at another slab,
// because tiles that walk rows a power of two apart in step meet on the same
// memory channels (one token through 8 of 64 experts 28.9 -> 26.1 us).  e4m3
// operands are widened to bf16, whose sums are those of fp32: the matrix cores
// have time.
__device__ __forceinline__ u32x4 loadRaw16(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t soff) {
  return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(r, (int)voff, (int)soff, 0));
}
__device__ __forceinline__ float loadRaw4(__amdgpu_buffer_rsrc_t r, uint32_t voff, uint32_t soff) {
  return __builtin_bit_cast(float, __builtin_amdgcn_raw_buffer_load_b32(r, (int)voff, (int)soff, 0));
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t bufferAt(const void *p) {
  const uint64_t at = (uint64_t)(uintptr_t)p;
  const uint64_t u = (uint64_t)uniform((uint32_t)at) | ((uint64_t)uniform((uint32_t)(at >> 32)) << 32);
  return __builtin_amdgcn_make_buffer_rsrc((void *)(uintptr_t)u, 0, 0x7fffffff, 0x00020000);
}

// ODD: rows at any byte.  Loads that are not a multiple of four bytes from the start
// of memory's words run at half the rate, so the words that hold a chunk are loaded,
// a fifth one where it ends in one, and shifted before they are multiplied (4 rows
// each of 16 experts, 2053 x 2053: 53 -> 32 us; 2048 x 2048: 24).
template <class T, int RN, int FM, int NW, int U, bool ODD>
struct Thin {
  static constexpr int ES = kBytes<T>, kElems = 16 / ES;
  static constexpr bool kScaled = ES == 1;
  static constexpr uint32_t kSlab = 128 / ES;
  struct Batch {
    u32x4 w[U][RN][2], x[U][FM][2];
    float sx[U][FM], sb[U][RN];
    float wEnd[ODD ? U : 1][RN][2], xEnd[ODD ? U : 1][FM][2];   // bits of the fifth words
  };
  uint32_t wEndAt[RN], xEndAt[FM], wShift[RN], xShift[FM];
  f32x4 acc[RN][FM];
  __amdgpu_buffer_rsrc_t bw, bx, bs, bb;
  uint32_t ow[RN], ox[FM], os[FM], ob[RN];
  uint32_t full, turn;            // whole slabs; the slab this tile starts at

  __device__ __forceinline__ void load(Batch &b, uint32_t s0) const {
#pragma unroll
    for (int u = 0; u < U; u++) {
      uint32_t s = s0 + u * NW;
      const uint32_t out = s < full ? 0 : kOutside;
      s += turn;
      s = s >= full ? s - full : s;
#pragma unroll
      for (int h = 0; h < 2; h++) {
#pragma unroll
        for (int r = 0; r < RN; r++) b.w[u][r][h] = loadRaw16(bw, (ow[r] + h * 64) | out, s * 128);
#pragma unroll
        for (int f = 0; f < FM; f++) b.x[u][f][h] = loadRaw16(bx, (ox[f] + h * 64) | out, s * 128);
        if constexpr (ODD) {
#pragma unroll
          for (int r = 0; r < RN; r++) b.wEnd[u][r][h] = loadRaw4(bw, (wEndAt[r] + h * 64) | out, s * 128);
#pragma unroll
          for (int f = 0; f < FM; f++) b.xEnd[u][f][h] = loadRaw4(bx, (xEndAt[f] + h * 64) | out, s * 128);
        }
      }
      if constexpr (kScaled) {
#pragma unroll
        for (int f = 0; f < FM; f++) b.sx[u][f] = loadRaw4(bs, os[f] | out, s * 4);
#pragma unroll
        for (int r = 0; r < RN; r++) b.sb[u][r] = loadRaw4(bb, ob[r] | out, s * 4);
      }
    }
  }
  __device__ __forceinline__ static u32x4 shifted(u32x4 v, float end, uint32_t bytes) {
    const uint32_t e = __builtin_bit_cast(uint32_t, end);
    u32x4 o;
#pragma unroll
    for (int j = 0; j < 4; j++) o[j] = __builtin_amdgcn_alignbyte(j < 3 ? v[j < 3 ? j + 1 : 3] : e, v[j], bytes);
    return o;
  }
  __device__ __forceinline__ void multiply(const Batch &b) {
#pragma unroll
    for (int u = 0; u < U; u++) {
      u32x4 w[RN][2], x[FM][2];
#pragma unroll
      for (int h = 0; h < 2; h++) {
#pragma unroll
        for (int r = 0; r < RN; r++) w[r][h] = ODD ? shifted(b.w[u][r][h], b.wEnd[ODD ? u : 0][r][h], wShift[r]) : b.w[u][r][h];
#pragma unroll
        for (int f = 0; f < FM; f++) x[f][h] = ODD ? shifted(b.x[u][f][h], b.xEnd[ODD ? u : 0][f][h], xShift[f]) : b.x[u][f][h];
      }
#pragma unroll
      for (int f = 0; f < FM; f++)
#pragma unroll
        for (int r = 0; r < RN; r++) {
          if constexpr (kScaled) {
            const f32x4 p = mma8<E4m3Exact>(w[r], x[f]);
            const float sc = b.sx[u][f] * b.sb[u][r];
#pragma unroll
            for (int v = 0; v < 4; v++) acc[r][f][v] = __builtin_fmaf(p[v], sc, acc[r][f][v]);
          } else {
#pragma unroll
            for (int h = 0; h < 2; h++) acc[r][f] = mma<T>(w[r][h], x[f][h], acc[r][f]);
          }
        }
    }
  }
  // 16 bytes of a row from element c on, of which `cols` exist: from the row's last 16, shifted into place.
  __device__ __forceinline__ static u32x4 part(const char *row, uint32_t c, uint32_t cols) {
    u32x4 v = {};
    if (cols >= (uint32_t)kElems) {
      const uint32_t from = c < cols - kElems ? c : cols - kElems;
      return dropFront(*reinterpret_cast<const u32x4_anywhere *>(row + (size_t)from * ES), (c - from) * ES);
    }
#pragma unroll
    for (int j = 0; j < kElems; j++)
      if (c + j < cols) {
        if constexpr (ES == 2) v[j >> 1] |= (uint32_t) reinterpret_cast<const uint16_t *>(row)[c + j] << (16 * (j & 1));
        else v[j >> 2] |= (uint32_t) reinterpret_cast<const uint8_t *>(row)[c + j] << (8 * (j & 3));
      }
    return v;
  }

  __device__ __forceinline__ void run(const ProductArgs &a, const Tile &t, uint32_t wave, uint32_t i, uint32_t g) {
    const uint32_t own = t.mEnd - t.m0;
    full = a.k / kSlab;
    turn = full ? (t.n0 / (16 * RN) * 37 + t.expert * 11) % full : 0;
    const char *w0 = (const char *)a.pn + ((size_t)t.expert * a.expertN + (size_t)t.n0 * a.ldn) * ES;
    const char *x0 = (const char *)a.pm + (size_t)t.m0 * a.ldm * ES;
    const uint32_t w3 = ODD ? (uint32_t)(uintptr_t)w0 & 3 : 0, x3 = ODD ? (uint32_t)(uintptr_t)x0 & 3 : 0;
    bw = bufferAt(w0 - w3);
    bx = bufferAt(x0 - x3);
#pragma unroll
    for (int r = 0; r < RN; r++) {
      ow[r] = t.n0 + 16 * r + i < a.n ? (uint32_t)((16 * r + i) * a.ldn * ES) + g * 16 + w3 : kOutside;
      wShift[r] = ow[r] & 3;
      ow[r] &= ~3u;
      wEndAt[r] = wShift[r] ? ow[r] + 16 : kOutside;
    }
#pragma unroll
    for (int f = 0; f < FM; f++) {
      ox[f] = 16 * f + i < own ? (uint32_t)((16 * f + i) * a.ldm * ES) + g * 16 + x3 : kOutside;
      xShift[f] = ox[f] & 3;
      ox[f] &= ~3u;
      xEndAt[f] = xShift[f] ? ox[f] + 16 : kOutside;
    }
    const float *s0 = nullptr, *b0 = nullptr;
    if constexpr (kScaled) {
      s0 = a.sm + (size_t)t.m0 * a.ldsm;
      b0 = a.sn + (size_t)t.expert * a.expertSn;
      bs = bufferAt(s0);
      bb = bufferAt(b0);
#pragma unroll
      for (int f = 0; f < FM; f++) os[f] = 16 * f + i < own ? (uint32_t)((16 * f + i) * a.ldsm * 4) : kOutside;
#pragma unroll
      for (int r = 0; r < RN; r++) ob[r] = t.n0 + 16 * r < a.n ? (uint32_t)((t.n0 + 16 * r) / FX_SCALE_GROUP * a.ldsn * 4) : kOutside;
    }
#pragma unroll
    for (int r = 0; r < RN; r++)
#pragma unroll
      for (int f = 0; f < FM; f++) acc[r][f] = f32x4{};
    Batch b[2];
    load(b[0], wave);
    for (uint32_t s = wave; s < full; s += 2 * U * NW) {
      load(b[1], s + U * NW);
      multiply(b[0]);
      load(b[0], s + 2 * U * NW);
      multiply(b[1]);
    }
    // what is left behind the whole slabs: one wavefront, element by element
    if (a.k % kSlab && wave == full % NW) {
      Thin<T, RN, FM, NW, 1, false> last;
      typename Thin<T, RN, FM, NW, 1, false>::Batch e;
#pragma unroll
      for (int h = 0; h < 2; h++) {
        const uint32_t c = full * kSlab + (h * 4 + g) * kElems;
#pragma unroll
        for (int r = 0; r < RN; r++)
          e.w[0][r][h] = ow[r] < kOutside ? part(w0 + (size_t)(16 * r + i) * a.ldn * ES, c, a.k) : u32x4{};
#pragma unroll
        for (int f = 0; f < FM; f++)
          e.x[0][f][h] = ox[f] < kOutside ? part(x0 + (size_t)(16 * f + i) * a.ldm * ES, c, a.k) : u32x4{};
      }
      if constexpr (kScaled) {
#pragma unroll
        for (int f = 0; f < FM; f++) e.sx[0][f] = loadRaw4(bs, os[f], full * 4);
#pragma unroll
        for (int r = 0; r < RN; r++) e.sb[0][r] = loadRaw4(bb, ob[r], full * 4);
      }
#pragma unroll
      for (int r = 0; r < RN; r++)
#pragma unroll
        for (int f = 0; f < FM; f++) last.acc[r][f] = acc[r][f];
      last.multiply(e);
#pragma unroll
      for (int r = 0; r < RN; r++)
#pragma unroll
        for (int f = 0; f < FM; f++) acc[r][f] = last.acc[r][f];
    }
  }
};

// FM = 4 holds three bodies, for 16, 32 and 64 rows: what of a tile exists is
// known on the device only.
template <class T, class Out, int RN, int FM, int NW, int U, bool ODD>
__global__ void __launch_bounds__(NW * 64) productThin(ProductArgs a) {
  __shared__ f32x4 lds[NW][RN * FM][64];
  Tile t;
  if (!findTile<16 * RN, 16 * FM, false>(a, &t)) return;
  const uint32_t wave = uniform(threadIdx.x >> 6), lane = threadIdx.x & 63, i = lane & 15, g = lane >> 4;
  const uint32_t own = t.mEnd - t.m0, live = own >= 16 * FM ? FM : (own + 15) / 16;
  auto body = [&](auto rows) {
    constexpr int F = decltype(rows)::value;
    Thin<T, RN, F, NW, (F == FM ? U : F == 1 ? 4 * U : 2 * U), ODD> p;
    p.run(a, t, wave, i, g);
#pragma unroll
    for (int r = 0; r < RN; r++)
#pragma unroll
      for (int f = 0; f < F; f++) lds[wave][r * FM + f][lane] = p.acc[r][f];
  };
  if constexpr (FM == 4) {
    if (live == 1) body(std::integral_constant<int, 1>());
    else if (live == 2) body(std::integral_constant<int, 2>());
    else body(std::integral_constant<int, 4>());
  } else {
    body(std::integral_constant<int, FM>());
  }
  __syncthreads();
  for (uint32_t q = wave; q < RN * FM; q += NW) {
    const uint32_t r = q / FM, f = q % FM;
    if (f >= live) continue;
    f32x4 sum = lds[0][q][lane];
#pragma unroll
    for (int w = 1; w < NW; w++) sum += lds[w][q][lane];
    const uint32_t m = t.m0 + 16 * f + i;
    if (m < t.mEnd) {
      const float v[4] = {sum[0], sum[1], sum[2], sum[3]};
      storeRun((Out *)a.y + (size_t)m * a.ldy, t.n0 + 16 * r + 4 * g, a.n, v);
    }
  }
}

// ------------------------------------------------------------- launch tables

enum ProductForm { kFormNK = 0, kFormKN = 1, kFormDw = 2 };

// Implemented once per operand type (fx_product_*.hip).
flagcxResult_t launchProductBf16(const ProductArgs &a, int form, bool outF32, hipStream_t s);
flagcxResult_t launchProductF16(const ProductArgs &a, int form, bool outF32, hipStream_t s);
flagcxResult_t launchProductE4m3(const ProductArgs &a, int outDtype, hipStream_t s);

// A launch takes less than 2^32 threads: calls that need more (4096 experts with a row
// each and 64,000 columns) go through their columns in several.  colBytes, outBytes:
// from one column of the n side and of the output to the next; es: of an operand.
inline flagcxResult_t launchGrid(const void *kernel, ProductArgs a, uint32_t bn, uint32_t bm, bool dw, uint32_t threads, size_t es,
                                 size_t colBytes, size_t outBytes, hipStream_t s) {
  if (dw) a.mTiles = (a.m + bm - 1) / bm;
  else if (!a.offsets) a.mTiles = (a.rows + bm - 1) / bm;
  else a.mTiles = a.rows / bm + (a.experts < a.rows ? a.experts : a.rows);   // every expert's last tile may be partial
  const uint32_t reached = a.experts < a.rows ? a.experts : a.rows;
  const uint64_t column = (uint64_t)a.mTiles * (dw ? a.experts : 1) * threads, most = 0xffffffffu / column;   // of tiles
  const uint64_t unit = es == 1 && bn < FX_SCALE_GROUP ? FX_SCALE_GROUP : bn, columns = most * bn / unit * unit;
  if (columns == 0 && (a.n + bn - 1) / bn > most) return flagcxNotSupported;
  flagcxResult_t rc = flagcxSuccess;
  for (uint64_t left = a.n; left && rc == flagcxSuccess;) {
    a.n = (uint32_t)((left + bn - 1) / bn <= most ? left : columns);
    a.nTiles = (a.n + bn - 1) / bn;
    a.group = (uint64_t)a.nTiles * (a.rows / bm + reached / 2) <= 2 * kUnits ? 8 : 4;
    void *argv[] = {&a};
    if (hipLaunchKernel(kernel, dim3(a.nTiles * (uint32_t)(column / threads)), dim3(threads), argv, 0, s) != hipSuccess)
      rc = flagcxUnhandledDeviceError;
    left -= a.n;
    a.pn = (const char *)a.pn + a.n * colBytes;
    a.y = (char *)a.y + a.n * outBytes;
    if (a.sn) a.sn += a.n / FX_SCALE_GROUP * a.ldsn;
  }
  return rc;
}

// SN = 1: any alignment; SN = 0: rows of less than a chunk
template <class T, class Out, int BN, int BM, int WN, int WM, int SN, int SM, bool NACROSS, bool MACROSS, bool DW, bool TOUCH = false>
flagcxResult_t launchTiles(ProductArgs a, hipStream_t s) {
  const void *kernel;
  if constexpr (SN == 1) kernel = reinterpret_cast<const void *>(productNear<T, Out, BN, BM, WN, WM, NACROSS, MACROSS, DW>);
  else if constexpr (SN != 0) kernel = reinterpret_cast<const void *>(productDirect<T, Out, BN, BM, WN, WM, SN, SM, NACROSS, MACROSS, DW, TOUCH>);
  else kernel = reinterpret_cast<const void *>(productGuarded<T, Out, BN, BM, WN, WM, NACROSS, MACROSS, DW>);
  const size_t es = kBytes<T>;
  return launchGrid(kernel, a, BN, BM, DW, WN * WM * 64, es, (NACROSS ? 1 : a.ldn) * es, sizeof(Out), s);
}

template <class T, class Out, int RN, int FM, int NW, int U>
flagcxResult_t launchThin(ProductArgs a, hipStream_t s) {
  const size_t es = kBytes<T>;
  const bool odd = ((uintptr_t)a.pn | (uintptr_t)a.pm | a.ldn * es | a.ldm * es | a.expertN * es) & 3;
  const void *kernel = odd ? reinterpret_cast<const void *>(productThin<T, Out, RN, FM, NW, U, true>)
                           : reinterpret_cast<const void *>(productThin<T, Out, RN, FM, NW, U, false>);
  return launchGrid(kernel, a, 16 * RN, 16 * FM, false, NW * 64, es, a.ldn * es, sizeof(Out), s);
}

// Whole 16-byte chunks everywhere: what the direct kernels assume.  `inner` is the
// contiguous extent of the operand's rows.
inline bool wholeChunks(const void *p, size_t ld, size_t expert, size_t inner, size_t es) {
  const size_t e = 16 / es;
  return ((uintptr_t)p & 15) == 0 && ld % e == 0 && expert % e == 0 && inner % e == 0 && ld * es < (1u << 22);
}

// The tiles of the direct kernels: extent, workgroups that a compute unit holds,
// what one slab takes a workgroup, in tenths of a microsecond: alone on its
// compute unit (`alone`, from calls with fewer workgroups than units: 64 .. 256 rows,
// n = k = 8192) and with all units full (`full`, from 8192^3), and the rate at which
// weights arrive (`rate`, TB/s, from 8 rows each of 32 experts, 4096 x 4096).  Large
// tiles multiply and read faster, small ones fill the chip with less; a smaller tile
// is taken where this account puts it a fifth ahead (it does not know that smaller
// tiles read their operands more often: 128 rows each of 32 experts take 228 us in
// tiles of 256 and 278 us in tiles of 128, where the account says 207 and 184).  Nor does
// it know what storing dw takes, which is most of a tile's life where experts have few
// rows (16 experts, 4096 x 4096: one row each 150 us, 64 each 181, of which 83 and 85 are
// the memory's).  productNear and widened e4m3 operands have no figures of their own: they
// go by those of the direct kernels with operands as they are.
struct TileCost {
  uint32_t bn, bm, held;
  float alone, full, rate;
};
enum { kTile256, kTile128, kTile128x64, kTile64, kTiles };
constexpr TileCost kCost16[kTiles] = {{256, 256, 1, 13.3f, 16.2f, 6.1f}, {128, 128, 2, 8.2f, 4.7f, 5.9f},
                                      {128, 64, 2, 4.6f, 2.9f, 5.1f}, {64, 64, 2, 3.4f, 1.9f, 4.3f}};
constexpr TileCost kCost8[kTiles] = {{256, 256, 1, 20.f, 20.5f, 6.1f}, {128, 128, 2, 10.1f, 5.8f, 5.9f},
                                     {128, 64, 2, 8.1f, 3.7f, 5.1f}, {64, 64, 2, 7.4f, 3.0f, 4.3f}};

inline int cheapestTile(const ProductArgs &a, bool dw, size_t es, const TileCost *cost, int first) {
  const float reached = (float)(a.experts < a.rows ? a.experts : a.rows);
  const float slabs = dw ? (float)a.rows / a.experts / 64 : (float)a.k * es / 128;
  const float bytes = dw ? 0.f : reached * a.n * a.k * es;
  int best = first;
  float least = 0.f;
  for (int c = first; c < kTiles; c++) {
    // an expert's last tile is half full on average, and takes half the time
    const float m = dw ? (float)((a.m + cost[c].bm - 1) / cost[c].bm) * a.experts
                       : (a.offsets ? (float)a.rows / cost[c].bm + 0.5f * reached : (float)((a.rows + cost[c].bm - 1) / cost[c].bm));
    const float tiles = m * (float)((a.n + cost[c].bn - 1) / cost[c].bn);
    const uint32_t slots = kUnits * cost[c].held, rounds = (uint32_t)(tiles / slots);
    const float rest = tiles - (float)rounds * slots;
    const float deep = (float)(uint32_t)((rest + kUnits - 1) / kUnits) * cost[c].full;   // workgroups sharing a unit in the last round
    const float multiply = slabs * 0.1f * (rounds * cost[c].held * cost[c].full + (rest > 0 ? (deep > cost[c].alone ? deep : cost[c].alone) : 0.f));
    const float read = bytes / (cost[c].rate * 1e6f);
    const float t = multiply > read ? multiply : read;
    if (c == first || t < 0.8f * least) {
      least = t;
      best = c;
    }
  }
  return best;
}

template <class T, class Out, bool NACROSS, bool MACROSS, bool DW>
flagcxResult_t launchShapes(const ProductArgs &a, hipStream_t s) {
  const size_t es = kBytes<T>;
  if constexpr (!NACROSS && !DW) {
    // Few rows.  (a) up to 8 an expert, 16 of a single one: 16 at a time, 32 columns a
    // workgroup, or 16 where that leaves units without one (one row, n = k = 4096: 12.2 ->
    // 8.3 us); eight wavefronts share the reduction, for e4m3 four (16 rows, 8192 x 8192:
    // 19.1 -> 17.0 us; bf16 31.3 -> 28.5 us the other way).  (b) up to 32 rows of one
    // expert, 64 in e4m3 (35 us against 48 with tiles).  Of several experts up to 4 rows
    // each, or 12 where tiles of 128 columns would not fill the chip (8 each of 16 experts,
    // 1024 x 4096: 24 us against 40; 8 each of 32, 4096 x 4096: 191 against 180).
    // The lanes' offsets have 31 bits.
    const bool near = a.ldn * es < (1u << 24) && a.ldm * es < (1u << 24) && a.ldsm < (1u << 22) &&
                      a.ldsn * (a.n / FX_SCALE_GROUP + 1) < (1u << 28) && (uint64_t)a.k * es < (1u << 30);
    const uint64_t reached = a.experts < a.rows ? a.experts : a.rows, each = a.rows / a.experts;
    const uint64_t most = a.experts == 1 ? (es == 1 ? 64 : 32) : reached * ((a.n + 127) / 128) < 2 * kUnits ? 12 : 4;
    const uint64_t m = a.offsets ? a.rows / 16 + reached : (a.rows + 15) / 16;
    const bool wide = m * ((a.n + 31) / 32) >= kUnits;
    constexpr int NW = kBytes<T> == 1 ? 4 : 8;
    if (near && each <= most) {
      if (each > (a.experts == 1 ? 16 : 8)) return launchThin<T, Out, 2, 4, 4, 1>(a, s);
      return wide ? launchThin<T, Out, 2, 1, NW, 2>(a, s) : launchThin<T, Out, 1, 1, NW, 2>(a, s);
    }
  }
  const bool direct = wholeChunks(a.pn, a.ldn, a.expertN, NACROSS ? a.n : a.k, es) &&
                      wholeChunks(a.pm, a.ldm, 0, MACROSS ? a.m : a.k, es) && a.ldsm < (1u << 20);
  if (!direct) {
    const size_t inner = (NACROSS ? a.n : a.k) < (MACROSS ? a.m : a.k) ? (NACROSS ? a.n : a.k) : (MACROSS ? a.m : a.k);
    if (inner * es < 16) return launchTiles<T, Out, 128, 128, 2, 2, 0, 0, NACROSS, MACROSS, DW>(a, s);
    if (cheapestTile(a, DW, es, es == 1 ? kCost8 : kCost16, kTile128) != kTile128)
      return launchTiles<T, Out, 64, 64, 1, 2, 1, 1, NACROSS, MACROSS, DW>(a, s);
    return launchTiles<T, Out, 128, 128, 2, 2, 1, 1, NACROSS, MACROSS, DW>(a, s);
  }
  // widened e4m3 operands leave no registers for the largest tile
  constexpr bool kLargest = !__is_same(T, E4m3Exact);
  switch (cheapestTile(a, DW, es, es == 1 ? kCost8 : kCost16, kLargest ? kTile256 : kTile128)) {
    case kTile256:
      if constexpr (__is_same(T, E4m3))
        if (a.rows / a.experts >= 2048) return launchTiles<T, Out, 256, 256, 4, 2, 2, 2, NACROSS, MACROSS, DW, true>(a, s);
      if constexpr (kLargest) return launchTiles<T, Out, 256, 256, 4, 2, kBytes<T> == 1 ? 2 : 3, 2, NACROSS, MACROSS, DW>(a, s);
    case kTile128: return launchTiles<T, Out, 128, 128, 2, 2, 2, 2, NACROSS, MACROSS, DW>(a, s);
    case kTile128x64: return launchTiles<T, Out, 128, 64, 2, 2, 3, 3, NACROSS, MACROSS, DW>(a, s);
    default: return launchTiles<T, Out, 64, 64, 1, 2, 4, 4, NACROSS, MACROSS, DW>(a, s);
  }
}

template <class T, class Out>
flagcxResult_t launchForm(const ProductArgs &a, int form, hipStream_t s) {
  switch (form) {
    case kFormNK: return launchShapes<T, Out, false, false, false>(a, s);
    case kFormKN: return launchShapes<T, Out, true, false, false>(a, s);
    default: return launchShapes<T, Out, true, true, true>(a, s);
  }
}

}  // namespace fx
