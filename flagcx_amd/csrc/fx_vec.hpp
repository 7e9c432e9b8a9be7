// Eight consecutive elements ("octet") of bf16, fp16 or fp32 in registers: raw
// loads and stores at any element boundary, widening to fp32, one rounding back.
#pragma once
#include "fx_common.hpp"

namespace fx {

typedef float f32x4 __attribute__((ext_vector_type(4)));

template <class T>
struct Octet;   // raw bits of eight elements

template <>
struct Octet<__bf16> {
  u32x4 v;
  __device__ __forceinline__ float get(int j) const {
    const uint32_t w = v[j >> 1];
    return __builtin_bit_cast(float, (j & 1) ? (w & 0xffff0000u) : (w << 16));
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
#pragma unroll
    for (int j = 0; j < 4; j++)
      v[j] = (uint32_t)__builtin_bit_cast(uint16_t, (__bf16)f[2 * j]) |
             ((uint32_t)__builtin_bit_cast(uint16_t, (__bf16)f[2 * j + 1]) << 16);
  }
};

template <>
struct Octet<_Float16> {
  u32x4 v;
  __device__ __forceinline__ float get(int j) const {
    return (float)__builtin_bit_cast(_Float16, (uint16_t)(v[j >> 1] >> (16 * (j & 1))));
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
#pragma unroll
    for (int j = 0; j < 4; j++)
      v[j] = (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[2 * j]) |
             ((uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f[2 * j + 1]) << 16);
  }
};

template <>
struct Octet<float> {
  u32x4 v[2];
  __device__ __forceinline__ float get(int j) const { return __builtin_bit_cast(float, (uint32_t)v[j >> 2][j & 3]); }
  __device__ __forceinline__ void set(const float (&f)[8]) {
#pragma unroll
    for (int j = 0; j < 8; j++) v[j >> 2][j & 3] = __builtin_bit_cast(uint32_t, f[j]);
  }
};

// STREAM: past the caches.
template <bool STREAM>
__device__ __forceinline__ u32x4 loadVec(const u32x4_anywhere *p) {
  if constexpr (STREAM) return __builtin_nontemporal_load(p);
  else return *p;
}
typedef uint32_t u32x2_anywhere __attribute__((ext_vector_type(2), aligned(1)));
template <bool STREAM>
__device__ __forceinline__ void storeVec(u32x4_anywhere *p, u32x4 v) {
  if constexpr (STREAM) __builtin_nontemporal_store(v, p);
  else *p = v;
}
template <bool STREAM>
__device__ __forceinline__ void storeVec(u32x2_anywhere *p, u32x2_anywhere v) {
  if constexpr (STREAM) __builtin_nontemporal_store(v, p);
  else *p = v;
}
// Octet at columns [c, c + 8) of a row of `cols` elements.  gfx950 serves 128-bit
// accesses at any element boundary, so rows of odd length need no path of their own:
// an octet that the row ends in is loaded from the row's last eight elements (no
// branch around the load, nothing behind the row touched) and shifted into place by
// settle(), which is called where the octet is first used; columns behind the last
// are zero then.  APART: element by element instead, for passes that have written
// other columns of the row already.
template <bool STREAM = false, bool APART = false, class T>
__device__ __forceinline__ Octet<T> loadOctet(const T *row, uint32_t c, uint32_t cols) {
  Octet<T> o = {};
  if (APART ? c + 8 <= cols : cols >= 8) {
    const u32x4_anywhere *p = reinterpret_cast<const u32x4_anywhere *>(row + (c < cols - 8 ? c : cols - 8));
    if constexpr (sizeof(T) == 4) {
      o.v[0] = loadVec<STREAM>(p);
      o.v[1] = loadVec<STREAM>(p + 1);
    } else {
      o.v = loadVec<STREAM>(p);
    }
  } else if (c < cols) {
    float f[8];
#pragma unroll
    for (int j = 0; j < 8; j++) f[j] = c + j < cols ? (float)row[c + j] : 0.f;   // exact both ways, NaN stays NaN
    o.set(f);
  }
  return o;
}

template <bool APART = false, class T>
__device__ __forceinline__ void settle(Octet<T> &o, uint32_t c, uint32_t cols) {
  if (APART || cols < 8 || c + 8 <= cols) return;
  const uint32_t s = c + 8 - cols;            // elements to drop in front
  if (s >= 8) {
    o = Octet<T>{};
    return;
  }
  if constexpr (sizeof(T) == 4) {
    uint32_t w[8];
#pragma unroll
    for (int j = 0; j < 8; j++) w[j] = o.v[j >> 2][j & 3];
#pragma unroll
    for (int b = 1; b < 8; b <<= 1)
#pragma unroll
      for (int j = 0; j < 8; j++) w[j] = (s & b) ? (j + b < 8 ? w[j + b] : 0u) : w[j];
#pragma unroll
    for (int j = 0; j < 8; j++) o.v[j >> 2][j & 3] = w[j];
  } else {
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; j++) w[j] = o.v[j];
#pragma unroll
    for (int b = 1; b < 4; b <<= 1)
#pragma unroll
      for (int j = 0; j < 4; j++) w[j] = (s >> 1 & b) ? (j + b < 4 ? w[j + b] : 0u) : w[j];
    if (s & 1)
#pragma unroll
      for (int j = 0; j < 4; j++) w[j] = w[j] >> 16 | (j < 3 ? w[j < 3 ? j + 1 : 3] << 16 : 0u);
#pragma unroll
    for (int j = 0; j < 4; j++) o.v[j] = w[j];
  }
}

template <bool STREAM = false, class T>
__device__ __forceinline__ void storeOctet(T *row, uint32_t c, uint32_t cols, const float (&f)[8]) {
  if (c + 8 <= cols) {
    Octet<T> o;
    o.set(f);
    u32x4_anywhere *p = reinterpret_cast<u32x4_anywhere *>(row + c);
    if constexpr (sizeof(T) == 4) {
      storeVec<STREAM>(p, o.v[0]);
      storeVec<STREAM>(p + 1, o.v[1]);
    } else {
      storeVec<STREAM>(p, o.v);
    }
  } else if (c < cols) {
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (c + j < cols) row[c + j] = (T)f[j];
  }
}

// Eight floats as e4m3 codes (round to nearest even), columns behind the last left alone.
template <bool STREAM>
__device__ __forceinline__ void storeE4m3(uint8_t *row, uint32_t c, uint32_t cols, const float (&f)[8]) {
  uint32_t w[2];
#pragma unroll
  for (int h = 0; h < 2; h++) {
    int q = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * h], f[4 * h + 1], 0, false);
    q = __builtin_amdgcn_cvt_pk_fp8_f32(f[4 * h + 2], f[4 * h + 3], q, true);
    w[h] = (uint32_t)q;
  }
  if (c + 8 <= cols) {
    u32x2_anywhere v;
    v[0] = w[0];
    v[1] = w[1];
    storeVec<STREAM>(reinterpret_cast<u32x2_anywhere *>(row + c), v);
  } else if (c < cols) {
#pragma unroll
    for (int j = 0; j < 8; j++)
      if (c + j < cols) row[c + j] = (uint8_t)(w[j >> 2] >> (8 * (j & 3)));
  }
}

__device__ __forceinline__ float waveSum(float x) {
#pragma unroll
  for (int d = 32; d; d >>= 1) x += __shfl_xor(x, d);
  return x;
}

}  // namespace fx
