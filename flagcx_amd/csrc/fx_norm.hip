// k-way sum + residual + root-mean-square norm (fx_reduce_norm) and its gradients
// (fx_reduce_norm_grad).
//
// A row of C columns is held in the registers of its threads, V octets each (octet
// i * threads + t belongs to thread t, so 16 neighbouring lanes hold one scale group
// of 128 columns): inputs are read once, the row's sum of squares is reduced over
// the threads, and the results leave from the same registers.  The arithmetic is a
// few operations per element; HBM bounds it.  Rows of up to 64 V octets are a
// wavefront's, four to a workgroup; longer ones a workgroup's, with as many
// wavefronts as they need; rows longer than the registers hold are read twice.  fp32
// rows of more than 16384 columns (gradients: 8192) do not quite fit: up to 116 bytes a
// lane go to scratch memory (gradients of 4096 x 16384: fp32 275 us, 3.9 TB/s; bf16 109,
// 4.9 TB/s).
// Measured: 16384 x 8192, two bf16 inputs and the residual to e4m3, 215 us (5.6 TB/s of
// exactly the operands' bytes); gradients of 8192 x 4096 bf16 47 us (5.7 TB/s); one row of
// 8192 with eight inputs 6 us, a launch being 4.
#include "flagcx_amd/fx_kernels.h"
#include "flagcx_amd/fx_model.h"
#include "fx_vec.hpp"

using namespace fx;

namespace {

constexpr uint32_t kHeld = 1024 * 4 * 8;      // widest row held in registers: 1024 threads, 4 octets each
constexpr float kE4m3Max = 448.f;
constexpr float kTinyScale = 0x1p-126f;

struct NormArgs {
  const void *in[FX_MAX_INPUTS + 1];          // k inputs and the residual, if any, behind them
  void *total, *out;
  float *scale;
  const void *weight;
  size_t ldIn, ldRes, ldTotal, ldOut, ldScale;
  uint32_t row0, rows, cols, n;               // rows [row0, rows) of this launch; n = entries of `in`
  uint32_t k;
  float eps;
  uint32_t weightF32;
};

__device__ __forceinline__ float blockSum(float x, float *lds, uint32_t nWaves) {
  x = waveSum(x);
  if (nWaves == 1) return x;
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = x;
  __syncthreads();
  float s = 0.f;
  for (uint32_t w = 0; w < nWaves; w++) s += lds[w];
  __syncthreads();
  return s;
}

// The octet's sum over all inputs, left to right.  B inputs are loaded before the
// first is used.
template <class T, int V, int B, bool APART = false>
__device__ __forceinline__ void sumInputs(const NormArgs &a, uint32_t row, const uint32_t (&c)[V], float (&f)[V][8]) {
#pragma unroll
  for (int i = 0; i < V; i++)
#pragma unroll
    for (int j = 0; j < 8; j++) f[i][j] = 0.f;
  for (uint32_t p0 = 0; p0 < a.n; p0 += B) {
    Octet<T> v[B][V];
#pragma unroll
    for (int b = 0; b < B; b++)
      if (p0 + b < a.n) {
        const T *r = (const T *)a.in[p0 + b] + (size_t)row * (p0 + b < a.k ? a.ldIn : a.ldRes);
#pragma unroll
        for (int i = 0; i < V; i++) v[b][i] = loadOctet<false, APART>(r, c[i], a.cols);
      }
#pragma unroll
    for (int b = 0; b < B; b++)
      if (p0 + b < a.n) {
        const bool first = p0 + b == 0;       // 0 + x would turn -0 into +0
#pragma unroll
        for (int i = 0; i < V; i++) settle<APART>(v[b][i], c[i], a.cols);
#pragma unroll
        for (int i = 0; i < V; i++)
#pragma unroll
          for (int j = 0; j < 8; j++) f[i][j] = first ? v[b][i].get(j) : f[i][j] + v[b][i].get(j);
      }
  }
}

template <class T>
__device__ __forceinline__ void weights(const NormArgs &a, uint32_t c, float (&w)[8]) {
  if (!a.weight) {
#pragma unroll
    for (int j = 0; j < 8; j++) w[j] = 1.f;
  } else if (sizeof(T) == 4 || a.weightF32) {
    Octet<float> o = loadOctet((const float *)a.weight, c, a.cols);
    settle(o, c, a.cols);
#pragma unroll
    for (int j = 0; j < 8; j++) w[j] = o.get(j);
  } else {
    Octet<T> o = loadOctet((const T *)a.weight, c, a.cols);
    settle(o, c, a.cols);
#pragma unroll
    for (int j = 0; j < 8; j++) w[j] = o.get(j);
  }
}

template <class T, bool QUANT, bool STREAM>
__device__ __forceinline__ void finishOctet(const NormArgs &a, uint32_t row, uint32_t c, const float (&f)[8], float r) {
  float w[8], y[8];
  weights<T>(a, c, w);
#pragma unroll
  for (int j = 0; j < 8; j++) y[j] = f[j] * r * w[j];
  if (a.total) storeOctet<STREAM>((T *)a.total + (size_t)row * a.ldTotal, c, a.cols, f);
  if constexpr (QUANT) {
    // The largest magnitude as an integer: NaN > infinity > finite, so a NaN gets through.
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const uint32_t b = c + j < a.cols ? (__builtin_bit_cast(uint32_t, y[j]) & 0x7fffffffu) : 0u;
      m = m > b ? m : b;
    }
#pragma unroll
    for (int d = 8; d; d >>= 1) {
      const uint32_t o = (uint32_t)__shfl_xor((int)m, d);
      m = m > o ? m : o;
    }
    const float amax = __builtin_bit_cast(float, m);
    float scale = amax / kE4m3Max;
    scale = scale < kTinyScale ? kTinyScale : scale;          // NaN compares false and stays
    const float inv = 1.f / scale;
#pragma unroll
    for (int j = 0; j < 8; j++) y[j] *= inv;
    storeE4m3<STREAM>((uint8_t *)a.out + (size_t)row * a.ldOut, c, a.cols, y);
    if ((threadIdx.x & 15) == 0 && c < a.cols) a.scale[(size_t)row * a.ldScale + c / FX_SCALE_GROUP] = scale;
  } else {
    storeOctet<STREAM>((T *)a.out + (size_t)row * a.ldOut, c, a.cols, y);
  }
}

template <class T, int V, bool WAVE, bool QUANT, bool STREAM>
__global__ void __launch_bounds__(WAVE ? 256 : 1024) normRows(NormArgs a) {
  __shared__ float lds[16];
  const uint32_t threads = WAVE ? 64 : blockDim.x, t = WAVE ? threadIdx.x & 63 : threadIdx.x;
  const uint32_t row = a.row0 + (WAVE ? blockIdx.x * 4 + (threadIdx.x >> 6) : blockIdx.x);
  if (row >= a.rows) return;                  // whole wavefronts leave, and there is no barrier then
  uint32_t c[V];
#pragma unroll
  for (int i = 0; i < V; i++) c[i] = (i * threads + t) * 8;
  float f[V][8];
  sumInputs<T, V, (V == 1 ? (sizeof(T) == 4 ? 8 : 16) : V == 2 ? 4 : 2)>(a, row, c, f);
  float q = 0.f;
#pragma unroll
  for (int i = 0; i < V; i++)
#pragma unroll
    for (int j = 0; j < 8; j++) q = __builtin_fmaf(f[i][j], f[i][j], q);
  q = blockSum(q, lds, threads / 64);
  const float r = 1.f / sqrtf(q / (float)a.cols + a.eps);
#pragma unroll
  for (int i = 0; i < V; i++) finishOctet<T, QUANT, STREAM>(a, row, c[i], f[i], r);
}

// Rows wider than the registers hold: the sum is formed twice.  Every element is
// read and written by one thread in the second pass, so exact aliasing is safe (and
// the octet that the row ends in must not be read together with its neighbour).
template <class T, bool QUANT>
__global__ void __launch_bounds__(1024) normLongRows(NormArgs a) {
  __shared__ float lds[16];
  const uint32_t row = a.row0 + blockIdx.x;
  const uint32_t steps = (a.cols + 1024 * 8 - 1) / (1024 * 8);
  float q = 0.f;
  for (uint32_t s = 0; s < steps; s++) {
    const uint32_t c[1] = {(s * 1024 + threadIdx.x) * 8};
    float f[1][8];
    sumInputs<T, 1, 8>(a, row, c, f);
#pragma unroll
    for (int j = 0; j < 8; j++) q = __builtin_fmaf(f[0][j], f[0][j], q);
  }
  q = blockSum(q, lds, 16);
  const float r = 1.f / sqrtf(q / (float)a.cols + a.eps);
  for (uint32_t s = 0; s < steps; s++) {
    const uint32_t c[1] = {(s * 1024 + threadIdx.x) * 8};
    float f[1][8];
    sumInputs<T, 1, 8, true>(a, row, c, f);
    finishOctet<T, QUANT, true>(a, row, c[0], f[0], r);
  }
}

// ------------------------------------------------------------------ gradients

struct NormGradArgs {
  const void *dy, *x, *dtotal, *weight;
  void *dx;
  float *partial;                             // sums of dweight, one row of ldPartial floats per part, or NULL
  uint32_t ldPartial;                         // columns rounded up to 32
  float *rms;                                 // long rows: 1 / rms per row for the column kernel
  size_t ldDy, ldX, ldDtotal, ldDx;
  uint32_t row0, rows, cols;                  // row0: long rows
  float eps;
  uint32_t weightF32;
};

template <class T>
__device__ __forceinline__ void gradWeights(const NormGradArgs &a, uint32_t c, float (&w)[8]) {
  NormArgs n;
  n.weight = a.weight;
  n.weightF32 = a.weightF32;
  n.cols = a.cols;
  weights<T>(n, c, w);
}

template <class T, int V, bool STREAM, bool APART = false>
struct GradRow {
  Octet<T> x[V], dy[V], dt[V];
  __device__ __forceinline__ void load(const NormGradArgs &a, uint32_t row, const uint32_t (&c)[V]) {
#pragma unroll
    for (int i = 0; i < V; i++) {
      x[i] = loadOctet<STREAM, APART>((const T *)a.x + (size_t)row * a.ldX, c[i], a.cols);
      dy[i] = loadOctet<STREAM, APART>((const T *)a.dy + (size_t)row * a.ldDy, c[i], a.cols);
    }
    if (a.dtotal && a.dx)
#pragma unroll
      for (int i = 0; i < V; i++) dt[i] = loadOctet<STREAM, APART>((const T *)a.dtotal + (size_t)row * a.ldDtotal, c[i], a.cols);
  }
  __device__ __forceinline__ void ready(const NormGradArgs &a, const uint32_t (&c)[V]) {
#pragma unroll
    for (int i = 0; i < V; i++) {
      settle<APART>(x[i], c[i], a.cols);
      settle<APART>(dy[i], c[i], a.cols);
      if (a.dtotal && a.dx) settle<APART>(dt[i], c[i], a.cols);
    }
  }
};

// Row r, r + gridDim.x, ... of a workgroup (WAVE: of each of its four wavefronts):
// the next row is loaded while this one is reduced (a workgroup of 1024 has no
// registers for that), and the columns' share of dweight stays in registers until the
// end.
template <class T, int V, bool WAVE, int THREADS, bool STREAM>
__global__ void __launch_bounds__(THREADS) normGradRows(NormGradArgs a) {
  constexpr bool kAhead = THREADS <= 512;
  __shared__ float lds[2][2][16];
  __shared__ float joined[WAVE ? 3 : 1][WAVE ? 64 * V * 8 : 1];
  const uint32_t threads = WAVE ? 64 : blockDim.x, t = WAVE ? threadIdx.x & 63 : threadIdx.x, wave = threadIdx.x >> 6;
  const uint32_t step = gridDim.x * (WAVE ? 4 : 1);
  uint32_t c[V], row = WAVE ? blockIdx.x * 4 + wave : blockIdx.x;
  float w[V][8], dw[V][8];
#pragma unroll
  for (int i = 0; i < V; i++) c[i] = (i * threads + t) * 8;
  GradRow<T, V, STREAM> next;
  if (kAhead && row < a.rows) next.load(a, row, c);
#pragma unroll
  for (int i = 0; i < V; i++) {
    gradWeights<T>(a, c[i], w[i]);
#pragma unroll
    for (int j = 0; j < 8; j++) dw[i][j] = 0.f;
  }
  const float invC = 1.f / (float)a.cols;
  for (uint32_t turn = 0; row < a.rows; row += step, turn ^= 1) {
    if (!kAhead) next.load(a, row, c);
    GradRow<T, V, STREAM> g = next;
    if (kAhead && row + step < a.rows) next.load(a, row + step, c);
    g.ready(a, c);
    float q = 0.f, m = 0.f;
#pragma unroll
    for (int i = 0; i < V; i++)
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float x = g.x[i].get(j);
        q = __builtin_fmaf(x, x, q);
        m = __builtin_fmaf(g.dy[i].get(j) * w[i][j], x, m);
      }
    q = waveSum(q);
    m = waveSum(m);
    if constexpr (!WAVE) {
      if (t % 64 == 0) {                      // two sets in turn: one barrier a row
        lds[turn][0][wave] = q;
        lds[turn][1][wave] = m;
      }
      __syncthreads();
      q = m = 0.f;
      for (uint32_t s = 0; s < threads / 64; s++) {
        q += lds[turn][0][s];
        m += lds[turn][1][s];
      }
    }
    const float r = 1.f / sqrtf(q * invC + a.eps);
    const float h = m * invC * r * r;         // mean(g xh) / rms: dx = r (g - x h)
#pragma unroll
    for (int i = 0; i < V; i++) {
      float d[8];
#pragma unroll
      for (int j = 0; j < 8; j++) {
        const float x = g.x[i].get(j), dy = g.dy[i].get(j);
        dw[i][j] = __builtin_fmaf(dy, x * r, dw[i][j]);
        d[j] = r * __builtin_fmaf(-x, h, dy * w[i][j]);
        if (a.dtotal) d[j] += g.dt[i].get(j);
      }
      if (a.dx) storeOctet<STREAM>((T *)a.dx + (size_t)row * a.ldDx, c[i], a.cols, d);
    }
  }
  if (!a.partial) return;
  if constexpr (WAVE) {                       // the four wavefronts' sums, in order
    if (wave)
#pragma unroll
      for (int i = 0; i < V; i++)
#pragma unroll
        for (int j = 0; j < 8; j++) joined[wave - 1][c[i] + j] = dw[i][j];
    __syncthreads();
    if (wave) return;
#pragma unroll
    for (int i = 0; i < V; i++)
#pragma unroll
      for (int j = 0; j < 8; j++)
#pragma unroll
        for (int s = 0; s < 3; s++) dw[i][j] += joined[s][c[i] + j];
  }
#pragma unroll
  for (int i = 0; i < V; i++)
    if (c[i] < a.ldPartial) storeOctet(a.partial + (size_t)blockIdx.x * a.ldPartial, c[i], a.ldPartial, dw[i]);   // zeros behind the last column
}

template <class T>
__global__ void __launch_bounds__(1024) normGradLongRows(NormGradArgs a) {
  __shared__ float lds[16];
  const uint32_t row = a.row0 + blockIdx.x;
  const uint32_t steps = (a.cols + 1024 * 8 - 1) / (1024 * 8);
  float q = 0.f, m = 0.f;
  for (uint32_t s = 0; s < steps; s++) {
    const uint32_t c[1] = {(s * 1024 + threadIdx.x) * 8};
    GradRow<T, 1, false> g;
    g.load(a, row, c);
    g.ready(a, c);
    float w[8];
    gradWeights<T>(a, c[0], w);
#pragma unroll
    for (int j = 0; j < 8; j++) {
      const float x = g.x[0].get(j);
      q = __builtin_fmaf(x, x, q);
      m = __builtin_fmaf(g.dy[0].get(j) * w[j], x, m);
    }
  }
  q = blockSum(q, lds, 16);
  m = blockSum(m, lds, 16);
  const float invC = 1.f / (float)a.cols;
  const float r = 1.f / sqrtf(q * invC + a.eps);
  const float h = m * invC * r * r;
  if (a.rms && threadIdx.x == 0) a.rms[row] = r;
  if (!a.dx) return;
  for (uint32_t s = 0; s < steps; s++) {
    const uint32_t c[1] = {(s * 1024 + threadIdx.x) * 8};
    GradRow<T, 1, false, true> g;
    g.load(a, row, c);
    g.ready(a, c);
    float w[8], d[8];
    gradWeights<T>(a, c[0], w);
#pragma unroll
    for (int j = 0; j < 8; j++) {
      d[j] = r * __builtin_fmaf(-g.x[0].get(j), h, g.dy[0].get(j) * w[j]);
      if (a.dtotal) d[j] += g.dt[0].get(j);
    }
    storeOctet((T *)a.dx + (size_t)row * a.ldDx, c[0], a.cols, d);
  }
}

// Must run before dx is written when dx equals dy: it reads dy again.  Workgroup
// (x, y): 2048 columns, every gridDim.y-th row from row y.
template <class T>
__global__ void __launch_bounds__(256) normGradLongColumns(NormGradArgs a) {
  const uint32_t c = (blockIdx.x * 256 + threadIdx.x) * 8;
  float dw[8] = {};
  for (uint32_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    Octet<T> x = loadOctet((const T *)a.x + (size_t)row * a.ldX, c, a.cols);
    Octet<T> dy = loadOctet((const T *)a.dy + (size_t)row * a.ldDy, c, a.cols);
    settle(x, c, a.cols);
    settle(dy, c, a.cols);
    const float r = a.rms[row];
#pragma unroll
    for (int j = 0; j < 8; j++) dw[j] = __builtin_fmaf(dy.get(j), x.get(j) * r, dw[j]);
  }
  if (c < a.ldPartial) storeOctet(a.partial + (size_t)blockIdx.y * a.ldPartial, c, a.ldPartial, dw);
}

// dweight = sum of `n` rows of partial sums, in a fixed order: 32 columns a
// workgroup, every 32nd row to each of 32 groups of eight lanes, eight rows on their
// way at a time; the groups meet in LDS.
template <class W>
__global__ void __launch_bounds__(256) normGradJoin(const float *partial, uint32_t n, uint32_t ld, uint32_t cols, W *dweight) {
  __shared__ float lds[32][33];
  const uint32_t part = threadIdx.x >> 3, c = (threadIdx.x & 7) * 4;
  const float *p = partial + blockIdx.x * 32 + c;
  f32x4 s = {};
  for (uint32_t r0 = part; r0 < n; r0 += 256) {
    f32x4 v[8];
#pragma unroll
    for (int u = 0; u < 8; u++) {
      const uint32_t r = r0 + 32 * u;
      v[u] = r < n ? *reinterpret_cast<const f32x4 *>(p + (size_t)r * ld) : f32x4{};
    }
#pragma unroll
    for (int u = 0; u < 8; u++)
#pragma unroll
      for (int j = 0; j < 4; j++) s[j] += v[u][j];
  }
#pragma unroll
  for (int j = 0; j < 4; j++) lds[part][c + j] = s[j];
  __syncthreads();
  if (threadIdx.x < 32 && blockIdx.x * 32 + threadIdx.x < cols) {
    float t = 0.f;
#pragma unroll
    for (int q = 0; q < 32; q++) t += lds[q][threadIdx.x];
    dweight[blockIdx.x * 32 + threadIdx.x] = (W)t;
  }
}

// ----------------------------------------------------------------- host side

template <class... P, class... A>
flagcxResult_t launchShape(void (*kernel)(P...), dim3 grid, uint32_t block, hipStream_t s, const A &...args) {
  std::tuple<P...> vals{static_cast<P>(args)...};
  void *argv[sizeof...(P)];
  argPointers(vals, argv, std::index_sequence_for<P...>{});
  return hipLaunchKernel(reinterpret_cast<const void *>(kernel), grid, dim3(block), argv, 0, s) == hipSuccess
             ? flagcxSuccess
             : flagcxUnhandledDeviceError;
}

size_t elementSize(int dt) {
  return dt == FX_E4M3 ? 1 : (dt == flagcxBfloat16 || dt == flagcxFloat16) ? 2 : dt == flagcxFloat32 ? 4 : 0;
}
bool known(int dt) { return (dt >= 0 && dt < flagcxNumTypes) || dt == FX_E4M3; }
bool at(const void *p, size_t es) { return p && ((uintptr_t)p & (es - 1)) == 0; }

// dtype / weight_dtype of both entry points
flagcxResult_t screenTypes(int dtype, int weightDtype) {
  if (!known(dtype) || !known(weightDtype)) return flagcxInvalidArgument;
  if (dtype == FX_E4M3 || !elementSize(dtype)) return flagcxNotSupported;
  if (weightDtype != dtype && weightDtype != flagcxFloat32) return flagcxNotSupported;
  return flagcxSuccess;
}

constexpr size_t kMaxExtent = 0x7fffffff;
constexpr size_t kMaxGradCols = 1u << 28;    // dweight's join has eight threads a column, and a launch less than 2^32
constexpr uint32_t kFewRows = 512;
constexpr uint64_t kStreamBytes = 32u << 20, kGradStreamBytes = 128u << 20;

// One launch for every kRowsAtATime rows, `per` of them to a workgroup: the runtime
// takes less than 2^32 threads.
constexpr uint32_t kRowsAtATime = 1u << 21;
template <class K, class A>
flagcxResult_t launchByRow(K kernel, A a, uint32_t per, uint32_t threads, hipStream_t s) {
  const uint32_t rows = a.rows;
  flagcxResult_t rc = flagcxSuccess;
  for (uint32_t r = 0; r < rows && rc == flagcxSuccess; r += kRowsAtATime) {
    a.row0 = r;
    a.rows = rows - r < kRowsAtATime ? rows : r + kRowsAtATime;
    rc = launchShape(kernel, dim3((a.rows - r + per - 1) / per), threads, s, a);
  }
  return rc;
}

// Wavefronts that hold `octets`, v to a lane, in threads.
uint32_t threadsFor(uint32_t octets, uint32_t v) { return ((octets + v - 1) / v + 63) / 64 * 64; }

template <class T, bool QUANT, bool STREAM>
flagcxResult_t launchNormRows(const NormArgs &a, hipStream_t s) {
  const uint32_t octets = (a.cols + 7) / 8;
  if (octets <= 64) return launchByRow(normRows<T, 1, true, QUANT, STREAM>, a, 4, 256, s);
  // Few rows: one octet to a lane, so that all inputs of a row are on their way at once (one row of 8192 with eight
  // inputs 8.4 -> 6.4 us).
  if constexpr (!STREAM)
    if (octets <= 1024 && a.rows <= kFewRows) return launchByRow(normRows<T, 1, false, QUANT, STREAM>, a, 1, threadsFor(octets, 1), s);
  if (octets <= 128) return launchByRow(normRows<T, 2, true, QUANT, STREAM>, a, 4, 256, s);
  if (octets <= (sizeof(T) == 4 ? 2048 : 512)) return launchByRow(normRows<T, 2, false, QUANT, STREAM>, a, 1, threadsFor(octets, 2), s);
  return launchByRow(normRows<T, 4, false, QUANT, STREAM>, a, 1, threadsFor(octets, 4), s);
}

// Results that the dies' L2s (32 MiB) cannot hold are streamed (16384 x 8192, two bf16
// inputs and the residual to e4m3: 216 -> 208 us; 4096 x 4096, four inputs: 47 -> 45
// us); smaller ones stay for whoever reads them next.  Loads are left to the caches:
// streaming them gained 5 % from memory and cost 30 % when the inputs had just been
// written (1024 x 4096).
template <class T, bool QUANT>
flagcxResult_t launchNorm(const NormArgs &a, hipStream_t s) {
  if (a.cols > kHeld) return launchByRow(normLongRows<T, QUANT>, a, 1, 1024, s);
  const uint64_t written = (uint64_t)a.rows * a.cols * ((a.total ? sizeof(T) : 0) + (QUANT ? 1 : sizeof(T)));
  return written > kStreamBytes ? launchNormRows<T, QUANT, true>(a, s) : launchNormRows<T, QUANT, false>(a, s);
}

template <class T>
flagcxResult_t launchNormOut(const NormArgs &a, bool quant, hipStream_t s) {
  return quant ? launchNorm<T, true>(a, s) : launchNorm<T, false>(a, s);
}

// Workgroups of the gradients, each with a row of partial sums: one per compute unit
// (8192 x 8192 bf16: 89 us, with 384 105, with 512 94), or as many as give each the same
// number of rows, with fewer partial sums to join (260 x 8192: 13.3 -> 11.6 us; 777 x 5003
// fp16: 16.9 -> 16.4).
constexpr uint32_t kGradWgs = 256;
constexpr uint32_t kLongParts = 64;
constexpr uint32_t kGradHeld = 1024 * 2 * 8;   // widest row that the gradients hold

uint32_t partialStride(size_t cols) { return (uint32_t)((cols + 31) / 32 * 32); }
bool waveRows(size_t cols) { return cols <= 64 * 2 * 8; }
uint32_t gradParts(size_t rows, size_t cols) {
  const size_t most = cols > kGradHeld ? kLongParts : kGradWgs;
  const size_t want = waveRows(cols) ? (rows + 3) / 4 : rows;
  const size_t rounds = (want + most - 1) / most;
  return (uint32_t)((want + rounds - 1) / rounds);
}
// What one call uses; and what every call of at most so many rows and columns can do with, for callers that keep one
// workspace: fewer rows may well have more parts, and the widest rows that are held more than wider ones.
size_t gradBytes(size_t rows, size_t cols) {
  return ((size_t)gradParts(rows, cols) * partialStride(cols) + (cols > kGradHeld ? rows : 0)) * sizeof(float);
}
size_t gradBytesUpTo(size_t rows, size_t cols) {
  const size_t want = waveRows(cols) ? (rows + 3) / 4 : rows;
  const size_t held = (want < kGradWgs ? want : kGradWgs) * partialStride(cols < kGradHeld ? cols : kGradHeld);
  const size_t wide = cols > kGradHeld ? (rows < kLongParts ? rows : kLongParts) * partialStride(cols) + rows : 0;
  return (held > wide ? held : wide) * sizeof(float);
}

template <class T, bool STREAM>
flagcxResult_t launchGradRows(const NormGradArgs &a, uint32_t parts, hipStream_t s) {
  const uint32_t octets = (a.cols + 7) / 8;
  if (octets <= 64) return launchShape(normGradRows<T, 1, true, 256, STREAM>, dim3(parts), 256, s, a);
  if (waveRows(a.cols)) return launchShape(normGradRows<T, 2, true, 256, STREAM>, dim3(parts), 256, s, a);
  if (octets <= 512) return launchShape(normGradRows<T, 1, false, 512, STREAM>, dim3(parts), threadsFor(octets, 1), s, a);
  if (octets <= 1024) return launchShape(normGradRows<T, 2, false, 512, STREAM>, dim3(parts), threadsFor(octets, 2), s, a);
  return launchShape(normGradRows<T, 2, false, 1024, STREAM>, dim3(parts), threadsFor(octets, 2), s, a);
}

template <class T>
flagcxResult_t launchGrad(NormGradArgs a, void *dweight, bool weightF32, void *workspace, hipStream_t s) {
  const uint32_t parts = a.rows ? gradParts(a.rows, a.cols) : 0;
  flagcxResult_t rc = flagcxSuccess;
  a.partial = dweight ? (float *)workspace : nullptr;
  a.ldPartial = partialStride(a.cols);
  a.rms = nullptr;
  if (a.rows && a.cols > kGradHeld) {
    // The column kernel reads dy and x again, so it goes before the pass that writes dx (which may equal dy):
    // rms first, without dx; then the columns; then dx.
    if (dweight) {
      a.rms = (float *)workspace + (size_t)parts * a.ldPartial;
      NormGradArgs b = a;
      b.dx = nullptr;
      rc = launchByRow(normGradLongRows<T>, b, 1, 1024, s);
      if (rc != flagcxSuccess) return rc;
      rc = launchShape(normGradLongColumns<T>, dim3((a.cols + 2047) / 2048, parts), 256, s, b);
      if (rc != flagcxSuccess) return rc;
    }
    if (a.dx) rc = launchByRow(normGradLongRows<T>, a, 1, 1024, s);
  } else if (a.rows) {
    // What the memory-side cache cannot keep is streamed both ways (8192 x 4096 bf16: 54 -> 50 us, 8192 x 8192: 107 ->
    // 95 us).
    const uint64_t bytes = (uint64_t)a.rows * a.cols * sizeof(T) * (2 + (a.dx ? 1 + (a.dtotal != nullptr) : 0));
    rc = bytes > kGradStreamBytes ? launchGradRows<T, true>(a, parts, s) : launchGradRows<T, false>(a, parts, s);
  }
  if (rc != flagcxSuccess || !dweight) return rc;
  const dim3 grid(a.ldPartial / 32);
  if (weightF32)
    return launchShape(normGradJoin<float>, grid, 256, s, (const float *)workspace, parts, a.ldPartial, a.cols, (float *)dweight);
  return launchShape(normGradJoin<T>, grid, 256, s, (const float *)workspace, parts, a.ldPartial, a.cols, (T *)dweight);
}

}  // namespace

extern "C" {
#pragma GCC visibility push(default)

int fx_reduce_norm(void *out, float *scale, void *total, const void *const *in, int k, const void *residual,
                   const void *weight, size_t rows, size_t cols, const fxNormStrides *strides, int dtype,
                   int weight_dtype, int out_dtype, float eps, void *stream) {
  const flagcxResult_t rc = screenTypes(dtype, weight_dtype);
  if (rc != flagcxSuccess) return rc;
  if (!known(out_dtype)) return flagcxInvalidArgument;
  if (out_dtype != dtype && out_dtype != FX_E4M3) return flagcxNotSupported;
  if (!in || k < 1 || k > FX_MAX_INPUTS || rows > kMaxExtent || cols > kMaxExtent || !(eps >= 0.f)) return flagcxInvalidArgument;
  const bool quant = out_dtype == FX_E4M3;
  if (quant != (scale != nullptr)) return flagcxInvalidArgument;
  if (rows == 0 || cols == 0) return flagcxSuccess;
  const size_t es = elementSize(dtype), groups = (cols + FX_SCALE_GROUP - 1) / FX_SCALE_GROUP;
  const fxNormStrides st = strides ? *strides : fxNormStrides{cols, cols, cols, cols, groups};
  if (st.in < cols || st.out < cols || (residual && st.residual < cols) || (total && st.total < cols) || (quant && st.scale < groups))
    return flagcxInvalidArgument;
  if (!at(out, quant ? 1 : es) || total == out || (total && !at(total, es)) || (residual && !at(residual, es)) ||
      (weight && !at(weight, elementSize(weight_dtype))) || (quant && !at(scale, 4)))
    return flagcxInvalidArgument;
  NormArgs a;
  for (int p = 0; p < k; p++) {
    if (!at(in[p], es)) return flagcxInvalidArgument;
    a.in[p] = in[p];
  }
  for (int p = k; p <= FX_MAX_INPUTS; p++) a.in[p] = residual;
  a.total = total;
  a.out = out;
  a.scale = scale;
  a.weight = weight;
  a.ldIn = st.in;
  a.ldRes = st.residual;
  a.ldTotal = st.total;
  a.ldOut = st.out;
  a.ldScale = st.scale;
  a.row0 = 0;
  a.rows = (uint32_t)rows;
  a.cols = (uint32_t)cols;
  a.k = (uint32_t)k;
  a.n = (uint32_t)k + (residual ? 1 : 0);
  a.eps = eps;
  a.weightF32 = weight_dtype == flagcxFloat32;
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case flagcxBfloat16: return launchNormOut<__bf16>(a, quant, s);
    case flagcxFloat16: return launchNormOut<_Float16>(a, quant, s);
    default: return launchNormOut<float>(a, quant, s);
  }
}

size_t fx_reduce_norm_grad_workspace(size_t rows, size_t cols) {
  if (rows == 0 || cols == 0) return 0;
  if (rows > kMaxExtent || cols > kMaxGradCols) return 0;
  return gradBytesUpTo(rows, cols);
}

int fx_reduce_norm_grad(void *dx, void *dweight, const void *dy, const void *x, const void *dtotal, const void *weight,
                        size_t rows, size_t cols, const fxNormGradStrides *strides, int dtype, int weight_dtype, float eps,
                        void *workspace, size_t workspace_bytes, void *stream) {
  const flagcxResult_t rc = screenTypes(dtype, weight_dtype);
  if (rc != flagcxSuccess) return rc;
  if (rows > kMaxExtent || cols > kMaxGradCols || !(eps >= 0.f)) return flagcxInvalidArgument;
  if (cols == 0 || (!dx && !dweight)) return flagcxSuccess;
  const size_t es = elementSize(dtype);
  if (dweight && !at(dweight, elementSize(weight_dtype))) return flagcxInvalidArgument;
  const fxNormGradStrides st = strides ? *strides : fxNormGradStrides{cols, cols, cols, cols};
  if (rows) {
    if (!at(dy, es) || !at(x, es) || (dx && !at(dx, es)) || (dtotal && !at(dtotal, es)) ||
        (weight && !at(weight, elementSize(weight_dtype))))
      return flagcxInvalidArgument;
    if (st.dy < cols || st.x < cols || (dtotal && st.dtotal < cols) || (dx && st.dx < cols)) return flagcxInvalidArgument;
    if (dweight && (!at(workspace, 16) || workspace_bytes < gradBytes(rows, cols)))
      return flagcxInvalidArgument;
  }
  NormGradArgs a;
  a.dy = dy;
  a.x = x;
  a.dtotal = dtotal;
  a.weight = weight;
  a.dx = dx;
  a.ldDy = st.dy;
  a.ldX = st.x;
  a.ldDtotal = st.dtotal;
  a.ldDx = st.dx;
  a.row0 = 0;
  a.rows = (uint32_t)rows;
  a.cols = (uint32_t)cols;
  a.eps = eps;
  a.weightF32 = weight_dtype == flagcxFloat32;
  hipStream_t s = (hipStream_t)stream;
  if (rows == 0 && !dweight) return flagcxSuccess;
  switch (dtype) {
    case flagcxBfloat16: return launchGrad<__bf16>(a, dweight, a.weightF32, workspace, s);
    case flagcxFloat16: return launchGrad<_Float16>(a, dweight, a.weightF32, workspace, s);
    default: return launchGrad<float>(a, dweight, a.weightF32, workspace, s);
  }
}

#pragma GCC visibility pop
}
