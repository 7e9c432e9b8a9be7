/*
 * Operators of a model that stand directly behind a collective: what a
 * tensor-parallel layer does with the ranks' partial results (the k-way sum of
 * fx_reduce_copy, the residual's addition and the root-mean-square norm in one
 * pass), and what an expert-parallel layer does with the rows that an
 * all-to-all-v delivers (matrix products grouped by expert).  FlagCX has no
 * counterpart: there a framework calls its own kernels between the collectives.
 *
 * The conventions are those of fx_kernels.h: plain pointers and sizes, every
 * function returns a flagcxResult_t value (0 success, 1 device error,
 * 4 invalid argument, 9 not supported), `stream` is a raw hipStream_t, calls
 * only enqueue.  All arguments are checked on the host before anything is
 * enqueued; nothing is allocated, so every call can be captured into a graph.
 * Element types are FlagCX's (bf16 = 9, fp16 = 6, fp32 = 7) and FX_E4M3.
 * Strides are in elements; a NULL stride block means dense rows.
 */
#ifndef FLAGCX_AMD_FX_MODEL_H_
#define FLAGCX_AMD_FX_MODEL_H_

#include "flagcx_amd/fx_types.h"

#ifdef __cplusplus
extern "C" {
#endif

/* 8-bit float with 4 exponent and 3 mantissa bits (OCP e4m3: largest value 448,
 * no infinities).  Not a FlagCX datatype: collectives move it as flagcxUint8. */
#define FX_E4M3 0x40
/* Consecutive columns that share one scale (and rows, for weights). */
#define FX_SCALE_GROUP 128

/*
 * Sum of k partial results, residual addition and root-mean-square norm:
 *   s[r,c]     = in[0][r,c] + ... + in[k-1][r,c] + residual[r,c]
 *   total[r,c] = s rounded to dtype                     (total may be NULL)
 *   y[r,c]     = s[r,c] / sqrt(mean_c(s[r,:]^2) + eps) * weight[c]
 *   out        = y rounded to out_dtype
 * in fp32, the inputs added left to right as fx_reduce_copy does, the residual
 * last; the norm is taken of the unrounded s.  residual and weight may be NULL
 * (none; ones).  dtype (inputs, residual, total): bf16, fp16 or fp32.
 * weight_dtype: dtype or fp32.  out_dtype: dtype, or FX_E4M3, then
 *   scale[r,g] = max(max_{c in group g} |y[r,c]| / 448, 2^-126)
 *   out[r,c]   = e4m3(y[r,c] / scale[r, c / 128])        (round to nearest even)
 * with the division done as a product with the fp32 reciprocal, and scale (fp32,
 * ceil(cols / 128) per row) is required; otherwise scale must be NULL.  A NaN
 * in a group makes its scale and all its values NaN.
 * total and out may each equal an input or the residual exactly (same stride,
 * same element size), but not each other; any other overlap is undefined.
 * k <= FX_MAX_INPUTS (64); rows and cols < 2^31.
 */
typedef struct fxNormStrides {
  size_t in, residual, total, out, scale; /* elements from row to row */
} fxNormStrides;
int fx_reduce_norm(void *out, float *scale, void *total,
                   const void *const *in, int k, const void *residual,
                   const void *weight, size_t rows, size_t cols,
                   const fxNormStrides *strides, int dtype, int weight_dtype,
                   int out_dtype, float eps, void *stream);

/*
 * Gradients of that norm.  x is what the forward call stored as `total`, dy the
 * gradient of `out` (in dtype), dtotal the gradient that reaches `total` from
 * elsewhere (the residual stream; may be NULL).  With r = 1 / sqrt(mean(x^2) + eps):
 *   g  = dy * weight
 *   dx = r * g - x * r^3 * mean_c(g * x) + dtotal
 *   dweight[c] = sum_r dy[r,c] * x[r,c] * r[r]
 * dx is the gradient of every in[p] and of the residual alike.  dx or dweight
 * (weight_dtype) may be NULL: not computed.  Sums run in fp32 in an order that
 * depends on the sizes alone, so equal calls give equal bits.  dx may equal dy
 * or dtotal exactly.  With rows = 0 dweight is filled with zeros.  rows < 2^31,
 * cols <= 2^28.
 * `workspace` (device memory, 16-byte aligned) is needed when dweight is asked
 * for.  fx_reduce_norm_grad_workspace(rows, cols) bytes do for every call of at
 * most that many rows and at most that many columns, so one workspace sized for
 * the largest serves them all; a call refuses one that is smaller than what it
 * uses itself.  It holds nothing between calls, and calls that may run at the same
 * time need one each.
 */
typedef struct fxNormGradStrides {
  size_t dy, x, dtotal, dx;
} fxNormGradStrides;
size_t fx_reduce_norm_grad_workspace(size_t rows, size_t cols);
int fx_reduce_norm_grad(void *dx, void *dweight, const void *dy, const void *x,
                        const void *dtotal, const void *weight, size_t rows,
                        size_t cols, const fxNormGradStrides *strides,
                        int dtype, int weight_dtype, float eps,
                        void *workspace, size_t workspace_bytes, void *stream);

/*
 * Matrix products grouped by expert: the rows of x [rows, k] lie sorted by
 * expert, as fx_unpack leaves what an all-to-all-v delivered, and expert e's are
 * offsets[e] .. offsets[e+1]-1:
 *   y[r, j] = sum_c x[r, c] * W_e[j, c]     FX_WEIGHT_NK: w is [experts][n][k]
 *   y[r, j] = sum_c x[r, c] * W_e[c, j]     FX_WEIGHT_KN: w is [experts][k][n]
 * x's gradient is the same product of dy with the other layout of the same
 * weights.  Accumulated in fp32, rounded once to out_dtype.
 * `offsets` is a DEVICE array of experts + 1 ascending int32 values, read when
 * the call executes (routing need not reach the host); an expert may have no
 * rows.  Values outside [0, rows] are clamped and a descending pair is an empty
 * expert: nothing outside the buffers is ever touched (rows that several experts
 * claim then get one's results, or none).  Rows of y before offsets[0] or from
 * offsets[experts] on are left as they were.  offsets = NULL with experts = 1: all
 * rows, the plain product.
 * dtype (x, w): bf16 or fp16; out_dtype: dtype or fp32.  y overlaps nothing else.
 * Extents and experts < 2^31.  A launch takes less than 2^32 threads; calls with more
 * columns than that go through them in several.  Where the rows of up to 256 columns
 * need as many by themselves, the call is not supported (9): that takes four million
 * experts with rows of their own, for dw eight million experts or 2^31 rows of dw.
 */
enum { FX_WEIGHT_NK = 0, FX_WEIGHT_KN = 1 };
typedef struct fxProductStrides {
  size_t x, w, y;       /* elements from row to row */
  size_t expert_w;      /* elements from one expert's weights to the next's */
} fxProductStrides;
int fx_expert_product(void *y, const void *x, const void *w,
                      const int32_t *offsets, size_t experts, size_t rows,
                      size_t n, size_t k, int layout,
                      const fxProductStrides *strides, int dtype,
                      int out_dtype, void *stream);

/*
 * The weights' gradient, dw [experts][n][k] (rows of k, also for weights used
 * as FX_WEIGHT_KN with n and k, dy and x exchanged):
 *   dw[e][j, c] = sum over expert e's rows r of dy[r, j] * x[r, c]
 * in fp32, rounded once to out_dtype (dtype or fp32).  Experts without rows get
 * zeros.  offsets as above.
 */
typedef struct fxProductDwStrides {
  size_t dy, x, dw, expert_dw;
} fxProductDwStrides;
int fx_expert_product_dw(void *dw, const void *dy, const void *x,
                         const int32_t *offsets, size_t experts, size_t rows,
                         size_t n, size_t k,
                         const fxProductDwStrides *strides, int dtype,
                         int out_dtype, void *stream);

/*
 * The same product of e4m3 operands with fp32 scales: x [rows, k] with one scale
 * per row and 128 columns (what fx_reduce_norm writes, and what an all-to-all-v
 * of bytes delivers), w [experts][n][k] with one per 128 x 128 block:
 *   y[r, j] = sum_g xscale[r, g] * wscale[e][j / 128, g] * sum_{c in group g} x[r, c] * w[e][j, c]
 * Groups and blocks at the ends may be partial.  out_dtype: bf16, fp16 or fp32.
 * For fp32 the products and sums are those of fp32 arithmetic.  For a 16-bit
 * out_dtype large calls (more than 64 rows of one expert, more than about 4 to 12
 * each of several) use the 8-bit matrix instructions, which take a group's columns
 * in runs of eight: a run's products are cut, towards zero, to multiples of
 * 2^(e-13), e being the largest sum of both factors' exponents among those that are
 * not zero (a subnormal's exponent is -6).  So a run's sum is off by less than 2^-10
 * of its largest product, subnormal factors counted as 2^-6: about 2^-16 of the
 * result for ordinary data, against the 2^-8 or 2^-11 of the rounding that follows,
 * but all of it where large terms cancel within a run and small ones ought to
 * remain.  Runs and groups are summed in fp32.  Who needs more asks for fp32 results
 * (2.2 to 3.4 times as long in large calls).
 */
typedef struct fxProductE4m3Strides {
  size_t x, w, y, expert_w;
  size_t xscale, wscale, expert_wscale;
} fxProductE4m3Strides;
int fx_expert_product_e4m3(void *y, const void *x, const float *xscale,
                           const void *w, const float *wscale,
                           const int32_t *offsets, size_t experts, size_t rows,
                           size_t n, size_t k,
                           const fxProductE4m3Strides *strides, int out_dtype,
                           void *stream);

#ifdef __cplusplus
}
#endif
#endif /* FLAGCX_AMD_FX_MODEL_H_ */
