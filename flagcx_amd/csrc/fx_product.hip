// C entry points of the products grouped by expert: argument checks, then the launch.
#include "fx_product.hpp"

using namespace fx;

namespace {

constexpr size_t kMaxExtent = 0x7fffffff;

bool known(int dt) { return (dt >= 0 && dt < flagcxNumTypes) || dt == FX_E4M3; }
bool sixteen(int dt) { return dt == flagcxBfloat16 || dt == flagcxFloat16; }
bool at(const void *p, size_t es) { return p && ((uintptr_t)p & (es - 1)) == 0; }

flagcxResult_t screenTypes(int dtype, int outDtype) {
  if (!known(dtype) || !known(outDtype)) return flagcxInvalidArgument;
  if (!sixteen(dtype) || (outDtype != dtype && outDtype != flagcxFloat32)) return flagcxNotSupported;
  return flagcxSuccess;
}

// Sizes and offsets of all three entry points.  *empty: nothing to compute.
flagcxResult_t screenSizes(const int32_t *offsets, size_t experts, size_t rows, size_t n, size_t k) {
  if (experts > kMaxExtent || rows > kMaxExtent || n > kMaxExtent || k > kMaxExtent) return flagcxInvalidArgument;
  if (!offsets && experts != 1) return flagcxInvalidArgument;
  if (offsets && !at(offsets, 4)) return flagcxInvalidArgument;
  return flagcxSuccess;
}

flagcxResult_t launch(const ProductArgs &a, int form, int dtype, bool outF32, void *stream) {
  return dtype == flagcxBfloat16 ? launchProductBf16(a, form, outF32, (hipStream_t)stream)
                                 : launchProductF16(a, form, outF32, (hipStream_t)stream);
}

}  // namespace

extern "C" {
#pragma GCC visibility push(default)

int fx_expert_product(void *y, const void *x, const void *w, const int32_t *offsets, size_t experts, size_t rows, size_t n,
                      size_t k, int layout, const fxProductStrides *strides, int dtype, int out_dtype, void *stream) {
  flagcxResult_t rc = screenTypes(dtype, out_dtype);
  if (rc != flagcxSuccess) return rc;
  if (layout != FX_WEIGHT_NK && layout != FX_WEIGHT_KN) return flagcxInvalidArgument;
  rc = screenSizes(offsets, experts, rows, n, k);
  if (rc != flagcxSuccess) return rc;
  if (experts == 0 || rows == 0 || n == 0) return flagcxSuccess;
  const bool nk = layout == FX_WEIGHT_NK;
  const size_t wCols = nk ? k : n;
  const fxProductStrides st = strides ? *strides : fxProductStrides{k, wCols, n, n * k};
  if (st.x < k || st.w < wCols || st.y < n) return flagcxInvalidArgument;
  if (!at(y, out_dtype == flagcxFloat32 ? 4 : 2) || (k && (!at(x, 2) || !at(w, 2)))) return flagcxInvalidArgument;
  ProductArgs a = {};
  a.pn = w;
  a.pm = x;
  a.y = y;
  a.offsets = offsets;
  a.ldn = st.w;
  a.ldm = st.x;
  a.ldy = st.y;
  a.expertN = st.expert_w;
  a.experts = (uint32_t)experts;
  a.rows = (uint32_t)rows;
  a.n = (uint32_t)n;
  a.k = (uint32_t)k;
  return launch(a, nk ? kFormNK : kFormKN, dtype, out_dtype == flagcxFloat32, stream);
}

int fx_expert_product_dw(void *dw, const void *dy, const void *x, const int32_t *offsets, size_t experts, size_t rows,
                         size_t n, size_t k, const fxProductDwStrides *strides, int dtype, int out_dtype, void *stream) {
  flagcxResult_t rc = screenTypes(dtype, out_dtype);
  if (rc != flagcxSuccess) return rc;
  rc = screenSizes(offsets, experts, rows, n, k);
  if (rc != flagcxSuccess) return rc;
  if (experts == 0 || n == 0 || k == 0) return flagcxSuccess;
  const fxProductDwStrides st = strides ? *strides : fxProductDwStrides{n, k, k, n * k};
  if (st.dy < n || st.x < k || st.dw < k) return flagcxInvalidArgument;
  if (!at(dw, out_dtype == flagcxFloat32 ? 4 : 2) || (rows && (!at(dy, 2) || !at(x, 2)))) return flagcxInvalidArgument;
  ProductArgs a = {};
  a.pn = x;
  a.pm = dy;
  a.y = dw;
  a.offsets = offsets;
  a.ldn = st.x;
  a.ldm = st.dy;
  a.ldy = st.dw;
  a.expertY = st.expert_dw;
  a.experts = (uint32_t)experts;
  a.rows = (uint32_t)rows;
  a.n = (uint32_t)k;
  a.m = (uint32_t)n;
  return launch(a, kFormDw, dtype, out_dtype == flagcxFloat32, stream);
}

int fx_expert_product_e4m3(void *y, const void *x, const float *xscale, const void *w, const float *wscale,
                           const int32_t *offsets, size_t experts, size_t rows, size_t n, size_t k,
                           const fxProductE4m3Strides *strides, int out_dtype, void *stream) {
  if (!known(out_dtype)) return flagcxInvalidArgument;
  if (!sixteen(out_dtype) && out_dtype != flagcxFloat32) return flagcxNotSupported;
  const flagcxResult_t rc = screenSizes(offsets, experts, rows, n, k);
  if (rc != flagcxSuccess) return rc;
  if (experts == 0 || rows == 0 || n == 0) return flagcxSuccess;
  const size_t kg = (k + FX_SCALE_GROUP - 1) / FX_SCALE_GROUP, ng = (n + FX_SCALE_GROUP - 1) / FX_SCALE_GROUP;
  const fxProductE4m3Strides st = strides ? *strides : fxProductE4m3Strides{k, k, n, n * k, kg, kg, ng * kg};
  if (st.x < k || st.w < k || st.y < n || st.xscale < kg || st.wscale < kg) return flagcxInvalidArgument;
  if (!at(y, out_dtype == flagcxFloat32 ? 4 : 2) || (k && (!x || !w || !at(xscale, 4) || !at(wscale, 4))))
    return flagcxInvalidArgument;
  ProductArgs a = {};
  a.pn = w;
  a.pm = x;
  a.y = y;
  a.sn = wscale;
  a.sm = xscale;
  a.offsets = offsets;
  a.ldn = st.w;
  a.ldm = st.x;
  a.ldy = st.y;
  a.expertN = st.expert_w;
  a.ldsn = st.wscale;
  a.ldsm = st.xscale;
  a.expertSn = st.expert_wscale;
  a.experts = (uint32_t)experts;
  a.rows = (uint32_t)rows;
  a.n = (uint32_t)n;
  a.k = (uint32_t)k;
  return launchProductE4m3(a, out_dtype, (hipStream_t)stream);
}

#pragma GCC visibility pop
}
