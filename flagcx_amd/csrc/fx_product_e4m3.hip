#include "fx_product.hpp"
namespace fx {
flagcxResult_t launchProductE4m3(const ProductArgs &a, int outDtype, hipStream_t s) {
  switch (outDtype) {
    case flagcxBfloat16: return launchShapes<E4m3, __bf16, false, false, false>(a, s);
    case flagcxFloat16: return launchShapes<E4m3, _Float16, false, false, false>(a, s);
    default: return launchShapes<E4m3Exact, float, false, false, false>(a, s);
  }
}
}  // namespace fx
