#include "fx_product.hpp"
namespace fx {
flagcxResult_t launchProductF16(const ProductArgs &a, int form, bool outF32, hipStream_t s) {
  return outF32 ? launchForm<_Float16, float>(a, form, s) : launchForm<_Float16, _Float16>(a, form, s);
}
}  // namespace fx
