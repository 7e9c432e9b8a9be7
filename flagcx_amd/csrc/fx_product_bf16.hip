#include "fx_product.hpp"
namespace fx {
flagcxResult_t launchProductBf16(const ProductArgs &a, int form, bool outF32, hipStream_t s) {
  return outF32 ? launchForm<__bf16, float>(a, form, s) : launchForm<__bf16, __bf16>(a, form, s);
}
}  // namespace fx
