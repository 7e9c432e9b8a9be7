#include "fx_product.hpp"
namespace fx {
flagcxResult_t launchProductE4m3(const ProductArgs &a, int outDtype, hipStream_t s) {
  switch (outDtype) {
    case flagcxBfloat16: return launchForm<E4m3, __bf16>(a, kFormNK, s);
    case flagcxFloat16: return launchForm<E4m3, _Float16>(a, kFormNK, s);
    default: return launchForm<E4m3Exact, float>(a, kFormNK, s);
  }
}
}  // namespace fx
