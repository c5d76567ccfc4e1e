// The big tiles of ff_big.hpp in bfloat16.
#include "ff_big.hpp"

namespace w4a16 {

hipError_t configure_product_big_bf16() { return configure_big<true>(); }
void launch_product_big_bf16(const ProductArgs& a, int rows, Layout layout, hipStream_t stream) {
  launch_big<true>(a, rows, layout, stream);
}

}  // namespace w4a16
