// The big tiles of ff_big.hpp in fp16.
#include "ff_big.hpp"

namespace w4a16 {

hipError_t configure_product_big_f16() { return configure_big<false>(); }
void launch_product_big_f16(const ProductArgs& a, int rows, Layout layout, hipStream_t stream) {
  launch_big<false>(a, rows, layout, stream);
}

}  // namespace w4a16
