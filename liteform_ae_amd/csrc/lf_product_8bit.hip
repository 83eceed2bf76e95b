#include "lf_product.h"

namespace lf {
// (8-bit operands are those of the forward product: both along k)
ProductFn product_e4m3(bool, bool, int tile, bool aligned, bool deep) { return kernel_of<e4m3_t, false, false>(tile, aligned, deep); }
ProductFn product_i8(bool, bool, int tile, bool aligned, bool deep) { return kernel_of<int8_t, false, false>(tile, aligned, deep); }
ProductFn gated_e4m3(int tile, bool aligned, bool deep) { return gated_of<e4m3_t>(tile, aligned, deep); }
ProductFn gated_i8(int tile, bool aligned, bool deep) { return gated_of<int8_t>(tile, aligned, deep); }
}  // namespace lf
