#include "lf_product.h"

namespace lf {
ProductFn product_f16(bool px, bool qx, int tile, bool aligned, bool deep) { return kernel_of<_Float16>(px, qx, tile, aligned, deep); }
ProductFn gated_f16(int tile, bool aligned, bool deep) { return gated_of<_Float16>(tile, aligned, deep); }
}  // namespace lf
