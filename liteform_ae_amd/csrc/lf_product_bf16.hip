#include "lf_product.h"

namespace lf {
ProductFn product_bf16(bool px, bool qx, int tile, bool aligned, bool deep) { return kernel_of<__bf16>(px, qx, tile, aligned, deep); }
}  // namespace lf
