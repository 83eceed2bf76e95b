#include "lf_product.h"

namespace lf {
ProductFn product_f32(bool px, bool qx, int tile, bool aligned, bool deep) { return kernel_of<float>(px, qx, tile, aligned, deep); }
}  // namespace lf
