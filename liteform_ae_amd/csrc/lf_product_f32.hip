#include "lf_product.h"

namespace lf {
ProductFn product_f32(bool px, bool qx, int tile) { return kernel_of<float>(px, qx, tile); }
}  // namespace lf
