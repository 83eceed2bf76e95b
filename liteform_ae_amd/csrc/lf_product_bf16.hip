#include "lf_product.h"

namespace lf {
ProductFn product_bf16(bool px, bool qx, int tile, bool aligned, bool deep) { return kernel_of<__bf16>(px, qx, tile, aligned, deep); }
ProductFn gated_bf16(int tile, bool aligned, bool deep) { return gated_of<__bf16>(tile, aligned, deep); }
}  // namespace lf
