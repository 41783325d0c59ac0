// The products that read the gradient of the logits (product.h): a file of their own, for the compiler's sake.
#include "product.h"

namespace moda {

hipError_t launch_grad_rows(const ProductArgs& a, int dtype, ProductTile tile, int compute_units, hipStream_t stream) { return launch_product<kGradRows>(a, dtype, tile, compute_units, stream); }
hipError_t launch_grad_weight(const ProductArgs& a, int dtype, ProductTile tile, int compute_units, hipStream_t stream) {
  return launch_product<kGradWeight>(a, dtype, tile, compute_units, stream);
}

}  // namespace moda
