// feat_product_f32.hip — the matrix products of the feature operators in fp32.
#include "feat_product_kernel.cuh"

namespace pwc {
namespace feat {
template hipError_t product_t<float>(const ProductArgs&, const ProductPlan&, hipStream_t);
}  // namespace feat
}  // namespace pwc
