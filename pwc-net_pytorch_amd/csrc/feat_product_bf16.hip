// feat_product_bf16.hip — the matrix products of the feature operators in bf16.
#include "feat_product_kernel.cuh"

namespace pwc {
namespace feat {
template hipError_t product_t<__hip_bfloat16>(const ProductArgs&, const ProductPlan&, hipStream_t);
}  // namespace feat
}  // namespace pwc
