// feat_product_f16.hip — the matrix products of the feature operators in fp16.
#include "feat_product_kernel.cuh"

namespace pwc {
namespace feat {
template hipError_t product_t<__half>(const ProductArgs&, const ProductPlan&, hipStream_t);
}  // namespace feat
}  // namespace pwc
