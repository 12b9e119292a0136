// feat_product.cuh — the argument block of the feature operators' matrix product.
#pragma once

#include "feat_common.cuh"

namespace pwc {
namespace feat {

enum ProductMode : int {
  kLinear = 0,    // act(sum + bias) + other
  kLinearDz = 1,  // other * act'(sum + bias)
  kGated = 2,     // act(gate) * up
  kGatedDz = 3,   // [other * up * act'(gate), other * act(gate)]
  kPartial = 4,   // 32-bit sums of one split of k, and the sums of B's rows
};

// Out(i, j) = sum_k A(i, k) B(j, k), at out[j * ldo + i]; strides in elements.
struct ProductArgs {
  const void* a;
  const void* b;
  void* out;
  const void* bias;   // along i (bias_i) or j, or NULL
  const void* other;  // residual or output gradient, or NULL; at ldother
  float* sums;        // kPartial: [splits][J] sums over k of B(j, k), or NULL
  long long lda, ldb, ldo, ldother;
  long long a_batch, b_batch, out_batch, other_batch;
  long long a_segment, b_segment;  // k runs over `segments` segments of K
  int I, J, K, segments, batches, splits;
  int a_k, b_k;        // the operand lies along k
  int pair_side;       // 0, or 1 (A) / 2 (B): that operand is [gate; up], `pair` rows each
  int pair;
  int bias_i, mode, act;
  float slope;
  int tiles_i, tiles_j;  // set by the launcher
};

hipError_t product_launch(const ProductArgs& g, int dtype, hipStream_t stream);
int product_splits(long long I, long long J, int segments, long long K, int dtype);
hipError_t product_add_splits(const float* part, void* out, long long n, int splits, int dtype,
                              hipStream_t stream);

}  // namespace feat
}  // namespace pwc
