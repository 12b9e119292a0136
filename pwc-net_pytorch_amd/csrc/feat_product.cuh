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
  kPlain = 5,     // the sum
  kPartial = 4,   // 32-bit sums of one split of k; one split alone: the result
};

// Out(i, j) = sum_k A(i, k) B(j, k), at out[j * ldo + i]; strides in elements.
struct ProductArgs {
  const void* a;
  const void* b;
  void* out;
  const void* bias;   // along the channels, or NULL
  const void* other;  // residual or output gradient, or NULL; at ldother
  float* part;        // workspace for 32-bit sums of the splits of k (kPartial's are its output)
  size_t part_bytes;  // its size, or kPartial's output's
  float* sums;        // k*Dz: partial sums of dz over the tokens, product_sum_rows rows, or NULL
  long long lda, ldb, ldo, ldother;
  long long a_batch, b_batch, out_batch, other_batch;
  long long a_segment, b_segment;  // k runs over `segments` segments of K
  long long low;      // k*Dz in 16 bits, 64-tiles and few tokens: where what rounding took goes, or 0
  int a_halves;       // pairs of segments share A's
  int I, J, K, segments, batches, splits;
  int a_k, b_k;        // the operand lies along k
  int a_pad, b_pad;    // its rows are filled up with zeros to whole 16 bytes
  int pair;            // kGated*: W is [gate; up], `pair` rows each
  int channel_i;       // forward / dz: the channels lie along i (tokens) or j (maps)
  int mode, act;
  float slope;
  int tiles_i, tiles_j;  // set by the launcher
};

// The kernels.  Direct loads from aligned rows; Any reads through registers.
enum ProductKernel : int {
  kFew16,  // passes over W for at most 16, 32, 64 tokens
  kFew32,
  kFew64,
  kTile64,
  kTile64Deep,  // three steps in LDS
  kTile64Any,
  kTile128,
  kTile256,
};
struct ProductPlan {
  int kernel;
  int bi, bj, passes;  // the tile; column halves that the epilogue takes it in
  int splits;        // of k: kPartial, or summed and finished by a kernel of its own
};
ProductPlan product_plan(const ProductArgs& g, int dtype);
template <typename T>
hipError_t product_t(const ProductArgs& g, const ProductPlan& p, hipStream_t stream);

hipError_t product_launch(const ProductArgs& g, int dtype, hipStream_t stream);
size_t product_part_bytes(const ProductArgs& g, int dtype);
int product_sum_rows(const ProductArgs& g, int dtype);
int product_column_parts(int layout, long long B, long long P, int C);
hipError_t product_column_sums(const void* dy, float* part, int layout, long long B, long long P,
                               int C, int parts, int dtype, hipStream_t stream);

// Several small passes over memory in one launch, each with a share of the grid.
constexpr int kJobs = 3;
// dst: `rows` rows of `cols` values, zeros up to the next 16 bytes; src: rows `row` apart, groups of
// `per_image` rows `image` apart.  Without src the zeros alone.  rows 0: no job
struct LayJob {
  const void* src;
  void* dst;
  long long row, image, per_image, rows, cols;
};
hipError_t product_lay_out(const LayJob (&jobs)[kJobs], int dtype, hipStream_t stream);
// out[n] = sum over `parts` rows of n values, in a fixed order (zeros for none).  n 0: no job
struct SumJob {
  const float* part;
  void* out;
  long long n;
  int parts;
};
hipError_t product_sum(const SumJob (&jobs)[kJobs], int dtype, hipStream_t stream);

}  // namespace feat
}  // namespace pwc
