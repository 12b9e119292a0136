// feat_norm.cuh — the argument block of layer norm.
#pragma once

#include "feat_common.cuh"

namespace pwc {
namespace feat {

struct NormArgs {
  const void *x, *w, *b, *dy;
  void *y, *dx, *dw, *db;
  float *mean, *rstd;  // [M]; NULL in a forward pass without a backward one
  float* part;         // [2][parts][C], or NULL: no weight or bias gradient
  long long x_stride;  // between x's tokens / images; the other tensors are dense
  long long B, P, M;   // maps: B images of P pixels; tokens: P = M tokens
  int C, layout;
  float eps;
};

int norm_parts(int layout, long long B, long long P, int C, int dtype);
hipError_t norm_forward(const NormArgs& a, int dtype, hipStream_t s);
hipError_t norm_no_rows(const NormArgs& a, int dtype, hipStream_t s);  // dw = db = 0
hipError_t norm_backward(const NormArgs& a, int parts, int dtype, hipStream_t s);

}  // namespace feat
}  // namespace pwc
