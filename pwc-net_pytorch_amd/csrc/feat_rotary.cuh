// feat_rotary.cuh — the argument block of the rotary positions.
#pragma once

#include "feat_common.cuh"

namespace pwc {
namespace feat {

constexpr int kMaxAxes = 4;

struct RotaryArgs {
  const void* x;
  void* y;
  const void* positions;   // [B][N][axes] by strides, or NULL: raster places of `grid`
  const double* inv_freq;  // [R]
  const int* axis;         // [R]
  long long xs_b, xs_n, xs_h, xs_d, ys_b, ys_n, ys_h, ys_d;
  long long pos_b, pos_n, pos_a;
  long long B, N;
  int H, D, R, axes, pos_type, interleaved;  // pos_type: 0 float, 1 int32, 2 int64
  long long grid[kMaxAxes], origin[kMaxAxes];
  float sign;              // 1 forward, -1 backward
  uint32_t inner[kMaxAxes];               // set by the launcher
  int heads_each, head_groups;
  long long batch_each, batch_groups;
};

hipError_t rotary_launch(const RotaryArgs& a, int dtype, hipStream_t stream);

}  // namespace feat
}  // namespace pwc
