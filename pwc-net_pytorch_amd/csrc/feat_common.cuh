// feat_common.cuh — shared pieces of the feature operators (layer norm, rotary positions, linear,
// gated linear): 16-byte vectors, reductions over a wave, the activations and their derivatives.
//
// Two layouts of the same M x C matrix of tokens and channels:
//   map    [B][C][P]: the pixels of an image are contiguous, an image may sit at any stride
//   tokens [M][C]:    the channels of a token are contiguous, a token may sit at any stride
#pragma once

#include "pwc_common.cuh"

namespace pwc {
namespace feat {

enum Layout : int { kMap = 0, kTokens = 1 };

// ---- 16-byte vectors of the storage type ----
template <typename T> struct alignas(16) Vec16 {
  static constexpr int N = 16 / (int)sizeof(T);
  T v[N];
};
template <typename T, int N> struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

// Sum over the `W` neighbouring lanes (a power of two) that share a row.
template <int W> __device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = W / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}

// ---- activations (the codes of `activation` in the C ABI) ----
enum Act : int {
  kActNone = 0,
  kActRelu = 1,
  kActLeaky = 2,
  kActSigmoid = 3,
  kActTanh = 4,
  kActSilu = 5,
  kActGelu = 6,      // x * Phi(x)
  kActGeluTanh = 7,  // x * sigmoid(2 a), a = sqrt(2 / pi) (x + 0.044715 x^3)
};

// 1 / (1 + exp(-z)): exp overflows to infinity for z < -88, where the quotient is the right 0.
__device__ __forceinline__ float sigmoid_f(float z) { return 1.f / (1.f + expf(-z)); }

constexpr float kSqrt2OverPi = 0.7978845608028654f;

__device__ __forceinline__ float act_value(int act, float z, float slope) {
  switch (act) {
    case kActRelu: return z > 0.f ? z : (z != z ? z : 0.f);
    case kActLeaky: return z > 0.f ? z : z * slope;
    case kActSigmoid: return sigmoid_f(z);
    case kActTanh: return tanhf(z);
    case kActSilu: return z * sigmoid_f(z);
    case kActGelu: return 0.5f * z * erfcf(-0.7071067811865476f * z);
    case kActGeluTanh:
      return z * sigmoid_f(2.f * kSqrt2OverPi * (z + 0.044715f * z * z * z));
    default: return z;
  }
}

__device__ __forceinline__ float act_slope(int act, float z, float slope) {
  switch (act) {
    case kActRelu: return z > 0.f ? 1.f : 0.f;
    case kActLeaky: return z > 0.f ? 1.f : slope;
    case kActSigmoid: {
      const float p = sigmoid_f(z);
      return p * (1.f - p);
    }
    case kActTanh: {
      const float t = tanhf(z);
      return 1.f - t * t;
    }
    case kActSilu: {
      const float p = sigmoid_f(z);
      return p * (1.f + z * (1.f - p));
    }
    case kActGelu:
      return 0.5f * erfcf(-0.7071067811865476f * z) +
             z * 0.3989422804014327f * expf(-0.5f * z * z);
    case kActGeluTanh: {
      const float p = sigmoid_f(2.f * kSqrt2OverPi * (z + 0.044715f * z * z * z));
      return p + z * p * (1.f - p) * 2.f * kSqrt2OverPi * (1.f + 0.134145f * z * z);
    }
    default: return 1.f;
  }
}

inline size_t align256(size_t n) { return (n + 255) / 256 * 256; }
inline bool aligned_to(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

}  // namespace feat
}  // namespace pwc
