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

template <typename T, int N> struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

// The rounding to storage, with the conversion instructions that this target has for bfloat16.
template <typename T> __device__ __forceinline__ T narrow(float v) { return from_f32<T>(v); }
template <> __device__ __forceinline__ __hip_bfloat16 narrow<__hip_bfloat16>(float v) {
  return __builtin_bit_cast(__hip_bfloat16, (__bf16)v);
}

// 16 bytes at any alignment of their values
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_at2 __attribute__((ext_vector_type(4), aligned(2)));
typedef uint32_t u32x4_at4 __attribute__((ext_vector_type(4), aligned(4)));
template <typename T> struct Any16 { typedef u32x4_at2 type; };
template <> struct Any16<float> { typedef u32x4_at4 type; };
template <typename T> __device__ __forceinline__ u32x4 load16(const T* p) {
  return *(const typename Any16<T>::type*)p;
}
// the first `have` values of 16 bytes, zeros behind them
template <typename T> __device__ __forceinline__ u32x4 load_some(const T* p, int have) {
  u32x4 v = {0u, 0u, 0u, 0u};
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      if (e < have) v[e] = ((const uint32_t*)p)[e];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < have) v[e / 2] |= (uint32_t)((const uint16_t*)p)[e] << (e % 2 * 16);
  }
  return v;
}
// V values of 16 bytes as floats
template <typename T, int V> __device__ __forceinline__ void as_floats(u32x4 p, float (&v)[V]) {
  static_assert(V * sizeof(T) == 16, "");
  const Pack<T, V> o = __builtin_bit_cast(Pack<T, V>, p);
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = to_f32(o.v[e]);
}
// V values (16 bytes, or one) as floats
template <typename T, int V>
__device__ __forceinline__ void load_values(const T* p, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = to_f32(*p);
  } else {
    as_floats<T, V>(load16(p), v);
  }
}
template <typename T, int V>
__device__ __forceinline__ void store_values(T* p, const float (&v)[V]) {
  if constexpr (V == 1) {
    *p = narrow<T>(v[0]);
  } else {
    static_assert(V * sizeof(T) == 16, "");
    Pack<T, V> o;
#pragma unroll
    for (int e = 0; e < V; ++e) o.v[e] = narrow<T>(v[e]);
    *(typename Any16<T>::type*)p = __builtin_bit_cast(u32x4, o);
  }
}

// Four neighbouring values at any alignment, zeros (nothing) from `left` on
typedef uint32_t u32x2_at2 __attribute__((ext_vector_type(2), aligned(2)));
template <typename T>
__device__ __forceinline__ void load_four(const T* p, int left, float (&v)[4]) {
  u32x4 q = {0u, 0u, 0u, 0u};
  if (left >= 4) {
    if constexpr (sizeof(T) == 4) {
      q = load16(p);
    } else {
      const u32x2_at2 h = *(const u32x2_at2*)p;
      q = u32x4{h[0], h[1], 0u, 0u};
    }
  } else if (left > 0) {
    q = load_some(p, left);
  }
  const Pack<T, 16 / sizeof(T)> o = __builtin_bit_cast(Pack<T, 16 / sizeof(T)>, q);
#pragma unroll
  for (int e = 0; e < 4; ++e) v[e] = to_f32(o.v[e]);
}
template <typename T>
__device__ __forceinline__ void store_four(T* p, const float (&v)[4], int left) {
  Pack<T, 16 / sizeof(T)> o = {};
#pragma unroll
  for (int e = 0; e < 4; ++e) o.v[e] = narrow<T>(v[e]);
  const u32x4 q = __builtin_bit_cast(u32x4, o);
  if (left >= 4) {
    if constexpr (sizeof(T) == 4)
      *(u32x4_at4*)p = q;
    else
      *(u32x2_at2*)p = u32x2_at2{q[0], q[1]};
  } else {
#pragma unroll
    for (int e = 0; e < 3; ++e)
      if (e < left) p[e] = o.v[e];
  }
}
// what rounding takes from the values; nothing where it gives an infinity or a NaN
template <typename T, int V> __device__ __forceinline__ void rounded_off(float (&v)[V]) {
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const float h = to_f32(narrow<T>(v[e]));
    v[e] = fabsf(h) < __builtin_inff() ? v[e] - h : 0.f;
  }
}

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

// The functions for 32-bit results are the device library's.  For 16-bit results (FAST) they are
// the hardware's exponential and reciprocal: the exponent is rounded before it is raised, so exp(-x)
// is off by |x| 2^-24 of its value and a step or two, against an output's rounding of 2^-11 or 2^-8.
template <bool FAST> __device__ __forceinline__ float exp_neg(float x) {  // exp(-x)
  return FAST ? __builtin_amdgcn_exp2f(-1.4426950408889634f * x) : expf(-x);
}
template <bool FAST> __device__ __forceinline__ float recip(float x) {
  return FAST ? __builtin_amdgcn_rcpf(x) : 1.f / x;
}
// exp overflows to infinity for z < -88.7, where the reciprocal gives 0 for what is below 2^-127
template <bool FAST> __device__ __forceinline__ float sigmoid_f(float z) {
  return recip<FAST>(1.f + exp_neg<FAST>(z));
}
// Phi(-|z|), the normal distribution's tail, given gauss = exp(-z^2 / 2), which it falls with: the
// quotient is a polynomial in t = 1 / (1 + 0.34 |z|) without a constant, fitted to 64-bit values for
// |z| up to 14 so that the tail is off by at most 1.1e-5 of itself everywhere and 1.6e-8 absolutely.
// (With 32-bit rounding 1.4e-5 at |z| = 13, where gauss is off by as much: a 300th of bf16's half
// step.  The best five terms are off by 7e-4 of the tail and 5e-7, for 4 us of the 347 of a training
// pass of 8192 x 1024 -> 4096.)
__device__ __forceinline__ float tail_f(float z, float gauss) {
  const float t = recip<true>(1.f + 0.34f * fabsf(z));
  float p = 0.043755324f;
  p = p * t - 0.19595344f;
  p = p * t + 0.256176078f;
  p = p * t - 0.0237047643f;
  p = p * t + 0.153229921f;
  p = p * t + 0.130545621f;
  p = p * t + 0.135951245f;
  return p * t * gauss;
}

constexpr float kSqrt2OverPi = 0.7978845608028654f;

// f = act(z) and, where SLOPE, d = act'(z), for N values: one branch for all of them.  `slope` is
// leaky relu's.
template <bool FAST, bool SLOPE, int N>
__device__ __forceinline__ void activate(int act, const float (&z)[N], float (&f)[N],
                                         float (&d)[N], float slope) {
  if (act == kActSilu) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float p = sigmoid_f<FAST>(z[e]);
      f[e] = z[e] * p;
      if (SLOPE) d[e] = p * (1.f + z[e] * (1.f - p));
    }
  } else if (act == kActGelu) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      const float z2 = z[e] * z[e];
      if (FAST) {
        const float g = __builtin_amdgcn_exp2f(-0.7213475204444817f * z2);
        const float t = tail_f(z[e], g);
        const float p = z[e] > 0.f ? 1.f - t : t;
        f[e] = z[e] * p;
        if constexpr (SLOPE) d[e] = p + z[e] * (0.3989422804014327f * g);
      } else {
        const float p = 0.5f * erfcf(-0.7071067811865476f * z[e]);
        f[e] = z[e] * p;
        if (SLOPE) d[e] = p + z[e] * 0.3989422804014327f * expf(-0.5f * z2);
      }
    }
  } else if (act == kActGeluTanh) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      // (from 100 on p is 0 or 1 whatever z^2 is; as infinity it would make 0 * inf of the slope)
      const float q = fminf(z[e] * z[e], 1e4f);
      const float p = sigmoid_f<FAST>(2.f * kSqrt2OverPi * (z[e] + 0.044715f * z[e] * q));
      f[e] = z[e] * p;
      if (SLOPE) d[e] = p + f[e] * (1.f - p) * 2.f * kSqrt2OverPi * (1.f + 0.134145f * q);
    }
  } else if (act == kActRelu || act == kActLeaky) {
    const float s = act == kActRelu ? 0.f : slope;
#pragma unroll
    for (int e = 0; e < N; ++e) {
      f[e] = z[e] > 0.f ? z[e] : act == kActRelu ? (z[e] != z[e] ? z[e] : 0.f) : z[e] * s;
      if (SLOPE) d[e] = z[e] > 0.f ? 1.f : s;
    }
  } else if (act == kActSigmoid) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      f[e] = sigmoid_f<FAST>(z[e]);
      if (SLOPE) d[e] = f[e] * (1.f - f[e]);
    }
  } else if (act == kActTanh) {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      // (2 sigmoid(2 z) - 1 would lose a small z's digits)
      f[e] = tanhf(z[e]);
      if (SLOPE) d[e] = 1.f - f[e] * f[e];
    }
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) {
      f[e] = z[e];
      if (SLOPE) d[e] = 1.f;
    }
  }
}

// A grid of any number of blocks: one dimension holds 2^24 of 256 threads.  Blocks behind the last
// have work of their own to check for.
__device__ __forceinline__ long long block_id() {
  return blockIdx.y * (long long)gridDim.x + blockIdx.x;
}
inline dim3 grid_of(long long blocks) {
  const long long x = blocks < (1 << 20) ? blocks : 1 << 20;
  return dim3((unsigned)x, (unsigned)((blocks + x - 1) / x));
}

inline size_t align256(size_t n) { return (n + 255) / 256 * 256; }
inline bool aligned_to(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

}  // namespace feat
}  // namespace pwc
