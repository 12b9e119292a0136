// feat_norm.hip — layer norm over the channels of feature maps and tokens.
//
//   forward   mu = mean_c x,  r = 1 / sqrt(mean_c (x - mu)^2 + eps),  y = (x - mu) r w + b
//   backward  with xh = (x - mu) r and h = w dy:
//             dx = r (h - mean_c h - xh mean_c (h xh)),  dw = sum_m dy xh,  db = sum_m dy
//
// Both are bound by memory: one read of x (and dy), one write of y (dx).  A row's values stay in
// registers between the statistics and the result, the variance is summed from x - mu (so a large
// mean costs no digits), every sum is in 32 bits.  The weight's gradient is summed by each thread
// for its own channels over the rows of a block that stays on its CU, then over the blocks in
// their order: no atomics, the same sums each time.
//
// Measured: 16383 x 2048 bf16 tokens 29 us forward (4.6 TB/s) and 46 backward (4.4; a 1 GiB copy does
// 5.2), a block a row; the 8 x 32 x 96 x 112 fp32 map 6.5 and 9.6 us, 64 pixels a block, and 4 us for
// the sums over blocks.
#include "feat_common.cuh"
#include "feat_norm.cuh"

namespace pwc {
namespace feat {

// ------------------------------------------------------------------------------ tokens [M][C]
// TPR threads share a row; each has NV vectors of V channels, TPR * V apart.
template <int TPR> __device__ __forceinline__ float row_sum(float v, float* red) {
  v = lanes_sum<(TPR < 64 ? TPR : 64)>(v);
  if constexpr (TPR > 64) {  // the whole block: waves joined through LDS
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int w = 0; w < TPR / 64; ++w) v += red[w];
  }
  return v;
}

// V values of a row, of which `have` exist (WHOLE: all or none do, and the caller has looked): rows of
// odd lengths are read in 16-byte pieces too, from any address.
template <typename T, int V, bool WHOLE>
__device__ __forceinline__ void load_row(const T* p, int have, float (&v)[V]) {
  if constexpr (WHOLE) {
    load_values<T, V>(p, v);
  } else {
    as_floats<T, V>(have >= V ? load16(p) : load_some(p, have), v);
  }
}
template <typename T, int V, bool WHOLE>
__device__ __forceinline__ void store_row(T* p, int have, const float (&v)[V]) {
  if (WHOLE || have >= V) {
    store_values<T, V>(p, v);
  } else {
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (e < have) p[e] = narrow<T>(v[e]);
  }
}

template <typename T, int TPR, int NV, int V, bool WHOLE>
__global__ __launch_bounds__(256) void norm_tokens(const NormArgs a) {
  __shared__ float red[4];
  constexpr int RPB = 256 / TPR;
  const int t = threadIdx.x % TPR;
  const long long m = block_id() * RPB + threadIdx.x / TPR;
  const bool row = m < a.M;
  const T* x = (const T*)a.x + (row ? m : 0) * a.x_stride;
  float v[NV][V];
  float s = 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (k * TPR + t) * V;
    if (c < a.C) {
      load_row<T, V, WHOLE>(x + c, a.C - c, v[k]);
#pragma unroll
      for (int e = 0; e < V; ++e) s += v[k][e];
    }
  }
  const float mu = row_sum<TPR>(s, red) / a.C;
  s = 0.f;
#pragma unroll
  for (int k = 0; k < NV; ++k)
    if ((k * TPR + t) * V < a.C)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        v[k][e] -= mu;
        if (WHOLE || (k * TPR + t) * V + e < a.C) s += v[k][e] * v[k][e];
      }
  const float r = 1.f / sqrtf(row_sum<TPR>(s, red) / a.C + a.eps);
  if (!row) return;
  if (a.mean && t == 0) {
    a.mean[m] = mu;
    a.rstd[m] = r;
  }
  T* y = (T*)a.y + m * a.C;
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (k * TPR + t) * V;
    if (c < a.C) {
      float w[V], b[V];
      if (a.w) load_row<T, V, WHOLE>((const T*)a.w + c, a.C - c, w);
      if (a.b) load_row<T, V, WHOLE>((const T*)a.b + c, a.C - c, b);
#pragma unroll
      for (int e = 0; e < V; ++e) v[k][e] = v[k][e] * r * (a.w ? w[e] : 1.f) + (a.b ? b[e] : 0.f);
      store_row<T, V, WHOLE>(y + c, a.C - c, v[k]);
    }
  }
}

template <typename T, int TPR, int NV, int V, bool WHOLE>
__global__ __launch_bounds__(256) void norm_tokens_backward(const NormArgs a) {
  extern __shared__ float lds[];
  constexpr int RPB = 256 / TPR;
  float* red = lds;
  const int t = threadIdx.x % TPR;
  float w[NV][V], dw[NV][V], db[NV][V];
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (k * TPR + t) * V;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      w[k][e] = 1.f;
      dw[k][e] = db[k][e] = 0.f;
    }
    if (a.w && c < a.C) load_row<T, V, WHOLE>((const T*)a.w + c, a.C - c, w[k]);
  }
  for (long long m0 = (long long)blockIdx.x * RPB; m0 < a.M; m0 += (long long)gridDim.x * RPB) {
    const long long m = m0 + threadIdx.x / TPR;
    const bool row = m < a.M;
    const T* x = (const T*)a.x + (row ? m : 0) * a.x_stride;
    const T* dy = (const T*)a.dy + (row ? m : 0) * a.C;
    const float mu = row ? a.mean[m] : 0.f, r = row ? a.rstd[m] : 0.f;
    float xh[NV][V], h[NV][V];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int k = 0; k < NV; ++k) {
      const int c = (k * TPR + t) * V;
      if (row && c < a.C) {
        load_row<T, V, WHOLE>(x + c, a.C - c, xh[k]);
        load_row<T, V, WHOLE>(dy + c, a.C - c, h[k]);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          xh[k][e] = WHOLE || c + e < a.C ? (xh[k][e] - mu) * r : 0.f;
          dw[k][e] += h[k][e] * xh[k][e];
          db[k][e] += h[k][e];
          h[k][e] *= w[k][e];
          s1 += h[k][e];
          s2 += h[k][e] * xh[k][e];
        }
      }
    }
    s1 = row_sum<TPR>(s1, red) / a.C;
    s2 = row_sum<TPR>(s2, red) / a.C;
    if (row && a.dx) {
#pragma unroll
      for (int k = 0; k < NV; ++k) {
        const int c = (k * TPR + t) * V;
        if (c < a.C) {
#pragma unroll
          for (int e = 0; e < V; ++e) h[k][e] = r * (h[k][e] - s1 - xh[k][e] * s2);
          store_row<T, V, WHOLE>((T*)a.dx + m * a.C + c, a.C - c, h[k]);
        }
      }
    }
  }
  if (!a.part) return;
  // rows of the wave, then waves of the block, then [2][blocks][C]
  float* acc = lds + 4;  // RPB > 1: [4][2][C]
#pragma unroll
  for (int k = 0; k < NV; ++k) {
    const int c = (k * TPR + t) * V;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if constexpr (TPR < 64) {
#pragma unroll
        for (int o = TPR; o < 64; o <<= 1) {
          dw[k][e] += __shfl_xor(dw[k][e], o, 64);
          db[k][e] += __shfl_xor(db[k][e], o, 64);
        }
      }
      if (c + e < a.C) {
        if constexpr (RPB == 1) {
          a.part[(long long)blockIdx.x * a.C + c + e] = dw[k][e];
          a.part[((long long)gridDim.x + blockIdx.x) * a.C + c + e] = db[k][e];
        } else if ((threadIdx.x & 63) < TPR) {
          acc[(threadIdx.x >> 6) * 2 * a.C + c + e] = dw[k][e];
          acc[((threadIdx.x >> 6) * 2 + 1) * a.C + c + e] = db[k][e];
        }
      }
    }
  }
  if constexpr (RPB > 1) {
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * a.C; i += 256) {
      const float v = acc[i] + acc[2 * a.C + i] + acc[4 * a.C + i] + acc[6 * a.C + i];
      const int c = i < a.C ? i : i - a.C;
      a.part[((long long)(i < a.C ? 0 : gridDim.x) + blockIdx.x) * a.C + c] = v;
    }
  }
}

// ------------------------------------------------------------------------------ maps [B][C][P]
// A block takes 64 PV pixels, a lane PV neighbours (4 bytes of 16-bit values where P is even); wave
// g of G holds NC channels g, g + G, ... in registers; more than 256 channels go by the loops below.

template <int G, int PV>
__device__ __forceinline__ void pixel_sum(float (&v)[PV], float (*red)[64 * PV]) {
  if constexpr (G > 1) {
    const int l = threadIdx.x & 63, g = threadIdx.x >> 6;
    __syncthreads();
#pragma unroll
    for (int e = 0; e < PV; ++e) red[g][l * PV + e] = v[e];
    __syncthreads();
#pragma unroll
    for (int e = 0; e < PV; ++e) {
      v[e] = 0.f;
#pragma unroll
      for (int k = 0; k < G; ++k) v[e] += red[k][l * PV + e];
    }
  }
}
// Sums over a wave of N values a lane (N a power of two): halves are exchanged, so N + 6 shuffles do
// what 6 N would.  Lane l returns the sum of value l / (64 / N).  (Steps by recursion: with a step
// count that the compiler does not see through, the values move to LDS.)
template <int N, int BIT, int M> __device__ __forceinline__ float fold_from(float (&v)[M]) {
  if constexpr (N > 1) {
    const bool up = threadIdx.x & BIT;
#pragma unroll
    for (int k = 0; k < N / 2; ++k) {
      const float give = up ? v[k] : v[k + N / 2], keep = up ? v[k + N / 2] : v[k];
      v[k] = keep + __shfl_xor(give, BIT, 64);
    }
    return fold_from<N / 2, BIT / 2>(v);
  } else {
    return lanes_sum<2 * BIT>(v[0]);
  }
}
template <int N> __device__ __forceinline__ float fold_lanes(float (&v)[N]) {
  return fold_from<N, 32>(v);
}
template <typename T, int PV>
__device__ __forceinline__ void load_pixels(const T* p, uint32_t at, bool ok, float (&v)[PV]) {
  Pack<T, PV> o;
#pragma unroll
  for (int e = 0; e < PV; ++e) o.v[e] = narrow<T>(0.f);
  if (ok) o = *(const Pack<T, PV>*)(p + at);
#pragma unroll
  for (int e = 0; e < PV; ++e) v[e] = to_f32(o.v[e]);
}
// A wave's channels g, g + G, ...: lane k holds channel k's value (`otherwise` where there is none),
// so that one load fetches all; a load a channel would be waited for one after the other.
template <typename T>
__device__ __forceinline__ float wave_channels(const void* p, int g, int G, int C,
                                               float otherwise) {
  const int c = (int)(threadIdx.x & 63) * G + g;
  return p && c < C ? to_f32(((const T*)p)[c]) : otherwise;
}
__device__ __forceinline__ float channel_of(float held, int k) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, held), k));
}
template <typename T, int PV>
__device__ __forceinline__ void store_pixels(T* p, uint32_t at, const float (&v)[PV]) {
  Pack<T, PV> o;
#pragma unroll
  for (int e = 0; e < PV; ++e) o.v[e] = narrow<T>(v[e]);
  *(Pack<T, PV>*)(p + at) = o;
}

template <typename T, int G, int NC, int PV>
__global__ __launch_bounds__(64 * G) void norm_map(const NormArgs a) {
  __shared__ float red[G][64 * PV];
  const int l = threadIdx.x & 63;
  const int g = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);  // channels: uniform
  const uint32_t P = (uint32_t)a.P;  // (an image's offsets fit 32 bits)
  const long long tiles = (a.P + 64 * PV - 1) / (64 * PV);
  const long long id = block_id(), img = id / tiles;
  const uint32_t p = (uint32_t)((id % tiles * 64 + l) * PV);
  const bool ok = p < P && img < a.B;
  const T* x = (const T*)a.x + img * a.x_stride;
  const float weights = wave_channels<T>(a.w, g, G, a.C, 1.f);
  const float biases = wave_channels<T>(a.b, g, G, a.C, 0.f);
  float v[NC][PV], s[PV], r[PV], mu[PV];
#pragma unroll
  for (int e = 0; e < PV; ++e) s[e] = 0.f;
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    const int c = k * G + g;
    load_pixels<T, PV>(x, c * P + p, ok && c < a.C, v[k]);
#pragma unroll
    for (int e = 0; e < PV; ++e) s[e] += v[k][e];
  }
  pixel_sum<G, PV>(s, red);
#pragma unroll
  for (int e = 0; e < PV; ++e) {
    mu[e] = s[e] / a.C;
    s[e] = 0.f;
  }
#pragma unroll
  for (int k = 0; k < NC; ++k)
    if (k * G + g < a.C)
#pragma unroll
      for (int e = 0; e < PV; ++e) {
        v[k][e] -= mu[e];
        s[e] += v[k][e] * v[k][e];
      }
  pixel_sum<G, PV>(s, red);
#pragma unroll
  for (int e = 0; e < PV; ++e) r[e] = 1.f / sqrtf(s[e] / a.C + a.eps);
  if (!ok) return;
  if (a.mean && g == 0)
#pragma unroll
    for (int e = 0; e < PV; ++e) {
      a.mean[img * a.P + p + e] = mu[e];
      a.rstd[img * a.P + p + e] = r[e];
    }
  T* y = (T*)a.y + img * a.C * a.P;
#pragma unroll
  for (int k = 0; k < NC; ++k) {
    const int c = k * G + g;
    if (c < a.C) {
      const float w = channel_of(weights, k), b = channel_of(biases, k);
#pragma unroll
      for (int e = 0; e < PV; ++e) v[k][e] = v[k][e] * r[e] * w + b;
      store_pixels<T, PV>(y, c * P + p, v[k]);
    }
  }
}

template <typename T, int G, int NC, int PV>
__global__ __launch_bounds__(64 * G) void norm_map_backward(const NormArgs a) {
  __shared__ float red[G][64 * PV];
  const int l = threadIdx.x & 63;
  const int g = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);  // channels: uniform
  const uint32_t P = (uint32_t)a.P;  // (an image's offsets fit 32 bits)
  const long long tiles = (a.P + 64 * PV - 1) / (64 * PV);
  const float weights = wave_channels<T>(a.w, g, G, a.C, 1.f);
  float dw[NC], db[NC];
#pragma unroll
  for (int k = 0; k < NC; ++k) dw[k] = db[k] = 0.f;
  for (long long t = blockIdx.x; t < tiles * a.B; t += gridDim.x) {
    const long long img = t / tiles;
    const uint32_t p = (uint32_t)((t % tiles * 64 + l) * PV);
    const bool ok = p < P;
    const T* x = (const T*)a.x + img * a.x_stride;
    const T* dy = (const T*)a.dy + img * a.C * a.P;
    float xh[NC][PV], h[NC][PV], mu[PV], r[PV], s1[PV], s2[PV];
#pragma unroll
    for (int k = 0; k < NC; ++k) {
      const bool have = ok && k * G + g < a.C;
      load_pixels<T, PV>(x, (k * G + g) * P + p, have, xh[k]);
      load_pixels<T, PV>(dy, (k * G + g) * P + p, have, h[k]);
    }
#pragma unroll
    for (int e = 0; e < PV; ++e) {
      mu[e] = ok ? a.mean[img * a.P + p + e] : 0.f;
      r[e] = ok ? a.rstd[img * a.P + p + e] : 0.f;
      s1[e] = s2[e] = 0.f;
    }
#pragma unroll
    for (int k = 0; k < NC; ++k)
      if (k * G + g < a.C) {
        const float w = channel_of(weights, k);
#pragma unroll
        for (int e = 0; e < PV; ++e) {
          xh[k][e] = (xh[k][e] - mu[e]) * r[e];
          dw[k] += h[k][e] * xh[k][e];
          db[k] += h[k][e];
          h[k][e] *= w;
          s1[e] += h[k][e];
          s2[e] += h[k][e] * xh[k][e];
        }
      }
    pixel_sum<G, PV>(s1, red);
    pixel_sum<G, PV>(s2, red);
#pragma unroll
    for (int e = 0; e < PV; ++e) {
      s1[e] /= a.C;
      s2[e] /= a.C;
    }
    if (ok && a.dx) {
      T* dx = (T*)a.dx + img * a.C * a.P;
#pragma unroll
      for (int k = 0; k < NC; ++k) {
        const int c = k * G + g;
        if (c < a.C) {
#pragma unroll
          for (int e = 0; e < PV; ++e) h[k][e] = r[e] * (h[k][e] - s1[e] - xh[k][e] * s2[e]);
          store_pixels<T, PV>(dx, c * P + p, h[k]);
        }
      }
    }
  }
  if (!a.part) return;
  const float sw = fold_lanes<NC>(dw), sb = fold_lanes<NC>(db);
  constexpr int each = 64 / NC;  // lanes that hold a channel's sum
  const int c = l / each * G + g;
  if (l % each == 0 && c < a.C) {
    a.part[(long long)blockIdx.x * a.C + c] = sw;
    a.part[((long long)gridDim.x + blockIdx.x) * a.C + c] = sb;
  }
}

// ------------------------------------------------------------------------------ any C
// Rows longer than the registers are read again for each pass, mostly from the caches, and bound by
// those reads: S threads share a row -- a whole block, V channels each (tokens), or 16 that have one
// of 64 pixels (maps) -- with several loads under way.  16384 x 9000 bf16 tokens: 156 us forward (3.8
// TB/s of what one read and one write are), 242 backward; the 8 x 300 x 2688 bf16 map 16 and 34.
struct RowAt {
  long long base, y, stride;  // first value in x, in y / dy / dx; between channels
  long long m;
  bool ok;
};
template <bool MAP> __device__ __forceinline__ RowAt row_at(const NormArgs& a) {
  RowAt r;
  if (MAP) {
    const long long tiles = (a.P + 63) / 64, id = block_id(), img = id / tiles;
    const long long p = id % tiles * 64 + (threadIdx.x & 63);
    r.ok = p < a.P && img < a.B;
    r.base = r.ok ? img * a.x_stride + p : 0;
    r.y = r.ok ? img * a.C * a.P + p : 0;
    r.stride = a.P;
    r.m = img * a.P + p;
  } else {
    r.m = block_id();
    r.ok = r.m < a.M;
    r.base = r.ok ? r.m * a.x_stride : 0;
    r.y = r.ok ? r.m * a.C : 0;
    r.stride = 1;
  }
  return r;
}
constexpr int any_threads(bool map) { return map ? 1024 : 256; }
template <bool MAP> __device__ __forceinline__ float any_sum(float v, float (*red)[64]) {
  if constexpr (MAP) {
    float s[1] = {v};
    pixel_sum<16, 1>(s, red);
    return s[0];
  } else {
    return row_sum<256>(v, red[0]);
  }
}

template <typename T, bool MAP, int V>
__global__ __launch_bounds__(any_threads(MAP)) void norm_any(const NormArgs a) {
  __shared__ float red[MAP ? 16 : 1][64];
  const RowAt r = row_at<MAP>(a);
  const int first = MAP ? threadIdx.x >> 6 : threadIdx.x * V, S = MAP ? 16 : 256 * V;
  const T* x = (const T*)a.x + r.base;
  float s = 0.f;
#pragma unroll 4
  for (int c = first; c < a.C; c += S) {
    float v[V];
    load_values<T, V>(x + c * r.stride, v);
#pragma unroll
    for (int e = 0; e < V; ++e) s += v[e];
  }
  const float mu = any_sum<MAP>(s, red) / a.C;
  s = 0.f;
#pragma unroll 4
  for (int c = first; c < a.C; c += S) {
    float v[V];
    load_values<T, V>(x + c * r.stride, v);
#pragma unroll
    for (int e = 0; e < V; ++e) s += (v[e] - mu) * (v[e] - mu);
  }
  const float rs = 1.f / sqrtf(any_sum<MAP>(s, red) / a.C + a.eps);
  if (!r.ok) return;
  if (a.mean && first == 0) {
    a.mean[r.m] = mu;
    a.rstd[r.m] = rs;
  }
  T* y = (T*)a.y + r.y;
#pragma unroll 2
  for (int c = first; c < a.C; c += S) {
    float v[V], w[V], b[V];
    load_values<T, V>(x + c * r.stride, v);
    if (a.w) load_values<T, V>((const T*)a.w + c, w);
    if (a.b) load_values<T, V>((const T*)a.b + c, b);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = (v[e] - mu) * rs * (a.w ? w[e] : 1.f) + (a.b ? b[e] : 0.f);
    store_values<T, V>(y + c * r.stride, v);
  }
}

template <typename T, bool MAP, int V>
__global__ __launch_bounds__(any_threads(MAP)) void norm_any_dx(const NormArgs a) {
  __shared__ float red[MAP ? 16 : 1][64];
  const RowAt r = row_at<MAP>(a);
  const int first = MAP ? threadIdx.x >> 6 : threadIdx.x * V, S = MAP ? 16 : 256 * V;
  const T* x = (const T*)a.x + r.base;
  const T* dy = (const T*)a.dy + r.y;
  const float mu = r.ok ? a.mean[r.m] : 0.f, rs = r.ok ? a.rstd[r.m] : 0.f;
  float s1 = 0.f, s2 = 0.f;
  auto take = [&](int c, float(&h)[V], float(&xh)[V]) __attribute__((always_inline)) {
    float w[V];
    load_values<T, V>(dy + c * r.stride, h);
    load_values<T, V>(x + c * r.stride, xh);
    if (a.w) load_values<T, V>((const T*)a.w + c, w);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      if (a.w) h[e] *= w[e];
      xh[e] = (xh[e] - mu) * rs;
    }
  };
#pragma unroll 2
  for (int c = first; c < a.C; c += S) {
    float h[V], xh[V];
    take(c, h, xh);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      s1 += h[e];
      s2 += h[e] * xh[e];
    }
  }
  s1 = any_sum<MAP>(s1, red) / a.C;
  s2 = any_sum<MAP>(s2, red) / a.C;
  if (!r.ok) return;
  T* dx = (T*)a.dx + r.y;
#pragma unroll 2
  for (int c = first; c < a.C; c += S) {
    float h[V], xh[V];
    take(c, h, xh);
#pragma unroll
    for (int e = 0; e < V; ++e) h[e] = rs * (h[e] - s1 - xh[e] * s2);
    store_values<T, V>(dx + c * r.stride, h);
  }
}

// dw, db of one channel over a share of the rows: tokens, a thread V channels; maps, a block one
template <typename T, bool MAP, int V>
__global__ __launch_bounds__(256) void norm_any_dw(const NormArgs a, int parts) {
  __shared__ float red[4];
  const long long part = blockIdx.y;
  const long long lo = a.M * part / parts, hi = a.M * (part + 1) / parts;
  float sw[V], sb[V];
#pragma unroll
  for (int e = 0; e < V; ++e) sw[e] = sb[e] = 0.f;
  const long long c = MAP ? blockIdx.x : (blockIdx.x * 256LL + threadIdx.x) * V;
  if (MAP) {
#pragma unroll 2
    for (long long m = lo + threadIdx.x; m < hi; m += 256) {
      const long long img = m / a.P, p = m - img * a.P;
      const float d = to_f32(((const T*)a.dy)[(img * a.C + c) * a.P + p]);
      sw[0] += d * (to_f32(((const T*)a.x)[img * a.x_stride + c * a.P + p]) - a.mean[m]) * a.rstd[m];
      sb[0] += d;
    }
    sw[0] = row_sum<256>(sw[0], red);
    sb[0] = row_sum<256>(sb[0], red);
    if (threadIdx.x != 0) return;
  } else {
    if (c >= a.C) return;
#pragma unroll 4
    for (long long m = lo; m < hi; ++m) {
      float d[V], x[V];
      load_values<T, V>((const T*)a.dy + m * a.C + c, d);
      load_values<T, V>((const T*)a.x + m * a.x_stride + c, x);
      const float mu = a.mean[m], rs = a.rstd[m];
#pragma unroll
      for (int e = 0; e < V; ++e) {
        sw[e] += d[e] * (x[e] - mu) * rs;
        sb[e] += d[e];
      }
    }
  }
#pragma unroll
  for (int e = 0; e < V; ++e) {
    a.part[part * a.C + c + e] = sw[e];
    a.part[(parts + part) * a.C + c + e] = sb[e];
  }
}

// dw, db: the blocks' sums [2][blocks][C] in a fixed order; 32 channels by 32 shares of the blocks.
// A share is eight sums, and they and the shares are joined in pairs, so a value goes through blocks /
// 256 + 8 additions: one after the other, the rounding of 32-bit gradients would be the sum's.
template <typename T>
__global__ __launch_bounds__(1024) void norm_add_parts(const float* __restrict__ part,
                                                       T* __restrict__ dw, T* __restrict__ db,
                                                       int C, int blocks) {
  __shared__ float red[32][33];
  const int l = threadIdx.x & 31, g = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + l;
  const float* p = part + (long long)blockIdx.y * blocks * C;
  float s[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) s[k] = 0.f;
  if (c < C) {
    int b = g;
    for (; b + 32 * 7 < blocks; b += 256)  // (whole rounds: eight loads under way)
#pragma unroll
      for (int k = 0; k < 8; ++k) s[k] += p[(long long)(b + 32 * k) * C + c];
#pragma unroll
    for (int k = 0; k < 7; ++k)
      if (b + 32 * k < blocks) s[k] += p[(long long)(b + 32 * k) * C + c];
  }
  red[g][l] = ((s[0] + s[1]) + (s[2] + s[3])) + ((s[4] + s[5]) + (s[6] + s[7]));
  __syncthreads();
  // half a wave a channel: lane l has share l of channel g
  const float v = lanes_sum<32>(red[l][g]);
  const int at = blockIdx.x * 32 + g;
  T* out = blockIdx.y == 0 ? dw : db;
  if (l == 0 && at < C && out) out[at] = narrow<T>(v);
}

// ------------------------------------------------------------------------------ launches
// Threads of a row and vectors of a thread for C channels in vectors of V: the fewest threads that
// hold a row in 16 values each (32 where the whole block shares it), so that short rows share a
// wave.  128, 1024 and 8192 channels end the three; 0 = too long.
constexpr int most_values(int tpr) { return tpr == 256 ? 32 : 16; }
struct RowPlan {
  int tpr, nv;
};
static RowPlan row_plan(int C, int V) {
  const int n = (C + V - 1) / V;
  for (int tpr : {8, 64, 256})
    for (int nv = 1; nv * V <= most_values(tpr); nv *= 2)
      if (n <= tpr * nv) return {tpr, nv};
  return {0, 0};
}

template <typename T> static bool vector_rows(const NormArgs& a) {
  constexpr int V = 16 / (int)sizeof(T);
  return a.C % V == 0;
}

// Blocks of the backward pass, each with a row of partial sums: tokens, four of 256 threads that stay
// on each of 256 CUs, fewer where a row takes a whole block and they would have less than eight (4096 x
// 8192 bf16: 85 us with 1024 blocks, whose sums are as much traffic as the rows, 59 with 512; 16383 x
// 2048: 46 and 55); maps, twice that (a tile of 64 pixels each up to 131072 pixels: with 1024 blocks
// the l4 map's 1344 tiles took two turns and twice the time).
constexpr int kBlocksTokens = 1024, kBlocksMaps = 2048;

// maps whose pixels' channels are held in registers
static bool map_held(long long P, int C) { return C <= 256 && C * P < 1LL << 30; }

int norm_parts(int layout, long long B, long long P, int C, int dtype) {
  const long long M = layout == kMap ? B * P : P;
  const RowPlan p = layout == kMap ? RowPlan{} : row_plan(C, dtype == 0 ? 4 : 8);
  if (layout == kMap ? !map_held(P, C) : !p.tpr) {
    // norm_any_dw's blocks have a channel or some, and share the rows: thousands (maps) or dozens each
    const long long n = M / (layout == kMap ? 4096 : 32) + 1;
    const long long most = layout == kMap ? kBlocksMaps : kBlocksTokens;
    return (int)(M == 0 ? 0 : n < most ? n : most);
  }
  const long long rows = layout == kMap ? 64 : 256 / p.tpr;  // of a block's turn
  const long long n = (M + rows - 1) / rows;
  long long most = layout == kMap ? kBlocksMaps : kBlocksTokens;
  if (layout == kTokens && rows == 1 && n / 8 < most) most = n / 8 > 256 ? n / 8 : 256;
  return (int)(n < most ? n : most);
}

template <typename T, int TPR, bool WHOLE, int NV = 1>
static void tokens_nv(const NormArgs& a, int nv, bool back, int parts, hipStream_t s) {
  constexpr int V = 16 / (int)sizeof(T);
  if constexpr (NV * V <= most_values(TPR)) {
    if (nv != NV) return tokens_nv<T, TPR, WHOLE, 2 * NV>(a, nv, back, parts, s);
    const dim3 grid = grid_of((a.M + 256 / TPR - 1) / (256 / TPR));
    const size_t lds = 16 + (TPR < 256 ? 8 * sizeof(float) * a.C : 0);
    if (back)
      norm_tokens_backward<T, TPR, NV, V, WHOLE><<<parts, 256, lds, s>>>(a);
    else
      norm_tokens<T, TPR, NV, V, WHOLE><<<grid, 256, 0, s>>>(a);
  }
}
template <typename T, bool WHOLE>
static bool tokens_whole(const NormArgs& a, bool back, int parts, hipStream_t s) {
  const RowPlan p = row_plan(a.C, 16 / (int)sizeof(T));
  if (p.tpr == 0) return false;
  p.tpr == 8    ? tokens_nv<T, 8, WHOLE>(a, p.nv, back, parts, s)
  : p.tpr == 64 ? tokens_nv<T, 64, WHOLE>(a, p.nv, back, parts, s)
                : tokens_nv<T, 256, WHOLE>(a, p.nv, back, parts, s);
  return true;
}
template <typename T> static bool tokens(const NormArgs& a, bool back, int parts, hipStream_t s) {
  return vector_rows<T>(a) ? tokens_whole<T, true>(a, back, parts, s)
                           : tokens_whole<T, false>(a, back, parts, s);
}

template <typename T, int PV>
static void map_pv(const NormArgs& a, bool back, int parts, hipStream_t s) {
  const dim3 grid = grid_of(a.B * ((a.P + 64 * PV - 1) / (64 * PV)));
#define NORM_MAP(G, NC)                                                    \
  (back ? norm_map_backward<T, G, NC, PV><<<parts, 64 * G, 0, s>>>(a)      \
        : norm_map<T, G, NC, PV><<<grid, 64 * G, 0, s>>>(a))
  // eight channels a thread where sixteen waves hold them: the backward pass keeps five values a
  // channel, and more of them leave fewer waves on a CU (16 x 128 x 7168 bf16 by 8 waves 92 us, by 16
  // 47; 16 x 256 x 7168 373 and 121)
  if (a.C <= 8) {
    NORM_MAP(1, 8);
  } else if (a.C <= 32) {
    NORM_MAP(4, 8);
  } else if (a.C <= 64) {
    NORM_MAP(8, 8);
  } else if (a.C <= 128) {
    NORM_MAP(16, 8);
  } else if constexpr (PV == 1) {
    NORM_MAP(16, 16);
  } else {  // (forward alone: the backward pass of more channels would not fit the registers)
    norm_map<T, 16, 16, PV><<<grid, 1024, 0, s>>>(a);
  }
#undef NORM_MAP
}
template <typename T> static bool map(const NormArgs& a, bool back, int parts, hipStream_t s) {
  if (!map_held(a.P, a.C)) return false;
  if constexpr (sizeof(T) == 2) {
    bool pairs = (a.C <= 128 || !back) && a.P % 2 == 0 && (a.B == 1 || a.x_stride % 2 == 0);
    for (const void* p : {a.x, a.dy, (const void*)a.y, (const void*)a.dx})
      pairs = pairs && aligned_to(p, 4);
    if (pairs) {
      map_pv<T, 2>(a, back, parts, s);
      return true;
    }
  }
  map_pv<T, 1>(a, back, parts, s);
  return true;
}

template <typename T, bool MAP, int V>
static void any_c(const NormArgs& a, bool back, int parts, hipStream_t s) {
  const dim3 grid = grid_of(MAP ? a.B * ((a.P + 63) / 64) : a.M);
  if (!back) {
    norm_any<T, MAP, V><<<grid, any_threads(MAP), 0, s>>>(a);
    return;
  }
  if (a.dx) norm_any_dx<T, MAP, V><<<grid, any_threads(MAP), 0, s>>>(a);
  if (a.part)
    norm_any_dw<T, MAP, V>
        <<<dim3(MAP ? a.C : (a.C + 256 * V - 1) / (256 * V), parts), 256, 0, s>>>(a, parts);
}
template <typename T> static void any_c(const NormArgs& a, bool back, int parts, hipStream_t s) {
  constexpr int V = 16 / (int)sizeof(T);
  if (a.layout == kMap)
    any_c<T, true, 1>(a, back, parts, s);
  else if (vector_rows<T>(a))
    any_c<T, false, V>(a, back, parts, s);
  else
    any_c<T, false, 1>(a, back, parts, s);
}

template <typename T> static hipError_t forward_t(const NormArgs& a, hipStream_t s) {
  if (!(a.layout == kMap ? map<T>(a, false, 0, s) : tokens<T>(a, false, 0, s)))
    any_c<T>(a, false, 0, s);
  return hipGetLastError();
}

template <typename T> static hipError_t backward_t(const NormArgs& a, int parts, hipStream_t s) {
  if (!(a.layout == kMap ? map<T>(a, true, parts, s) : tokens<T>(a, true, parts, s)))
    any_c<T>(a, true, parts, s);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !a.part) return e;
  norm_add_parts<T><<<dim3((a.C + 31) / 32, 2), 1024, 0, s>>>(a.part, (T*)a.dw, (T*)a.db, a.C,
                                                             parts);
  return hipGetLastError();
}

template <typename T> static hipError_t no_rows_t(const NormArgs& a, hipStream_t s) {
  norm_add_parts<T><<<dim3((a.C + 31) / 32, 2), 1024, 0, s>>>(nullptr, (T*)a.dw, (T*)a.db, a.C, 0);
  return hipGetLastError();
}

hipError_t norm_no_rows(const NormArgs& a, int dtype, hipStream_t s) {
  return dtype == 0   ? no_rows_t<float>(a, s)
         : dtype == 1 ? no_rows_t<__half>(a, s)
                      : no_rows_t<__hip_bfloat16>(a, s);
}
hipError_t norm_forward(const NormArgs& a, int dtype, hipStream_t s) {
  return dtype == 0   ? forward_t<float>(a, s)
         : dtype == 1 ? forward_t<__half>(a, s)
                      : forward_t<__hip_bfloat16>(a, s);
}
hipError_t norm_backward(const NormArgs& a, int parts, int dtype, hipStream_t s) {
  return dtype == 0   ? backward_t<float>(a, parts, s)
         : dtype == 1 ? backward_t<__half>(a, parts, s)
                      : backward_t<__hip_bfloat16>(a, parts, s);
}

}  // namespace feat
}  // namespace pwc
