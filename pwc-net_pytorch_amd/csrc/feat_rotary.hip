// feat_rotary.hip — rotary positions with several axes (t, y, x).
//
//   pair j of R turns by a_j = position[axis_j] * inv_freq_j:
//   (u, v) -> (u cos a - v sin a, u sin a + v cos a);  channels from 2 R on pass unchanged
//   pairs are (j, R + j), or (2j, 2j + 1) where `interleaved`.  The backward pass turns by -a.
//
// Bound by memory: one read and one write of x.  The angle is a product in 64 bits, taken modulo a
// whole turn before it is rounded to 32: at position 40000 the angle of the first pair keeps
// 2^-24 of a turn, where a product in 32 bits has lost 2^-9.  Its sine and cosine serve all heads
// (tokens) or all images with the same positions (maps).
#include "feat_common.cuh"
#include "feat_rotary.cuh"

namespace pwc {
namespace feat {

__device__ __forceinline__ double position(const RotaryArgs& a, long long b, long long n, int ax) {
  if (a.positions == nullptr) {  // raster place in the grid
    long long r = n;
    for (int k = a.axes - 1; k > ax; --k) r /= a.grid[k];
    return (double)(a.origin[ax] + r % a.grid[ax]);
  }
  const long long i = b * a.pos_b + n * a.pos_n + ax * a.pos_a;
  return a.pos_type == 0   ? (double)((const float*)a.positions)[i]
         : a.pos_type == 1 ? (double)((const int*)a.positions)[i]
                           : (double)((const long long*)a.positions)[i];
}

__device__ __forceinline__ void turn(const RotaryArgs& a, long long b, long long n, int j, float& s,
                                     float& c) {
  const int ax = min(max(a.axis[j], 0), a.axes - 1);  // whatever the caller wrote: in bounds
  double t = position(a, b, n, ax) * (a.inv_freq[j] * 0.15915494309189535);
  t -= rint(t);
  sincospif(2.f * (float)t, &s, &c);
  s *= a.sign;
}

// one thread: V pairs of one token, over `hpt` heads (D contiguous, V * sizeof(T) aligned)
template <typename T, int V, bool INTER>
__global__ __launch_bounds__(256) void rotary_rows(const RotaryArgs a) {
  const int units = (a.R + V - 1) / V;              // of a token's pairs
  const int rest = (a.D - 2 * a.R + 2 * V - 1) / (2 * V);  // units of the channels that pass
  const long long per = (units + rest) * (long long)a.head_groups;
  const long long id = blockIdx.x * 256LL + threadIdx.x;
  if (id >= a.B * a.N * per) return;
  const int u = (int)(id % (units + rest));
  const int hg = (int)(id / (units + rest) % a.head_groups);
  const long long bn = id / per, b = bn / a.N, n = bn - b * a.N;
  const int h0 = hg * a.heads_each, h1 = min(a.H, h0 + a.heads_each);
  const T* x = (const T*)a.x + b * a.xs_b + n * a.xs_n;
  T* y = (T*)a.y + b * a.ys_b + n * a.ys_n;
  if (u >= units) {
    const int c0 = 2 * a.R + (u - units) * 2 * V;
    for (int h = h0; h < h1; ++h)
#pragma unroll
      for (int e = 0; e < 2 * V; ++e)
        if (c0 + e < a.D) y[h * a.ys_h + c0 + e] = x[h * a.xs_h + c0 + e];
    return;
  }
  const int j0 = u * V;
  float s[V], c[V];
#pragma unroll
  for (int e = 0; e < V; ++e)
    if (j0 + e < a.R) turn(a, b, n, j0 + e, s[e], c[e]);
  for (int h = h0; h < h1; ++h) {
    const T* xp = x + h * a.xs_h;
    T* yp = y + h * a.ys_h;
    if constexpr (V == 1) {
      const int p = INTER ? 2 * j0 : j0, q = INTER ? p + 1 : a.R + j0;
      const float f = to_f32(xp[p]), g = to_f32(xp[q]);
      yp[p] = narrow<T>(f * c[0] - g * s[0]);
      yp[q] = narrow<T>(f * s[0] + g * c[0]);
    } else {
      const int p = INTER ? 2 * j0 : j0, q = INTER ? p + V : a.R + j0;
      Pack<T, V> f = *(const Pack<T, V>*)(xp + p), g = *(const Pack<T, V>*)(xp + q);
#pragma unroll
      for (int e = 0; e < V; ++e) {
        // interleaved: pair e is values 2e, 2e + 1 of (f, g) laid end to end
        T& tu = INTER ? (2 * e < V ? f.v[2 * e % V] : g.v[2 * e % V]) : f.v[e];
        T& tv = INTER ? (2 * e < V ? f.v[(2 * e + 1) % V] : g.v[(2 * e + 1) % V]) : g.v[e];
        const float fu = to_f32(tu), fv = to_f32(tv);
        tu = narrow<T>(fu * c[e] - fv * s[e]);
        tv = narrow<T>(fu * s[e] + fv * c[e]);
      }
      *(Pack<T, V>*)(yp + p) = f;
      *(Pack<T, V>*)(yp + q) = g;
    }
  }
}

// any strides: one thread takes one pair (or two passing channels) of V neighbouring tokens, over
// the images that share its positions; lanes run along the tokens (maps: pixels)
template <typename T, int V>
__global__ __launch_bounds__(256) void rotary_pixels(const RotaryArgs a) {
  const long long nv = (a.N + V - 1) / V;
  const long long id = blockIdx.x * 256LL + threadIdx.x;
  const int units = a.R + (a.D - 2 * a.R + 1) / 2;
  if (id >= nv * units * a.H * a.batch_groups) return;
  const long long n0 = id % nv * V;
  const int u = (int)(id / nv % units), h = (int)(id / (nv * units) % a.H);
  const long long bg = id / (nv * units * a.H);
  const long long b0 = bg * a.batch_each, b1 = min(a.B, b0 + a.batch_each);
  const bool turned = u < a.R;
  const int p = !turned ? 2 * u : a.interleaved ? 2 * u : u;
  const int q = !turned ? 2 * u + 1 : a.interleaved ? 2 * u + 1 : a.R + u;
  float s[V], c[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    s[e] = 0.f;
    c[e] = 1.f;
    if (turned && n0 + e < a.N) turn(a, b0, n0 + e, u, s[e], c[e]);
  }
  for (long long b = b0; b < b1; ++b) {
    const T* x = (const T*)a.x + b * a.xs_b + h * a.xs_h + n0 * a.xs_n;
    T* y = (T*)a.y + b * a.ys_b + h * a.ys_h + n0 * a.ys_n;
    if constexpr (V == 1) {
      const float f = to_f32(x[p * a.xs_d]), g = q < a.D ? to_f32(x[q * a.xs_d]) : 0.f;
      // a passing value is not multiplied: infinity times zero is none
      y[p * a.ys_d] = turned ? narrow<T>(f * c[0] - g * s[0]) : x[p * a.xs_d];
      if (q < a.D) y[q * a.ys_d] = turned ? narrow<T>(f * s[0] + g * c[0]) : x[q * a.xs_d];
    } else {
      Pack<T, V> f = *(const Pack<T, V>*)(x + p * a.xs_d), g;
      if (q < a.D) g = *(const Pack<T, V>*)(x + q * a.xs_d);
      if (turned) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float fu = to_f32(f.v[e]), fv = to_f32(g.v[e]);
          f.v[e] = narrow<T>(fu * c[e] - fv * s[e]);
          g.v[e] = narrow<T>(fu * s[e] + fv * c[e]);
        }
      }
      *(Pack<T, V>*)(y + p * a.ys_d) = f;
      if (q < a.D) *(Pack<T, V>*)(y + q * a.ys_d) = g;
    }
  }
}

template <typename T> static hipError_t rotary_t(RotaryArgs a, hipStream_t stream) {
  constexpr int V = 16 / (int)sizeof(T);
  auto every = [](std::initializer_list<long long> v, int n) {
    for (long long x : v)
      if (x % n) return false;
    return true;
  };
  const bool base = aligned_to(a.x, 16) && aligned_to(a.y, 16);
  constexpr long long kThreads = 256LL * 1024;  // enough to fill 256 CUs
  if (a.xs_d == 1 && a.ys_d == 1) {
    const bool vec = base && a.R % V == 0 && a.D % V == 0 &&
                     every({a.xs_b, a.xs_n, a.xs_h, a.ys_b, a.ys_n, a.ys_h}, V);
    const int v = vec ? V : 1;
    const long long units = (a.R + v - 1) / v + (a.D - 2 * a.R + 2 * v - 1) / (2 * v);
    // heads in one thread share its angles, as long as the threads fill the card
    long long groups = kThreads / (a.B * a.N * units) + 1;
    if (groups > a.H) groups = a.H;
    a.heads_each = (int)((a.H + groups - 1) / groups);
    a.head_groups = (a.H + a.heads_each - 1) / a.heads_each;
    const long long blocks = (a.B * a.N * units * a.head_groups + 255) / 256;
    if (blocks > 0x7fffffffLL) return hipErrorInvalidConfiguration;
    if (a.interleaved)
      vec ? rotary_rows<T, V, true><<<(unsigned)blocks, 256, 0, stream>>>(a)
          : rotary_rows<T, 1, true><<<(unsigned)blocks, 256, 0, stream>>>(a);
    else
      vec ? rotary_rows<T, V, false><<<(unsigned)blocks, 256, 0, stream>>>(a)
          : rotary_rows<T, 1, false><<<(unsigned)blocks, 256, 0, stream>>>(a);
    return hipGetLastError();
  }
  const bool vec = base && a.xs_n == 1 && a.ys_n == 1 && a.N % V == 0 &&
                   every({a.xs_b, a.xs_d, a.xs_h, a.ys_b, a.ys_d, a.ys_h}, V);
  const long long nv = vec ? a.N / V : a.N;
  const long long one = nv * (a.R + (a.D - 2 * a.R + 1) / 2) * a.H;
  const bool shared = a.positions == nullptr || a.pos_b == 0;
  long long groups = shared ? kThreads / one + 1 : a.B;
  if (groups > a.B) groups = a.B;
  a.batch_each = (a.B + groups - 1) / groups;
  a.batch_groups = (a.B + a.batch_each - 1) / a.batch_each;
  const long long blocks = (one * a.batch_groups + 255) / 256;
  if (blocks > 0x7fffffffLL) return hipErrorInvalidConfiguration;
  vec ? rotary_pixels<T, V><<<(unsigned)blocks, 256, 0, stream>>>(a)
      : rotary_pixels<T, 1><<<(unsigned)blocks, 256, 0, stream>>>(a);
  return hipGetLastError();
}

hipError_t rotary_launch(const RotaryArgs& a, int dtype, hipStream_t stream) {
  return dtype == 0   ? rotary_t<float>(a, stream)
         : dtype == 1 ? rotary_t<__half>(a, stream)
                      : rotary_t<__hip_bfloat16>(a, stream);
}

}  // namespace feat
}  // namespace pwc
