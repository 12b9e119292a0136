// feat_rotary.hip — rotary positions with several axes (t, y, x).
//
//   pair j of R turns by a_j = position[axis_j] * inv_freq_j:
//   (u, v) -> (u cos a - v sin a, u sin a + v cos a);  channels from 2 R on pass unchanged
//   pairs are (j, R + j), or (2j, 2j + 1) where `interleaved`.  The backward pass turns by -a.
//
// Bound by memory: one read and one write of x.  The angle is a product in 64 bits, taken modulo a
// whole turn before it is rounded to 32: at position 40000 the angle of the first pair keeps
// 2^-24 of a turn, where a product in 32 bits has lost 2^-9.  Its sine and cosine serve all heads
// (tokens) or all images with the same positions (maps).  Measured: 2 x 9603 x 24 x 128 bf16 tokens
// 54 us (4.4 TB/s; a 1 GiB copy does 5.2), the 16 x 32 x 112 x 256 fp16 map 15.3 us (3.8).
#include "feat_common.cuh"
#include "feat_rotary.cuh"

namespace pwc {
namespace feat {

// The angle `place` * inv_freq_j, modulo a whole turn before it is rounded.
__device__ __forceinline__ void turn(const RotaryArgs& a, double place, int j, float& s, float& c) {
  double t = place * (a.inv_freq[j] * 0.15915494309189535);
  t -= rint(t);
  sincospif(2.f * (float)t, &s, &c);
  s *= a.sign;
}
__device__ __forceinline__ int axis_of(const RotaryArgs& a, int j) {
  return min(max(a.axis[j], 0), a.axes - 1);  // whatever the caller wrote: in bounds
}
__device__ __forceinline__ double given_place(const RotaryArgs& a, long long b, long long n,
                                              int ax) {
  const long long i = b * a.pos_b + n * a.pos_n + ax * a.pos_a;
  return a.pos_type == 0   ? (double)((const float*)a.positions)[i]
         : a.pos_type == 1 ? (double)((const int*)a.positions)[i]
                           : (double)((const long long*)a.positions)[i];
}
// raster place of token n in the grid, and what is left of n within the axis's step
__device__ __forceinline__ uint32_t grid_place(const RotaryArgs& a, uint32_t n, int ax,
                                               uint32_t& rest) {
  const uint32_t q = n / a.inner[ax];
  rest = n - q * a.inner[ax];
  return q % (uint32_t)a.grid[ax];
}

// one thread: V pairs of one token, over `heads_each` heads (D contiguous, rows at 16-byte places
// where V > 1), four heads' loads under way at a time
template <typename T, int V, bool INTER>
__global__ __launch_bounds__(256) void rotary_rows(const RotaryArgs a) {
  const int units = (a.R + V - 1) / V;                     // of a token's pairs
  const int rest = (a.D - 2 * a.R + 2 * V - 1) / (2 * V);  // units of the channels that pass
  const long long per = (units + rest) * (long long)a.head_groups;
  const long long id = block_id() * 256 + threadIdx.x;
  if (id >= a.B * a.N * per) return;
  const long long bn = id / per;
  const uint32_t in = (uint32_t)(id - bn * per);
  const int hg = (int)(in / (uint32_t)(units + rest)), u = (int)(in - hg * (units + rest));
  const long long b = bn / a.N, n = bn - b * a.N;
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
  // Values p .. p + V and q .. q + V of a head.  Apart, pair j0 + e is their values e; interleaved,
  // both hold pairs of their own, half a head apart so that neighbouring lanes read neighbouring
  // bytes.
  const int j0 = INTER && V > 1 ? u * (V / 2) : u * V;
  const int p = INTER ? 2 * j0 : j0, q = INTER ? (V > 1 ? p + a.R : p + 1) : a.R + j0;
  float s[V], c[V];
  int last = -1;
  double place = 0.;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    const int j = INTER && V > 1 && e >= V / 2 ? a.R / 2 + j0 + e - V / 2 : j0 + e;
    if (j < a.R) {
      const int ax = axis_of(a, j);
      if (ax != last) {
        uint32_t left;
        place = a.positions ? given_place(a, b, n, ax)
                            : (double)(a.origin[ax] + grid_place(a, (uint32_t)n, ax, left));
        last = ax;
      }
      turn(a, place, j, s[e], c[e]);
    }
  }
  constexpr int HB = 4;
  for (int h = h0; h < h1; h += HB) {
    Pack<T, V> f[HB], g[HB];
#pragma unroll
    for (int k = 0; k < HB; ++k)
      if (h + k < h1) {
        const T* xp = x + (h + k) * a.xs_h;
        f[k] = *(const Pack<T, V>*)(xp + p);
        g[k] = *(const Pack<T, V>*)(xp + q);
      }
#pragma unroll
    for (int k = 0; k < HB; ++k)
      if (h + k < h1) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          // interleaved: pair e is values 2e, 2e + 1 of f, then of g
          T& tu = !INTER || V == 1 ? f[k].v[e] : 2 * e < V ? f[k].v[2 * e % V] : g[k].v[2 * e % V];
          T& tv = !INTER || V == 1 ? g[k].v[e]
                  : 2 * e < V      ? f[k].v[(2 * e + 1) % V]
                                   : g[k].v[(2 * e + 1) % V];
          const float fu = to_f32(tu), fv = to_f32(tv);
          tu = narrow<T>(fu * c[e] - fv * s[e]);
          tv = narrow<T>(fu * s[e] + fv * c[e]);
        }
        T* yp = y + (h + k) * a.ys_h;
        *(Pack<T, V>*)(yp + p) = f[k];
        *(Pack<T, V>*)(yp + q) = g[k];
      }
  }
}

// any strides: one thread takes one pair (or two passing channels) of V neighbouring tokens, over
// the images that share its positions, four at a time; lanes run along the tokens (maps: pixels)
template <typename T, int V>
__global__ __launch_bounds__(256) void rotary_pixels(const RotaryArgs a) {
  const uint32_t nv = (uint32_t)((a.N + V - 1) / V);
  const long long id = block_id() * 256 + threadIdx.x;
  const int units = a.R + (a.D - 2 * a.R + 1) / 2;
  if (id >= (long long)nv * units * a.H * a.batch_groups) return;
  const long long rows = id / nv;
  const long long n0 = (id - rows * nv) * V;
  const int u = (int)(rows % units), h = (int)(rows / units % a.H);
  const long long bg = rows / units / a.H;
  const long long b0 = bg * a.batch_each, b1 = min(a.B, b0 + a.batch_each);
  const bool turned = u < a.R;
  const int p = !turned ? 2 * u : a.interleaved ? 2 * u : u;
  const int q = !turned ? 2 * u + 1 : a.interleaved ? 2 * u + 1 : a.R + u;
  float s[V], c[V];
#pragma unroll
  for (int e = 0; e < V; ++e) {
    s[e] = 0.f;
    c[e] = 1.f;
  }
  if (turned) {
    const int ax = axis_of(a, u);
    uint32_t left = 0;
    uint32_t at = a.positions ? 0 : grid_place(a, (uint32_t)n0, ax, left);
#pragma unroll
    for (int e = 0; e < V; ++e)
      if (n0 + e < a.N) {
        if (e > 0 && !a.positions) {  // the next raster place
          if (++left == a.inner[ax]) {
            left = 0;
            if (++at == (uint32_t)a.grid[ax]) at = 0;
          }
          if (left > 0) {  // same place on this axis as its neighbour
            s[e] = s[e - 1];
            c[e] = c[e - 1];
            continue;
          }
        }
        turn(a, a.positions ? given_place(a, b0, n0 + e, ax) : (double)(a.origin[ax] + at), u,
             s[e], c[e]);
      }
  }
  constexpr int BB = 4;
  const bool second = q < a.D;
  for (long long b = b0; b < b1; b += BB) {
    Pack<T, V> f[BB], g[BB];
#pragma unroll
    for (int k = 0; k < BB; ++k)
      if (b + k < b1) {
        const T* x = (const T*)a.x + (b + k) * a.xs_b + h * a.xs_h + n0 * a.xs_n;
        f[k] = *(const Pack<T, V>*)(x + p * a.xs_d);
        if (second) g[k] = *(const Pack<T, V>*)(x + q * a.xs_d);
      }
#pragma unroll
    for (int k = 0; k < BB; ++k)
      if (b + k < b1) {
        if (turned) {  // (a passing value is not multiplied: infinity times zero is none)
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float fu = to_f32(f[k].v[e]), fv = to_f32(g[k].v[e]);
            f[k].v[e] = narrow<T>(fu * c[e] - fv * s[e]);
            g[k].v[e] = narrow<T>(fu * s[e] + fv * c[e]);
          }
        }
        T* y = (T*)a.y + (b + k) * a.ys_b + h * a.ys_h + n0 * a.ys_n;
        *(Pack<T, V>*)(y + p * a.ys_d) = f[k];
        if (second) *(Pack<T, V>*)(y + q * a.ys_d) = g[k];
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
  uint32_t inner = 1;  // tokens between neighbours on an axis (the launch entry bounds them)
  for (int k = a.axes - 1; k >= 0 && a.positions == nullptr; --k) {
    a.inner[k] = inner;
    inner *= (uint32_t)a.grid[k];
  }
  const bool base = aligned_to(a.x, 16) && aligned_to(a.y, 16);
  if (a.xs_d == 1 && a.ys_d == 1) {
    const bool vec = base && a.R % V == 0 && a.D % V == 0 &&
                     every({a.xs_b, a.xs_n, a.xs_h, a.ys_b, a.ys_n, a.ys_h}, V);
    const int v = vec ? V : 1;
    const long long units = (a.R + v - 1) / v + (a.D - 2 * a.R + 2 * v - 1) / (2 * v);
    // Heads in one thread share its angles, which bound calls whose rows come from the cache, as long
    // as the threads fill the card (2 x 4096 x 8 x 128 bf16: 10 us with 128 thousand threads, 15 with
    // 512); rows from memory want more loads under way (2 x 9603 x 24 x 128: 57 and 54 us).
    const long long bytes = 2 * a.B * a.N * a.H * a.D * (long long)sizeof(T);
    const long long threads = bytes > (128LL << 20) ? 512LL << 10 : 128LL << 10;
    long long groups = threads / (a.B * a.N * units) + 1;
    if (groups > a.H) groups = a.H;
    a.heads_each = (int)((a.H + groups - 1) / groups);
    a.head_groups = (a.H + a.heads_each - 1) / a.heads_each;
    const long long blocks = (a.B * a.N * units * a.head_groups + 255) / 256;
    const dim3 grid = grid_of(blocks);
    if (a.interleaved)
      vec ? rotary_rows<T, V, true><<<grid, 256, 0, stream>>>(a)
          : rotary_rows<T, 1, true><<<grid, 256, 0, stream>>>(a);
    else
      vec ? rotary_rows<T, V, false><<<grid, 256, 0, stream>>>(a)
          : rotary_rows<T, 1, false><<<grid, 256, 0, stream>>>(a);
    return hipGetLastError();
  }
  const bool vec = base && a.xs_n == 1 && a.ys_n == 1 && a.N % V == 0 &&
                   every({a.xs_b, a.xs_d, a.xs_h, a.ys_b, a.ys_d, a.ys_h}, V);
  const long long nv = vec ? a.N / V : a.N;
  const long long one = nv * (a.R + (a.D - 2 * a.R + 1) / 2) * a.H;
  // Images in one thread share its angles; 16 x 32 x 112 x 256 fp16 took 15.1 us with 170 thousand
  // threads, 16.7 with 115, 19.7 with 460.
  const bool shared = a.positions == nullptr || a.pos_b == 0;
  long long groups = shared ? (128LL << 10) / one + 1 : a.B;
  if (groups > a.B) groups = a.B;
  a.batch_each = (a.B + groups - 1) / groups;
  a.batch_groups = (a.B + a.batch_each - 1) / a.batch_each;
  const long long blocks = (one * a.batch_groups + 255) / 256;
  const dim3 grid = grid_of(blocks);
  vec ? rotary_pixels<T, V><<<grid, 256, 0, stream>>>(a)
      : rotary_pixels<T, 1><<<grid, 256, 0, stream>>>(a);
  return hipGetLastError();
}

hipError_t rotary_launch(const RotaryArgs& a, int dtype, hipStream_t stream) {
  return dtype == 0   ? rotary_t<float>(a, stream)
         : dtype == 1 ? rotary_t<__half>(a, stream)
                      : rotary_t<__hip_bfloat16>(a, stream);
}

}  // namespace feat
}  // namespace pwc
