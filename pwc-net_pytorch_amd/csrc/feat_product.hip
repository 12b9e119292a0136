// feat_product.hip — the matrix products of the feature operators linear and gated linear.
//
//   linear:        y = act(x W^T + b) + res
//   gated linear:  y = act(x Wg^T + bg) * (x Wu^T + bu),  W = [Wg; Wu]
//   backward:      dz = dy act'(z)                  (linear)
//                  dz = [dy u act'(g), dy act(g)]   (gated)
//                  dx = dz W,  dW = dz^T x,  db = sum over tokens of dz
//
// z is not kept by the forward pass: the backward multiplies again and turns the 32-bit sums into
// dz in the epilogue, so dz is rounded once (a z kept in 16 bits would be a second rounding, in 32
// bits 8 bytes a value of traffic that costs more than the product below 700 channels).
//
// ONE kernel computes Out(i, j) = sum_k A(i, k) B(j, k).  i is the dimension of the output that is
// contiguous in memory: the matrix instruction leaves four consecutive i in a lane.  Each operand
// lies either along k ("K": rows of contiguous k) or along its own row index ("N"):
//              tokens                               map
//   forward    i = out channel  A = W (K), B = x (K)   i = pixel    A = x (N),  B = W (K)
//   dx         i = in channel   A = W (N), B = dz (K)  i = pixel    A = dz (N), B = W (N)
//   dW         i = in channel   A = x (N), B = dz (N)  i = in chan. A = x (K),  B = dz (K)
// The gated forms interleave 16 gate rows with 16 up rows in W's tile, so both halves of a value
// end in neighbouring accumulators of one lane.
//
// A k step is 128 bytes of either operand's k (64 values of 16 bits, 32 of 32).  A K tile lies in
// LDS as rows of 128 bytes, an N tile as rows of contiguous i; 16-byte chunks are exclusive-ored
// with bits of the row so that the reads of a wave fall into different banks.  A fragment is 16
// bytes a lane: eight k of one row (16 bits, one 16x16x32 instruction) or four (32 bits, four
// 16x16x4 instructions).  The order of k within a fragment does not matter as long as both
// operands share it; N tiles of 16 bits are turned by the transposing LDS read.
//
// What bounds them (bf16, 8192 x K -> 4096): the matrix units in the steps, 1520 to 1565 TFLOP/s by
// 256-tiles between K = 512 and 8192 (the largest library product, 8192^3, has 1583), and the memory at
// a tile's end, where a CU writes 128 KiB and nothing multiplies: 34 us of the 79 at K = 1024 (a library
// product 59) with nothing else to do there, 105 with gelu where the operands come from memory.  Tiles of half that size would overlap the two, and
// lose more in the steps; a tile's sums stored from the registers, without the turn through LDS,
// were no faster.  Few tokens are bound by the bytes of W (few_tokens), some hundred by latency.

#include "feat_product.cuh"
#include "feat_steps.cuh"

namespace pwc {
namespace feat {

constexpr int kStepBytes = 128;  // of either operand's k, as in the kernel

// Direct loads want whole 16-byte chunks at 16-byte places and offsets within 31 bits.
template <typename T> static bool direct_loads(const ProductArgs& g, int bi, int bj) {
  constexpr int E = 16 / (int)sizeof(T);
  auto fits = [&](const void* p, long long ld, long long batch, long long seg, bool kc, int n,
                  int rows, int pair, int pad) {
    const long long far = (long long)(kc ? rows + pair : kStepBytes / (int)sizeof(T)) * ld;
    return aligned_to(p, 16) && ld % E == 0 && batch % E == 0 && seg % E == 0 &&
           (pad || (kc ? g.K : n) % E == 0) && far * (long long)sizeof(T) < (1LL << 31) - (1 << 20);
  };
  return fits(g.a, g.lda, g.a_batch, g.a_segment, g.a_k, g.I, bi,
              g.channel_i ? g.pair : 0, g.a_pad) &&
         fits(g.b, g.ldb, g.b_batch, g.b_segment, g.b_k, g.J, bj, g.channel_i ? 0 : g.pair,
              g.b_pad);
}

// Which kernel: the one with the least modelled time.  A step of 128 bytes of k costs a block at
// least `far` (loads, barrier, latency; `near` where both operands stay in the L2 caches), and the
// blocks of a CU share its matrix units, `work` a block; a tile's epilogue and start cost `fixed`
// for every round of tiles over the card.  The figures are fitted to measured calls (us, bf16, by
// 64-, deep 64-, 128- and 256-tiles: 512 tokens 4096 -> 4096 36, 28, 33, 43; 1024 tokens 51, 53, 47,
// 53; 8192 tokens 4096 -> 1024 95, 98, 66, 76; 1024 -> 4096 111, 115, 83, 73; 128 -> 1024 12, 13,
// 10, 18; fp32 4096 tokens 1024 -> 1024 by 64- and 128-tiles 73, 75; 8192 1024 -> 4096 520, 513).
struct TileCost {
  int kernel, bi, bj, passes, blocks;  // blocks that a CU holds
  double far, near, work, fixed;
};
static constexpr TileCost kCost16[] = {{kTile64, 64, 64, 1, 4, 0.50, 0.20, 0.175, 3.5},
                                       {kTile64Deep, 64, 64, 1, 3, 0.35, 0.20, 0.19, 3.5},
                                       {kTile128, 128, 128, 1, 2, 0.66, 0.46, 0.47, 4.4},
                                       {kTile256, 256, 256, 2, 1, 1.39, 1.39, 1.39, 14.0}};
// Through registers, both operands along k or not (rows at odd places that are read across k cost
// most; bf16, 1024 x 1021 -> 1021: forward 15, in four parts 23; dx 27, in four parts 20).
static constexpr TileCost kCostAnyK16 = {kTile64Any, 64, 64, 1, 4, 0.60, 0.60, 0.21, 3.5};
static constexpr TileCost kCostAnyK32 = {kTile64Any, 64, 64, 1, 4, 1.00, 1.00, 0.55, 3.5};
static constexpr TileCost kCostAny = {kTile64Any, 64, 64, 1, 4, 1.35, 1.35, 0.60, 3.5};
static constexpr TileCost kCost32[] = {{kTile64, 64, 64, 1, 4, 0.65, 0.60, 0.53, 3.0},
                                       {kTile128, 128, 128, 1, 2, 2.00, 2.00, 1.96, 6.0}};
constexpr int kCUs = 256;
constexpr double kNear = 8e6;  // bytes of both operands

static bool direct_any(const ProductArgs& g, const TileCost& c, int dtype) {
  return dtype == 0   ? direct_loads<float>(g, c.bi, c.bj)
         : dtype == 1 ? direct_loads<__half>(g, c.bi, c.bj)
                      : direct_loads<__hip_bfloat16>(g, c.bi, c.bj);
}

ProductPlan product_plan(const ProductArgs& g, int dtype) {
  const bool pair = g.mode == kGated || g.mode == kGatedDz;
  const long long pairs = ((long long)g.pair + 15) / 16 * 32;
  const long long ri = pair && g.channel_i ? pairs : g.I, rj = pair && !g.channel_i ? pairs : g.J;
  const double bytes = dtype == 0 ? 4.0 : 2.0;  // bytes of a value
  ProductPlan best = {};
  double least = 1e300;
  if (g.channel_i && g.J <= 64) {
    // A pass over W: a CU takes 50 bytes of W and x a ns (64 tokens, 4096 -> 4096: 13.6 us, by
    // tiles 16.0; 4096 -> 16384: 45, by tiles 30), and up to 32 tokens nothing is faster.
    best = {g.J <= 16 ? kFew16 : g.J <= 32 ? kFew32 : kFew64, 16, 16, 1, 1};
    if (g.J <= 32) return best;
    const int blocks = ((pair ? g.pair : g.I) + 15) / 16;
    least = 2.0 + (double)((blocks + kCUs - 1) / kCUs) * (g.J + (pair ? 32 : 16)) * g.K *
                      bytes / 50e3;
  }
  const TileCost* costs = dtype == 0 ? kCost32 : kCost16;
  const bool near = ((double)g.I + g.J) * g.K * g.segments * g.batches * bytes <= kNear;
  for (int n = 0; n < (dtype == 0 ? 2 : 4); ++n) {
    const bool direct = direct_any(g, costs[n], dtype);
    if (!direct && n > 0) break;
    const TileCost& c = direct               ? costs[n]
                        : !(g.a_k && g.b_k) ? kCostAny
                        : dtype == 0        ? kCostAnyK32
                                            : kCostAnyK16;
    const int ks = kStepBytes / (dtype == 0 ? 4 : 2);
    const double steps = (double)g.segments * Steps::of(g.K, ks);
    const double tiles =
        (double)((ri + c.bi - 1) / c.bi) * ((rj + c.bj - 1) / c.bj) * g.batches;
    for (int splits = 1; splits <= (g.mode == kPartial || g.channel_i ? 512 : 1); splits *= 2) {
      if (splits > 1 && splits * 4 > steps) break;  // some steps each
      const double blocks = tiles * splits, each = steps / splits;
      const double rounds = blocks / (kCUs * c.blocks);
      double t = each * (near ? c.near : c.far);
      if (t < blocks / kCUs * each * c.work) t = blocks / kCUs * each * c.work;
      t += 2.0 + c.fixed * (rounds < 1 ? 1 : rounds);
      // the partial sums go out and come back, and one more launch, with the epilogue if there is
      // one (128 tokens, 4096 -> 4096: 40 us in one part, 20 in eight)
      if (splits > 1) t += 5.5 + (double)g.I * g.J * splits * 8 / (direct ? 6.5e6 : 3.2e6);
      if (t < least) {
        least = t;
        best = {c.kernel, c.bi, c.bj, c.passes, splits};
      }
    }
  }
  return best;
}

// The epilogue of a product that was summed in parts, bound by reading them: a lane takes four
// channels, a wave 256 of a token, `each` tokens of every fourth.  (128 tokens, 4096 -> 4096 in eight
// parts: 16 us with the product, 40 by tiles that see all of k.)
template <typename T, int MODE>
__global__ __launch_bounds__(256) void finish_parts(const ProductArgs g, int splits, int each) {
  constexpr bool kPair = MODE == kGated || MODE == kGatedDz;
  constexpr bool kDz = MODE == kLinearDz || MODE == kGatedDz;
  __shared__ float red[kDz ? 3 : 1][kPair ? 2 : 1][256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const int outs = kPair ? g.pair : g.I, i = (blockIdx.x * 64 + lane) * 4, left = outs - i;
  const T* bias = (const T*)g.bias;
  float b[4], c[4], sv[4], sw[4];
  load_four(bias + i, bias ? left : 0, b);
  load_four(bias + g.pair + i, bias && kPair ? left : 0, c);
#pragma unroll
  for (int e = 0; e < 4; ++e) sv[e] = sw[e] = 0.f;
  for (int r = 0; r < each; ++r) {
    const int j = (blockIdx.y * each + r) * 4 + wave;
    if (j >= g.J || left <= 0) break;
    float v[4], w[4], d[4], t[4], o[4];
    load_four((const T*)g.other + (long long)j * g.ldother + i, g.other ? left : 0, o);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = b[e];
      w[e] = c[e];
    }
    const float* p = g.part + (long long)j * g.I + i;
#pragma unroll 4
    for (int s = 0; s < splits; ++s, p += (long long)g.I * g.J) {
      load_four(p, left, t);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[e] += t[e];
      if constexpr (kPair) {
        load_four(p + g.pair, left, t);
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] += t[e];
      }
    }
    float f[4];
    activate<sizeof(T) == 2, kDz>(g.act, v, f, d, g.slope);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if constexpr (MODE == kLinear) {
        v[e] = f[e] + o[e];
      } else if constexpr (MODE == kGated) {
        v[e] = f[e] * w[e];
      } else if constexpr (MODE == kLinearDz) {
        v[e] = o[e] * d[e];
      } else {
        v[e] = o[e] * w[e] * d[e];
        w[e] = o[e] * f[e];
      }
      if (kDz && e < left) {
        sv[e] += v[e];
        sw[e] += w[e];
      }
    }
    T* out = (T*)g.out + (long long)j * g.ldo + i;
#pragma unroll
    for (int n = 0; n < (kDz && sizeof(T) == 2 ? 2 : 1); ++n) {
      if (n && !g.low) break;
      if (n) {
        rounded_off<T, 4>(v);
        rounded_off<T, 4>(w);
        out += g.low;
      }
      store_four(out, v, left);
      if (MODE == kGatedDz) store_four(out + g.pair, w, left);
    }
  }
  if constexpr (kDz) {
    if (!g.sums) return;
    if (wave)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        red[wave - 1][0][lane * 4 + e] = sv[e];
        if (kPair) red[wave - 1][kPair][lane * 4 + e] = sw[e];
      }
    __syncthreads();
    if (wave) return;
    float* sums = g.sums + (long long)blockIdx.y * g.I + i;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      if (e >= left) break;
      sums[e] = sv[e] + red[0][0][lane * 4 + e] + red[1][0][lane * 4 + e] + red[2][0][lane * 4 + e];
      if (kPair)
        sums[g.pair + e] = sw[e] + red[0][kPair][lane * 4 + e] + red[1][kPair][lane * 4 + e] +
                           red[2][kPair][lane * 4 + e];
    }
  }
}
// some blocks a CU where there are that many tokens
static int finish_each(const ProductArgs& g) {
  const int outs = g.mode == kGated || g.mode == kGatedDz ? g.pair : g.I;
  const long long blocks = (outs + 255LL) / 256 * ((g.J + 3) / 4);
  return (int)((blocks + 2047) / 2048);
}
static int finish_rows(const ProductArgs& g) {
  const int each = finish_each(g) * 4;
  return (g.J + each - 1) / each;
}
template <typename T>
static hipError_t finish_t(const ProductArgs& g, int splits, hipStream_t stream) {
  const int outs = g.mode == kGated || g.mode == kGatedDz ? g.pair : g.I;
  const dim3 grid((outs + 255) / 256, finish_rows(g));
  const int each = finish_each(g);
#define FINISH(MODE) finish_parts<T, MODE><<<grid, 256, 0, stream>>>(g, splits, each)
  switch (g.mode) {
    case kLinear: FINISH(kLinear); break;
    case kLinearDz: FINISH(kLinearDz); break;
    case kGated: FINISH(kGated); break;
    case kGatedDz: FINISH(kGatedDz); break;
    default: return hipErrorInvalidValue;
  }
#undef FINISH
  return hipGetLastError();
}
template <typename T>
static hipError_t launch_t(const ProductArgs& g, const ProductPlan& p, hipStream_t stream) {
  const int splits = g.mode == kPartial ? g.splits : p.splits;
  if (splits > 1 && (size_t)splits * g.I * g.J * sizeof(float) > g.part_bytes)
    return hipErrorInvalidValue;  // not the workspace of this plan
  if (g.mode == kPartial || splits == 1) return product_t<T>(g, p, stream);
  ProductArgs parts = g;
  parts.mode = kPartial;
  parts.out = g.part;
  parts.splits = p.splits;
  const hipError_t e = product_t<T>(parts, p, stream);
  return e == hipSuccess ? finish_t<T>(g, p.splits, stream) : e;
}
hipError_t product_launch(const ProductArgs& g, int dtype, hipStream_t stream) {
  const ProductPlan p = product_plan(g, dtype);
  return dtype == 0   ? launch_t<float>(g, p, stream)
         : dtype == 1 ? launch_t<__half>(g, p, stream)
                      : launch_t<__hip_bfloat16>(g, p, stream);
}
size_t product_part_bytes(const ProductArgs& g, int dtype) {
  const int splits = product_plan(g, dtype).splits;
  return splits > 1 ? align256((size_t)splits * g.I * g.J * sizeof(float)) : 0;
}

// Rows of partial sums that a kLinearDz / kGatedDz launch writes.
int product_sum_rows(const ProductArgs& g, int dtype) {
  const ProductPlan p = product_plan(g, dtype);
  if (p.splits > 1) return finish_rows(g);
  if (p.kernel <= kFew64) return 1 << (p.kernel - kFew16);
  if (g.channel_i) return (g.J + p.bj - 1) / p.bj * 2 * p.passes;
  return (g.I + p.bi - 1) / p.bi * 2 * g.batches;
}

// ---- rows at 16-byte places ----
// Copies bound by memory, or by their launch (a 5 x 96 x 1961 fp16 map: 4 us).
struct LayJobs {
  LayJob job[kJobs];
};
template <typename T> __global__ __launch_bounds__(256) void lay_out(const LayJobs jobs) {
  constexpr int E = 16 / (int)sizeof(T);
  const LayJob& j = jobs.job[blockIdx.y];
  T* dst = (T*)j.dst;
  const long long chunks = (j.cols + E - 1) / E, pitch = chunks * E;
  const long long first = blockIdx.x * 256LL + threadIdx.x, next = gridDim.x * 256LL;
  if (!j.src) {
    for (long long r = first; r < j.rows; r += next)
      for (long long c = j.cols; c < pitch; ++c) dst[r * pitch + c] = narrow<T>(0.f);
    return;
  }
  for (long long id = first; id < j.rows * chunks; id += next) {
    const long long r = id / chunks, c = (id - r * chunks) * E;
    const long long m = r / j.per_image;
    const T* p = (const T*)j.src + m * j.image + (r - m * j.per_image) * j.row + c;
    *(u32x4*)(dst + id * E) = j.cols - c >= E ? load16(p) : load_some(p, (int)(j.cols - c));
  }
}
hipError_t product_lay_out(const LayJob (&jobs)[kJobs], int dtype, hipStream_t stream) {
  LayJobs all = {};
  long long blocks = 0;
  int n = 0;
  const long long e = dtype == 0 ? 4 : 8;
  for (const LayJob& j : jobs) {
    const long long chunks = (j.cols + e - 1) / e;
    if (j.rows == 0 || (!j.src && chunks * e == j.cols)) continue;
    all.job[n++] = j;
    const long long b = ((j.src ? j.rows * chunks : j.rows) + 255) / 256;
    if (blocks < b) blocks = b;
  }
  if (n == 0) return hipSuccess;
  const dim3 grid((unsigned)(blocks < 16384 ? blocks : 16384), n);
  if (dtype == 0)
    lay_out<float><<<grid, 256, 0, stream>>>(all);
  else  // 16 bits are moved as they are
    lay_out<__half><<<grid, 256, 0, stream>>>(all);
  return hipGetLastError();
}

// ---- sums of parts ----
// Bound by memory (two parts of 4096 x 1024 values and a bias gradient, 34 MB read: 10.5 us).  Few
// parts of many values: a thread takes four values.  Many parts of few values:
// `groups` threads share a value, eight parts each, and join through LDS; the order is the same
// whatever runs first.
struct SumJobs {
  SumJob job[kJobs];
  int groups[kJobs], first[kJobs + 1];  // first: blocks before the job's
};
template <typename T> __global__ __launch_bounds__(512) void sum_parts(const SumJobs jobs) {
  __shared__ float red[512];
  int which = 0;
#pragma unroll
  for (int k = 1; k < kJobs; ++k) which += (int)blockIdx.x >= jobs.first[k];
  const SumJob& j = jobs.job[which];
  const int groups = jobs.groups[which], blocks = jobs.first[which + 1] - jobs.first[which];
  const long long block = (int)blockIdx.x - jobs.first[which];
  T* out = (T*)j.out;
  if (groups == 1) {
    for (long long c = (block * 512 + threadIdx.x) * 4; c < j.n; c += blocks * 2048LL) {
      const int have = j.n - c < 4 ? (int)(j.n - c) : 4;
      float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
      for (int k = 0; k < j.parts; ++k) {
        const float* p = j.part + k * j.n + c;
        const Pack<float, 4> v =
            __builtin_bit_cast(Pack<float, 4>, have == 4 ? load16(p) : load_some(p, have));
#pragma unroll
        for (int e = 0; e < 4; ++e) s[e] += v.v[e];
      }
      store_four(out + c, s, have);
    }
    return;
  }
  const int cols = 512 / groups, col = threadIdx.x % cols, group = threadIdx.x / cols;
  for (long long c0 = block * cols; c0 < j.n; c0 += (long long)blocks * cols) {
    const long long c = c0 + col;
    float s = 0.f;
    if (c < j.n) {
#pragma unroll 8
      for (int k = group; k < j.parts; k += groups) s += j.part[k * j.n + c];
    }
    __syncthreads();
    red[threadIdx.x] = s;
    __syncthreads();
    if (group > 0 || c >= j.n) continue;
    for (int k = 1; k < groups; ++k) s += red[k * cols + col];
    out[c] = narrow<T>(s);
  }
}
hipError_t product_sum(const SumJob (&jobs)[kJobs], int dtype, hipStream_t stream) {
  SumJobs all = {};
  int n = 0;
  long long blocks = 0;
  for (const SumJob& j : jobs) {
    if (j.n == 0) continue;
    int groups = 1;
    while (groups < 32 && groups * 16 <= j.parts) groups *= 2;
    const long long each = groups == 1 ? 2048 : 512 / groups, b = (j.n + each - 1) / each;
    all.job[n] = j;
    all.groups[n] = groups;
    all.first[n] = (int)blocks;
    blocks += b < 65536 ? b : 65536;
    ++n;
  }
  if (n == 0) return hipSuccess;
  for (int k = n; k <= kJobs; ++k) all.first[k] = (int)blocks;
  if (dtype == 0)
    sum_parts<float><<<(unsigned)blocks, 512, 0, stream>>>(all);
  else if (dtype == 1)
    sum_parts<__half><<<(unsigned)blocks, 512, 0, stream>>>(all);
  else
    sum_parts<__hip_bfloat16><<<(unsigned)blocks, 512, 0, stream>>>(all);
  return hipGetLastError();
}

// Partial column sums of dy, for a linear without an activation: tokens [M][C], a wave V channels
// of a lane by 4 waves' rows; maps [B][C][P], a block a channel.  Bound by reading dy (8192 x 4096
// bf16, 67 MB: 15 us with the sums over the parts).
template <typename T, int V>
__global__ __launch_bounds__(256) void sum_tokens(const T* __restrict__ dy,
                                                  float* __restrict__ part, long long M, int C) {
  __shared__ float red[3][64 * V];
  const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
  const int c = (blockIdx.x * 64 + lane) * V;
  const long long lo = M * blockIdx.y / gridDim.y, hi = M * (blockIdx.y + 1) / gridDim.y;
  float s[V];
#pragma unroll
  for (int e = 0; e < V; ++e) s[e] = 0.f;
  if (c < C)
    for (long long m = lo + w; m < hi; m += 4) {
      float v[V];
      load_values<T, V>(dy + m * C + c, v);
#pragma unroll
      for (int e = 0; e < V; ++e) s[e] += v[e];
    }
  if (w > 0)
#pragma unroll
    for (int e = 0; e < V; ++e) red[w - 1][lane * V + e] = s[e];
  __syncthreads();
  if (w == 0 && c < C)
#pragma unroll
    for (int e = 0; e < V; ++e)
      part[(long long)blockIdx.y * C + c + e] =
          s[e] + red[0][lane * V + e] + red[1][lane * V + e] + red[2][lane * V + e];
}
template <typename T>
__global__ __launch_bounds__(256) void sum_map(const T* __restrict__ dy, float* __restrict__ part,
                                               long long B, long long P, int C) {
  __shared__ float red[4];
  const int c = blockIdx.x;
  // this part's share of the B * P pixels, image by image
  const long long lo = B * P * blockIdx.y / gridDim.y, hi = B * P * (blockIdx.y + 1) / gridDim.y;
  float s = 0.f;
  for (long long b = lo / P; b * P < hi; ++b) {
    const long long from = lo > b * P ? lo - b * P : 0, to = hi < (b + 1) * P ? hi - b * P : P;
    const T* p = dy + (b * C + c) * P;
    for (long long i = from + threadIdx.x; i < to; i += 256) s += to_f32(p[i]);
  }
  s = lanes_sum<64>(s);
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = s;
  __syncthreads();
  if (threadIdx.x == 0) part[(long long)blockIdx.y * C + c] = red[0] + red[1] + red[2] + red[3];
}
int product_column_parts(int layout, long long B, long long P, int C) {
  const long long M = layout == kMap ? B * P : P;
  // about 1024 blocks, with some thousands of values each
  const long long across = layout == kMap ? C : (C + 511) / 512;
  long long parts = 1024 / across + 1, most = layout == kMap ? M / 2048 + 1 : M / 64 + 1;
  return (int)(parts < most ? parts : most);
}
template <typename T>
static hipError_t column_sums_t(const void* dy, float* part, int layout, long long B, long long P,
                                int C, int parts, hipStream_t stream) {
  constexpr int V = 16 / (int)sizeof(T);
  if (layout == kMap)
    sum_map<T><<<dim3(C, parts), 256, 0, stream>>>((const T*)dy, part, B, P, C);
  else if (C % V == 0)
    sum_tokens<T, V><<<dim3((C + 64 * V - 1) / (64 * V), parts), 256, 0, stream>>>((const T*)dy,
                                                                                  part, P, C);
  else
    sum_tokens<T, 1><<<dim3((C + 63) / 64, parts), 256, 0, stream>>>((const T*)dy, part, P, C);
  return hipGetLastError();
}
hipError_t product_column_sums(const void* dy, float* part, int layout, long long B, long long P,
                               int C, int parts, int dtype, hipStream_t stream) {
  return dtype == 0   ? column_sums_t<float>(dy, part, layout, B, P, C, parts, stream)
         : dtype == 1 ? column_sums_t<__half>(dy, part, layout, B, P, C, parts, stream)
                      : column_sums_t<__hip_bfloat16>(dy, part, layout, B, P, C, parts, stream);
}

}  // namespace feat
}  // namespace pwc
