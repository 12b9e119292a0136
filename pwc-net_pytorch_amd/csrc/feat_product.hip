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
#include "feat_common.cuh"
#include "feat_product.cuh"

namespace pwc {
namespace feat {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 h16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 b16x8 __attribute__((ext_vector_type(8)));

template <typename T> struct Frag;
template <> struct Frag<float> { typedef f32x4 type; };
template <> struct Frag<__half> { typedef s16x8 type; };
template <> struct Frag<__hip_bfloat16> { typedef s16x8 type; };

__device__ __forceinline__ f32x4 mma(const f32x4& a, const f32x4& b, f32x4 c, float) {
#pragma unroll
  for (int s = 0; s < 4; ++s) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[s], b[s], c, 0, 0, 0);
  return c;
}
__device__ __forceinline__ f32x4 mma(const s16x8& a, const s16x8& b, f32x4 c, __half) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(h16x8, a),
                                                __builtin_bit_cast(h16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(const s16x8& a, const s16x8& b, f32x4 c, __hip_bfloat16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(b16x8, a),
                                                 __builtin_bit_cast(b16x8, b), c, 0, 0, 0);
}
// a fragment of ones: its product with B leaves the sums of B's rows (db)
__device__ __forceinline__ void ones(f32x4& f, float) { f = f32x4{1.f, 1.f, 1.f, 1.f}; }
__device__ __forceinline__ void ones(s16x8& f, __half) {
  for (int e = 0; e < 8; ++e) f[e] = 0x3C00;
}
__device__ __forceinline__ void ones(s16x8& f, __hip_bfloat16) {
  for (int e = 0; e < 8; ++e) f[e] = 0x3F80;
}

constexpr int kStepBytes = 128;           // bytes of k in a step
constexpr uint32_t kOOB = 0x80000000u;    // beyond every buffer range: the load returns zeros

// The chunk (16 bytes) of row `r` where logical chunk c lies.
// K tile: 8 chunks a row; a wave's 16-byte reads take 16 rows at one logical chunk.
__device__ __forceinline__ int swz_k(int r, int c) { return c ^ ((r >> 1) & 7); }
// N tile, 16 bits: a transposing read takes, per 16 lanes, 4 rows of 32 bytes; lanes 0-31 take
// rows 0-3 and 8-11.  32 bits: rows q*4+s of the four lane groups q, 64 bytes each.
template <typename T, int CHUNKS> __device__ __forceinline__ int swz_n(int k, int c) {
  const int g = sizeof(T) == 2 ? ((k & 3) | ((k >> 1) & 4)) * 2 : ((k >> 2) & 3) * 4;
  return c ^ (g & (CHUNKS - 1));
}

// One operand's tile: R rows (its i or j) times a k step, loaded by NW waves.
template <typename T, int R, bool KC, int NW> struct Tile {
  static constexpr int E = 16 / (int)sizeof(T);             // values in a chunk
  static constexpr int KS = kStepBytes / (int)sizeof(T);    // k in a step
  static constexpr int BYTES = R * kStepBytes;
  static constexpr int ROWB = KC ? kStepBytes : R * (int)sizeof(T);
  static constexpr int CHUNKS = ROWB / 16;
  static constexpr int LOADS = BYTES / 16 / (NW * 64);      // chunks of a thread
  static_assert(LOADS * NW * 64 * 16 == BYTES, "tile splits over the threads");

  // Chunk n of this thread: its place in LDS is linear (what a wave's direct load wants).
  static __device__ __forceinline__ int place(int n) {
    return ((n * NW * 64) + (int)threadIdx.x) * 16;
  }
  // row of memory and value within it (relative to the tile) that belong there
  static __device__ __forceinline__ void source(int n, int& row, int& at) {
    const int p = place(n);
    row = p / ROWB;
    const int c = (p % ROWB) / 16;
    at = (KC ? swz_k(row, c) : swz_n<T, CHUNKS>(row, c)) * E;
  }
  // fragment of 16 rows from r0 (K: rows, N: columns), k part kk (of 2)
  static __device__ __forceinline__ typename Frag<T>::type frag(const char* lds, int r0, int kk) {
    const int lane = threadIdx.x & 63, l = lane & 15, q = lane >> 4;
    if constexpr (KC) {
      const int r = r0 + l;
      return *(const typename Frag<T>::type*)(lds + r * ROWB + swz_k(r, kk * 4 + q) * 16);
    } else if constexpr (sizeof(T) == 2) {
      s16x8 f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int k = kk * 32 + q * 8 + h * 4 + (l >> 2);
        const int col = r0 + (l & 3) * 4;
        const char* p = lds + k * ROWB + swz_n<T, CHUNKS>(k, col / 8) * 16 + (col % 8) * 2;
        const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) s16x4*)p);
#pragma unroll
        for (int e = 0; e < 4; ++e) f[h * 4 + e] = v[e];
      }
      return f;
    } else {
      f32x4 f;
#pragma unroll
      for (int s = 0; s < 4; ++s) {
        const int k = kk * 16 + q * 4 + s, col = r0 + l;
        f[s] = *(const float*)(lds + k * ROWB + swz_n<T, CHUNKS>(k, col / 4) * 16 + (col % 4) * 4);
      }
      return f;
    }
  }
};

// The loads of one operand.  DIRECT: memory -> LDS by the buffer unit, whose range check gives the
// zeros outside; it wants 16-byte aligned rows.  Otherwise through registers from any address;
// a chunk that crosses the end of its row is read value by value.
template <typename T, int R, bool KC, int NW, bool DIRECT> struct Loader {
  typedef Tile<T, R, KC, NW> Tl;
  const T* base;      // of the tile's first row and this batch
  long long ld;
  int K, limit;       // k in a segment; N: rows left of the tile's own dimension
  uint32_t off[Tl::LOADS];  // DIRECT: bytes from base, or kOOB
  int at[Tl::LOADS];        // first k (K) or row k (N) of the chunk within the step
  long long row[DIRECT ? 1 : Tl::LOADS];
  int left[DIRECT ? 1 : Tl::LOADS];  // N: valid values from the chunk's start; K: 0 or 1 (row valid)
  Vec16<T> reg[DIRECT ? 1 : Tl::LOADS];

  // `pair` > 0: rows alternate in groups of 16 between the halves of a matrix of 2 * pair rows
  __device__ __forceinline__ void init(const T* b, long long ld_, int K_, int r0, int rows,
                                       int pair) {
    ld = ld_;
    K = K_;
    base = KC ? b + (pair ? (long long)(r0 / 2) : (long long)r0) * ld : b + r0;
    limit = rows - r0;
#pragma unroll
    for (int n = 0; n < Tl::LOADS; ++n) {
      int r, c;
      Tl::source(n, r, c);
      if constexpr (KC) {
        long long rr = r;
        bool ok = r < limit;
        if (pair) {
          const int o = (r >> 5) * 16 + (r & 15);
          ok = r0 / 2 + o < pair;
          rr = o + ((r >> 4) & 1) * (long long)pair;
        }
        at[n] = c;
        if constexpr (DIRECT) {
          off[n] = ok ? (uint32_t)(rr * ld + c) * (uint32_t)sizeof(T) : kOOB;
        } else {
          row[n] = rr * ld + c;
          left[n] = ok;
        }
      } else {
        at[n] = r;
        if constexpr (DIRECT) {
          off[n] = c < limit ? (uint32_t)(r * ld + c) * (uint32_t)sizeof(T) : kOOB;
        } else {
          row[n] = r * ld + c;
          left[n] = limit - c;
        }
      }
    }
  }

  // start loading the step at k0 of the segment at `seg` values from base
  __device__ __forceinline__ void load(char* lds, long long seg, int k0) {
    const T* b = base + seg + (KC ? (long long)k0 : (long long)k0 * ld);
    if constexpr (DIRECT) {
      const uint64_t a = (uint64_t)(uintptr_t)b;
      const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)a);
      const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32));
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
          (void*)(uintptr_t)(((uint64_t)hi << 32) | lo), (short)0, 0x7fffffff, 0x00020000);
      const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
#pragma unroll
      for (int n = 0; n < Tl::LOADS; ++n) {
        const uint32_t o = k0 + at[n] < K ? off[n] : kOOB;
        __builtin_amdgcn_raw_ptr_buffer_load_lds(
            rs, (__attribute__((address_space(3))) void*)(lds + (n * NW + wave) * 1024), 16, o, 0, 0,
            0);
      }
    } else {
#pragma unroll
      for (int n = 0; n < Tl::LOADS; ++n) {
        // K: k0 + at .. < K;  N: row k0 + at < K, `left` values of it
        const int have = KC ? (left[n] ? K - k0 - at[n] : 0) : (k0 + at[n] < K ? left[n] : 0);
        const T* p = b + row[n];
        if (have >= Tl::E) {
          __builtin_memcpy(&reg[n], p, 16);  // any alignment
        } else {
#pragma unroll
          for (int e = 0; e < Tl::E; ++e) {
            reg[n].v[e] = from_f32<T>(0.f);
            if (e < have) reg[n].v[e] = p[e];
          }
        }
      }
    }
  }
  __device__ __forceinline__ void finish(char* lds) {
    if constexpr (!DIRECT) {
#pragma unroll
      for (int n = 0; n < Tl::LOADS; ++n) *(Vec16<T>*)(lds + Tl::place(n)) = reg[n];
    }
  }
};

// N values at any alignment, `n` of them there (the rest 0 / not written)
template <typename T, int N>
__device__ __forceinline__ void put(T* p, const float (&v)[N], int n) {
  Pack<T, N> o;
#pragma unroll
  for (int e = 0; e < N; ++e) o.v[e] = from_f32<T>(v[e]);
  if (n >= N) {
    __builtin_memcpy(p, &o, sizeof(o));
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e < n) p[e] = o.v[e];
  }
}
template <typename T, int N>
__device__ __forceinline__ void get(const T* p, float (&v)[N], int n) {
  Pack<T, N> o;
  if (n >= N) {
    __builtin_memcpy(&o, p, sizeof(o));
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) o.v[e] = e < n ? p[e] : from_f32<T>(0.f);
  }
#pragma unroll
  for (int e = 0; e < N; ++e) v[e] = to_f32(o.v[e]);
}

// Epilogue of one wave's WI x WJ sums, which lie in LDS as rows of i (`tile`, pitch in floats):
// V consecutive i of one j a lane, so that rows leave in 16-byte pieces.
template <typename T, int WI, int WJ, int PITCH>
__device__ __forceinline__ void finish_tile(const ProductArgs& g, const float* tile, int i0, int j0,
                                            int z) {
  constexpr int V = 16 / (int)sizeof(T);
  const int lane = threadIdx.x & 63;
  if (g.mode == kPartial) {
    float* out = (float*)g.out + (long long)z * g.I * g.J;
    for (int u = lane; u < WI / 4 * WJ; u += 64) {
      const int i = i0 + u % (WI / 4) * 4, j = j0 + u / (WI / 4);
      const float* p = tile + u / (WI / 4) * PITCH + u % (WI / 4) * 4;
      const float v[4] = {p[0], p[1], p[2], p[3]};
      if (i < g.I && j < g.J) put(out + (long long)j * g.I + i, v, g.I - i);
    }
    return;
  }
  T* out = (T*)g.out + z * g.out_batch;
  const T* bias = (const T*)g.bias;
  const T* other = g.other ? (const T*)g.other + z * g.other_batch : nullptr;
  if (g.pair_side == 0) {
    constexpr int U = WI / V;
    for (int u = lane; u < U * WJ; u += 64) {
      const int i = i0 + u % U * V, j = j0 + u / U, n = g.I - i;
      if (n <= 0 || j >= g.J) continue;
      const float* p = tile + u / U * PITCH + u % U * V;
      float v[V], o[V], b[V];
      if (other) get(other + (long long)j * g.ldother + i, o, n);
      if (bias && g.bias_i) get(bias + i, b, n);
      const float bj = bias && !g.bias_i ? to_f32(bias[j]) : 0.f;
#pragma unroll
      for (int e = 0; e < V; ++e) {
        v[e] = p[e] + (bias && g.bias_i ? b[e] : bj);
        if (g.mode == kLinearDz)
          v[e] = o[e] * act_slope(g.act, v[e], g.slope);
        else
          v[e] = act_value(g.act, v[e], g.slope) + (other ? o[e] : 0.f);
      }
      put(out + (long long)j * g.ldo + i, v, n);
    }
    return;
  }
  // gated: 16 gate rows, 16 up rows in turn along the paired side
  const bool along_i = g.pair_side == 1, back = g.mode == kGatedDz;
  const int U = (along_i ? WI / 2 : WI) / V, R = along_i ? WJ : WJ / 2;
  const int oi = along_i ? i0 / 2 : i0, oj = along_i ? j0 : j0 / 2;
  const int most_i = along_i ? g.pair : g.I, most_j = along_i ? g.J : g.pair;
  for (int u = lane; u < U * R; u += 64) {
    const int ui = u % U * V, uj = u / U;
    const int i = oi + ui, j = oj + uj, n = most_i - i;
    if (n <= 0 || j >= most_j) continue;
    const int ti = along_i ? (ui >> 4) * 32 + (ui & 15) : ui;
    const int tj = along_i ? uj : (uj >> 4) * 32 + (uj & 15);
    const float* pg = tile + tj * PITCH + ti;
    const float* pu = pg + (along_i ? 16 : 16 * PITCH);
    float d[V], v[V], w[V], bg[V], bu[V];
    if (back) get(other + (long long)j * g.ldother + i, d, n);
    if (bias && along_i) {
      get(bias + i, bg, n);
      get(bias + g.pair + i, bu, n);
    }
    const float bgj = bias && !along_i ? to_f32(bias[j]) : 0.f;
    const float buj = bias && !along_i ? to_f32(bias[g.pair + j]) : 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float xg = pg[e] + (bias && along_i ? bg[e] : bgj);
      const float xu = pu[e] + (bias && along_i ? bu[e] : buj);
      w[e] = act_value(g.act, xg, g.slope);
      if (back) {
        v[e] = d[e] * xu * act_slope(g.act, xg, g.slope);
        w[e] *= d[e];
      } else {
        v[e] = w[e] * xu;
      }
    }
    T* p = out + (long long)j * g.ldo + i;
    put(p, v, n);
    if (back) put(p + (along_i ? (long long)g.pair : (long long)g.pair * g.ldo), w, n);
  }
}

template <typename T, int BI, int BJ, int NWI, int NWJ, int PASSES, bool AKC, bool BKC, bool DIRECT>
__global__ __launch_bounds__(NWI* NWJ * 64) void product(const ProductArgs g) {
  constexpr int NW = NWI * NWJ;
  constexpr int WI = BI / NWI, WJ = BJ / NWJ, FI = WI / 16, FJ = WJ / 16;
  typedef Tile<T, BI, AKC, NW> TA;
  typedef Tile<T, BJ, BKC, NW> TB;
  typedef typename Frag<T>::type frag_t;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  constexpr int STAGE = TA::BYTES + TB::BYTES;

  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, l = lane & 15, q = lane >> 4;
  const int wi = (wave % NWI) * WI, wj = (wave / NWI) * WJ;

  // tile (ti, tj) of batch / k split z; neighbouring tiles on one XCD
  int id = xcd_remap(blockIdx.x, gridDim.x);
  const int ti = id % g.tiles_i;
  id /= g.tiles_i;
  const int tj = id % g.tiles_j, z = id / g.tiles_j;
  const int i0 = ti * BI, j0 = tj * BJ;
  const bool partial = g.mode == kPartial;
  const int batch = partial ? 0 : z;

  Loader<T, BI, AKC, NW, DIRECT> la;
  Loader<T, BJ, BKC, NW, DIRECT> lb;
  la.init((const T*)g.a + batch * g.a_batch, g.lda, g.K, i0, g.I, g.pair_side == 1 ? g.pair : 0);
  lb.init((const T*)g.b + batch * g.b_batch, g.ldb, g.K, j0, g.J, g.pair_side == 2 ? g.pair : 0);

  // steps of this block: all of K, or its share of the segments' steps
  const int per_seg = (g.K + TA::KS - 1) / TA::KS;
  const int total = g.segments * per_seg;
  int s = 0, end = total;
  if (partial) {
    s = (int)((long long)total * z / g.splits);
    end = (int)((long long)total * (z + 1) / g.splits);
  }

  f32x4 acc[FI][FJ];
  f32x4 sums[FJ];
#pragma unroll
  for (int j = 0; j < FJ; ++j) {
    sums[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < FI; ++i) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  const bool row_sums = partial && g.sums != nullptr && ti == 0 && wi == 0;
  frag_t one;
  ones(one, T());

  auto start = [&](int step, int buf) {
    const int seg = step / per_seg, k0 = (step - seg * per_seg) * TA::KS;
    char* p = lds + buf * STAGE;
    la.load(p, seg * g.a_segment, k0);
    lb.load(p + TA::BYTES, seg * g.b_segment, k0);
  };
  auto settle = [&](int buf) {
    la.finish(lds + buf * STAGE);
    lb.finish(lds + buf * STAGE + TA::BYTES);
    if constexpr (DIRECT) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
  };

  if (s < end) {
    start(s, 0);
    settle(0);
  }
  for (int buf = 0; s < end; ++s, buf ^= 1) {
    if (s + 1 < end) start(s + 1, buf ^ 1);
    const char* pa = lds + buf * STAGE;
    const char* pb = pa + TA::BYTES;
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      frag_t fa[FI], fb[FJ];
#pragma unroll
      for (int i = 0; i < FI; ++i) fa[i] = TA::frag(pa, wi + i * 16, kk);
#pragma unroll
      for (int j = 0; j < FJ; ++j) fb[j] = TB::frag(pb, wj + j * 16, kk);
#pragma unroll
      for (int i = 0; i < FI; ++i)
#pragma unroll
        for (int j = 0; j < FJ; ++j) acc[i][j] = mma(fa[i], fb[j], acc[i][j], T());
      if (row_sums) {
#pragma unroll
        for (int j = 0; j < FJ; ++j) sums[j] = mma(one, fb[j], sums[j], T());
      }
    }
    if (s + 1 < end) settle(buf ^ 1);
  }

  // lane (l, q) holds i = 16 fi + 4 q + r, j = 16 fj + l
  if (row_sums && q == 0) {
#pragma unroll
    for (int fj = 0; fj < FJ; ++fj) {
      const int j = j0 + wj + fj * 16 + l;
      if (j < g.J) g.sums[(long long)z * g.J + j] = sums[fj][0];
    }
  }
  // the sums turn through this wave's own part of LDS, HJ of the FJ columns of fragments at a time
  constexpr int PITCH = WI + 4, HJ = FJ / PASSES;
  float* tile = (float*)lds + wave * (PITCH * HJ * 16);
  __syncthreads();
#pragma unroll
  for (int h = 0; h < PASSES; ++h) {
#pragma unroll
    for (int fj = 0; fj < HJ; ++fj)
#pragma unroll
      for (int fi = 0; fi < FI; ++fi)
        *(f32x4*)(tile + (fj * 16 + l) * PITCH + fi * 16 + q * 4) = acc[fi][h * HJ + fj];
    __builtin_amdgcn_wave_barrier();
    finish_tile<T, WI, HJ * 16, PITCH>(g, tile, i0 + wi, j0 + wj + h * HJ * 16, z);
    __builtin_amdgcn_wave_barrier();
  }
}

// out[n] = sum over the splits, in their order (the same sums whatever ran first)
template <typename T>
__global__ __launch_bounds__(256) void add_splits(const float* __restrict__ part,
                                                  T* __restrict__ out, long long n, int splits) {
  for (long long i = blockIdx.x * 256LL + threadIdx.x; i < n; i += gridDim.x * 256LL) {
    float v = 0.f;
    for (int s = 0; s < splits; ++s) v += part[s * n + i];
    out[i] = from_f32<T>(v);
  }
}

template <typename T, int BI, int BJ, int NWI, int NWJ, int PASSES, bool AKC, bool BKC, bool DIRECT>
static hipError_t launch(ProductArgs g, hipStream_t stream) {
  const auto kernel = product<T, BI, BJ, NWI, NWJ, PASSES, AKC, BKC, DIRECT>;
  constexpr int stages = 2 * (BI + BJ) * kStepBytes;
  constexpr int turned = NWJ * (BI + 4 * NWI) * (BJ / NWJ / PASSES) * 4;
  constexpr int bytes = stages > turned ? stages : turned;
  hipError_t e = lds_limit((const void*)kernel, bytes);
  if (e != hipSuccess) return e;
  const long long ri = g.pair_side == 1 ? (g.pair + 15) / 16 * 32 : g.I;
  const long long rj = g.pair_side == 2 ? (g.pair + 15) / 16 * 32 : g.J;
  g.tiles_i = (int)((ri + BI - 1) / BI);
  g.tiles_j = (int)((rj + BJ - 1) / BJ);
  const long long blocks =
      (long long)g.tiles_i * g.tiles_j * (g.mode == kPartial ? g.splits : g.batches);
  if (blocks > 0x7fffffffLL) return hipErrorInvalidConfiguration;
  kernel<<<(unsigned)blocks, NWI * NWJ * 64, bytes, stream>>>(g);
  return hipGetLastError();
}

template <typename T, int BI, int BJ, int NWI, int NWJ, int PASSES>
static hipError_t by_operands(const ProductArgs& g, hipStream_t stream) {
  // direct loads: whole 16-byte chunks at 16-byte places, offsets within 31 bits
  constexpr int E = 16 / (int)sizeof(T);
  auto direct = [&](const void* p, long long ld, long long batch, long long seg, bool kc, int n,
                    int rows, int pair) {
    const long long far = (long long)(kc ? rows + pair : kStepBytes / (int)sizeof(T)) * ld;
    return aligned_to(p, 16) && ld % E == 0 && batch % E == 0 && seg % E == 0 &&
           (kc ? g.K : n) % E == 0 && far * (long long)sizeof(T) < (1LL << 31) - (1 << 20);
  };
  const bool d = direct(g.a, g.lda, g.a_batch, g.a_segment, g.a_k, g.I, BI,
                        g.pair_side == 1 ? g.pair : 0) &&
                 direct(g.b, g.ldb, g.b_batch, g.b_segment, g.b_k, g.J, BJ,
                        g.pair_side == 2 ? g.pair : 0);
  if (g.a_k && g.b_k)
    return d ? launch<T, BI, BJ, NWI, NWJ, PASSES, true, true, true>(g, stream)
             : launch<T, BI, BJ, NWI, NWJ, PASSES, true, true, false>(g, stream);
  if (!g.a_k && g.b_k)
    return d ? launch<T, BI, BJ, NWI, NWJ, PASSES, false, true, true>(g, stream)
             : launch<T, BI, BJ, NWI, NWJ, PASSES, false, true, false>(g, stream);
  return d ? launch<T, BI, BJ, NWI, NWJ, PASSES, false, false, true>(g, stream)
           : launch<T, BI, BJ, NWI, NWJ, PASSES, false, false, false>(g, stream);
}

template <typename T> static hipError_t product_t(const ProductArgs& g, hipStream_t stream) {
  return by_operands<T, 128, 128, 2, 2, 1>(g, stream);
}

template <typename T>
static hipError_t add_splits_t(const float* part, void* out, long long n, int splits,
                               hipStream_t stream) {
  const long long blocks = (n + 255) / 256;
  add_splits<T><<<(unsigned)(blocks < 65536 ? blocks : 65536), 256, 0, stream>>>(part, (T*)out, n,
                                                                               splits);
  return hipGetLastError();
}

hipError_t product_launch(const ProductArgs& g, int dtype, hipStream_t stream) {
  return dtype == 0   ? product_t<float>(g, stream)
         : dtype == 1 ? product_t<__half>(g, stream)
                      : product_t<__hip_bfloat16>(g, stream);
}

// Blocks that share a weight gradient's k: enough for every CU, a step or more each.
int product_splits(long long I, long long J, int segments, long long K, int dtype) {
  const int ks = dtype == 0 ? 32 : 64;
  const long long tiles = ((I + 127) / 128) * ((J + 127) / 128);
  const long long steps = segments * ((K + ks - 1) / ks);
  long long splits = (512 + tiles - 1) / tiles;
  if (splits > (steps + 3) / 4) splits = (steps + 3) / 4;
  return (int)(splits < 1 ? 1 : splits);
}

hipError_t product_add_splits(const float* part, void* out, long long n, int splits, int dtype,
                              hipStream_t stream) {
  return dtype == 0   ? add_splits_t<float>(part, out, n, splits, stream)
         : dtype == 1 ? add_splits_t<__half>(part, out, n, splits, stream)
                      : add_splits_t<__hip_bfloat16>(part, out, n, splits, stream);
}

}  // namespace feat
}  // namespace pwc
