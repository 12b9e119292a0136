// feat_product_kernel.cuh — the matrix product kernel of feat_product.hip, instantiated per type.
#pragma once

#include <type_traits>

#include "feat_product.cuh"
#include "feat_steps.cuh"

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
// The same with the sums pinned to the accumulation registers: left to itself the compiler moves
// a 256 x 256 tile's sums between the two register files, 350 moves a step.  Nothing but these
// instructions touches the sums until the waits behind the loop have let the last of them finish, and
// no operand is written right before one: the compiler keeps no wait states for inline asm, so the
// build looks at what it made (check_pinned.py).
__device__ __forceinline__ void mma_pinned(const s16x8& a, const s16x8& b, f32x4& c, __half) {
  asm("v_mfma_f32_16x16x32_f16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
__device__ __forceinline__ void mma_pinned(const s16x8& a, const s16x8& b, f32x4& c,
                                           __hip_bfloat16) {
  asm("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(c) : "v"(a), "v"(b));
}
__device__ __forceinline__ void mma_pinned(const f32x4& a, const f32x4& b, f32x4& c, float) {
  c = mma(a, b, c, 0.f);
}
constexpr int kStepBytes = 128;           // bytes of k in a step
constexpr uint32_t kOOB = 0x80000000u;    // beyond every buffer range: the load returns zeros

// The chunk (16 bytes) of row `r` where logical chunk c lies.
// K tile: a wave's 16-byte reads take 16 rows at one logical chunk of the 8 of a row.
__device__ __forceinline__ int swz_k(int r, int c) { return c ^ ((r >> 1) & 7); }
// N tile, 16 bits: a transposing read takes, per 16 lanes, 4 rows of 32 bytes; lanes 0-31 take
// rows 0-3 and 8-11.  32 bits: rows q*4+s of the four lane groups q, 64 bytes each.
template <typename T, int CHUNKS> __device__ __forceinline__ int swz_n(int k, int c) {
  const int g = sizeof(T) == 2 ? ((k & 3) | ((k >> 1) & 4)) * 2 : ((k >> 2) & 3) * 4;
  return c ^ (g & (CHUNKS - 1));
}

// Chunk c of four sums of row j in the turned tile: 16 neighbouring rows write one chunk each.
template <int WI> __device__ __forceinline__ int swz_turn(int j, int c) {
  return c ^ (j & (WI / 4 < 16 ? WI / 4 - 1 : 15));
}

// V neighbouring sums of row j of the turned tile, from column i on
template <int WI, int V>
__device__ __forceinline__ void turned(const float* tile, int j, int i, float (&v)[V]) {
  if constexpr (V == 1) {
    v[0] = tile[j * WI + swz_turn<WI>(j, i / 4) * 4 + i % 4];
  } else {
#pragma unroll
    for (int c = 0; c < V / 4; ++c) {
      const f32x4 q = *(const f32x4*)(tile + j * WI + swz_turn<WI>(j, i / 4 + c) * 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) v[c * 4 + e] = q[e];
    }
  }
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
  int limit;          // N: rows left of the tile's own dimension
  uint32_t off[Tl::LOADS];  // DIRECT: bytes from base, or kOOB
  int at[Tl::LOADS];        // first k (K) or row k (N) of the chunk within the step
  long long row[DIRECT ? 1 : Tl::LOADS];
  int left[DIRECT ? 1 : Tl::LOADS];  // N: valid values from the chunk's start; K: row valid, 0 or 1
  u32x4 reg[DIRECT ? 1 : Tl::LOADS];

  // `pair` > 0: rows alternate in groups of 16 between the halves of a matrix of 2 * pair rows
  __device__ __forceinline__ void init(const T* b, long long ld_, int r0, int rows, int pair) {
    ld = ld_;
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

  // the step at k0 of the segment at `seg` values from base, which has `have` values of k: where it
  // lies, then its loads
  const T* from;
  int left_k;
  __device__ __forceinline__ void aim(long long seg, int k0, int have) {
    from = base + seg + (KC ? (long long)k0 : (long long)k0 * ld);
    left_k = have;
  }
  __device__ __forceinline__ void load(char* lds, int n) {
    if constexpr (DIRECT) {
      const uint64_t a = (uint64_t)(uintptr_t)from;
      const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)a);
      const uint32_t hi = __builtin_amdgcn_readfirstlane((uint32_t)(a >> 32));
      const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc(
          (void*)(uintptr_t)(((uint64_t)hi << 32) | lo), (short)0, 0x7fffffff, 0x00020000);
      const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
      const uint32_t o = at[n] < left_k ? off[n] : kOOB;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(
          rs, (__attribute__((address_space(3))) void*)(lds + (n * NW + wave) * 1024), 16, o, 0, 0,
          0);
    } else {
      // K: k0 + at .. < K;  N: row k0 + at < K, `left` values of it
      const int have = KC ? (left[n] ? left_k - at[n] : 0) : (at[n] < left_k ? left[n] : 0);
      const T* p = from + row[n];
      if (have >= Tl::E) {
        reg[n] = load16(p);
      } else {
        reg[n] = u32x4{0u, 0u, 0u, 0u};
        if (have > 0) reg[n] = load_some(p, have);
      }
    }
  }
  __device__ __forceinline__ void finish(char* lds) {
    if constexpr (!DIRECT) {
#pragma unroll
      for (int n = 0; n < Tl::LOADS; ++n) *(u32x4*)(lds + Tl::place(n)) = reg[n];
    }
  }
};

// What the epilogue needs of one wave's sums: they lie in LDS as rows of i (`tile`, WI long).
struct Finish {
  const float* tile;
  float* row_sums;   // LDS, this wave's: sums of dz over the tokens of a row (maps)
  int i0, j0;        // first output column and row; gated: counted in outputs
  int i_end, j_end;  // the output's bounds
};

// A lane keeps V neighbouring i, so that whole rows leave in 16-byte pieces, and goes over the rows
// j in batches whose loads are all under way before the first is used: there may be one wave a
// SIMD, and nothing else would hide them.  V = 1 takes the columns behind the last whole piece.
template <typename T, int MODE, bool CI, int WI, int WJ, int V>
__device__ __forceinline__ void finish_columns(const ProductArgs& g, const Finish& f, T* out,
                                               const T* other, int sum_row) {
  constexpr bool kFast = sizeof(T) == 2, kPair = MODE == kGated || MODE == kGatedDz;
  constexpr bool kDz = MODE == kLinearDz || MODE == kGatedDz;
  constexpr bool kLow = kDz && sizeof(T) == 2 && WI == 32;  // small tiles
  constexpr int E = 16 / (int)sizeof(T);                    // columns of a whole piece
  constexpr int COLS = kPair && CI ? WI / 2 : WI, ROWS = kPair && !CI ? WJ / 2 : WJ;
  constexpr int U = V == 1 ? E : COLS / V, RS = 64 / U, N = ROWS / RS;
  constexpr int NB = V == 1 ? 1 : (kPair ? 2 : 4) < N ? (kPair ? 2 : 4) : N;
  const int lane = threadIdx.x & 63, ul = lane % U, uj = lane / U;
  const int have = min(COLS, f.i_end - f.i0);               // columns that exist
  const int ui = V == 1 ? have / E * E + ul : ul * V, i = f.i0 + ui;
  const bool column = ui + V <= have;
  const int ti = kPair && CI ? (ui >> 4) * 32 + (ui & 15) : ui;
  const T* bias = (const T*)g.bias;
  const long long ldo = g.ldo, ldother = g.ldother;
  const int act = g.act;
  const float slope = g.slope;

  // Bias: of a lane's own channels (along i), or of the row
  float b[V], c[V];
#pragma unroll
  for (int e = 0; e < V; ++e) b[e] = c[e] = 0.f;
  if (MODE != kPlain && CI && bias && column) {
    load_values<T, V>(bias + i, b);
    if (kPair) load_values<T, V>(bias + g.pair + i, c);
  }
  // Bias gradient: sums of dz before it is rounded
  float sv[V], sw[V];
#pragma unroll
  for (int e = 0; e < V; ++e) sv[e] = sw[e] = 0.f;

  // the residual or output gradient, a batch ahead
  constexpr bool kOther = MODE != kGated && MODE != kPlain;
  u32x4 ahead[kOther && V > 1 ? NB : 1];
  auto fetch = [&](int r0) __attribute__((always_inline)) {
    if constexpr (kOther && V > 1) {
#pragma unroll
      for (int r = 0; r < NB; ++r) {
        const int j = f.j0 + uj + (r0 + r) * RS;
        ahead[r] = u32x4{0u, 0u, 0u, 0u};
        if (other && column && r0 < N && j < f.j_end)
          ahead[r] = load16(other + (long long)j * ldother + i);
      }
    }
  };
  fetch(0);
#pragma unroll 1
  for (int r0 = 0; r0 < N; r0 += NB) {
    float v[NB][V], w[NB][V], o[NB][V], bj[NB], cj[NB];
    bool ok[NB];
#pragma unroll
    for (int r = 0; r < NB; ++r) {
      const int j = f.j0 + uj + (r0 + r) * RS;
      ok[r] = column && j < f.j_end;
      bj[r] = cj[r] = 0.f;
      if (MODE != kPlain && !CI && bias && ok[r]) {
        bj[r] = to_f32(bias[j]);
        if (kPair) cj[r] = to_f32(bias[g.pair + j]);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) o[r][e] = 0.f;
      if constexpr (kOther && V > 1) {
        as_floats<T, V>(ahead[r], o[r]);
      } else if constexpr (kOther) {
        if (other && ok[r]) o[r][0] = to_f32(other[(long long)j * ldother + i]);
      }
    }
    fetch(r0 + NB);
#pragma unroll
    for (int r = 0; r < NB; ++r) {
      const int rj = uj + (r0 + r) * RS;
      const int tj = kPair && !CI ? (rj >> 4) * 32 + (rj & 15) : rj;
      turned<WI, V>(f.tile, tj, ti, v[r]);
      if constexpr (MODE != kPlain) {
#pragma unroll
        for (int e = 0; e < V; ++e) v[r][e] += CI ? b[e] : bj[r];
      }
      if constexpr (kPair) {
        turned<WI, V>(f.tile, CI ? tj : tj + 16, CI ? ti + 16 : ti, w[r]);
#pragma unroll
        for (int e = 0; e < V; ++e) w[r][e] += CI ? c[e] : cj[r];
      }
      if constexpr (MODE == kLinear) {
        if (act != kActNone) activate<kFast, false>(act, v[r], v[r], sv, slope);
        if (other) {
#pragma unroll
          for (int e = 0; e < V; ++e) v[r][e] += o[r][e];
        }
      } else if constexpr (MODE == kLinearDz) {
        float a[V], s[V];
        activate<kFast, true>(act, v[r], a, s, slope);
#pragma unroll
        for (int e = 0; e < V; ++e) v[r][e] = ok[r] ? o[r][e] * s[e] : 0.f;
      } else if constexpr (MODE == kGated) {
        activate<kFast, false>(act, v[r], v[r], sv, slope);
#pragma unroll
        for (int e = 0; e < V; ++e) v[r][e] *= w[r][e];
      } else if constexpr (MODE == kGatedDz) {
        float a[V], s[V];
        activate<kFast, true>(act, v[r], a, s, slope);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          v[r][e] = ok[r] ? o[r][e] * w[r][e] * s[e] : 0.f;
          w[r][e] = ok[r] ? o[r][e] * a[e] : 0.f;
        }
      }
      if constexpr (kDz && CI) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          sv[e] += v[r][e];
          if (kPair) sw[e] += w[r][e];
        }
      } else if constexpr (kDz) {
        if (g.sums) {
          float s = 0.f, t = 0.f;
#pragma unroll
          for (int e = 0; e < V; ++e) {
            s += v[r][e];
            if (kPair) t += w[r][e];
          }
#pragma unroll
          for (int d = U / 2; d > 0; d >>= 1) {
            s += __shfl_xor(s, d, 64);
            if (kPair) t += __shfl_xor(t, d, 64);
          }
          if (ul == 0) {
            f.row_sums[rj] += s;
            if (kPair) f.row_sums[ROWS + rj] += t;
          }
        }
      }
    }
#pragma unroll
    for (int r = 0; r < NB; ++r) {
      T* p = out + (long long)(f.j0 + uj + (r0 + r) * RS) * ldo + i;
      if (!ok[r]) continue;
      T* const up = p + (CI ? (long long)g.pair : g.pair * ldo);
      store_values<T, V>(p, v[r]);
      if (MODE == kGatedDz) store_values<T, V>(up, w[r]);
      if constexpr (kLow) {
        if (g.low) {
          rounded_off<T, V>(v[r]);
          store_values<T, V>(p + g.low, v[r]);
          if (MODE == kGatedDz) {
            rounded_off<T, V>(w[r]);
            store_values<T, V>(up + g.low, w[r]);
          }
        }
      }
    }
  }
  if constexpr (kDz && CI) {
    if (g.sums) {
      float* sums = g.sums + (long long)sum_row * (kPair ? 2 * g.pair : g.I);
#pragma unroll
      for (int e = 0; e < V; ++e) {
#pragma unroll
        for (int d = U; d < 64; d <<= 1) {
          sv[e] += __shfl_xor(sv[e], d, 64);
          if (kPair) sw[e] += __shfl_xor(sw[e], d, 64);
        }
        if (uj == 0 && column) {
          sums[i + e] = sv[e];
          if (kPair) sums[g.pair + i + e] = sw[e];
        }
      }
    }
  }
}

template <typename T, int MODE, bool CI, int WI, int WJ>
__device__ __forceinline__ void finish_tile(const ProductArgs& g, const float* tile,
                                            float* row_sums, int i0, int j0, int z, int sum_row) {
  constexpr bool kPair = MODE == kGated || MODE == kGatedDz;
  constexpr bool kDz = MODE == kLinearDz || MODE == kGatedDz;
  constexpr int E = 16 / (int)sizeof(T);
  const int lane = threadIdx.x & 63;
  if constexpr (MODE == kPartial) {
    if (g.splits > 1) {
      float* out = (float*)g.out + (long long)z * g.I * g.J;
#pragma unroll 4
      for (int u = lane; u < WI / 4 * WJ; u += 64) {
        const int i = i0 + u % (WI / 4) * 4, j = j0 + u / (WI / 4);
        float v[4];
        turned<WI, 4>(tile, u / (WI / 4), u % (WI / 4) * 4, v);
        if (j >= g.J) continue;
        if (i + 4 <= g.I) {
          store_values<float, 4>(out + (long long)j * g.I + i, v);
        } else {
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (i + e < g.I) out[(long long)j * g.I + i + e] = v[e];
        }
      }
      return;
    }
  }
  Finish f;
  f.tile = tile;
  f.row_sums = row_sums;
  f.i0 = kPair && CI ? i0 / 2 : i0;
  f.j0 = kPair && !CI ? j0 / 2 : j0;
  f.i_end = kPair && CI ? g.pair : g.I;
  f.j_end = kPair && !CI ? g.pair : g.J;
  constexpr int COLS = kPair && CI ? WI / 2 : WI, ROWS = kPair && !CI ? WJ / 2 : WJ;
  if constexpr (kDz && !CI) {
    for (int r = lane; r < (kPair ? 2 : 1) * ROWS; r += 64) row_sums[r] = 0.f;
    __builtin_amdgcn_wave_barrier();
  }
  const int batch = MODE == kPartial ? 0 : z;
  T* out = (T*)g.out + batch * g.out_batch;
  const T* other = g.other ? (const T*)g.other + batch * g.other_batch : nullptr;
  // one instance of the body for whole pieces, one for what is left of a row
  constexpr int M = MODE == kPartial ? kPlain : MODE;
  const int have = min(COLS, f.i_end - f.i0);
  if (have >= E) finish_columns<T, M, CI, WI, WJ, E>(g, f, out, other, sum_row);
  if (have > 0 && have % E) finish_columns<T, M, CI, WI, WJ, 1>(g, f, out, other, sum_row);
  if constexpr (kDz && !CI) {
    if (g.sums) {
      __builtin_amdgcn_wave_barrier();
      float* sums = g.sums + (long long)sum_row * (kPair ? 2 * g.pair : g.J);
      for (int r = lane; r < ROWS; r += 64)
        if (f.j0 + r < f.j_end) {
          sums[f.j0 + r] = row_sums[r];
          if (kPair) sums[g.pair + f.j0 + r] = row_sums[ROWS + r];
        }
    }
  }
}

template <typename T, int BI, int BJ, int NWI, int NWJ, int PASSES, int STAGES, bool AKC, bool BKC,
          int MODE, bool DIRECT>
__global__ __launch_bounds__(NWI* NWJ * 64, BI* BJ > 128 * 128 ? 1 : 2)
    void product(const ProductArgs g) {
  constexpr int NW = NWI * NWJ;
  constexpr bool PART = MODE == kPartial, CI = BKC && AKC && !PART;  // channels along i: tokens
  constexpr int WI = BI / NWI, WJ = BJ / NWJ, FI = WI / 16, FJ = WJ / 16;
  constexpr bool kPair = MODE == kGated || MODE == kGatedDz;
  constexpr bool kPinned = FI * FJ >= 64;  // one block a CU, one wave a SIMD
  typedef Tile<T, BI, AKC, NW> TA;
  typedef Tile<T, BJ, BKC, NW> TB;
  typedef typename Frag<T>::type frag_t;
  // Each buffer is a variable: the compiler then sees that a read of one does not have to wait for
  // the direct loads that are under way into another.
  static_assert(STAGES >= 2 && STAGES <= 3 && (DIRECT || STAGES == 2), "stages");
  constexpr int A2 = STAGES > 2 ? TA::BYTES : 16, B2 = STAGES > 2 ? TB::BYTES : 16;
  __shared__ __attribute__((aligned(16))) char a0[TA::BYTES], b0[TB::BYTES], a1[TA::BYTES],
      b1[TB::BYTES], a2[A2], b2[B2];
  __shared__ float row_sums[NW][WJ];

  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, l = lane & 15, q = lane >> 4;
  const int wi = (wave % NWI) * WI, wj = (wave / NWI) * WJ;

  // tile (ti, tj) of batch / k split z; neighbouring tiles on one XCD
  // (4 tiles along j at a time: 32 tiles in flight on an XCD share 8 tiles of A and 4 of B)
  const int plane = g.tiles_i * g.tiles_j, blocks = plane * (PART ? g.splits : g.batches);
  if (block_id() >= blocks) return;
  const int id = xcd_remap((int)block_id(), blocks), z = id / plane, at = id - z * plane;
  const int group = at / (4 * g.tiles_i), first = group * 4, in = at - group * 4 * g.tiles_i;
  const int deep = min(4, g.tiles_j - first);
  const int ti = in / deep, tj = first + in % deep;
  const int i0 = ti * BI, j0 = tj * BJ;
  const int batch = PART ? 0 : z;

  Loader<T, BI, AKC, NW, DIRECT> la;
  Loader<T, BJ, BKC, NW, DIRECT> lb;
  la.init((const T*)g.a + batch * g.a_batch, g.lda, i0, g.I, kPair && CI ? g.pair : 0);
  lb.init((const T*)g.b + batch * g.b_batch, g.ldb, j0, g.J, kPair && !CI ? g.pair : 0);

  // steps of this block: all of K, or its share of the segments' steps
  Steps at_step;  // the one whose loads start next
  at_step.init(g.segments, g.K, TA::KS, PART ? z : 0, PART ? g.splits : 1);
  int s = 0;
  const int end = at_step.left;
  auto aim = [&]() __attribute__((always_inline)) {
    // past the end every chunk is outside: zeros, without an access to memory
    const int have = at_step.have(g.K);
    la.aim((at_step.seg >> g.a_halves) * g.a_segment, at_step.k0, have);
    lb.aim(at_step.seg * g.b_segment, at_step.k0, have);
    at_step.next(g.K, TA::KS);
  };
  constexpr int LOADS = TA::LOADS + TB::LOADS;  // of a step
  auto start = [&](char* pa, char* pb) __attribute__((always_inline)) {
    aim();
#pragma unroll
    for (int n = 0; n < TA::LOADS; ++n) la.load(pa, n);
#pragma unroll
    for (int n = 0; n < TB::LOADS; ++n) lb.load(pb, n);
  };
  // the loads into these are in LDS, `behind` steps' loads may be under way, and this wave's reads
  // so far are done
  auto settle = [&](char* pa, char* pb, auto behind) __attribute__((always_inline)) {
    la.finish(pa);
    lb.finish(pb);
    constexpr int flying = DIRECT ? decltype(behind)::value * LOADS : 0;
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(flying) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
  };

  f32x4 acc[FI][FJ];
#pragma unroll
  for (int j = 0; j < FJ; ++j)
#pragma unroll
    for (int i = 0; i < FI; ++i) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  // Two fragment sets: while one is multiplied the other is read.  A step has two halves of k:
  //   multiply half 0, reading half 1 | wait for the next step's loads, barrier |
  //   multiply half 1, reading half 0 of the next step and starting the loads of the step STAGES on
  //   into the buffer that all waves have read
  // so the loads have STAGES - 1 steps, the reads half a step, and one barrier a step is enough.
  // Where one wave a SIMD has to feed the matrix unit alone, reads and loads stand between its
  // instructions, a row of fragments at a time: issued in one go they fill the queues and it waits
  // behind them (8192 x K -> 4096 tokens: 1430 -> 1520 TFLOP/s).  With two waves a SIMD one
  // multiplies while the other issues, and the same order costs a third of the rate.
  frag_t fa[2][FI], fb[2][FJ];
  auto read = [&](const char* pa, const char* pb, int kk) __attribute__((always_inline)) {
#pragma unroll
    for (int j = 0; j < FJ; ++j) fb[kk][j] = TB::frag(pb, wj + j * 16, kk);
#pragma unroll
    for (int i = 0; i < FI; ++i) fa[kk][i] = TA::frag(pa, wi + i * 16, kk);
  };
  // half kk is multiplied, half 1 - kk is read from (pa, pb); LOAD: loads start into (qa, qb)
  auto half = [&](int kk, const char* pa, const char* pb, auto load, char* qa, char* qb)
      __attribute__((always_inline)) {
    constexpr bool LOAD = decltype(load)::value;
    if constexpr (!kPinned) {
      read(pa, pb, 1 - kk);
      if (LOAD) start(qa, qb);
#pragma unroll
      for (int i = 0; i < FI; ++i)
#pragma unroll
        for (int j = 0; j < FJ; ++j) acc[i][j] = mma(fa[kk][i], fb[kk][j], acc[i][j], T());
      __builtin_amdgcn_sched_barrier(0);
    } else {
      if (LOAD) aim();
#pragma unroll
      for (int i = 0; i < FI; ++i) {
#pragma unroll
        for (int j = 0; j < FJ; ++j)
          if (j * FI / FJ == i) fb[1 - kk][j] = TB::frag(pb, wj + j * 16, 1 - kk);
        fa[1 - kk][i] = TA::frag(pa, wi + i * 16, 1 - kk);
        if (LOAD) {
#pragma unroll
          for (int n = 0; n < TA::LOADS; ++n)
            if (n * FI / TA::LOADS == i) la.load(qa, n);
#pragma unroll
          for (int n = 0; n < TB::LOADS; ++n)
            if (n * FI / TB::LOADS == i) lb.load(qb, n);
        }
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int j = 0; j < FJ; ++j) mma_pinned(fa[kk][i], fb[kk][j], acc[i][j], T());
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  auto step = [&](char* pa, char* pb, char* qa, char* qb) __attribute__((always_inline)) {
    half(0, pa, pb, std::false_type(), nullptr, nullptr);
    settle(qa, qb, std::integral_constant<int, STAGES - 2>());
    __builtin_amdgcn_sched_barrier(0);
    half(1, qa, qb, std::true_type(), pa, pb);
  };
  // (the sums stand in their registers before the wait, and are taken from them behind the next)
  auto pin = [&]() __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < FI; ++i)
#pragma unroll
      for (int j = 0; j < FJ; ++j) asm volatile("" : "+a"(acc[i][j]));
  };
  if constexpr (kPinned) {
    // written sums before the first matrix instruction reads them
    pin();
    asm volatile("s_nop 7" ::: "memory");
  }
  start(a0, b0);
  if constexpr (DIRECT) {
    // the next steps' loads follow at once; the first is there when only they are under way
    start(a1, b1);
    if constexpr (STAGES > 2) start(a2, b2);
    settle(a0, b0, std::integral_constant<int, STAGES - 1>());
    read(a0, b0, 0);
  } else {
    settle(a0, b0, std::integral_constant<int, 0>());
    read(a0, b0, 0);
    start(a1, b1);
  }
  // the steps of all buffers, or of the first `left`
  auto round = [&](int left) __attribute__((always_inline)) {
    step(a0, b0, a1, b1);
    if constexpr (STAGES == 2) {
      if (left > 1) step(a1, b1, a0, b0);
    } else {
      if (left > 1) step(a1, b1, a2, b2);
      if (left > 2) step(a2, b2, a0, b0);
    }
  };
  if constexpr (kPinned) {
    // (a step past the end multiplies zeros)
    for (; s < end; s += STAGES) round(STAGES);
  } else if constexpr (DIRECT) {
    // (written out: with exchanged pointers a read waits for the loads into the other buffers too)
    for (; s + STAGES <= end; s += STAGES) round(STAGES);
    if (s < end) round(end - s);
  } else {
    char *pa = a0, *pb = b0, *qa = a1, *qb = b1;
    for (; s < end; ++s) {
      step(pa, pb, qa, qb);
      char* t = pa;
      pa = qa;
      qa = t;
      t = pb;
      pb = qb;
      qb = t;
    }
  }
  // the last matrix instructions (16 cycles each by the counters) before their sums are read: any
  // instruction of the matrix unit would be done
  if constexpr (kPinned) {
    asm volatile("s_nop 15\n\ts_nop 15\n\ts_nop 15" ::: "memory");
    pin();
  }
  // what is still under way into LDS (zeros, or nothing) arrives before LDS is used otherwise
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
  __syncthreads();

  // lane (l, q) holds i = 16 fi + 4 q + r, j = 16 fj + l
  // the sums turn through this wave's own part of LDS, HJ of the FJ columns of fragments at a time
  constexpr int HJ = FJ / PASSES;
  constexpr int SHARE = WI * HJ * 16 * 4;
  static_assert(NW == 4 && SHARE <= (TA::BYTES < TB::BYTES ? TA::BYTES : TB::BYTES),
                "a buffer a wave");
  float* tile = (float*)(wave == 0 ? a0 : wave == 1 ? b0 : wave == 2 ? a1 : b1);
  auto pass = [&](auto which) __attribute__((always_inline)) {
    constexpr int h = decltype(which)::value;
#pragma unroll
    for (int fj = 0; fj < HJ; ++fj)
#pragma unroll
      for (int fi = 0; fi < FI; ++fi) {
        const int j = fj * 16 + l;
        *(f32x4*)(tile + j * WI + swz_turn<WI>(j, fi * 4 + q) * 4) = acc[fi][h * HJ + fj];
      }
    __builtin_amdgcn_wave_barrier();
    // this wave's row of the bias gradient's partial sums
    const int row = CI ? (tj * NWJ + wave / NWI) * PASSES + h
                       : (z * g.tiles_i + ti) * NWI + wave % NWI;
    finish_tile<T, MODE, CI, WI, HJ * 16>(g, tile, row_sums[wave], i0 + wi,
                                          j0 + wj + h * HJ * 16, z, row);
    __builtin_amdgcn_wave_barrier();
  };
  static_assert(PASSES <= 2, "passes are written out: the sums have to stay in registers");
  pass(std::integral_constant<int, 0>());
  if constexpr (PASSES == 2) pass(std::integral_constant<int, 1>());
}

// ---- few tokens: a pass over W ----
// At most 16 JB tokens: the time is W's bytes.  A block takes 16 FR output channels (gated: of each
// half) and its 8 waves take an eighth of k each; then the waves' sums are added in their order.
// Eight lanes read 128 bytes of a row, whole lines, a group of steps ahead of its use, and a
// wave turns them into fragments through its own part of LDS, without a barrier: read as the
// fragments want them, four neighbouring lanes ask for four lines, and the L1 cache gives 16 of its
// 64 bytes a cycle (4096 -> 4096 bf16, 33.6 MB: 1 token 8.6 us, 64 tokens 22; by lines 6.9 and 14).
constexpr int kFewWaves = 8;

template <typename T, int FR, int JB, int MODE>
__global__ __launch_bounds__(kFewWaves * 64, JB < 4 ? 4 : 2) void few_tokens(const ProductArgs g) {
  constexpr bool kPair = MODE == kGated || MODE == kGatedDz;
  constexpr bool kDz = MODE == kLinearDz || MODE == kGatedDz;
  constexpr int E = 16 / (int)sizeof(T), HALVES = kPair ? 2 : 1, FA = FR * HALVES;
  constexpr int STEP = 8 * E;  // k of a step: 128 bytes of a row
  constexpr int DEPTH = FA + JB > 2 ? 1 : 2;
  constexpr int REGION = ((FA + JB) * 2 > FA * JB ? (FA + JB) * 2 : FA * JB) * 1024;
  typedef typename Frag<T>::type frag_t;
  __shared__ __attribute__((aligned(16))) char lds[kFewWaves][REGION];
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, l = lane & 15, q = lane >> 4;
  const int outs = kPair ? g.pair : g.I, i0 = blockIdx.x * 16 * FR;

  // this lane's chunk of rows 8 n + lane / 8 of each fragment
  const T* pa[FA][2];
  const T* pb[JB][2];
  bool oa[FA][2], ob[JB][2];
#pragma unroll
  for (int n = 0; n < 2; ++n) {
    const int r = n * 8 + lane / 8, at = lane % 8 * E;
#pragma unroll
    for (int f = 0; f < FA; ++f) {
      const int i = i0 + f / HALVES * 16 + r;
      oa[f][n] = i < outs;
      const long long row = (long long)(kPair && f % 2 ? g.pair : 0) + (oa[f][n] ? i : 0);
      pa[f][n] = (const T*)g.a + row * g.lda + at;
    }
#pragma unroll
    for (int f = 0; f < JB; ++f) {
      ob[f][n] = f * 16 + r < g.J;
      pb[f][n] = (const T*)g.b + (ob[f][n] ? f * 16 + r : 0) * g.ldb + at;
    }
  }
  f32x4 acc[FA][JB];
#pragma unroll
  for (int f = 0; f < FA; ++f)
#pragma unroll
    for (int j = 0; j < JB; ++j) acc[f][j] = f32x4{0.f, 0.f, 0.f, 0.f};

  struct Step {
    u32x4 a[FA][2], b[JB][2];
  };
  const u32x4 none = {0u, 0u, 0u, 0u};
  auto take = [&](int k, bool whole, Step& v) __attribute__((always_inline)) {
    const int have = whole ? E : g.K - k - lane % 8 * E;
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
      for (int f = 0; f < FA; ++f) {
        v.a[f][n] = none;
        if (oa[f][n] && have >= E) v.a[f][n] = load16(pa[f][n] + k);
        if (!whole && oa[f][n] && have > 0 && have < E) v.a[f][n] = load_some(pa[f][n] + k, have);
      }
#pragma unroll
      for (int f = 0; f < JB; ++f) {
        v.b[f][n] = none;
        if (ob[f][n] && have >= E) v.b[f][n] = load16(pb[f][n] + k);
        if (!whole && ob[f][n] && have > 0 && have < E) v.b[f][n] = load_some(pb[f][n] + k, have);
      }
    }
  };
  // a fragment is 16 rows of 128 bytes, its chunks exclusive-ored with the row
  char* const mine = lds[wave];
  const int put = lane / 8 * 128 + ((lane % 8) ^ (lane / 8)) * 16;
  auto use = [&](const Step& v) __attribute__((always_inline)) {
#pragma unroll
    for (int n = 0; n < 2; ++n) {
#pragma unroll
      for (int f = 0; f < FA; ++f) *(u32x4*)(mine + f * 2048 + n * 1024 + put) = v.a[f][n];
#pragma unroll
      for (int f = 0; f < JB; ++f) *(u32x4*)(mine + (FA + f) * 2048 + n * 1024 + put) = v.b[f][n];
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    frag_t a[FA][2], b[JB][2];
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int get = l * 128 + ((c * 4 + q) ^ (l & 7)) * 16;
#pragma unroll
      for (int f = 0; f < FA; ++f) a[f][c] = *(const frag_t*)(mine + f * 2048 + get);
#pragma unroll
      for (int f = 0; f < JB; ++f) b[f][c] = *(const frag_t*)(mine + (FA + f) * 2048 + get);
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int f = 0; f < FA; ++f)
#pragma unroll
        for (int j = 0; j < JB; ++j) acc[f][j] = mma(a[f][c], b[j][c], acc[f][j], T());
  };
  // whole steps in groups of DEPTH, the next group's loads before one is used; then what is left
  const int steps = (g.K + STEP - 1) / STEP, whole = g.K / STEP;
  int s = steps * wave / kFewWaves;
  const int end = steps * (wave + 1) / kFewWaves, fast = min(end, whole);
  if (s + DEPTH <= fast) {
    Step x[DEPTH], y[DEPTH];
    auto group = [&](Step(&v)[DEPTH], int at) __attribute__((always_inline)) {
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) take((at + d) * STEP, true, v[d]);
    };
    auto spend = [&](const Step(&v)[DEPTH]) __attribute__((always_inline)) {
#pragma unroll
      for (int d = 0; d < DEPTH; ++d) use(v[d]);
      s += DEPTH;
    };
    group(x, s);
    for (;;) {
      const bool more = s + 2 * DEPTH <= fast;
      if (more) group(y, s + DEPTH);
      spend(x);
      if (!more) break;
      const bool again = s + 2 * DEPTH <= fast;
      if (again) group(x, s + DEPTH);
      spend(y);
      if (!again) break;
    }
  }
  for (; s < end; ++s) {
    Step x;
    take(s * STEP, false, x);
    use(x);
  }

  f32x4(*join)[REGION / 16] = (f32x4(*)[REGION / 16])lds;
#pragma unroll
  for (int f = 0; f < FA; ++f)
#pragma unroll
    for (int j = 0; j < JB; ++j) join[wave][(f * JB + j) * 64 + lane] = acc[f][j];
  __syncthreads();
  // one wave a fragment; lane (l, q) holds token 16 fj + l, channels 16 fi + 4 q + 0..3
  for (int u = wave; u < FR * JB; u += kFewWaves) {
    const int fi = u / JB, fj = u % JB, j = fj * 16 + l, i = i0 + fi * 16 + q * 4;
    const int at = (fi * HALVES * JB + fj) * 64 + lane;
    f32x4 a = join[0][at], b = a;
    for (int w = 1; w < kFewWaves; ++w) a += join[w][at];
    if (kPair) {
      b = join[0][at + JB * 64];
      for (int w = 1; w < kFewWaves; ++w) b += join[w][at + JB * 64];
    }
    const T* bias = (const T*)g.bias;
    const T* other = (const T*)g.other + (long long)j * g.ldother;
    T* out = (T*)g.out + (long long)j * g.ldo;
    float z[4], v[4], w[4], d[4];
    bool ok[4];
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      ok[r] = j < g.J && i + r < outs;
      z[r] = a[r] + (bias && i + r < outs ? to_f32(bias[i + r]) : 0.f);
      w[r] = b[r];
      if (kPair && bias && i + r < outs) w[r] += to_f32(bias[g.pair + i + r]);
    }
    activate<sizeof(T) == 2, kDz>(g.act, z, v, d, g.slope);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const float o = g.other && ok[r] ? to_f32(other[i + r]) : 0.f;
      if constexpr (MODE == kLinear) {
        v[r] += o;
      } else if constexpr (MODE == kGated) {
        v[r] *= w[r];
      } else if constexpr (MODE == kLinearDz) {
        v[r] = ok[r] ? o * d[r] : 0.f;
      } else {
        const float dz = ok[r] ? o * w[r] * d[r] : 0.f;
        w[r] = ok[r] ? o * v[r] : 0.f;
        v[r] = dz;
      }
      if (kDz && g.sums) {
        // the bias gradient's row of these 16 tokens
        float sv = v[r], sw = w[r];
#pragma unroll
        for (int m = 1; m < 16; m <<= 1) {
          sv += __shfl_xor(sv, m, 64);
          if (kPair) sw += __shfl_xor(sw, m, 64);
        }
        float* sums = g.sums + (long long)fj * (kPair ? 2 * g.pair : g.I);
        if (l == 0 && i + r < outs) {
          sums[i + r] = sv;
          if (kPair) sums[g.pair + i + r] = sw;
        }
      }
    }
#pragma unroll
    for (int part = 0; part < (kDz && sizeof(T) == 2 ? 2 : 1); ++part) {
      if (part && !g.low) break;
      if (part) {
        rounded_off<T, 4>(v);
        rounded_off<T, 4>(w);
        out += g.low;
      }
#pragma unroll
      for (int r = 0; r < 4; ++r)
        if (ok[r]) {
          out[i + r] = narrow<T>(v[r]);
          if (MODE == kGatedDz) out[g.pair + i + r] = narrow<T>(w[r]);
        }
    }
  }
}

template <typename T, int FR, int JB>
static hipError_t launch_few(const ProductArgs& g, hipStream_t stream) {
  const int outs = g.mode == kGated || g.mode == kGatedDz ? g.pair : g.I;
  const unsigned blocks = (unsigned)((outs + 16 * FR - 1) / (16 * FR));
#define FEW(MODE) few_tokens<T, FR, JB, MODE><<<blocks, kFewWaves * 64, 0, stream>>>(g)
  switch (g.mode) {
    case kLinear: FEW(kLinear); break;
    case kLinearDz: FEW(kLinearDz); break;
    case kGated: FEW(kGated); break;
    case kGatedDz: FEW(kGatedDz); break;
    default: return hipErrorInvalidValue;
  }
#undef FEW
  return hipGetLastError();
}

template <typename T, int BI, int BJ, int NWI, int NWJ, int PASSES, int STAGES, bool AKC, bool BKC,
          int MODE, bool DIRECT>
static hipError_t launch(ProductArgs g, hipStream_t stream) {
  constexpr bool kPair = MODE == kGated || MODE == kGatedDz, CI = AKC && BKC;
  const long long pairs = (g.pair + 15) / 16 * 32;
  g.tiles_i = (int)(((kPair && CI ? pairs : g.I) + BI - 1) / BI);
  g.tiles_j = (int)(((kPair && !CI ? pairs : g.J) + BJ - 1) / BJ);
  const long long blocks =
      (long long)g.tiles_i * g.tiles_j * (g.mode == kPartial ? g.splits : g.batches);
  if (blocks > 0x7fffffffLL) return hipErrorInvalidConfiguration;
  product<T, BI, BJ, NWI, NWJ, PASSES, STAGES, AKC, BKC, MODE, DIRECT>
      <<<grid_of(blocks), NWI * NWJ * 64, 0, stream>>>(g);
  return hipGetLastError();
}

// the combinations of operands and epilogues that the calls use
template <typename T, int BI, int BJ, int NWI, int NWJ, int PASSES, int STAGES, bool DIRECT>
static hipError_t by_operands(const ProductArgs& g, hipStream_t stream) {
#define PRODUCT(AKC, BKC, MODE) \
  return launch<T, BI, BJ, NWI, NWJ, PASSES, STAGES, AKC, BKC, MODE, DIRECT>(g, stream)
  if (g.a_k && g.b_k) switch (g.mode) {
      case kLinear: PRODUCT(true, true, kLinear);
      case kLinearDz: PRODUCT(true, true, kLinearDz);
      case kGated: PRODUCT(true, true, kGated);
      case kGatedDz: PRODUCT(true, true, kGatedDz);
      case kPartial: PRODUCT(true, true, kPartial);
    }
  else if (g.b_k) switch (g.mode) {
      case kLinear: PRODUCT(false, true, kLinear);
      case kLinearDz: PRODUCT(false, true, kLinearDz);
      case kGated: PRODUCT(false, true, kGated);
      case kGatedDz: PRODUCT(false, true, kGatedDz);
      case kPartial: PRODUCT(false, true, kPartial);
    }
  else switch (g.mode) {
      case kPlain: PRODUCT(false, false, kPlain);
      case kPartial: PRODUCT(false, false, kPartial);
    }
#undef PRODUCT
  return hipErrorInvalidValue;
}

template <typename T>
hipError_t product_t(const ProductArgs& g, const ProductPlan& p, hipStream_t stream) {
  switch (p.kernel) {
    case kFew16: return launch_few<T, 1, 1>(g, stream);
    case kFew32: return launch_few<T, 1, 2>(g, stream);
    case kFew64: return launch_few<T, 1, 4>(g, stream);
    case kTile64: return by_operands<T, 64, 64, 2, 2, 1, 2, true>(g, stream);
    case kTile64Deep:
      if constexpr (sizeof(T) == 2) return by_operands<T, 64, 64, 2, 2, 1, 3, true>(g, stream);
      break;
    case kTile64Any: return by_operands<T, 64, 64, 2, 2, 1, 2, false>(g, stream);
    case kTile128: return by_operands<T, 128, 128, 2, 2, 1, 2, true>(g, stream);
    case kTile256:
      if constexpr (sizeof(T) == 2) return by_operands<T, 256, 256, 2, 2, 2, 2, true>(g, stream);
  }
  return hipErrorInvalidValue;
}

}  // namespace feat
}  // namespace pwc
