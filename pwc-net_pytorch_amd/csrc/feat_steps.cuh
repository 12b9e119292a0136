// feat_steps.cuh — the steps of k that one block of the product takes, in their order.
#pragma once

#ifdef __HIPCC__
#define PWC_STEPS_FN __host__ __device__ __forceinline__
#else
#define PWC_STEPS_FN inline
#endif

namespace pwc {
namespace feat {

// k runs over `segments` segments of K values (1 <= K < 2^31) in steps of KS.
struct Steps {
  int seg, k0;  // the step that comes next: values k0 .. of segment seg
  int left;     // steps still to come; loads run ahead of the sums, so it gets negative

  static PWC_STEPS_FN int of(int K, int KS) { return (K - 1) / KS + 1; }  // in a segment

  // part z of `splits`; the caller sees to segments * of(K, KS) < 2^31
  PWC_STEPS_FN void init(int segments, int K, int KS, int z, int splits) {
    const int each = of(K, KS), total = segments * each;
    const int first = (int)((long long)total * z / splits);
    left = (int)((long long)total * (z + 1) / splits) - first;
    seg = first / each;
    k0 = (first - seg * each) * KS;
  }
  // values of the segment from the step on: none past the end, whatever K is
  PWC_STEPS_FN int have(int K) const { return left > 0 ? K - k0 : 0; }
  PWC_STEPS_FN void next(int K, int KS) {
    --left;
    if (K - k0 <= KS) {
      k0 = 0;
      ++seg;
    } else {
      k0 += KS;
    }
  }
};

}  // namespace feat
}  // namespace pwc
