// Top-k of one token's expert logits by one warp, the logits held in registers: shared by the
// stand-alone router and the few-token layer, which therefore route alike to the last bit.
#pragma once

#include <float.h>

#include "common.cuh"

namespace bolt {

constexpr int kMaxPerLane = 32;  // experts per lane -> up to 1024 experts

// v[j]: this lane's logit of expert lane + 32 j.  Lane k < topk ends up with the k-th choice.
template <int NPL>
__device__ __forceinline__ void topk_of_row(float (&v)[NPL], int experts, int topk, int renormalize,
                                            int softmax, int lane, float& my_w, int& my_id) {
  const int per_lane = (experts + 31) / 32;
  float mx = -FLT_MAX;
#pragma unroll
  for (int j = 0; j < NPL; ++j) {
    const int e = lane + 32 * j;
    if (j >= per_lane || e >= experts) v[j] = -FLT_MAX;
    mx = fmaxf(mx, v[j]);
  }
  if (softmax) {
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
      const int e = lane + 32 * j;
      if (j < per_lane && e < experts) {
        v[j] = expf(v[j] - mx);
        sum += v[j];
      } else {
        v[j] = -3.f;  // never offered
      }
    }
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float inv = 1.0f / sum;
#pragma unroll
    for (int j = 0; j < NPL; ++j)
      if (v[j] >= 0.f) v[j] *= inv;
  } else {
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
      const int e = lane + 32 * j;
      v[j] = (j < per_lane && e < experts) ? 1.0f / (1.0f + expf(-v[j])) : -3.f;
    }
  }
  // top-k by repeated warp arg-max (ties: lowest expert index)
  my_w = 0.f;
  my_id = 0;
  int past_end = 0;
  float total = 0.f;
  for (int k = 0; k < topk; ++k) {
    float best = -2.f;
    int best_e = 0x7fffffff;
#pragma unroll
    for (int j = 0; j < NPL; ++j) {
      const int e = lane + 32 * j;
      if (v[j] > best) { best = v[j]; best_e = e; }
    }
    // (scores are not negative, and a lane that holds none offers -2: their bit patterns order
    // like the values as signed integers)
    const int top = __reduce_max_sync(0xffffffffu, __float_as_int(best));
    best_e = __reduce_min_sync(0xffffffffu, __float_as_int(best) == top ? best_e : 0x7fffffff);
    best = __int_as_float(top);
    if (top < 0) {   // all that is left is NaN: ids past the last expert, which the sort drops
      best_e = experts + past_end++;
      if (best_e < 32 * kMaxPerLane) best = -1.f;
      else best_e = 0x7fffffff;
    }
    if ((best_e & 31) == lane) {
#pragma unroll
      for (int j = 0; j < NPL; ++j)
        if (lane + 32 * j == best_e) v[j] = -3.f;  // taken
    }
    if (lane == k) { my_w = best; my_id = best_e; }
    total += best;
  }
  if (renormalize) my_w = my_w / total;
}

}  // namespace bolt
