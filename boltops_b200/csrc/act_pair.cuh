// The expert activations of one (gate, up) pair in fp32: the stand-alone kernels and the few-token
// layer's epilogue.
#pragma once

#include "common.cuh"

namespace bolt {

struct ActParams {
  int kind;
  int gated;
  float alpha;
  float limit;
};

__device__ __forceinline__ float gelu_erf(float x) {
  return x * 0.5f * (1.0f + erff(x * 0.7071067811865476f));
}
__device__ __forceinline__ float gelu_tanh(float x) {
  const float k = 0.7978845608028654f;  // sqrt(2/pi)
  return 0.5f * x * (1.0f + tanhf(k * (x + 0.044715f * x * x * x)));
}

// fp32 activation of one (gate, up) pair; `u` is ignored when not gated.
__device__ __forceinline__ float act_pair(const ActParams& p, float g, float u) {
  float a;
  switch (p.kind) {
    case BOLT_ACT_SILU: a = silu_f32(g); break;
    case BOLT_ACT_GELU: a = gelu_erf(g); break;
    case BOLT_ACT_GELU_TANH: a = gelu_tanh(g); break;
    case BOLT_ACT_RELU2: a = g > 0.f ? g * g : 0.f; break;
    case BOLT_ACT_SWIGLU_OAI: {
      const float gc = fminf(g, p.limit);
      const float uc = fminf(fmaxf(u, -p.limit), p.limit);
      return gc * (1.0f / (1.0f + expf(-p.alpha * gc))) * (uc + 1.0f);
    }
    case BOLT_ACT_SWIGLU_STEP:
      a = fminf(silu_f32(g), p.limit);
      u = fminf(fmaxf(u, -p.limit), p.limit);
      break;
    case BOLT_ACT_SILU_CLAMP:
      a = silu_f32(fminf(g, p.limit));
      u = fminf(fmaxf(u, -p.limit), p.limit);
      break;
    case BOLT_ACT_SWIGLU_OAI_INTERLEAVED: {
      const float gc = fminf(g, p.limit);
      const float uc = fminf(fmaxf(u, -p.limit), p.limit);
      return gc * (1.0f / (1.0f + expf(-p.alpha * gc))) * (uc + 1.0f);
    }
    case BOLT_ACT_SITU: {
      // tanh(x) = 2*sigmoid(2x) - 1, the reference's form
      const float tg = 2.0f / (1.0f + expf(-2.0f * (g / p.alpha))) - 1.0f;
      a = p.alpha * tg * (1.0f / (1.0f + expf(-g)));
      if (p.limit > 0.f) u = p.limit * (2.0f / (1.0f + expf(-2.0f * (u / p.limit))) - 1.0f);
      break;
    }
    default: a = g; break;
  }
  return p.gated ? a * u : a;
}

}  // namespace bolt
