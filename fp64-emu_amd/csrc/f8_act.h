// Activations of one matrix (those of a product's epilogue), and their slopes, in float32.
#pragma once
#include "f8_common.h"

namespace {

[[maybe_unused]] inline bool known_act(int a) { return a >= FP64EMU_ACT_NONE && a <= FP64EMU_ACT_GELU_TANH; }

// 2 sqrt(2 / pi) (1, 0.044715): gelu_tanh(h) = h sigmoid(h (kTanh1 + kTanh3 h^2)), since
// (1 + tanh u) / 2 is sigmoid(2 u).
constexpr float kTanh1 = 1.59576912f, kTanh3 = 0.0713548163f;
constexpr float kRoot = 0.707106781f;                          // sqrt(1 / 2)

// Of kN values; `act` is the same for all lanes.  NaN stays NaN.
template <int kN>
__device__ __forceinline__ void activate(int act, float (&v)[kN]) {
#pragma unroll
  for (int j = 0; j < kN; ++j) {
    const float h = v[j];
    switch (act) {
      case FP64EMU_ACT_RELU: v[j] = h < 0.0f ? 0.0f : h; break;
      case FP64EMU_ACT_RELU2: v[j] = h < 0.0f ? 0.0f : h * h; break;
      case FP64EMU_ACT_SILU: v[j] = h * sigmoid(h); break;
      case FP64EMU_ACT_GELU: v[j] = 0.5f * h * erfcf(-h * kRoot); break;
      case FP64EMU_ACT_GELU_TANH: v[j] = h * sigmoid(h * fmaf(kTanh3 * h, h, kTanh1)); break;
      default: break;
    }
  }
}

// d[j] times the slope at h[j].
template <int kN>
__device__ __forceinline__ void activate_back(int act, const float (&h)[kN], float (&d)[kN]) {
#pragma unroll
  for (int j = 0; j < kN; ++j) {
    const float x = h[j];
    switch (act) {
      case FP64EMU_ACT_RELU: d[j] = x > 0.0f ? d[j] : 0.0f; break;
      case FP64EMU_ACT_RELU2: d[j] *= 2.0f * (x < 0.0f ? 0.0f : x); break;
      case FP64EMU_ACT_SILU: {
        const float s = sigmoid(x);
        d[j] *= s * fmaf(x, 1.0f - s, 1.0f);
        break;
      }
      case FP64EMU_ACT_GELU:
        d[j] *= fmaf(x * 0.398942280f, expf(-0.5f * x * x), 0.5f * erfcf(-x * kRoot));
        break;
      case FP64EMU_ACT_GELU_TANH: {
        // (s (1 - s) is zero long before the clamp, which keeps its factor finite.)
        const float c = __builtin_amdgcn_fmed3f(x, -100.0f, 100.0f);
        const float s = sigmoid(x * fmaf(kTanh3 * x, x, kTanh1));
        d[j] *= fmaf(x * (s * (1.0f - s)), fmaf(3.0f * kTanh3 * c, c, kTanh1), s);
        break;
      }
      default: break;
    }
  }
}

}  // namespace
