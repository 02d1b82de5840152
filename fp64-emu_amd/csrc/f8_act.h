// Activations of one matrix (those of a product's epilogue), and their slopes, in float32.
#pragma once
#include "f8_common.h"

namespace {

[[maybe_unused]] inline bool known_act(int a) { return a >= FP64EMU_ACT_NONE && a <= FP64EMU_ACT_GELU_TANH; }

// Calls fn with `act` as a constant.  On the device `act` is the same for all lanes; a loop
// that is inside of fn does not branch by it.
template <class Fn>
__host__ __device__ __forceinline__ void with_act(int act, const Fn& fn) {
  switch (act) {
    case FP64EMU_ACT_RELU: fn(std::integral_constant<int, FP64EMU_ACT_RELU>{}); break;
    case FP64EMU_ACT_RELU2: fn(std::integral_constant<int, FP64EMU_ACT_RELU2>{}); break;
    case FP64EMU_ACT_SILU: fn(std::integral_constant<int, FP64EMU_ACT_SILU>{}); break;
    case FP64EMU_ACT_GELU: fn(std::integral_constant<int, FP64EMU_ACT_GELU>{}); break;
    case FP64EMU_ACT_GELU_TANH: fn(std::integral_constant<int, FP64EMU_ACT_GELU_TANH>{}); break;
    default: fn(std::integral_constant<int, FP64EMU_ACT_NONE>{}); break;
  }
}

// 2 sqrt(2 / pi) (1, 0.044715): gelu_tanh(h) = h sigmoid(h (kTanh1 + kTanh3 h^2)), since
// (1 + tanh u) / 2 is sigmoid(2 u).
constexpr float kTanh1 = 1.59576912f, kTanh3 = 0.0713548163f;

// kFine: float32 accuracy over the whole range.  Without it 2^t is taken of t rounded once, off by |g| 1.25
// 2^-24 of itself more: 2^-17 where an activation's tail ends, nothing beside the rounding of
// 16-bit values, and 5 instructions instead of 11 (8192^3 with silu: 7 us less).  So products to 16 bits on tiles
// without splits take it; few rows and sums of parts, where it would save nothing, and all float32 outputs do not.
template <bool kFine>
__device__ __forceinline__ float sigmoid_of(float g) {
  if constexpr (kFine) return sigmoid(g);
  return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(g * -1.44269502f));
}

// e^(-h^2 / 2); kFine: with the roundings of h^2 and of its product with log2(e) / 2 carried into the result.
template <bool kFine>
__device__ __forceinline__ float bell(float h) {
  constexpr float kL = 0.721347511f, kLlo = 9.62981517e-9f;    // log2(e) / 2 = kL + kLlo
  const float s = h * h, t = -s * kL;
  float e = __builtin_amdgcn_exp2f(t);
  if constexpr (kFine) {
    const float lo = fmaf(-s, kL, -t) - fmaf(fmaf(h, h, -s), kL, s * kLlo);
    if (t > -126.0f) e = fmaf(e, lo * 0.693147182f, e);        // (past that inf - inf)
  }
  return e;
}

// The normal distribution function Phi(h), from the bell at h: with x = |h| and t = 1 / (1 + 0.28 x),
// Phi(-x) = bell(x) t P(t).  P is a least-squares fit over 0 .. 200, reweighted until its largest
// relative error was least: 1.3e-7, and 4.6e-7 with its float32 arithmetic.  (The library's erfcf
// branches by lanes: 8192^3 with gelu took 52 us more.)
__device__ __forceinline__ float normal_cdf(float h, float bell) {
  const float t = __builtin_amdgcn_rcpf(fmaf(0.28f, fabsf(h), 1.0f));
  float p = 0.025377780f;
  p = fmaf(p, t, -0.0961872190f);
  p = fmaf(p, t, 0.0966112316f);
  p = fmaf(p, t, -0.0100027369f);
  p = fmaf(p, t, 0.0744824708f);
  p = fmaf(p, t, 0.0831677988f);
  p = fmaf(p, t, 0.103151247f);
  p = fmaf(p, t, 0.111695431f);
  p = fmaf(p, t, 0.111703947f);
  const float q = bell * (t * p);
  return h > 0.0f ? 1.0f - q : q;
}

// NaN stays NaN.
template <int kAct, bool kFine>
__device__ __forceinline__ float activated(float h) {
  if constexpr (kAct == FP64EMU_ACT_RELU) return h < 0.0f ? 0.0f : h;
  if constexpr (kAct == FP64EMU_ACT_RELU2) return h < 0.0f ? 0.0f : h * h;
  if constexpr (kAct == FP64EMU_ACT_SILU) return h * sigmoid_of<kFine>(h);
  if constexpr (kAct == FP64EMU_ACT_GELU) return h * normal_cdf(h, bell<kFine>(h));
  if constexpr (kAct == FP64EMU_ACT_GELU_TANH) return h * sigmoid_of<kFine>(h * fmaf(kTanh3 * h, h, kTanh1));
  return h;
}

// sigmoid(g) and 1 - sigmoid(g), the second as e^-g times the first where that nears 1: taken from 1 it would keep nothing of
// itself there, and gelu_tanh multiplies it by up to 500 (h from 4 to 8: its slope was off by up to 32 2^-24, now by 2).  Below
// that 1 - s is the nearer one: its error and s's go against each other.
struct Logistic { float s, rest; };
// (|g| below 2^23: e^-g is as sigmoid() has it, but what its argument's rounding was goes in as a factor, which stays positive
// up to there and which an infinite 2^t stands.)
__device__ __forceinline__ Logistic logistic(float g) {
  constexpr float kL = 1.44269502f, kLlo = 1.92596303e-8f;
  const float t = -g * kL, lo = fmaf(-g, kLlo, fmaf(-g, kL, -t));
  const float e = __builtin_amdgcn_exp2f(t) * fmaf(lo, 0.693147182f, 1.0f);
  const float s = __builtin_amdgcn_rcpf(1.0f + e);
  return {s, g > 2.0f ? e * s : 1.0f - s};
}

// d times the slope at h, to float32 accuracy whatever the operands' type: the bias's gradient and the 8-bit forms come
// from float32 values.
template <int kAct>
__device__ __forceinline__ float activated_back(float h, float d) {
  if constexpr (kAct == FP64EMU_ACT_RELU) return h > 0.0f ? d : 0.0f;
  if constexpr (kAct == FP64EMU_ACT_RELU2) return d * (2.0f * (h < 0.0f ? 0.0f : h));
  if constexpr (kAct == FP64EMU_ACT_SILU) {
    const Logistic l = logistic(__builtin_amdgcn_fmed3f(h, -1000.0f, 1000.0f));
    return d * (l.s * fmaf(h, l.rest, 1.0f));
  }
  if constexpr (kAct == FP64EMU_ACT_GELU) {
    const float e = bell<true>(h);
    return d * fmaf(h * 0.398942280f, e, normal_cdf(h, e));
  }
  if constexpr (kAct == FP64EMU_ACT_GELU_TANH) {
    // (s (1 - s) is zero long before the clamp, which keeps its factor finite; h itself brings a NaN along.)
    const float c = __builtin_amdgcn_fmed3f(h, -100.0f, 100.0f);
    const float q = c * c;
    const Logistic l = logistic(c * fmaf(kTanh3, q, kTanh1));
    return d * fmaf(h * (l.s * l.rest), fmaf(3.0f * kTanh3, q, kTanh1), l.s);
  }
  return d;
}

}  // namespace
