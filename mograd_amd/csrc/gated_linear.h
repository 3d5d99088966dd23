// A gated Linear layer: g = x Wg^T + bg, u = x Wu^T + bu, y = act(g) u, with W = [Wg; Wu] one (2 F, K) array and b = [bg; bu].
//
// Gradients, from dy and the kept g and u:
//   dg = dy u act'(g),  du = dy act(g);   dx = [dg du] W,  dW = [dg du]^T x,  db = column sums of [dg du]
#pragma once

#include "gemm_impl.h"

namespace mg {

// A product's arguments: B the weights, N the columns F of y, C y (M, F) without gaps.
template <typename T>
struct GatedProblem : Gemm16Problem<T> {
  T* gu = nullptr;  // (M, 2 F): g and u, rounded; may be null
  int gate = 0;
};

// Calls f with `gate` (an mg_gate) as a compile-time number.
template <typename F>
__host__ __device__ __forceinline__ void gated_with(int gate, F&& f) {
  switch (gate) {
    case MG_GATE_SILU: return f(std::integral_constant<int, MG_GATE_SILU>{});
    case MG_GATE_GELU: return f(std::integral_constant<int, MG_GATE_GELU>{});
    case MG_GATE_GELU_TANH: return f(std::integral_constant<int, MG_GATE_GELU_TANH>{});
    case MG_GATE_SIGMOID: return f(std::integral_constant<int, MG_GATE_SIGMOID>{});
    default: return f(std::integral_constant<int, MG_GATE_RELU>{});
  }
}

// s = 1 / (1 + e^-z) and t = 1 - s, either to a few units in its own last place: from e^-|z|, which neither overflows nor leaves
// anything to cancel.  FAST: e^z as 2^(z log2 e) with the hardware's exponential and reciprocal, |z| 2^-24 and 2^-23 off, which
// 16 bits do not see, and 0 below 2^-126; fp32 takes the exact ones.
template <bool FAST>
__device__ __forceinline__ void gated_sigmoid(float z, float& s, float& t) {
  float e, r;
  if constexpr (FAST) {
    e = __builtin_amdgcn_exp2f(-1.44269504f * fabsf(z));
    r = __builtin_amdgcn_rcpf(1.f + e);
  } else {
    e = expf(-fabsf(z));
    r = 1.f / (1.f + e);
  }
  const float small = e * r;
  s = z >= 0.f ? r : small;
  t = z >= 0.f ? small : r;
  if (z != z) s = t = z;
}

// The normal distribution's Phi(g), through erfc, whose tail keeps its digits.  FAST: erfc(x) = t P(t) e^(-x^2), t = 1 / (1 + x / 2), with P
// of degree 6 fitted to e^(x^2) erfc(x) / t over 0 <= x <= 9.3 for the least relative error: 1.4e-6 in fp32, which 16 bits do not see.
template <bool FAST>
__device__ __forceinline__ float gated_phi(float g) {
  if constexpr (!FAST) return 0.5f * erfcf(-0.70710678f * g);
  const float t = __builtin_amdgcn_rcpf(fmaf(0.35355339f, fabsf(g), 1.f));
  const float p = fmaf(fmaf(fmaf(fmaf(fmaf(fmaf(0.0895019994f, t, -0.361318171f), t, 0.395655721f), t, 0.033319734f), t, 0.283226967f), t, 0.277257442f), t, 0.282355189f);
  const float tail = 0.5f * t * p * __builtin_amdgcn_exp2f(-0.72134752f * g * g);
  return g > 0.f ? 1.f - tail : tail;
}

constexpr float kGeluTanh2C = 1.59576912f;  // 2 sqrt(2 / pi): 1/2 (1 + tanh(c v)) = sigmoid(2 c v)

// act(g)
template <bool FAST, int GATE>
__device__ __forceinline__ float gated_act(float g) {
  if constexpr (GATE == MG_GATE_RELU) return g > 0.f ? g : g != g ? g : 0.f;
  else if constexpr (GATE == MG_GATE_GELU) return g * gated_phi<FAST>(g);
  else {
    float s, t;
    gated_sigmoid<FAST>(GATE == MG_GATE_GELU_TANH ? kGeluTanh2C * g * (1.f + 0.044715f * g * g) : g, s, t);
    return GATE == MG_GATE_SIGMOID ? s : g * s;
  }
}

// act(g) and act'(g)
template <bool FAST, int GATE>
__device__ __forceinline__ void gated_act_slope(float g, float& act, float& slope) {
  if constexpr (GATE == MG_GATE_RELU) {
    act = gated_act<FAST, GATE>(g);
    slope = g > 0.f ? 1.f : g != g ? g : 0.f;
  } else if constexpr (GATE == MG_GATE_GELU) {
    const float phi = gated_phi<FAST>(g);
    act = g * phi;
    slope = phi + g * 0.39894228f * (FAST ? __builtin_amdgcn_exp2f(-0.72134752f * g * g) : expf(-0.5f * g * g));
  } else {
    float s, t;
    gated_sigmoid<FAST>(GATE == MG_GATE_GELU_TANH ? kGeluTanh2C * g * (1.f + 0.044715f * g * g) : g, s, t);
    const float st = s * t;
    if constexpr (GATE == MG_GATE_SIGMOID) act = s, slope = st;
    else if constexpr (GATE == MG_GATE_SILU) act = g * s, slope = s + g * st;
    else act = g * s, slope = s + g * st * kGeluTanh2C * (1.f + 0.134145f * fminf(g * g, 1e30f));  // (st is zero by then)
  }
}

// Calls f with act as a function for 16-bit outputs.  The three gates made of a sigmoid share their code, s times g or 1 with s the
// sigmoid of g (c1 + c3 g^2), so that a kernel's epilogue has three copies of its loops and not five.  (g or 1 is a choice and no sum
// a0 + a1 g: 0 g is NaN for an infinite g, where the sigmoid is 1 or 0.)
template <typename F>
__device__ __forceinline__ void gated_with_fast(int gate, F&& f) {
  if (gate == MG_GATE_RELU) return f([](float g) { return gated_act<true, MG_GATE_RELU>(g); });
  if (gate == MG_GATE_GELU) return f([](float g) { return gated_act<true, MG_GATE_GELU>(g); });
  const bool tanh = gate == MG_GATE_GELU_TANH, plain = gate == MG_GATE_SIGMOID;
  const float c1 = -1.44269504f * (tanh ? kGeluTanh2C : 1.f), c3 = tanh ? -1.44269504f * 0.044715f * kGeluTanh2C : 0.f;
  f([=](float g) {
    const float e = __builtin_amdgcn_exp2f(g * fmaf(c3, fminf(g * g, 1e30f), c1));
    return __builtin_amdgcn_rcpf(1.f + e) * (plain ? 1.f : g);
  });
}

// gemm_deep_*.hip: the products and y in one launch, operands on 16-byte chunks, `tile` kTile128 or kTile256 (64 and 128 columns of y).
template <typename T>
int launch_gated_deep(const GatedProblem<T>& pr, Gemm16Tile tile, hipStream_t stream);

}  // namespace mg
