// Optimizer updates as single streaming kernels over flat fp32 arrays: Adam / AdamW and
// SGD.  The reference builds each update from a chain of elementwise ops
// (mograd/nn/optim/adam.mojo:6-78, sgd.mojo:24-45); the arithmetic and its order are the
// same here, in one pass: 28 bytes moved per parameter for Adam, 12 for SGD.
#include "mg_device.h"
#include <cmath>

#include "mg_internal.h"

// No fused multiply-add contraction in this file: each operation of an update is rounded
// on its own, in the order the reference's chain of elementwise kernels applies them, so an
// fp32 emulation of that chain gives the same bits.
#pragma clang fp contract(off)

namespace mg {

struct AdamParams {
  float lr, beta1, beta2, eps, weight_decay;
  float one_minus_beta1, one_minus_beta2;
  float inv_bc1, inv_bc2;  // 1 / (1 - beta^t)
  float decay;             // 1 - lr * weight_decay
  int decoupled;
};

// Plain operators: compiled under the pragma above they carry no permission to contract
// (the header's __fmul_rn/__fadd_rn wrappers are compiled without it and would fuse).
__device__ __forceinline__ float mul_rn(float a, float b) { return a * b; }
__device__ __forceinline__ float add_rn(float a, float b) { return a + b; }
__device__ __forceinline__ float sub_rn(float a, float b) { return a - b; }

__device__ __forceinline__ void adam_one(float& w, float g, float& m, float& v, const AdamParams& p) {
  if (!p.decoupled && p.weight_decay > 0.f) g = add_rn(g, mul_rn(w, p.weight_decay));
  m = add_rn(mul_rn(m, p.beta1), mul_rn(g, p.one_minus_beta1));
  v = add_rn(mul_rn(v, p.beta2), mul_rn(mul_rn(g, g), p.one_minus_beta2));
  const float m_hat = mul_rn(m, p.inv_bc1);
  const float v_hat = mul_rn(v, p.inv_bc2);
  const float update = mul_rn(__fdiv_rn(m_hat, add_rn(__fsqrt_rn(v_hat), p.eps)), p.lr);
  const float base = (p.decoupled && p.weight_decay > 0.f) ? mul_rn(w, p.decay) : w;
  w = sub_rn(base, update);
}

// CLIP: the gradients are scaled on their way in (clip_scale); `norm` is their global norm.
template <bool CLIP>
__global__ __launch_bounds__(256) void adam_kernel(float* __restrict__ w, const float* __restrict__ g,
                                                   float* __restrict__ m, float* __restrict__ v, int64_t n,
                                                   AdamParams p, const float* __restrict__ norm, float max_norm) {
  const float scale = CLIP ? clip_scale(*norm, max_norm) : 1.f;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * 256 * 4;
  for (int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4; i < n; i += stride) {
    if (i + 4 <= n) {
      float4 w4 = *reinterpret_cast<const float4*>(w + i);
      float4 g4 = *reinterpret_cast<const float4*>(g + i);
      if constexpr (CLIP) g4 = make_float4(mul_rn(g4.x, scale), mul_rn(g4.y, scale), mul_rn(g4.z, scale), mul_rn(g4.w, scale));
      float4 m4 = *reinterpret_cast<const float4*>(m + i);
      float4 v4 = *reinterpret_cast<const float4*>(v + i);
      adam_one(w4.x, g4.x, m4.x, v4.x, p);
      adam_one(w4.y, g4.y, m4.y, v4.y, p);
      adam_one(w4.z, g4.z, m4.z, v4.z, p);
      adam_one(w4.w, g4.w, m4.w, v4.w, p);
      *reinterpret_cast<float4*>(w + i) = w4;
      *reinterpret_cast<float4*>(m + i) = m4;
      *reinterpret_cast<float4*>(v + i) = v4;
    } else {
      for (int64_t j = i; j < n; ++j) adam_one(w[j], CLIP ? mul_rn(g[j], scale) : g[j], m[j], v[j], p);
    }
  }
}

template <bool CLIP>
__global__ __launch_bounds__(256) void sgd_kernel(float* __restrict__ w, const float* __restrict__ g, int64_t n,
                                                  float lr, const float* __restrict__ norm, float max_norm) {
  const float scale = CLIP ? clip_scale(*norm, max_norm) : 1.f;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * 256 * 4;
  for (int64_t i = (static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x) * 4; i < n; i += stride) {
    if (i + 4 <= n) {
      float4 w4 = *reinterpret_cast<const float4*>(w + i);
      float4 g4 = *reinterpret_cast<const float4*>(g + i);
      if constexpr (CLIP) g4 = make_float4(mul_rn(g4.x, scale), mul_rn(g4.y, scale), mul_rn(g4.z, scale), mul_rn(g4.w, scale));
      w4.x = sub_rn(w4.x, mul_rn(g4.x, lr));
      w4.y = sub_rn(w4.y, mul_rn(g4.y, lr));
      w4.z = sub_rn(w4.z, mul_rn(g4.z, lr));
      w4.w = sub_rn(w4.w, mul_rn(g4.w, lr));
      *reinterpret_cast<float4*>(w + i) = w4;
    } else {
      for (int64_t j = i; j < n; ++j) w[j] = sub_rn(w[j], mul_rn(CLIP ? mul_rn(g[j], scale) : g[j], lr));
    }
  }
}

static unsigned optim_blocks(int64_t n) {
  int64_t blocks = ceil_div(n, 1024);
  const int64_t cap = static_cast<int64_t>(device_info().cu_count) * 16;
  if (blocks > cap) blocks = cap;
  return static_cast<unsigned>(blocks < 1 ? 1 : blocks);
}

static int adam_step(const char* who, void* w, const void* g, void* m, void* v, int64_t n, float lr, float beta1, float beta2, float eps,
                     float weight_decay, int64_t t, int decoupled_weight_decay, const float* norm, float max_norm, mg_stream stream) {
  if (n < 0) return fail(MG_ERR_INVALID, "%s: negative size", who);
  if (t < 1) return fail(MG_ERR_INVALID, "%s: step count t=%lld must be >= 1", who, static_cast<long long>(t));
  if (n == 0) return MG_OK;
  if (!w || !g || !m || !v) return fail(MG_ERR_INVALID, "%s: null pointer argument", who);
  if (!aligned16(w) || !aligned16(g) || !aligned16(m) || !aligned16(v))
    return fail(MG_ERR_INVALID, "%s: pointers must be 16-byte aligned", who);
  // Bias corrections `Float32(1.0) - beta**t` (mograd/nn/optim/adam.mojo:19-20).  The power is
  // taken in double and rounded to fp32 once: constant time in t, and within one fp32 rounding
  // of the exact value however large the step count (a chain of t fp32 multiplications costs
  // O(t) host time per call and drifts by up to t/2 ulp).
  const float b1t = static_cast<float>(std::pow(static_cast<double>(beta1), static_cast<double>(t)));
  const float b2t = static_cast<float>(std::pow(static_cast<double>(beta2), static_cast<double>(t)));
  AdamParams p{lr,
               beta1,
               beta2,
               eps,
               weight_decay,
               1.0f - beta1,
               1.0f - beta2,
               1.0f / (1.0f - b1t),
               1.0f / (1.0f - b2t),
               1.0f - lr * weight_decay,
               decoupled_weight_decay != 0};
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(optim_blocks(n)), dim3(256), 0, to_stream(stream), static_cast<float*>(w),
                       static_cast<const float*>(g), static_cast<float*>(m), static_cast<float*>(v), n, p, norm, max_norm);
  };
  if (norm) launch(adam_kernel<true>);
  else launch(adam_kernel<false>);
  MG_LAUNCH_CHECK();
  return MG_OK;
}

static int sgd_step(const char* who, void* w, const void* g, int64_t n, float lr, const float* norm, float max_norm, mg_stream stream) {
  if (n < 0) return fail(MG_ERR_INVALID, "%s: negative size", who);
  if (n == 0) return MG_OK;
  if (!w || !g) return fail(MG_ERR_INVALID, "%s: null pointer argument", who);
  if (!aligned16(w) || !aligned16(g)) return fail(MG_ERR_INVALID, "%s: pointers must be 16-byte aligned", who);
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(optim_blocks(n)), dim3(256), 0, to_stream(stream), static_cast<float*>(w),
                       static_cast<const float*>(g), n, lr, norm, max_norm);
  };
  if (norm) launch(sgd_kernel<true>);
  else launch(sgd_kernel<false>);
  MG_LAUNCH_CHECK();
  return MG_OK;
}

static int clip_check(const char* who, const float* norm, float max_norm) {
  if (!norm) return fail(MG_ERR_INVALID, "%s: null pointer argument", who);
  if (!(max_norm >= 0.f)) return fail(MG_ERR_INVALID, "%s: max_norm=%g", who, static_cast<double>(max_norm));
  return MG_OK;
}

}  // namespace mg

extern "C" {

int mg_adam_step(void* w, const void* g, void* m, void* v, int64_t n, float lr, float beta1, float beta2, float eps,
                 float weight_decay, int64_t t, int decoupled_weight_decay, mg_stream stream) {
  return mg::adam_step("adam_step", w, g, m, v, n, lr, beta1, beta2, eps, weight_decay, t, decoupled_weight_decay, nullptr, 0.f, stream);
}

int mg_adam_step_clipped(void* w, const void* g, void* m, void* v, int64_t n, float lr, float beta1, float beta2, float eps,
                         float weight_decay, int64_t t, int decoupled_weight_decay, const float* norm, float max_norm, mg_stream stream) {
  const char* const who = "adam_step_clipped";
  MG_TRY(mg::clip_check(who, norm, max_norm));
  return mg::adam_step(who, w, g, m, v, n, lr, beta1, beta2, eps, weight_decay, t, decoupled_weight_decay, norm, max_norm, stream);
}

int mg_sgd_step(void* w, const void* g, int64_t n, float lr, mg_stream stream) {
  return mg::sgd_step("sgd_step", w, g, n, lr, nullptr, 0.f, stream);
}

int mg_sgd_step_clipped(void* w, const void* g, int64_t n, float lr, const float* norm, float max_norm, mg_stream stream) {
  const char* const who = "sgd_step_clipped";
  MG_TRY(mg::clip_check(who, norm, max_norm));
  return mg::sgd_step(who, w, g, n, lr, norm, max_norm, stream);
}

}  // extern "C"
