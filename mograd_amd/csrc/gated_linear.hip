// C ABI of the gated Linear layer: argument checks, the choice of kernels, the gradient of the gate.
#include "gated_linear.h"

#include "gemm_pad.h"
#include "mg_deferred.h"
#include "mg_rows.h"

namespace mg {

int gemm_dispatch(const char* who, const GemmArgs& g, hipStream_t stream);  // gemm.hip

constexpr int kGatedThreads = 256;
constexpr int64_t kGatedBlocks = 1 << 23;  // of a launch, which counts its threads in 32 bits

// y = act(g) u of kept projections; a thread takes VEC columns of one row.  Bound by its bytes.
template <typename T, int VEC, int GATE>
__global__ __launch_bounds__(kGatedThreads) void gate_fwd_kernel(const T* __restrict__ gu, T* __restrict__ y, int64_t items, int F,
                                                                uint32_t per_row, int64_t first_block) {
  const int64_t item = (first_block + blockIdx.x) * kGatedThreads + threadIdx.x;
  if (item >= items) return;
  const int64_t row = item / per_row;
  const int c = static_cast<int>(item - row * per_row) * VEC;
  float g[VEC], u[VEC];
  VecIO<T, VEC>::load(gu + row * 2 * F + c, g);
  VecIO<T, VEC>::load(gu + row * 2 * F + F + c, u);
#pragma unroll
  for (int i = 0; i < VEC; ++i) g[i] = gated_act<sizeof(T) == 2, GATE>(g[i]) * u[i];
  VecIO<T, VEC>::store(y + row * F + c, g);
}

// [dg du] from dy, g and u, rounded to the tensors' type as the products take it.  Bound by its bytes, five values an output.
template <typename T, int VEC, int GATE>
__global__ __launch_bounds__(kGatedThreads) void gate_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ gu, T* __restrict__ dgu,
                                                                int64_t items, int F, uint32_t per_row, int64_t first_block) {
  const int64_t item = (first_block + blockIdx.x) * kGatedThreads + threadIdx.x;
  if (item >= items) return;
  const int64_t row = item / per_row;
  const int c = static_cast<int>(item - row * per_row) * VEC;
  float d[VEC], g[VEC], u[VEC];
  VecIO<T, VEC>::load(dy + row * F + c, d);
  VecIO<T, VEC>::load(gu + row * 2 * F + c, g);
  VecIO<T, VEC>::load(gu + row * 2 * F + F + c, u);
#pragma unroll
  for (int i = 0; i < VEC; ++i) {
    float act, slope;
    gated_act_slope<sizeof(T) == 2, GATE>(g[i], act, slope);
    g[i] = d[i] * u[i] * slope;
    u[i] = d[i] * act;
  }
  VecIO<T, VEC>::store(dgu + row * 2 * F + c, g);
  VecIO<T, VEC>::store(dgu + row * 2 * F + F + c, u);
}

// Calls launch(VEC, gate, items, items of a row, first workgroup, workgroups) for M rows of F columns, in as many launches as it takes.
template <typename T, typename L>
static int gate_launch(int64_t M, int64_t F, int gate, bool aligned, L&& launch) {
  auto with = [&](auto vec) -> int {
    constexpr int VEC = decltype(vec)::value;
    const int64_t per_row = F / VEC, items = M * per_row, blocks = ceil_div(items, kGatedThreads);
    for (int64_t first = 0; first < blocks; first += kGatedBlocks) {
      const dim3 grid(static_cast<unsigned>(std::min(blocks - first, kGatedBlocks)));
      gated_with(gate, [&](auto g) { launch(vec, g, items, static_cast<uint32_t>(per_row), first, grid); });
      MG_LAUNCH_CHECK();
    }
    return MG_OK;
  };
  if (aligned && F % WideVec<T>::value == 0) return with(std::integral_constant<int, WideVec<T>::value>{});
  return with(std::integral_constant<int, 1>{});
}

template <typename T>
static int gate_fwd(const void* gu, void* y, int64_t M, int64_t F, int gate, hipStream_t stream) {
  return gate_launch<T>(M, F, gate, aligned16(gu) && aligned16(y), [&](auto vec, auto g, int64_t items, uint32_t per_row, int64_t first, dim3 grid) {
    hipLaunchKernelGGL((gate_fwd_kernel<T, decltype(vec)::value, decltype(g)::value>), grid, dim3(kGatedThreads), 0, stream,
                       static_cast<const T*>(gu), static_cast<T*>(y), items, static_cast<int>(F), per_row, first);
  });
}

template <typename T>
static int gate_bwd(const void* dy, const void* gu, void* dgu, int64_t M, int64_t F, int gate, hipStream_t stream) {
  return gate_launch<T>(M, F, gate, aligned16(dy) && aligned16(gu), [&](auto vec, auto g, int64_t items, uint32_t per_row, int64_t first, dim3 grid) {
    hipLaunchKernelGGL((gate_bwd_kernel<T, decltype(vec)::value, decltype(g)::value>), grid, dim3(kGatedThreads), 0, stream,
                       static_cast<const T*>(dy), static_cast<const T*>(gu), static_cast<T*>(dgu), items, static_cast<int>(F), per_row, first);
  });
}

// 16 bits: both projections and y in one launch; y comes from the projections before they are rounded.
template <typename T>
static int gated_fwd_16bit(const void* x, const void* w, const void* bias, void* y, void* gu, int64_t M, int64_t F, int64_t K, int gate,
                           hipStream_t stream) {
  int64_t ldx = K, ldw = K, no_batch = 0;
  PadCopies<T> pads;
  if (K % 8 != 0 || !aligned16(x)) MG_TRY(pads.add(&x, 1, M, K, &ldx, &no_batch));
  if (K % 8 != 0 || !aligned16(w)) MG_TRY(pads.add(&w, 1, 2 * F, K, &ldw, &no_batch));
  MG_TRY(pads.launch(stream));
  GatedProblem<T> pr{};
  pr.A = static_cast<const T*>(x), pr.B = static_cast<const T*>(w), pr.bias = static_cast<const T*>(bias), pr.C = static_cast<T*>(y);
  pr.M = static_cast<int>(M), pr.N = static_cast<int>(F), pr.K = static_cast<int>(ceil_div(K, 8) * 8);  // (zeros behind K in an image)
  pr.lda = ldx, pr.ldb = ldw, pr.ldc = F, pr.batches = pr.splits = 1, pr.k_per_split = pr.K;
  pr.gu = static_cast<T*>(gu), pr.gate = gate;
  const int64_t large = ceil_div(M, 256) * ceil_div(F, 128);
  return launch_gated_deep<T>(pr, 2 * large >= device_info().cu_count ? kTile256 : kTile128, stream);
}

static int gated_check(const char* who, int64_t M, int64_t F, int64_t K, int gate, int dtype) {
  if (!is_float_dtype(dtype)) return fail(MG_ERR_INVALID, "%s: unsupported dtype %s", who, dtype_name(dtype));
  if (gate < MG_GATE_SILU || gate > MG_GATE_RELU) return fail(MG_ERR_INVALID, "%s: no such gate: %d", who, gate);
  if (M < 0 || F <= 0 || K <= 0 || M > 0x7fffffffLL || F > 0x3fffffffLL || K > 0x7fffffffLL)
    return fail(MG_ERR_INVALID, "%s: bad shape M=%lld F=%lld K=%lld", who, static_cast<long long>(M), static_cast<long long>(F),
                static_cast<long long>(K));
  if (dtype != MG_F32 && K + 64 > kGemmDeepMaxLd)
    return fail(MG_ERR_UNSUPPORTED, "%s: no kernel for 16-bit rows of %lld", who, static_cast<long long>(K));
  return MG_OK;
}

// The three gradients; `list`: that of a `_deferred` call, or null.
static int gated_bwd(const char* who, const void* dy, const void* gu, const void* x, const void* w, void* dx, void* dw, void* db, int64_t M,
                     int64_t F, int64_t K, int dx_accumulate, int gate, int dtype, int grad_dtype, DeferredList* list, mg_stream stream) {
  MG_TRY(gated_check(who, M, F, K, gate, dtype));
  if (!is_float_dtype(grad_dtype) || (grad_dtype != dtype && grad_dtype != MG_F32))
    return fail(MG_ERR_INVALID, "%s: grad_dtype must be the tensors' dtype or float32, got %s", who, dtype_name(grad_dtype));
  if (!dw || (M > 0 && (!dy || !gu || !x || (dx && !w)))) return fail(MG_ERR_INVALID, "%s: null pointer argument", who);
  if (M == 0) {
    MG_TRY(mg_fill(dw, 0.0, 2 * F * K, grad_dtype, stream));
    if (db) MG_TRY(mg_fill(db, 0.0, 2 * F, grad_dtype, stream));
    return MG_OK;
  }
  hipStream_t s = to_stream(stream);
  return without_exceptions(who, [&]() -> int {
    CaptureHold hold;
    if (!list) MG_TRY(hold.begin(s));  // (a list's blocks outlive the call, and go back to the pool with it)
    Scratch dgu;
    MG_TRY(dgu.take(M * 2 * F * dtype_size(dtype)));
    switch (dtype) {
      case MG_F32: MG_TRY(gate_bwd<float>(dy, gu, dgu.as<char>(), M, F, gate, s)); break;
      case MG_F16: MG_TRY(gate_bwd<f16_t>(dy, gu, dgu.as<char>(), M, F, gate, s)); break;
      default: MG_TRY(gate_bwd<bf16_t>(dy, gu, dgu.as<char>(), M, F, gate, s)); break;
    }
    auto products = [&] { return mg_linear_bwd_fused(dgu.as<char>(), x, w, dx, dw, db, M, 2 * F, K, dx_accumulate, 0, dtype, stream); };
    if (list) {
      DeferredScope scope(list, dtype, grad_dtype);
      return products();
    }
    if (grad_dtype == dtype) return products();
    DeferredList own;
    int rc;
    {
      DeferredScope scope(&own, dtype, grad_dtype);
      rc = products();
    }
    const int rc2 = mg_finish_deferred(&own, stream);
    return rc != MG_OK ? rc : rc2;
  });
}

}  // namespace mg

extern "C" {

int mg_gated_linear_fwd(const void* x, const void* w, const void* bias, void* y, void* gu, int64_t M, int64_t F, int64_t K, int gate,
                        int dtype, mg_stream stream) {
  const char* const who = "gated_linear_fwd";
  MG_TRY(mg::gated_check(who, M, F, K, gate, dtype));
  if (M == 0) return MG_OK;
  if (!x || !w || !y) return mg::fail(MG_ERR_INVALID, "%s: null pointer argument", who);
  hipStream_t s = mg::to_stream(stream);
  return mg::without_exceptions(who, [&]() -> int {
    mg::CaptureHold hold;
    MG_TRY(hold.begin(s));
    if (dtype == MG_BF16) return mg::gated_fwd_16bit<mg::bf16_t>(x, w, bias, y, gu, M, F, K, gate, s);
    if (dtype == MG_F16) return mg::gated_fwd_16bit<mg::f16_t>(x, w, bias, y, gu, M, F, K, gate, s);
    // fp32: the projections as one product, whose values are not rounded on the way; 3 M F values of 2 (K + 1) M F products' time.
    mg::Scratch kept;
    if (!gu) {
      MG_TRY(kept.take(M * 2 * F * static_cast<int64_t>(sizeof(float))));
      gu = kept.as<char>();
    }
    const mg::GemmArgs g{x, w, bias, gu, 1, M, 2 * F, K, K, 1, 1, K, 0, 0, MG_F32};
    MG_TRY(mg::gemm_dispatch(who, g, s));
    return mg::gate_fwd<float>(gu, y, M, F, gate, s);
  });
}

int mg_gated_linear_bwd(const void* dy, const void* gu, const void* x, const void* w, void* dx, void* dw, void* db, int64_t M, int64_t F,
                        int64_t K, int dx_accumulate, int gate, int dtype, int grad_dtype, mg_stream stream) {
  return mg::gated_bwd("gated_linear_bwd", dy, gu, x, w, dx, dw, db, M, F, K, dx_accumulate, gate, dtype, grad_dtype, nullptr, stream);
}

int mg_gated_linear_bwd_deferred(const void* dy, const void* gu, const void* x, const void* w, void* dx, void* dw, void* db, int64_t M,
                                 int64_t F, int64_t K, int dx_accumulate, int gate, int dtype, int grad_dtype, mg_deferred list,
                                 mg_stream stream) {
  const char* const who = "gated_linear_bwd_deferred";
  if (!list) return mg::fail(MG_ERR_INVALID, "%s: null deferred list", who);
  return mg::gated_bwd(who, dy, gu, x, w, dx, dw, db, M, F, K, dx_accumulate, gate, dtype, grad_dtype,
                       static_cast<mg::DeferredList*>(list), stream);
}

}  // extern "C"
