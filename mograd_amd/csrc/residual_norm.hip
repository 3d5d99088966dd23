// C ABI of the residual norm: argument checks and dtype dispatch.
#include "residual_norm.h"

#include "mg_act8.h"

namespace mg {

static int residual_norm_check(const char* who, int64_t rows, int64_t cols, int64_t gate_rows, bool gate, int dtype) {
  if (!is_float_dtype(dtype)) return fail(MG_ERR_INVALID, "%s: unsupported dtype %s", who, dtype_name(dtype));
  if (rows < 0 || cols <= 0 || cols > 0x3fffffffLL || rows > 0x7fffffffLL)
    return fail(MG_ERR_INVALID, "%s: bad shape rows=%lld cols=%lld", who, static_cast<long long>(rows),
                static_cast<long long>(cols));
  if (gate && rows > 0 && (gate_rows <= 0 || rows % gate_rows != 0))
    return fail(MG_ERR_INVALID, "%s: gate_rows=%lld does not divide rows=%lld", who, static_cast<long long>(gate_rows),
                static_cast<long long>(rows));
  return MG_OK;
}

// A norm's pointers: all of them or none.
static int norm_pointers(const char* who, const char* norm, std::initializer_list<const void*> ptrs) {
  size_t given = 0;
  for (const void* p : ptrs) given += p != nullptr;
  if (given != 0 && given != ptrs.size())
    return fail(MG_ERR_INVALID, "%s: the %s norm needs all of its arrays, or none", who, norm);
  return MG_OK;
}

template <typename T>
static const T* as(const void* p) {
  return static_cast<const T*>(p);
}

}  // namespace mg

extern "C" {

int mg_residual_norm_fwd(const void* f, const void* h, const void* gate, const void* post_gamma, const void* post_beta,
                         const void* pre_gamma, const void* pre_beta, void* h_out, void* x, float* post_mean, float* post_rstd,
                         float* pre_mean, float* pre_rstd, void* f8, void* x8, int64_t rows, int64_t cols, int64_t gate_rows,
                         float residual_scale, float eps, int dtype, mg_stream stream) {
  const char* const who = "residual_norm_fwd";
  MG_TRY(mg::residual_norm_check(who, rows, cols, gate_rows, gate != nullptr, dtype));
  if (rows == 0) return MG_OK;
  if (!f || !h || !h_out) return mg::fail(MG_ERR_INVALID, "%s: null pointer argument", who);
  MG_TRY(mg::norm_pointers(who, "post", {post_gamma, post_beta, post_mean, post_rstd}));
  MG_TRY(mg::norm_pointers(who, "pre", {pre_gamma, pre_beta, pre_mean, pre_rstd, x}));
  if (x8 && !x) return mg::fail(MG_ERR_INVALID, "%s: x8 without a pre norm", who);
  if (f8 || x8) MG_TRY(mg::act8_check(who, rows, cols, dtype));
  if (f8) MG_TRY(mg::act8_pointer_check(who, f8));
  if (x8) MG_TRY(mg::act8_pointer_check(who, x8));
  auto run = [&](auto zero) {
    using T = decltype(zero);
    const mg::ResidualNormFwd<T> a{mg::as<T>(f), mg::as<T>(h), mg::as<T>(gate), mg::as<T>(post_gamma), mg::as<T>(post_beta),
                                   mg::as<T>(pre_gamma), mg::as<T>(pre_beta), static_cast<T*>(h_out), static_cast<T*>(x),
                                   post_mean, post_rstd, pre_mean, pre_rstd, static_cast<uint8_t*>(f8),
                                   static_cast<uint8_t*>(x8), rows, mg::act8_ld(cols), static_cast<int>(cols),
                                   static_cast<uint32_t>(gate ? gate_rows : rows), residual_scale, eps};
    return mg::residual_norm_fwd<T>(a, dtype, mg::to_stream(stream));
  };
  switch (dtype) {
    case MG_F32: return run(float{});
    case MG_F16: return run(mg::f16_t{});
    default: return run(mg::bf16_t{});
  }
}

int mg_residual_norm_bwd(const void* dx, const void* dh_out, const void* f, const void* f8, const void* h_out, const void* gate,
                         const void* post_gamma, const void* post_beta, const void* pre_gamma, const float* post_mean,
                         const float* post_rstd, const float* pre_mean, const float* pre_rstd, void* df, void* dh, void* dgate,
                         void* dpost_gamma, void* dpost_beta, void* dpre_gamma, void* dpre_beta, int64_t rows, int64_t cols,
                         int64_t gate_rows, float residual_scale, int dtype, int grad_dtype, mg_stream stream) {
  const char* const who = "residual_norm_bwd";
  MG_TRY(mg::residual_norm_check(who, rows, cols, gate_rows, gate != nullptr, dtype));
  if (!mg::is_float_dtype(grad_dtype) || (grad_dtype != dtype && grad_dtype != MG_F32))
    return mg::fail(MG_ERR_INVALID, "%s: grad_dtype must be the tensors' dtype or float32, got %s", who,
                    mg::dtype_name(grad_dtype));
  if ((gate != nullptr) != (dgate != nullptr)) return mg::fail(MG_ERR_INVALID, "%s: gate and dgate come together", who);
  hipStream_t s = mg::to_stream(stream);
  // The column sums of empty matrices are zero.  (An empty batch has no gate rows of its own, but may have the one of all rows.)
  if (rows == 0) {
    MG_TRY(mg::norm_pointers(who, "post", {post_gamma, post_beta, dpost_gamma, dpost_beta}));
    MG_TRY(mg::norm_pointers(who, "pre", {pre_gamma, dpre_gamma, dpre_beta}));
    for (void* out : {dgate && gate_rows == 0 ? dgate : nullptr, dpost_gamma, dpost_beta, dpre_gamma, dpre_beta})
      if (out) MG_TRY(mg_fill(out, 0.0, cols, grad_dtype, stream));
    return MG_OK;
  }
  MG_TRY(mg::norm_pointers(who, "post", {post_gamma, post_beta, post_mean, post_rstd, dpost_gamma, dpost_beta}));
  MG_TRY(mg::norm_pointers(who, "pre", {pre_gamma, pre_mean, pre_rstd, dx, dpre_gamma, dpre_beta}));
  if (f && f8) return mg::fail(MG_ERR_INVALID, "%s: f or f8, not both", who);
  if (!f && !f8 && (gate || post_gamma)) return mg::fail(MG_ERR_INVALID, "%s: f or f8 is needed for a gate or a post norm", who);
  if (!df || !dh || (!dh_out && !dx) || (!h_out && dx)) return mg::fail(MG_ERR_INVALID, "%s: null pointer argument", who);
  if (f8) {
    MG_TRY(mg::act8_check(who, rows, cols, dtype));
    MG_TRY(mg::act8_pointer_check(who, f8));
  }
  mg::CaptureHold hold;
  MG_TRY(hold.begin(s));
  void* const out[4] = {dpost_gamma, dpost_beta, dpre_gamma, dpre_beta};
  auto run = [&](auto zero) {
    using T = decltype(zero);
    mg::ResidualNormBwd<T> a{};
    a.dx = mg::as<T>(dx);
    a.dh_out = mg::as<T>(dh_out);
    a.f = mg::as<T>(f);
    a.h_out = mg::as<T>(h_out);
    a.f8 = static_cast<const uint8_t*>(f8);
    a.gate = mg::as<T>(gate);
    a.post_gamma = mg::as<T>(post_gamma);
    a.post_beta = mg::as<T>(post_beta);
    a.pre_gamma = mg::as<T>(pre_gamma);
    a.post_mean = post_mean;
    a.post_rstd = post_rstd;
    a.pre_mean = pre_mean;
    a.pre_rstd = pre_rstd;
    a.df = static_cast<T*>(df);
    a.dh = static_cast<T*>(dh);
    a.dgate = dgate;
    a.grad_f32 = grad_dtype == MG_F32;
    a.rows = rows;
    a.ld = mg::act8_ld(cols);
    a.cols = static_cast<int>(cols);
    a.gate_rows = static_cast<uint32_t>(gate ? gate_rows : rows);
    a.gates = rows / a.gate_rows;
    a.scale = residual_scale;
    return mg::without_exceptions(who, [&] { return mg::residual_norm_bwd<T>(a, out, dtype, s); });
  };
  switch (dtype) {
    case MG_F32: return run(float{});
    case MG_F16: return run(mg::f16_t{});
    default: return run(mg::bf16_t{});
  }
}

}  // extern "C"
