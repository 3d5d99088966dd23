// The gradients of a Linear layer whose input was kept in 8 bits (format: mg_act8.h).
#include "linear_act8.h"
#include "mg_act8.h"
#include "mg_deferred.h"

extern "C" {

int mg_linear_bwd_act8(const void* dy, const void* x8, const void* w, void* dx, void* dw, void* db, int64_t M, int64_t N,
                       int64_t K, int dx_accumulate, int x_is_relu_output, int dtype, int grad_dtype, mg_stream stream) {
  const char* const who = "linear_bwd_act8";
  if (!mg::is_float_dtype(dtype)) return mg::fail(MG_ERR_INVALID, "%s: unsupported dtype %s", who, mg::dtype_name(dtype));
  if (!mg::is_float_dtype(grad_dtype) || (grad_dtype != dtype && grad_dtype != MG_F32))
    return mg::fail(MG_ERR_INVALID, "%s: grad_dtype must be the tensors' dtype or float32, got %s", who,
                    mg::dtype_name(grad_dtype));
  if (M < 0 || N <= 0 || K <= 0) return mg::fail(MG_ERR_INVALID, "%s: bad size", who);
  MG_TRY(mg::act8_check(who, M, K, dtype));
  if (!dw || (M > 0 && (!dy || !x8 || (dx && !w)))) return mg::fail(MG_ERR_INVALID, "%s: null pointer argument", who);
  hipStream_t s = mg::to_stream(stream);
  if (M == 0) {
    MG_TRY(mg_fill(dw, 0.0, N * K, grad_dtype, stream));
    if (db) MG_TRY(mg_fill(db, 0.0, N, grad_dtype, stream));
    return MG_OK;
  }
  MG_TRY(mg::act8_pointer_check(who, x8));
  return mg::without_exceptions(who, [&]() -> int {
    mg::CaptureHold hold;
    MG_TRY(hold.begin(s));
    const int64_t ld = mg::act8_ld(K);
    const uint8_t* const q = static_cast<const uint8_t*>(x8);
    bool done = false;
    MG_TRY(mg::linear_bwd_act8_products(dy, q, q + M * ld, ld, w, dx, dw, db, M, N, K, dx_accumulate != 0, x_is_relu_output != 0, dtype,
                                        grad_dtype, s, &done));
    if (done) return MG_OK;
    mg::Scratch x;
    MG_TRY(x.take(M * K * static_cast<int64_t>(mg::dtype_size(dtype))));
    auto run = [&] {
      return mg::linear_bwd_act8_copied(dy, mg::Act8Restore{x8, x.as<char>()}, w, dx, dw, db, M, N, K, dx_accumulate != 0,
                                        x_is_relu_output != 0, dtype, s);
    };
    if (grad_dtype == dtype) return run();
    mg::DeferredList list;
    int rc;
    {
      mg::DeferredScope scope(&list, dtype, grad_dtype);
      rc = run();
    }
    const int rc2 = mg_finish_deferred(&list, stream);
    return rc != MG_OK ? rc : rc2;
  });
}

}  // extern "C"
