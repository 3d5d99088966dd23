// Arguments of the products with an input in 8 bits (linear_act8_dw.h), shared with their host side (gemm.hip).
#pragma once

#include "gemm_impl.h"

namespace mg {

template <typename T>
struct Act8Dw {
  const T* dy;           // (M, N), rows ldy apart, any address of its elements
  const uint8_t *q, *e;  // (M, ldx) and (M, ldx / 32)
  float* partial;        // splits > 1: partial tiles as gemm16_partial_floats says
  T* dw;                 // splits == 1: the result, of T ...
  float* dw32;           // ... or, if not null, fp32
  float* db_part;        // not null: sums of dY over each range of rows, (splits, N)
  int64_t ldy, ldx;
  int M, N, K;
  int tiles_n, tiles_k, rows_per_split, splits;
  bool partial_stream;  // see Gemm16Problem
};

// The workgroups of dW and those of dX = dY W in one launch (n_dx == 0: dW alone); x_tile: 64 or 128, rows and columns of a tile of an
// fp32 dX.
template <typename T>
int launch_linear_act8(const Act8Dw<T>& dw, const Gemm16Problem<T>* dx, int x_tile, int64_t n_dw, int64_t n_dx, hipStream_t stream);

// gemm.hip: the three gradients from (M, K) bytes q, rows ldx apart, and their exponents e, sums left on `list`.
// *done = false: not such a layer, nothing launched.
int linear_bwd_act8_products(const void* dy, const uint8_t* q, const uint8_t* e, int64_t ldx, const void* w, void* dx, void* dw,
                             void* db, int64_t M, int64_t N, int64_t K, bool dx_accumulate, bool relu, int dtype, int grad_dtype,
                             hipStream_t stream, bool* done);

// An input that the products below read as T and that lies in 8 bits yet: M rows of K columns at `act8`, to be restored into `x`.
struct Act8Restore {
  const void* act8;
  void* x;
};
// The same by the kernels of any Linear backward, which read a copy of the input (it is restored into `restore.x`).
int linear_bwd_act8_copied(const void* dy, const Act8Restore& restore, const void* w, void* dx, void* dw, void* db, int64_t M, int64_t N,
                           int64_t K, bool dx_accumulate, bool relu, int dtype, hipStream_t stream);

}  // namespace mg
