// Arguments of the residual-norm kernels (residual_norm_impl.h), shared with the C ABI (residual_norm.hip).
#pragma once

#include "mg_device.h"
#include "mg_internal.h"

namespace mg {

template <typename T>
struct ResidualNormFwd {
  const T *f, *h;
  const T *gate, *post_gamma, *post_beta, *pre_gamma, *pre_beta;  // null: no gate, no post norm, no pre norm
  T *h_out, *x;
  float *post_mean, *post_rstd, *pre_mean, *pre_rstd;
  uint8_t *f8, *x8;  // null: not kept in 8 bits
  int64_t rows, ld;  // ld: bytes of a row of q
  int cols;
  uint32_t gate_rows;
  float scale, eps;
};

template <typename T>
struct ResidualNormBwd {
  const T *dx, *dh_out, *f, *h_out;
  const uint8_t* f8;
  const T *gate, *post_gamma, *post_beta, *pre_gamma;
  const float *post_mean, *post_rstd, *pre_mean, *pre_rstd;
  T *df, *dh;
  void* dgate;  // of T, or fp32
  int grad_f32;
  int64_t rows, ld;
  int cols;
  uint32_t gate_rows;
  float scale;
  // Workgroup (x, y) has piece x of the gate rows y gates_per_group and on: one gate row in several pieces, or several whole.
  // A piece's rows start piece * piece_start into the gate row's, are row_step apart for each of the rows in flight, and end
  // piece_span on or with the gate row.
  int64_t gates, gates_per_group, piece_start, piece_span, row_step;
  uint32_t pieces;
  int own;  // each of a workgroup's rows in flight has whole gate rows to itself
  // Column sums.  gate_sums [2][gates * pieces][cols]: of d and d fh over each piece of a gate row's rows; pre_sums
  // [2][workgroups][cols]: of dx xh and dx.  Null where nobody asks.
  float *gate_sums, *pre_sums, *post_sums;  // (post_sums: see ResidualNormFinish)
  float* row_sums;  // (rows, 2), the kernels of wide rows: the two means of the pre norm's gradient
};

// One row of the backward, value by value.
template <typename T>
struct ResidualNormRow {
  const ResidualNormBwd<T>& a;
  int64_t at;
  float pre_mean, pre_rstd, post_mean, post_rstd;
  __device__ __forceinline__ ResidualNormRow(const ResidualNormBwd<T>& args, int64_t row)
      : a(args), at(row * args.cols), pre_mean(args.pre_gamma ? args.pre_mean[row] : 0.f),
        pre_rstd(args.pre_gamma ? args.pre_rstd[row] : 1.f), post_mean(args.post_gamma ? args.post_mean[row] : 0.f),
        post_rstd(args.post_gamma ? args.post_rstd[row] : 1.f) {}
  __device__ __forceinline__ float pre_hat(int c) const { return (to_float(a.h_out[at + c]) - pre_mean) * pre_rstd; }
  __device__ __forceinline__ float post_hat(int c) const {
    return a.f ? (to_float(a.f[at + c]) - post_mean) * post_rstd : 0.f;
  }
  // The gradient of h', given the two means of the pre norm's.
  __device__ __forceinline__ float stream(int c, float c0, float c1) const {
    float d = a.dh_out ? to_float(a.dh_out[at + c]) : 0.f;
    if (a.pre_gamma) d += pre_rstd * (to_float(a.dx[at + c]) * to_float(a.pre_gamma[c]) - c0 - pre_hat(c) * c1);
    return d;
  }
};

template <typename T>
struct ResidualNormFinish {
  const float *gate_sums, *pre_sums;
  const T *gate, *post_gamma, *post_beta;
  void *dgate, *dpost_gamma, *dpost_beta, *dpre_gamma, *dpre_beta;
  float* post_sums;  // of many gate rows, [2][gridDim.z][cols]: the post norm's gradients over gates_per_block each; or null
  int64_t cols, groups, gates, gates_per_block, pieces;
  int64_t first_column;  // of the launch's columns
  int split;  // lanes to a gate row: a power of two, 1 .. 32
  int first;  // the first workgroups' job: 0 the gate and the post norm, 1 the pre norm
  int grad_f32;
};

template <typename T>
int residual_norm_fwd(const ResidualNormFwd<T>& a, int dtype, hipStream_t stream);
template <typename T>
int residual_norm_bwd(const ResidualNormBwd<T>& a, void* const (&out)[4], int dtype, hipStream_t stream);

}  // namespace mg
