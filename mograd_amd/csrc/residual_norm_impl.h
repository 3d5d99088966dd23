// What happens between two blocks of a transformer, for one storage type T: a block's output f is normalised, gated and added
// to the scaled residual stream h, and the sum is normalised for the next block.
//
//   z  = post_gamma (f - mean_f) rstd_f + post_beta      (z = f without a post norm)
//   h' = scale h + gate z                                (a gate row for every `gate_rows` rows; 1 without a gate)
//   x  = pre_gamma (h' - mean_h') rstd_h' + pre_beta     (no x without a pre norm)
//
// and the gradients, with fh and xh the normalised f and h':
//
//   d   = dh' + rstd_h' (pre_gamma dx - mean(pre_gamma dx) - xh mean(pre_gamma dx xh))
//   dh  = scale d
//   df  = rstd_f (post_gamma u - mean(post_gamma u) - fh mean(post_gamma u fh)),  u = gate d      (df = u without a post norm)
//   dpre_gamma = sum dx xh,  dpre_beta = sum dx,  and with A = sum d, B = sum d fh over the rows of one gate row
//   dgate = post_gamma B + post_beta A,  dpost_gamma = sum of gate B,  dpost_beta = sum of gate A over the gate rows
//   (without a post norm B = sum d f = dgate).
//
// One pass in either direction, every tensor read once and written once, a row held in registers: both are bound by HBM.
// Sums, statistics and the stream between the two norms are fp32; x is formed from the h' in registers, before h' is rounded
// for storing.  Row layout as in layer_norm_impl.h: chunks of 16 bytes dealt round-robin to the TPR threads of a row.
#pragma once

#include "mg_act8.h"
#include "mg_internal.h"
#include "mg_rows.h"
#include "residual_norm.h"

namespace mg {

// A row's chunks as loaded, unpacked where they are used: half the registers of fp32 values for 16-bit rows, so that the
// parameter vectors and the next row fit beside the present one.  Zeros past the row.
template <typename T, int TPR, int VPT, bool ANY>
struct RawRow {
  static constexpr int VEC = WideVec<T>::value;
  using Tile = RowTile<T, VEC, TPR, VPT, ANY>;
  uint32_t w[VPT][4];

  static __device__ __forceinline__ int col(int i, int t) { return (i * TPR + t) * VEC; }
  __device__ __forceinline__ void load(const T* row, int t, int cols) {
    const unsigned lane = static_cast<unsigned>(t) * VEC;
    const int full = Tile::full_chunks(cols);
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const T* const p = row + i * (TPR * VEC) + lane;
      if (i < full) {
        get(p, w[i]);
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) w[i][j] = 0;
        if (i == full && col(i, t) < cols) {
          if constexpr (ANY) VecAny<T, VEC>::words_end(p, max(col(i, t) + VEC - cols, 0), 0, w[i]);
          else get(p, w[i]);
        }
      }
    }
  }
  __device__ __forceinline__ void values(int i, float (&v)[VEC]) const { VecAny<T, VEC>::unpack(w[i], v); }
  // Whether element e of chunk i is one of the row's.
  static __device__ __forceinline__ bool in_row(int i, int e, int t, int cols) { return Tile::in_row(col(i, t), e, cols); }
  static __device__ __forceinline__ void store(T* row, int i, int t, int cols, const float (&v)[VEC]) {
    const int c = col(i, t);
    if (c < cols) Tile::store_end_stream(row + c, c, cols, v);
  }

 private:
  static __device__ __forceinline__ void get(const T* p, uint32_t (&to)[4]) {
    if constexpr (ANY) {
      const mg_u4_any r = *reinterpret_cast<const mg_u4_any*>(p);
#pragma unroll
      for (int j = 0; j < 4; ++j) to[j] = r[j];
    } else {
      const mg_u4 r = *reinterpret_cast<const mg_u4*>(p);
#pragma unroll
      for (int j = 0; j < 4; ++j) to[j] = r[j];
    }
  }
};

// A row kept in 8 bits, chunk by chunk as RawRow lays it out.
template <typename T, int TPR, int VPT>
struct Act8Row {
  static constexpr int VEC = WideVec<T>::value;
  uint32_t q[VPT][VEC / 4];
  uint32_t e[VPT];

  __device__ __forceinline__ void load(const uint8_t* q_row, const uint8_t* e_row, int t, int cols) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      const int c = (i * TPR + t) * VEC;
      e[i] = 7;
#pragma unroll
      for (int j = 0; j < VEC / 4; ++j) q[i][j] = 0;
      if (c < cols) {  // (a row of q is zeros to the end of its last block)
        if constexpr (VEC == 8) {
          const uint2 r = *reinterpret_cast<const uint2*>(q_row + c);
          q[i][0] = r.x;
          q[i][1] = r.y;
        } else {
          q[i][0] = *reinterpret_cast<const uint32_t*>(q_row + c);
        }
        e[i] = e_row[c / kAct8Block];
      }
    }
  }
  __device__ __forceinline__ void values(int i, float (&v)[VEC]) const {
    const float scale = act8_scale(e[i]);
#pragma unroll
    for (int j = 0; j < VEC / 4; ++j) {
      float x[4];
      act8_unpack4(q[i][j], scale, x);
#pragma unroll
      for (int k = 0; k < 4; ++k) v[4 * j + k] = x[k];
    }
  }
};

// One chunk of a row into its place in 8 bits.  The lanes of a block call it together.
template <typename T, int TPR>
__device__ __forceinline__ void act8_store_chunk(uint8_t* q_row, uint8_t* e_row, int i, int t, int cols,
                                                 const float (&v)[WideVec<T>::value]) {
  constexpr int VEC = WideVec<T>::value, LANES = kAct8Block / VEC;
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < VEC; ++e) m = max(m, act8_abs_bits(v[e]));
  const uint32_t ex = act8_exponent<T>(act8_lanes_max<LANES>(m));
  const float inverse = act8_inverse(ex);
  const int c = (i * TPR + t) * VEC;
  if (c / kAct8Block * kAct8Block >= cols) return;  // (the lanes past the columns of the last block write its zeros)
  uint32_t w[VEC / 4];
#pragma unroll
  for (int j = 0; j < VEC / 4; ++j) {
    const float x[4] = {v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]};
    w[j] = act8_pack4(x, inverse, false);
  }
  if constexpr (VEC == 8) *reinterpret_cast<uint2*>(q_row + c) = make_uint2(w[0], w[1]);
  else *reinterpret_cast<uint32_t*>(q_row + c) = w[0];
  if (t % LANES == 0) e_row[c / kAct8Block] = static_cast<uint8_t>(ex);
}

// Mean and rstd of a row: the mean first, then the squares about it (the row is in registers, and a first element far from
// the others would cost the one-pass sums their digits).  `v` is zero past the row.
template <typename Row, int TPR, int VPT, int WG>
__device__ __forceinline__ void row_moments(const float (&v)[VPT][Row::VEC], int t, int cols, float inv_n, float eps, float* slots,
                                            int& phase, float& mean, float& rstd) {
  float s[1] = {0.f};
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int e = 0; e < Row::VEC; ++e) s[0] += v[i][e];
  row_allreduce_sum<TPR, WG, 1>(s, slots, phase);
  mean = s[0] * inv_n;
  s[0] = 0.f;
#pragma unroll
  for (int i = 0; i < VPT; ++i)
#pragma unroll
    for (int e = 0; e < Row::VEC; ++e) {
      const float d = Row::in_row(i, e, t, cols) ? v[i][e] - mean : 0.f;
      s[0] += d * d;
    }
  row_allreduce_sum<TPR, WG, 1>(s, slots, phase);
  rstd = rsqrtf(s[0] * inv_n + eps);
}

template <typename T, int TPR, int VPT, int WG, bool ANY>
__global__ __launch_bounds__(WG) void residual_norm_fwd_kernel(const ResidualNormFwd<T> a) {
  using Row = RawRow<T, TPR, VPT, ANY>;
  constexpr int VEC = Row::VEC, RPW = WG / TPR;
  static_assert(TPR <= kWave || RPW == 1, "rows of several waves have a workgroup each");
  __shared__ float slots[2 * (WG / kWave)];
  int t, sub;
  row_thread<TPR, WG>(t, sub);
  int phase = 0;
  const int cols = a.cols;
  const float inv_n = 1.0f / static_cast<float>(cols);

  Row post_gamma, post_beta, pre_gamma, pre_beta, gate;
  if (a.post_gamma) {
    post_gamma.load(a.post_gamma, t, cols);
    post_beta.load(a.post_beta, t, cols);
  }
  if (a.pre_gamma) {
    pre_gamma.load(a.pre_gamma, t, cols);
    pre_beta.load(a.pre_beta, t, cols);
  }
  uint32_t gate_at = 0xffffffffu;

  const int64_t step = static_cast<int64_t>(gridDim.x) * RPW;
  int64_t row = static_cast<int64_t>(blockIdx.x) * RPW + sub;
  Row f, h, f_next, h_next;
  if (row < a.rows) {
    f.load(a.f + row * cols, t, cols);
    h.load(a.h + row * cols, t, cols);
  }
  for (; row < a.rows; row += step) {  // uniform per row of 16 lanes (TPR == 16), per wave (64) or per workgroup
    const int64_t next = row + step;
    if (next < a.rows) {
      f_next.load(a.f + next * cols, t, cols);
      h_next.load(a.h + next * cols, t, cols);
    }
    if (a.gate) {
      const uint32_t at = static_cast<uint32_t>(row) / a.gate_rows;
      if (at != gate_at) gate.load(a.gate + static_cast<int64_t>(at) * cols, t, cols);
      gate_at = at;
    }
    float v[VPT][VEC];
#pragma unroll
    for (int i = 0; i < VPT; ++i) f.values(i, v[i]);
    if (a.f8) {
      uint8_t* const e_row = a.f8 + a.rows * a.ld + row * (a.ld / kAct8Block);
#pragma unroll
      for (int i = 0; i < VPT; ++i) act8_store_chunk<T, TPR>(a.f8 + row * a.ld, e_row, i, t, cols, v[i]);
    }
    float mean, rstd;
    if (a.post_gamma) {
      row_moments<Row, TPR, VPT, WG>(v, t, cols, inv_n, a.eps, slots, phase, mean, rstd);
      if (t == 0) {
        a.post_mean[row] = mean;
        a.post_rstd[row] = rstd;
      }
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        float g[VEC], b[VEC];
        post_gamma.values(i, g);
        post_beta.values(i, b);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[i][e] = (v[i][e] - mean) * rstd * g[e] + b[e];  // (zero past the row: g and b are)
      }
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float hv[VEC];
      h.values(i, hv);
      if (a.gate) {
        float g[VEC];
        gate.values(i, g);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[i][e] *= g[e];
      }
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[i][e] = fmaf(a.scale, hv[e], v[i][e]);
      Row::store(a.h_out + row * cols, i, t, cols, v[i]);
    }
    if (a.pre_gamma) {
      row_moments<Row, TPR, VPT, WG>(v, t, cols, inv_n, a.eps, slots, phase, mean, rstd);
      if (t == 0) {
        a.pre_mean[row] = mean;
        a.pre_rstd[row] = rstd;
      }
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        float g[VEC], b[VEC];
        pre_gamma.values(i, g);
        pre_beta.values(i, b);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[i][e] = (v[i][e] - mean) * rstd * g[e] + b[e];
        Row::store(a.x + row * cols, i, t, cols, v[i]);
        if (a.x8) {  // of x as it is stored
#pragma unroll
          for (int e = 0; e < VEC; ++e) v[i][e] = to_float(from_float<T>(v[i][e]));
          act8_store_chunk<T, TPR>(a.x8 + row * a.ld, a.x8 + a.rows * a.ld + row * (a.ld / kAct8Block), i, t, cols, v[i]);
        }
      }
    }
    f = f_next;
    h = h_next;
  }
}

// Rows of fewer columns than a chunk has, or of more than registers hold: a workgroup a row, which is read again from the
// caches for every sum.  (Neither is a width that transformers have.)
template <typename T, int WG>
__global__ __launch_bounds__(WG) void residual_norm_fwd_wide_kernel(const ResidualNormFwd<T> a) {
  __shared__ float slots[2 * (WG / kWave)];
  int phase = 0;
  const int64_t row = blockIdx.x;
  const int cols = a.cols;
  const float inv_n = 1.0f / static_cast<float>(cols);
  const T* const f = a.f + row * cols;
  const T* const h = a.h + row * cols;
  const T* const gate = a.gate ? a.gate + static_cast<int64_t>(static_cast<uint32_t>(row) / a.gate_rows) * cols : nullptr;
  auto moments = [&](auto&& value, float& mean, float& rstd) {
    float s[1] = {0.f};
    for (int c = threadIdx.x; c < cols; c += WG) s[0] += value(c);
    block_allreduce<SumOp, WG / kWave, 1>(s, slots, phase);
    phase ^= 1;
    mean = s[0] * inv_n;
    s[0] = 0.f;
    for (int c = threadIdx.x; c < cols; c += WG) {
      const float d = value(c) - mean;
      s[0] += d * d;
    }
    block_allreduce<SumOp, WG / kWave, 1>(s, slots, phase);
    phase ^= 1;
    rstd = rsqrtf(s[0] * inv_n + a.eps);
  };
  float f_mean = 0.f, f_rstd = 1.f;
  if (a.post_gamma) {
    moments([&](int c) { return to_float(f[c]); }, f_mean, f_rstd);
    if (threadIdx.x == 0) {
      a.post_mean[row] = f_mean;
      a.post_rstd[row] = f_rstd;
    }
  }
  auto stream = [&](int c) {
    float z = to_float(f[c]);
    if (a.post_gamma) z = (z - f_mean) * f_rstd * to_float(a.post_gamma[c]) + to_float(a.post_beta[c]);
    if (gate) z *= to_float(gate[c]);
    return fmaf(a.scale, to_float(h[c]), z);
  };
  if (a.pre_gamma) {
    float mean, rstd;
    moments(stream, mean, rstd);
    if (threadIdx.x == 0) {
      a.pre_mean[row] = mean;
      a.pre_rstd[row] = rstd;
    }
    for (int c = threadIdx.x; c < cols; c += WG)
      a.x[row * cols + c] = from_float<T>((stream(c) - mean) * rstd * to_float(a.pre_gamma[c]) + to_float(a.pre_beta[c]));
  }
  // (last: h_out may be h, of which each value is read and written by one thread)
  for (int c = threadIdx.x; c < cols; c += WG) a.h_out[row * cols + c] = from_float<T>(stream(c));
}

// ------------------------------------------------------------------------------------
// Backward, stage 1: df, dh, and column sums of the workgroup's rows.  A workgroup has either one piece of the rows of one
// gate row, or several gate rows whole (the partition is the host's, ResidualNormBwd): the sums A and B are written out, as
// gradients of the gate and of the post norm's parameters, where the gate row changes.  No atomics, fixed orders.
// ------------------------------------------------------------------------------------

template <typename T, int TPR, int VPT, int WG, bool ANY, bool F8>
__global__ __launch_bounds__(WG) void residual_norm_bwd_kernel(const ResidualNormBwd<T> a) {
  using Row = RawRow<T, TPR, VPT, ANY>;
  constexpr int VEC = Row::VEC, RPW = WG / TPR, NW = WG / kWave;
  constexpr int TILE_COLS = VPT * TPR * VEC;
  constexpr int SETS = TPR < kWave ? NW : RPW;  // column sums to add in the workgroup: one set a wave, or one a row
  static_assert(TPR <= kWave || RPW == 1, "rows of several waves have a workgroup each");
  __shared__ float slots[2 * 2 * NW];
  __shared__ float combine[RPW > 1 ? SETS * TILE_COLS : 1];
  int t, sub;
  row_thread<TPR, WG>(t, sub);
  int phase = 0;
  const int cols = a.cols;
  const float inv_n = 1.0f / static_cast<float>(cols);
  const bool post = a.post_gamma != nullptr, pre = a.pre_gamma != nullptr;

  Row post_gamma, pre_gamma, gate;
  if (post) post_gamma.load(a.post_gamma, t, cols);
  if (pre) pre_gamma.load(a.pre_gamma, t, cols);
  float sum_d[VPT][VEC], sum_df[VPT][VEC], sum_g[VPT][VEC], sum_b[VPT][VEC];
  auto clear = [](float (&s)[VPT][VEC]) {
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) s[i][e] = 0.f;
  };
  clear(sum_g);
  clear(sum_b);

  // One column's sums over the present gate row's rows, out to memory.
  float* const part = a.part + static_cast<int64_t>(blockIdx.x) * cols;
  const int64_t set = a.part_stride;
  auto emit = [&](int c, float d, float df, int64_t gate_row, bool first) {
    if (post) {
      const float g = a.gate ? to_float(a.gate[gate_row * cols + c]) : 1.f;
      const float pg = g * df, pb = g * d;
      part[0 * set + c] = first ? pg : part[0 * set + c] + pg;
      part[1 * set + c] = first ? pb : part[1 * set + c] + pb;
      df = to_float(a.post_gamma[c]) * df + to_float(a.post_beta[c]) * d;
    }
    if (!a.gate) return;
    if (a.pieces > 1) part[4 * set + c] = df;
    else if (a.grad_f32) static_cast<float*>(a.dgate)[gate_row * cols + c] = df;
    else static_cast<T*>(a.dgate)[gate_row * cols + c] = from_float<T>(df);
  };
  // The workgroup's column sums of two tiles of its threads, handed column by column to `out`.
  auto columns = [&](float (&s0)[VPT][VEC], float (&s1)[VPT][VEC], auto&& out) {
    if constexpr (RPW == 1) {
#pragma unroll
      for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          const int c = Row::col(i, t) + e;
          if (c < cols) out(c, s0[i][e], s1[i][e]);
        }
    } else {
      constexpr int PER = (TILE_COLS + WG - 1) / WG;
      float total[2][PER];
      const int mine = TPR < kWave ? static_cast<int>(threadIdx.x / kWave) : sub;
#pragma unroll
      for (int which = 0; which < 2; ++which) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            float v = which == 0 ? s0[i][e] : s1[i][e];
            if constexpr (TPR < kWave) {
#pragma unroll
              for (int w = TPR; w < kWave; w *= 2) v += __shfl_xor(v, w);
            }
            if (TPR >= kWave || threadIdx.x % kWave < TPR) combine[mine * TILE_COLS + Row::col(i, t) + e] = v;
          }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < PER; ++k) {
          const int c = threadIdx.x + k * WG;
          float v = 0.f;
          if (c < TILE_COLS)
#pragma unroll
            for (int r = 0; r < SETS; ++r) v += combine[r * TILE_COLS + c];
          total[which][k] = v;
        }
      }
#pragma unroll
      for (int k = 0; k < PER; ++k) {
        const int c = threadIdx.x + k * WG;
        if (c < TILE_COLS && c < cols) out(c, total[0][k], total[1][k]);
      }
    }
  };

  const int64_t gate_first = a.pieces > 1 ? blockIdx.x / a.pieces : static_cast<int64_t>(blockIdx.x) * a.gates_per_group;
  const int64_t gate_last = a.pieces > 1 ? gate_first + 1 : min(gate_first + a.gates_per_group, a.gates);
  const int64_t piece = a.pieces > 1 ? blockIdx.x % a.pieces : 0;
  for (int64_t gate_row = gate_first; gate_row < gate_last; ++gate_row) {
    if (a.gate) gate.load(a.gate + gate_row * cols, t, cols);
    clear(sum_d);
    clear(sum_df);
    const int64_t end = min((gate_row + 1) * static_cast<int64_t>(a.gate_rows),
                            gate_row * static_cast<int64_t>(a.gate_rows) + piece * a.piece_start + a.piece_span);
    int64_t row = gate_row * static_cast<int64_t>(a.gate_rows) + piece * a.piece_start + sub;
    for (; row < end; row += a.row_step) {
      Row dx, dh, h, f;
      Act8Row<T, TPR, VPT> f8;
      if constexpr (F8) f8.load(a.f8 + row * a.ld, a.f8 + a.rows * a.ld + row * (a.ld / kAct8Block), t, cols);
      else f.load(a.f + row * cols, t, cols);
      if (a.dh_out) dh.load(a.dh_out + row * cols, t, cols);
      float d[VPT][VEC];
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        if (a.dh_out) dh.values(i, d[i]);
        else
#pragma unroll
          for (int e = 0; e < VEC; ++e) d[i][e] = 0.f;
      }
      if (pre) {
        dx.load(a.dx + row * cols, t, cols);
        h.load(a.h_out + row * cols, t, cols);
        const float mean = a.pre_mean[row], rstd = a.pre_rstd[row];
        float s[2] = {0.f, 0.f};
        float hat[VPT][VEC];
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          float dv[VEC], g[VEC];
          dx.values(i, dv);
          pre_gamma.values(i, g);
          h.values(i, hat[i]);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            hat[i][e] = (hat[i][e] - mean) * rstd;
            const float dg = dv[e] * g[e];  // zero past the row
            s[0] += dg;
            s[1] += dg * hat[i][e];
            sum_g[i][e] += dv[e] * hat[i][e];
            sum_b[i][e] += dv[e];
          }
        }
        row_allreduce_sum<TPR, WG, 2>(s, slots, phase);
        const float c1 = s[0] * inv_n, c2 = s[1] * inv_n;
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          float dv[VEC], g[VEC];
          dx.values(i, dv);
          pre_gamma.values(i, g);
#pragma unroll
          for (int e = 0; e < VEC; ++e) d[i][e] += rstd * (dv[e] * g[e] - c1 - hat[i][e] * c2);
        }
      }
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        float out[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) out[e] = a.scale * d[i][e];
        Row::store(a.dh + row * cols, i, t, cols, out);
      }
      // (from here on d is gate d; what stands past the row in d meets gamma = 0 or is not stored)
      float hat[VPT][VEC];
      float mean = 0.f, rstd = 1.f;
      if (post) {
        mean = a.post_mean[row];
        rstd = a.post_rstd[row];
      }
      float s[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        if constexpr (F8) f8.values(i, hat[i]);
        else f.values(i, hat[i]);
        float g[VEC], pg[VEC];
        if (a.gate) gate.values(i, g);
        if (post) post_gamma.values(i, pg);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          hat[i][e] = (hat[i][e] - mean) * rstd;
          sum_d[i][e] += d[i][e];
          sum_df[i][e] += d[i][e] * hat[i][e];
          if (a.gate) d[i][e] *= g[e];
          if (post) {
            d[i][e] *= pg[e];
            s[0] += d[i][e];
            s[1] += d[i][e] * hat[i][e];
          }
        }
      }
      if (post) {
        row_allreduce_sum<TPR, WG, 2>(s, slots, phase);
        const float c1 = s[0] * inv_n, c2 = s[1] * inv_n;
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
          for (int e = 0; e < VEC; ++e) d[i][e] = rstd * (d[i][e] - c1 - hat[i][e] * c2);
      }
#pragma unroll
      for (int i = 0; i < VPT; ++i) Row::store(a.df + row * cols, i, t, cols, d[i]);
    }
    columns(sum_d, sum_df, [&](int c, float d, float df) { emit(c, d, df, gate_row, gate_row == gate_first); });
  }
  if (pre) {
    columns(sum_g, sum_b, [&](int c, float g, float b) {
      part[2 * set + c] = g;
      part[3 * set + c] = b;
    });
  }
}

// The backward of rows that registers do not hold, a workgroup a row: df and dh.  f in the type T.
template <typename T, int WG>
__global__ __launch_bounds__(WG) void residual_norm_bwd_wide_kernel(const ResidualNormBwd<T> a) {
  __shared__ float slots[2 * 2 * (WG / kWave)];
  int phase = 0;
  const int64_t row = blockIdx.x, at = row * a.cols;
  const int cols = a.cols;
  const float inv_n = 1.0f / static_cast<float>(cols);
  const T* const gate = a.gate ? a.gate + row / a.gate_rows * cols : nullptr;
  const ResidualNormRow<T> r(a, row);
  float c[2] = {0.f, 0.f};
  if (a.pre_gamma) {
    for (int i = threadIdx.x; i < cols; i += WG) {
      const float dg = to_float(a.dx[at + i]) * to_float(a.pre_gamma[i]);
      c[0] += dg;
      c[1] += dg * r.pre_hat(i);
    }
    block_allreduce<SumOp, WG / kWave, 2>(c, slots, phase);
    phase ^= 1;
  }
  const float c0 = c[0] * inv_n, c1 = c[1] * inv_n;
  float s[2] = {0.f, 0.f};
  if (a.post_gamma) {
    for (int i = threadIdx.x; i < cols; i += WG) {
      const float u = r.stream(i, c0, c1) * (gate ? to_float(gate[i]) : 1.f) * to_float(a.post_gamma[i]);
      s[0] += u;
      s[1] += u * r.post_hat(i);
    }
    block_allreduce<SumOp, WG / kWave, 2>(s, slots, phase);
  }
  if (threadIdx.x == 0) {
    a.row_sums[2 * row] = c0;
    a.row_sums[2 * row + 1] = c1;
  }
  // dh last: it may be dh_out, of which each value is read and written by one thread ...
  for (int i = threadIdx.x; i < cols; i += WG) {
    const float d = r.stream(i, c0, c1);
    float u = d * (gate ? to_float(gate[i]) : 1.f);
    if (a.post_gamma) u = r.post_rstd * (u * to_float(a.post_gamma[i]) - s[0] * inv_n - r.post_hat(i) * (s[1] * inv_n));
    a.df[at + i] = from_float<T>(u);
  }
}

// ... and after the column sums, which need d too: a thread a column of one piece of one gate row's rows.
template <typename T, int WG>
__global__ __launch_bounds__(WG) void residual_norm_bwd_columns_kernel(const ResidualNormBwd<T> a) {
  const int c = static_cast<int>(blockIdx.x) * WG + threadIdx.x;
  if (c >= a.cols) return;
  const int64_t set = a.part_stride;
  const int64_t group = blockIdx.y;
  float* const part = a.part + group * a.cols;
  const int64_t gate_first = a.pieces > 1 ? group / a.pieces : group * a.gates_per_group;
  const int64_t gate_last = a.pieces > 1 ? gate_first + 1 : min(gate_first + a.gates_per_group, a.gates);
  const int64_t piece = a.pieces > 1 ? group % a.pieces : 0;
  float pg = 0.f, pb = 0.f, sg = 0.f, sb = 0.f;
  for (int64_t gate_row = gate_first; gate_row < gate_last; ++gate_row) {
    const int64_t end = min((gate_row + 1) * static_cast<int64_t>(a.gate_rows),
                            gate_row * static_cast<int64_t>(a.gate_rows) + piece * a.piece_start + a.piece_span);
    float sd = 0.f, sdf = 0.f;
    for (int64_t row = gate_row * static_cast<int64_t>(a.gate_rows) + piece * a.piece_start; row < end; ++row) {
      const ResidualNormRow<T> r(a, row);
      const float d = r.stream(c, a.row_sums[2 * row], a.row_sums[2 * row + 1]);
      sd += d;
      sdf += d * r.post_hat(c);
      if (a.pre_gamma) {
        const float dx = to_float(a.dx[row * a.cols + c]);
        sg += dx * r.pre_hat(c);
        sb += dx;
      }
      a.dh[row * a.cols + c] = from_float<T>(a.scale * d);
    }
    float dg = sdf;
    if (a.post_gamma) {
      const float g = a.gate ? to_float(a.gate[gate_row * a.cols + c]) : 1.f;
      pg += g * sdf;
      pb += g * sd;
      dg = to_float(a.post_gamma[c]) * sdf + to_float(a.post_beta[c]) * sd;
    }
    if (a.gate) {
      if (a.pieces > 1) part[4 * set + c] = dg;
      else if (a.grad_f32) static_cast<float*>(a.dgate)[gate_row * a.cols + c] = dg;
      else static_cast<T*>(a.dgate)[gate_row * a.cols + c] = from_float<T>(dg);
    }
  }
  part[0 * set + c] = pg;
  part[1 * set + c] = pb;
  part[2 * set + c] = sg;
  part[3 * set + c] = sb;
}

// Stage 2: the column sums over the workgroups' parts, in a fixed order.  32 columns by 32 lanes that share the parts;
// blockIdx.y: 0 .. 3 the norms' parameters, from 4 on the pieces of a gate row each.
template <typename T>
__global__ __launch_bounds__(1024) void residual_norm_finish_kernel(const ResidualNormFinish a) {
  __shared__ float tile[32][33];
  const int job = blockIdx.y < 4 ? blockIdx.y : 4;
  void* const out = a.out[job];
  if (!out) return;
  const int64_t gate_row = job == 4 ? blockIdx.y - 4 : 0;
  const float* part = a.part + job * a.part_stride + gate_row * a.pieces * a.cols;
  const int64_t count = job == 4 ? a.pieces : a.groups;
  const int cx = threadIdx.x % 32, ly = threadIdx.x / 32;
  const int64_t c = static_cast<int64_t>(blockIdx.x) * 32 + cx;
  float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
  if (c < a.cols) {
    int64_t g = ly;
    for (; g + 96 < count; g += 128) {
      s0 += part[g * a.cols + c];
      s1 += part[(g + 32) * a.cols + c];
      s2 += part[(g + 64) * a.cols + c];
      s3 += part[(g + 96) * a.cols + c];
    }
    for (; g < count; g += 32) s0 += part[g * a.cols + c];
  }
  tile[ly][cx] = (s0 + s1) + (s2 + s3);
  __syncthreads();
  if (ly == 0 && c < a.cols) {
    float s = 0.f;
#pragma unroll
    for (int k = 0; k < 32; ++k) s += tile[k][cx];
    const int64_t at = gate_row * a.cols + c;
    if (a.grad_f32) static_cast<float*>(out)[at] = s;
    else static_cast<T*>(out)[at] = from_float<T>(s);
  }
}

// ------------------------------------------------------------------------------------
// Host side
// ------------------------------------------------------------------------------------

template <typename T>
struct ResidualNormOps {
  static constexpr int VEC = WideVec<T>::value;
  struct Shape {
    int tpr, vpt;
  };
  // How a row of `chunks` chunks is laid over threads.
  static bool pick_shape(int64_t chunks, Shape* s) {
    if (chunks <= 16) *s = {16, 1};
    else if (chunks <= 32) *s = {16, 2};
    else if (chunks <= 64) *s = {64, 1};
    else if (chunks <= 128) *s = {64, 2};
    else if (chunks <= 256) *s = {256, 1};
    else if (chunks <= 512) *s = {512, 1};
    else if (chunks <= 1024) *s = {1024, 1};
    else if (chunks <= 2048) *s = {1024, 2};
    else return false;
    return true;
  }
  static bool aligned(int64_t cols, std::initializer_list<const void*> ptrs) {
    if (cols % VEC != 0) return false;
    for (const void* p : ptrs)
      if (p && !aligned16(p)) return false;
    return true;
  }

  template <int TPR, int VPT, bool ANY>
  static int launch_fwd(const ResidualNormFwd<T>& a, hipStream_t stream) {
    constexpr int WG = TPR <= 64 ? 256 : TPR;
    constexpr int RPW = WG / TPR;
    const int64_t want = ceil_div(a.rows, RPW);
    const int64_t cap = static_cast<int64_t>(device_info().cu_count) * (2048 / WG);
    hipLaunchKernelGGL((residual_norm_fwd_kernel<T, TPR, VPT, WG, ANY>), dim3(static_cast<unsigned>(std::min(want, cap))),
                       dim3(WG), 0, stream, a);
    MG_LAUNCH_CHECK();
    return MG_OK;
  }

#define MG_RESIDUAL_NORM_SHAPES(CALL) \
  CALL(16, 1);                        \
  CALL(16, 2);                        \
  CALL(64, 1);                        \
  CALL(64, 2);                        \
  CALL(256, 1);                       \
  CALL(512, 1);                       \
  CALL(1024, 1);                      \
  CALL(1024, 2)

  template <bool ANY>
  static int dispatch_fwd(Shape s, const ResidualNormFwd<T>& a, hipStream_t stream) {
#define MG_CASE(TPR_, VPT_) \
  if (s.tpr == TPR_ && s.vpt == VPT_) return launch_fwd<TPR_, VPT_, ANY>(a, stream)
    MG_RESIDUAL_NORM_SHAPES(MG_CASE);
#undef MG_CASE
    return fail(MG_ERR_UNSUPPORTED, "residual_norm_fwd: no kernel for row shape (%d, %d)", s.tpr, s.vpt);
  }

  static int fwd(const ResidualNormFwd<T>& a, int dtype, hipStream_t stream) {
    Shape s;
    if (a.cols >= VEC && pick_shape(ceil_div(a.cols, VEC), &s)) {
      if (aligned(a.cols, {a.f, a.h, a.gate, a.post_gamma, a.post_beta, a.pre_gamma, a.pre_beta, a.h_out, a.x}))
        return dispatch_fwd<false>(s, a, stream);
      return dispatch_fwd<true>(s, a, stream);
    }
    if (a.f8) MG_TRY(act8_store(a.f, a.f8, a.rows, a.cols, false, dtype, stream));
    hipLaunchKernelGGL((residual_norm_fwd_wide_kernel<T, 1024>), dim3(static_cast<unsigned>(a.rows)), dim3(1024), 0, stream, a);
    MG_LAUNCH_CHECK();
    if (a.x8) MG_TRY(act8_store(a.x, a.x8, a.rows, a.cols, false, dtype, stream));
    return MG_OK;
  }

  // Splits the rows over at most `most` workgroups of `rows_at_once` rows: fewer gate rows than workgroups are cut into
  // pieces, more are dealt out whole.
  static int64_t partition(ResidualNormBwd<T>& a, int64_t most, int rows_at_once, bool interleave) {
    const int64_t per_gate = std::max<int64_t>(1, std::min(most / a.gates, ceil_div(a.gate_rows, rows_at_once)));
    a.gates_per_group = ceil_div(a.gates, most);
    if (a.gates_per_group > 1 || per_gate == 1) {
      a.pieces = 1;
      a.piece_start = 0;
      a.piece_span = a.gate_rows;
      a.row_step = rows_at_once;
      return ceil_div(a.gates, a.gates_per_group);
    }
    a.gates_per_group = 1;
    const int64_t span = ceil_div(ceil_div(a.gate_rows, per_gate), rows_at_once) * rows_at_once;
    a.pieces = static_cast<uint32_t>(ceil_div(a.gate_rows, span));
    a.piece_start = interleave ? rows_at_once : span;
    a.piece_span = interleave ? a.gate_rows : span;
    a.row_step = interleave ? static_cast<int64_t>(a.pieces) * rows_at_once : rows_at_once;
    return a.gates * a.pieces;
  }

  static int finish(ResidualNormBwd<T>& a, int64_t groups, void* const (&out)[4], hipStream_t stream) {
    ResidualNormFinish f{};
    f.part = a.part;
    f.part_stride = a.part_stride;
    f.cols = a.cols;
    f.groups = groups;
    f.pieces = a.pieces;
    f.grad_f32 = a.grad_f32;
    for (int i = 0; i < 4; ++i) f.out[i] = out[i];
    f.out[4] = a.gate && a.pieces > 1 ? a.dgate : nullptr;
    if (!f.out[0] && !f.out[2] && !f.out[4]) return MG_OK;
    const unsigned jobs = 4 + (f.out[4] ? static_cast<unsigned>(a.gates) : 0u);
    hipLaunchKernelGGL((residual_norm_finish_kernel<T>), dim3(static_cast<unsigned>(ceil_div(a.cols, 32)), jobs), dim3(1024), 0,
                       stream, f);
    MG_LAUNCH_CHECK();
    return MG_OK;
  }

  template <int TPR, int VPT, bool ANY, bool F8>
  static int launch_bwd(ResidualNormBwd<T> a, void* const (&out)[4], hipStream_t stream) {
    constexpr int WG = TPR <= 64 ? (VPT == 1 ? 512 : 256) : TPR;
    constexpr int RPW = WG / TPR;
    const bool interleave = a.rows * a.cols * static_cast<int64_t>(sizeof(T)) >= (int64_t{16} << 20);
    const int64_t groups = partition(a, static_cast<int64_t>(device_info().cu_count) * (WG >= 1024 ? 1 : 2), RPW, interleave);
    a.part_stride = groups * a.cols;
    Scratch part;
    MG_TRY(part.take(5 * a.part_stride * static_cast<int64_t>(sizeof(float))));
    a.part = part.as<float>();
    hipLaunchKernelGGL((residual_norm_bwd_kernel<T, TPR, VPT, WG, ANY, F8>), dim3(static_cast<unsigned>(groups)), dim3(WG), 0,
                       stream, a);
    MG_LAUNCH_CHECK();
    return finish(a, groups, out, stream);
  }

  template <bool ANY>
  static int dispatch_bwd(Shape s, const ResidualNormBwd<T>& a, void* const (&out)[4], hipStream_t stream) {
#define MG_CASE(TPR_, VPT_)           \
  if (s.tpr == TPR_ && s.vpt == VPT_) \
  return a.f8 ? launch_bwd<TPR_, VPT_, ANY, true>(a, out, stream) : launch_bwd<TPR_, VPT_, ANY, false>(a, out, stream)
    MG_RESIDUAL_NORM_SHAPES(MG_CASE);
#undef MG_CASE
    return fail(MG_ERR_UNSUPPORTED, "residual_norm_bwd: no kernel for row shape (%d, %d)", s.tpr, s.vpt);
  }
#undef MG_RESIDUAL_NORM_SHAPES

  // out: dpost_gamma, dpost_beta, dpre_gamma, dpre_beta.
  static int bwd(ResidualNormBwd<T> a, void* const (&out)[4], int dtype, hipStream_t stream) {
    Shape s;
    if (a.cols >= VEC && pick_shape(ceil_div(a.cols, VEC), &s)) {
      if (aligned(a.cols, {a.dx, a.dh_out, a.f, a.h_out, a.gate, a.post_gamma, a.post_beta, a.pre_gamma, a.df, a.dh}))
        return dispatch_bwd<false>(s, a, out, stream);
      return dispatch_bwd<true>(s, a, out, stream);
    }
    Scratch f, sums, part;
    if (a.f8) {
      MG_TRY(f.take(a.rows * a.cols * static_cast<int64_t>(sizeof(T))));
      MG_TRY(act8_load(a.f8, f.as<T>(), a.rows, a.cols, dtype, stream));
      a.f = f.as<T>();
    }
    MG_TRY(sums.take(2 * a.rows * static_cast<int64_t>(sizeof(float))));
    a.row_sums = sums.as<float>();
    hipLaunchKernelGGL((residual_norm_bwd_wide_kernel<T, 1024>), dim3(static_cast<unsigned>(a.rows)), dim3(1024), 0, stream, a);
    MG_LAUNCH_CHECK();
    const int64_t blocks = ceil_div(a.cols, 256);
    const int64_t most = std::max<int64_t>(1, ceil_div(static_cast<int64_t>(device_info().cu_count) * 4, blocks));
    const int64_t groups = partition(a, std::min<int64_t>(most, 65535), 1, false);
    a.part_stride = groups * a.cols;
    MG_TRY(part.take(5 * a.part_stride * static_cast<int64_t>(sizeof(float))));
    a.part = part.as<float>();
    hipLaunchKernelGGL((residual_norm_bwd_columns_kernel<T, 256>), dim3(static_cast<unsigned>(blocks), static_cast<unsigned>(groups)),
                       dim3(256), 0, stream, a);
    MG_LAUNCH_CHECK();
    return finish(a, groups, out, stream);
  }
};

}  // namespace mg

// Defines the per-dtype functions that residual_norm.hip dispatches to.
#define MG_DEFINE_RESIDUAL_NORM(T)                                                                  \
  namespace mg {                                                                                    \
  template <>                                                                                       \
  int residual_norm_fwd<T>(const ResidualNormFwd<T>& a, int dtype, hipStream_t stream) {            \
    return ResidualNormOps<T>::fwd(a, dtype, stream);                                               \
  }                                                                                                 \
  template <>                                                                                       \
  int residual_norm_bwd<T>(const ResidualNormBwd<T>& a, void* const (&out)[4], int dtype, hipStream_t stream) { \
    return ResidualNormOps<T>::bwd(a, out, dtype, stream);                                          \
  }                                                                                                 \
  }
