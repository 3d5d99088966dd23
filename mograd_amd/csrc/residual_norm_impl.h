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
  // Keeps the compiler from carrying unpacked values into what comes after, or out of the loop: twice the registers.
  __device__ __forceinline__ void keep_packed() {
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) asm volatile("" : "+v"(w[i][j]));
  }
  __device__ __forceinline__ void zeros() {
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) w[i][j] = 0;
  }
  __device__ __forceinline__ void ones() {
    float v[VEC];
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = 1.f;
#pragma unroll
    for (int i = 0; i < VPT; ++i) VecAny<T, VEC>::pack(v, w[i]);
  }
  __device__ __forceinline__ void values(int i, float (&v)[VEC]) const { VecAny<T, VEC>::unpack(w[i], v); }
  // The values times `scale`, plus `shift`.
  __device__ __forceinline__ void normalised(int i, float scale, float shift, float (&v)[VEC]) const {
    values(i, v);
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] = fmaf(v[e], scale, shift);
  }
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
  __device__ __forceinline__ void keep_packed() {
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int j = 0; j < VEC / 4; ++j) asm volatile("" : "+v"(q[i][j]));
  }
  // The values times `scale`, plus `shift`.
  __device__ __forceinline__ void normalised(int i, float scale, float shift, float (&v)[VEC]) const {
    const float step = act8_scale(e[i]) * scale;
#pragma unroll
    for (int j = 0; j < VEC / 4; ++j)
#pragma unroll
      for (int k = 0; k < 4; ++k) v[4 * j + k] = fmaf(static_cast<float>(static_cast<int8_t>(q[i][j] >> 8 * k)), step, shift);
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

// row_thread, with a slot that the compiler knows to be the same for a whole wave: addresses and the row's statistics stay in
// scalar registers (the backward of (16384, 384) bf16 spent a tenth of its vector instructions on 64-bit addresses).
template <int TPR, int WG>
__device__ __forceinline__ void wave_row_thread(int& t, int& sub) {
  row_thread<TPR, WG>(t, sub);
  if constexpr (TPR == kWave) sub = __builtin_amdgcn_readfirstlane(sub);
}

// Mean and rstd of a row: the mean first, then the squares about it (the row is in registers, and a first element far from
// the others would cost the one-pass sums their digits).  `v` is zero past the row.
template <typename Row, int TPR, int VPT, int WG>
__device__ __forceinline__ void row_moments(const float (&v)[VPT][Row::VEC], int t, int cols, float inv_n, float eps,
                                            float* slots, int& phase, float& mean, float& rstd) {
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
    if (Row::col(i, t) < cols) {
#pragma unroll
      for (int e = 0; e < Row::VEC; ++e) {
        const float d = Row::in_row(i, e, t, cols) ? v[i][e] - mean : 0.f;
        s[0] = fmaf(d, d, s[0]);
      }
    }
  row_allreduce_sum<TPR, WG, 1>(s, slots, phase);
  rstd = rsqrtf(s[0] * inv_n + eps);
}

// Which norms there are, and whether f or x is kept in 8 bits, is known to the compiler: as branches in the kernel they cost
// small calls most, which wait for every line of code that a row passes through.
template <typename T, int TPR, int VPT, int WG, bool ANY, bool POST, bool PRE, bool KEEP>
__global__ __launch_bounds__(WG) void residual_norm_fwd_kernel(const ResidualNormFwd<T> a) {
  using Row = RawRow<T, TPR, VPT, ANY>;
  constexpr int VEC = Row::VEC, RPW = WG / TPR;
  static_assert(TPR <= kWave || RPW == 1, "rows of several waves have a workgroup each");
  __shared__ float slots[2 * (WG / kWave)];
  int t, sub;
  wave_row_thread<TPR, WG>(t, sub);
  int phase = 0;
  const int cols = a.cols;
  const float inv_n = 1.0f / static_cast<float>(cols);
  const int64_t step = static_cast<int64_t>(gridDim.x) * RPW;
  int64_t row = static_cast<int64_t>(blockIdx.x) * RPW + sub;
  if (row >= a.rows) return;  // (the whole workgroup, where its waves share a row)

  Row f, h, f_next, h_next, post_gamma, post_beta, pre_gamma, pre_beta, gate;
  f.load(a.f + row * cols, t, cols);
  h.load(a.h + row * cols, t, cols);
  uint32_t gate_at = static_cast<uint32_t>(row) / a.gate_rows;
  if (a.gate) gate.load(a.gate + static_cast<int64_t>(gate_at) * cols, t, cols);
  else gate.ones();
  if constexpr (POST) {
    post_gamma.load(a.post_gamma, t, cols);
    post_beta.load(a.post_beta, t, cols);
  }
  if constexpr (PRE) {
    pre_gamma.load(a.pre_gamma, t, cols);
    pre_beta.load(a.pre_beta, t, cols);
  }
  while (true) {  // uniform per row of 16 lanes (TPR == 16), per wave (64) or per workgroup
    const int64_t next = row + step;
    if (next < a.rows) {
      f_next.load(a.f + next * cols, t, cols);
      h_next.load(a.h + next * cols, t, cols);
    }
    float v[VPT][VEC];
#pragma unroll
    for (int i = 0; i < VPT; ++i) f.values(i, v[i]);
    if constexpr (KEEP) {
      if (a.f8) {
        uint8_t* const e_row = a.f8 + a.rows * a.ld + row * (a.ld / kAct8Block);
#pragma unroll
        for (int i = 0; i < VPT; ++i) act8_store_chunk<T, TPR>(a.f8 + row * a.ld, e_row, i, t, cols, v[i]);
      }
    }
    float mean, rstd;
    if constexpr (POST) {
      row_moments<Row, TPR, VPT, WG>(v, t, cols, inv_n, a.eps, slots, phase, mean, rstd);
      if (t == 0) {
        a.post_mean[row] = mean;
        a.post_rstd[row] = rstd;
      }
    }
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      float hv[VEC], gt[VEC];
      if constexpr (POST) {
        float g[VEC], b[VEC];
        post_gamma.values(i, g);
        post_beta.values(i, b);
#pragma unroll
        for (int e = 0; e < VEC; ++e) v[i][e] = fmaf((v[i][e] - mean) * rstd, g[e], b[e]);  // (zero past the row: g and b are)
      }
      h.values(i, hv);
      gate.values(i, gt);
#pragma unroll
      for (int e = 0; e < VEC; ++e) v[i][e] = fmaf(a.scale, hv[e], v[i][e] * gt[e]);
      Row::store(a.h_out + row * cols, i, t, cols, v[i]);
    }
    if constexpr (PRE) {
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
        for (int e = 0; e < VEC; ++e) v[i][e] = fmaf((v[i][e] - mean) * rstd, g[e], b[e]);
        Row::store(a.x + row * cols, i, t, cols, v[i]);
        if constexpr (KEEP) {
          if (a.x8) {  // of x as it is stored
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[i][e] = to_float(from_float<T>(v[i][e]));
            act8_store_chunk<T, TPR>(a.x8 + row * a.ld, a.x8 + a.rows * a.ld + row * (a.ld / kAct8Block), i, t, cols, v[i]);
          }
        }
      }
    }
    if (next >= a.rows) return;
    row = next;
    f = f_next;
    h = h_next;
    const uint32_t at = static_cast<uint32_t>(row) / a.gate_rows;
    if (a.gate && at != gate_at) gate.load(a.gate + static_cast<int64_t>(at) * cols, t, cols);
    gate_at = at;
  }
}

// Rows of fewer columns than a chunk has, or of more than registers hold: a workgroup a row, which is read again from the
// caches for every sum.  (Neither is a width that transformers have.)  Past kWideGroups rows a workgroup takes several: a launch
// counts its threads in 32 bits.
constexpr int64_t kWideGroups = 1 << 16;
template <typename T, int WG>
__global__ __launch_bounds__(WG) void residual_norm_fwd_wide_kernel(const ResidualNormFwd<T> a) {
  __shared__ float slots[2 * (WG / kWave)];
  int phase = 0;
  const int cols = a.cols;
  const float inv_n = 1.0f / static_cast<float>(cols);
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
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* const f = a.f + row * cols;
    const T* const h = a.h + row * cols;
    const T* const gate = a.gate ? a.gate + static_cast<int64_t>(static_cast<uint32_t>(row) / a.gate_rows) * cols : nullptr;
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
}

// ------------------------------------------------------------------------------------
// Backward, stage 1: df, dh, and column sums of the workgroup's rows.  A workgroup has either one piece of the rows of one
// gate row, or several gate rows whole (the partition is the host's, ResidualNormBwd); the sums A and B go out where the gate
// row changes.  Many gate rows of few rows (a gate a token) go to the rows in flight, which write A and B from their registers.
// No atomics, fixed orders.
// ------------------------------------------------------------------------------------

template <typename T, int TPR, int VPT, int WG, bool ANY, bool F8, bool POST, bool PRE>
__global__ __launch_bounds__(WG) void residual_norm_bwd_kernel(const ResidualNormBwd<T> a) {
  using Row = RawRow<T, TPR, VPT, ANY>;
  using FRow = std::conditional_t<F8, Act8Row<T, TPR, VPT>, Row>;
  constexpr int VEC = Row::VEC, RPW = WG / TPR, NW = WG / kWave;
  constexpr int TILE_COLS = VPT * TPR * VEC;
  constexpr int SETS = TPR < kWave ? NW : RPW;  // column sums to add in the workgroup: one set a wave, or one a row
  // (1024 threads have 128 registers each, and rows off the chunks take more: (2587, 1001) fp16 with | without 24.1 | 20.5 us)
  constexpr bool PREFETCH = WG < 1024 && VPT * VEC <= (ANY ? 8 : 16);
  static_assert(TPR <= kWave || RPW == 1, "rows of several waves have a workgroup each");
  __shared__ float slots[2 * 2 * NW];
  __shared__ __attribute__((aligned(16))) float combine[RPW > 1 ? 2 * SETS * TILE_COLS : 4];
  int t, sub;
  wave_row_thread<TPR, WG>(t, sub);
  int phase = 0;
  const int cols = a.cols;
  const float inv_n = 1.0f / static_cast<float>(cols);

  float sums[4][VPT][VEC];  // of d, d fh (over the rows of a gate row), dx xh, dx
#pragma unroll
  for (int k = 0; k < 4; ++k)
#pragma unroll
    for (int i = 0; i < VPT; ++i)
#pragma unroll
      for (int e = 0; e < VEC; ++e) sums[k][i][e] = 0.f;
  // Sums k and k + 1 over the workgroup's rows to `out` and, `set` floats on, to the second one's place; back to zero.
  auto flush = [&](int k, float* out, int64_t set, bool from_registers) {
    if (RPW == 1 || from_registers) {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        const int c = Row::col(i, t);
        if (c >= cols) continue;
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float* const to = out + j * set + c;
          if (!ANY) {
#pragma unroll
            for (int e = 0; e < VEC; e += 4) {
              const mg_f4 v = {sums[k + j][i][e], sums[k + j][i][e + 1], sums[k + j][i][e + 2], sums[k + j][i][e + 3]};
              *reinterpret_cast<mg_f4*>(to + e) = v;
            }
          } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e)
              if (c + e < cols) to[e] = sums[k + j][i][e];
          }
        }
      }
    } else if constexpr (RPW > 1) {
      // The rows of the workgroup hold sums for the same columns: added through LDS, after those that share a wave.
      const int mine = TPR < kWave ? static_cast<int>(threadIdx.x / kWave) : sub;
      __syncthreads();  // (the sums before these have been read)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          if constexpr (TPR < kWave) {
#pragma unroll
            for (int e = 0; e < VEC; ++e)
#pragma unroll
              for (int w = TPR; w < kWave; w *= 2) sums[k + j][i][e] += __shfl_xor(sums[k + j][i][e], w);
          }
          if (TPR >= kWave || threadIdx.x % kWave < TPR) {
#pragma unroll
            for (int e = 0; e < VEC; e += 4) {
              const mg_f4 v = {sums[k + j][i][e], sums[k + j][i][e + 1], sums[k + j][i][e + 2], sums[k + j][i][e + 3]};
              *reinterpret_cast<mg_f4*>(combine + (j * SETS + mine) * TILE_COLS + Row::col(i, t) + e) = v;
            }
          }
        }
      __syncthreads();
      for (int c = threadIdx.x; c < cols; c += WG) {
        float v0 = combine[c], v1 = combine[SETS * TILE_COLS + c];
#pragma unroll
        for (int r = 1; r < SETS; ++r) {
          v0 += combine[r * TILE_COLS + c];
          v1 += combine[(SETS + r) * TILE_COLS + c];
        }
        out[c] = v0;
        out[set + c] = v1;
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < VPT; ++i)
#pragma unroll
        for (int e = 0; e < VEC; ++e) sums[k + j][i][e] = 0.f;
  };

  Row pre_gamma;
  if constexpr (PRE) pre_gamma.load(a.pre_gamma, t, cols);
  const uint32_t piece = blockIdx.x, group = blockIdx.y * gridDim.x + blockIdx.x;
  const int64_t first = static_cast<int64_t>(blockIdx.y) * a.gates_per_group;
  const int64_t last = min(first + a.gates_per_group, a.gates);
  const bool own = RPW > 1 && a.own;
  for (int64_t gate_row = first + (own ? sub : 0); gate_row < last; gate_row += own ? RPW : 1) {
    const int64_t base = gate_row * static_cast<int64_t>(a.gate_rows) + piece * a.piece_start;
    const int64_t end = min((gate_row + 1) * static_cast<int64_t>(a.gate_rows), base + a.piece_span);
    int64_t row = base + (own ? 0 : sub);

    Row dx, dh, h, dx_next, dh_next, h_next;
    FRow f, f_next;
    float pre_mean = 0.f, pre_rstd = 1.f, post_mean = 0.f, post_rstd = 1.f;
    float pre_mean_next = 0.f, pre_rstd_next = 1.f, post_mean_next = 0.f, post_rstd_next = 1.f;
    auto load = [&](int64_t r, FRow& f_, Row& dh_, Row& dx_, Row& h_, float& m0, float& r0, float& m1, float& r1) {
      if constexpr (F8) f_.load(a.f8 + r * a.ld, a.f8 + a.rows * a.ld + r * (a.ld / kAct8Block), t, cols);
      else if (POST || a.f) f_.load(a.f + r * cols, t, cols);
      else f_.zeros();  // (only the sums of d f ask for it, and nobody for them)
      if constexpr (PRE) {
        dx_.load(a.dx + r * cols, t, cols);
        h_.load(a.h_out + r * cols, t, cols);
        m0 = a.pre_mean[r];
        r0 = a.pre_rstd[r];
      }
      if (!PRE || a.dh_out) dh_.load(a.dh_out + r * cols, t, cols);
      else dh_.zeros();
      if constexpr (POST) {
        m1 = a.post_mean[r];
        r1 = a.post_rstd[r];
      }
    };
    Row gate, post_gamma;
    float w[VPT][VEC];  // gate post_gamma, or the gate
    auto weights = [&] {
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        gate.values(i, w[i]);
        if constexpr (POST) {
          float g[VEC];
          post_gamma.values(i, g);
#pragma unroll
          for (int e = 0; e < VEC; ++e) w[i][e] *= g[e];
        }
      }
    };
    if (a.gate) gate.load(a.gate + gate_row * cols, t, cols);
    else gate.ones();
    if constexpr (POST) post_gamma.load(a.post_gamma, t, cols);
    // The next row is on its way while a row is computed, where registers hold both.
    if (PREFETCH && row < end) load(row, f, dh, dx, h, pre_mean, pre_rstd, post_mean, post_rstd);
    weights();
    for (; row < end; row += a.row_step) {
      if constexpr (PREFETCH) {
        const int64_t next = row + a.row_step;
        if (next < end)
          load(next, f_next, dh_next, dx_next, h_next, pre_mean_next, pre_rstd_next, post_mean_next, post_rstd_next);
      } else {
        load(row, f, dh, dx, h, pre_mean, pre_rstd, post_mean, post_rstd);
      }
      if constexpr (sizeof(T) == 2) {
        dh.keep_packed();
        f.keep_packed();
        if constexpr (PRE) {
          dx.keep_packed();
          h.keep_packed();
          pre_gamma.keep_packed();
        }
      }
      float d[VPT][VEC], hat[VPT][VEC];
      if constexpr (PRE) {
        const float pre_shift = -pre_mean * pre_rstd;
        float s[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          float g[VEC];
          dx.values(i, d[i]);
          pre_gamma.values(i, g);
          h.values(i, hat[i]);
#pragma unroll
          for (int e = 0; e < VEC; ++e) {
            hat[i][e] = fmaf(hat[i][e], pre_rstd, pre_shift);
            sums[2][i][e] = fmaf(d[i][e], hat[i][e], sums[2][i][e]);
            sums[3][i][e] += d[i][e];
            d[i][e] *= g[e];  // zero past the row
            s[0] += d[i][e];
            s[1] = fmaf(d[i][e], hat[i][e], s[1]);
          }
        }
        row_allreduce_sum<TPR, WG, 2>(s, slots, phase);
        const float c1 = -pre_rstd * (s[0] * inv_n), c2 = -pre_rstd * (s[1] * inv_n);
#pragma unroll
        for (int i = 0; i < VPT; ++i) {
          float dv[VEC];
          dh.values(i, dv);
#pragma unroll
          for (int e = 0; e < VEC; ++e) d[i][e] = dv[e] + fmaf(d[i][e], pre_rstd, fmaf(hat[i][e], c2, c1));
        }
      } else {
#pragma unroll
        for (int i = 0; i < VPT; ++i) dh.values(i, d[i]);
      }
      // (what stands past the row in d meets w = 0, or is not stored)
      const float post_shift = -post_mean * post_rstd;
      float s[2] = {0.f, 0.f};
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        float out[VEC];
#pragma unroll
        for (int e = 0; e < VEC; ++e) out[e] = a.scale * d[i][e];
        Row::store(a.dh + row * cols, i, t, cols, out);
        f.normalised(i, post_rstd, post_shift, hat[i]);
#pragma unroll
        for (int e = 0; e < VEC; ++e) {
          sums[0][i][e] += d[i][e];
          sums[1][i][e] = fmaf(d[i][e], hat[i][e], sums[1][i][e]);
          d[i][e] *= w[i][e];
          if constexpr (POST) {
            s[0] += d[i][e];
            s[1] = fmaf(d[i][e], hat[i][e], s[1]);
          }
        }
      }
      if constexpr (POST) {
        row_allreduce_sum<TPR, WG, 2>(s, slots, phase);
        const float c1 = -post_rstd * (s[0] * inv_n), c2 = -post_rstd * (s[1] * inv_n);
#pragma unroll
        for (int i = 0; i < VPT; ++i)
#pragma unroll
          for (int e = 0; e < VEC; ++e) d[i][e] = fmaf(d[i][e], post_rstd, fmaf(hat[i][e], c2, c1));
      }
#pragma unroll
      for (int i = 0; i < VPT; ++i) Row::store(a.df + row * cols, i, t, cols, d[i]);
      if constexpr (PREFETCH) {
        f = f_next;
        dh = dh_next;
        if constexpr (PRE) {
          dx = dx_next;
          h = h_next;
          pre_mean = pre_mean_next;
          pre_rstd = pre_rstd_next;
        }
        if constexpr (POST) {
          post_mean = post_mean_next;
          post_rstd = post_rstd_next;
        }
      }
    }
    const int64_t item = gate_row * a.pieces + piece;
    if (POST || a.gate) flush(0, a.gate_sums + item * cols, a.gates * a.pieces * cols, own);
  }
  const int64_t groups = gridDim.x * gridDim.y;
  if constexpr (PRE) flush(2, a.pre_sums + static_cast<int64_t>(group) * cols, groups * cols, false);
}

// The backward of rows that registers do not hold, a workgroup a row at a time: df and dh.  f in the type T.
template <typename T, int WG>
__global__ __launch_bounds__(WG) void residual_norm_bwd_wide_kernel(const ResidualNormBwd<T> a) {
  __shared__ float slots[2 * 2 * (WG / kWave)];
  int phase = 0;
  const int cols = a.cols;
  const float inv_n = 1.0f / static_cast<float>(cols);
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const int64_t at = row * cols;
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
      phase ^= 1;
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
}

// ... and after the column sums, which need d too: a thread a column of one piece of one gate row's rows.
template <typename T, int WG>
__global__ __launch_bounds__(WG) void residual_norm_bwd_columns_kernel(const ResidualNormBwd<T> a) {
  const int c = static_cast<int>(blockIdx.x) * WG + threadIdx.x;
  if (c >= a.cols) return;
  const uint32_t piece = blockIdx.y, group = blockIdx.z * gridDim.y + blockIdx.y, groups = gridDim.y * gridDim.z;
  const int64_t first = static_cast<int64_t>(blockIdx.z) * a.gates_per_group;
  const int64_t last = min(first + a.gates_per_group, a.gates);
  float sg = 0.f, sb = 0.f;
  for (int64_t gate_row = first; gate_row < last; ++gate_row) {
    const int64_t base = gate_row * static_cast<int64_t>(a.gate_rows) + piece * a.piece_start;
    const int64_t end = min((gate_row + 1) * static_cast<int64_t>(a.gate_rows), base + a.piece_span);
    float sd = 0.f, sdf = 0.f;
    for (int64_t row = base; row < end; ++row) {
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
    const int64_t item = gate_row * a.pieces + piece;
    if (a.gate_sums) {
      a.gate_sums[item * a.cols + c] = sd;
      a.gate_sums[(a.gates * a.pieces + item) * a.cols + c] = sdf;
    }
  }
  if (a.pre_sums) {
    a.pre_sums[static_cast<int64_t>(group) * a.cols + c] = sg;
    a.pre_sums[static_cast<int64_t>(groups + group) * a.cols + c] = sb;
  }
}

// Stage 2: from the workgroups' column sums to the parameters' gradients, in a fixed order.  A workgroup has 32 columns and
// 32 lanes for each; blockIdx.y: 0 the gate and the post norm, 1 the pre norm; blockIdx.z: a block of gate rows.  The lanes are
// `split` to a gate row, whose pieces they share, so that many gate rows are walked side by side, and the pieces of one are; whole
// gate rows go eight to a lane at once.
template <typename T>
__global__ __launch_bounds__(1024) void residual_norm_finish_kernel(const ResidualNormFinish<T> a) {
  __shared__ float tile[2][32][33];
  const int cx = threadIdx.x % 32, ly = threadIdx.x / 32;
  const int64_t cols = a.cols, c = a.first_column + static_cast<int64_t>(blockIdx.x) * 32 + cx;
  const bool mine = c < cols;
  // The sums of two arrays' rows first, first + step, ...: eight loads on their way at once, those past the end repeating the
  // last row, to no effect.
  auto walk = [&](const float* p0, const float* p1, int64_t first, int64_t count, int64_t step, float& s0, float& s1) {
    s0 = s1 = 0.f;
    if (!mine) return;
    for (int64_t i = first; i < count; i += 4 * step) {
      float v0[4], v1[4];
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int64_t at = min(i + k * step, count - 1) * cols;
        v0[k] = p0[at];
        v1[k] = p1[at];
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        s0 += i + k * step < count ? v0[k] : 0.f;
        s1 += i + k * step < count ? v1[k] : 0.f;
      }
    }
  };
  // Lanes 0 .. n - 1, n a power of two, of each `n` lanes added into the first one's.
  auto add_lanes = [&](int n, float& s0, float& s1) {
    tile[0][ly][cx] = s0;
    tile[1][ly][cx] = s1;
    for (int w = n / 2; w > 0; w /= 2) {
      __syncthreads();
      if (ly % n < w) {
        tile[0][ly][cx] += tile[0][ly + w][cx];
        tile[1][ly][cx] += tile[1][ly + w][cx];
      }
    }
    __syncthreads();
    s0 = tile[0][ly][cx];
    s1 = tile[1][ly][cx];
    __syncthreads();
  };
  // Over all 32 lanes, to lane 0: the two of a wave, then the sixteen waves.
  auto add_all = [&](float& s0, float& s1) {
    s0 += __shfl_xor(s0, 32);
    s1 += __shfl_xor(s1, 32);
    if (ly % 2 == 0) {
      tile[0][ly / 2][cx] = s0;
      tile[1][ly / 2][cx] = s1;
    }
    __syncthreads();
    if (ly != 0) return;
    s0 = s1 = 0.f;
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      s0 += tile[0][k][cx];
      s1 += tile[1][k][cx];
    }
  };
  auto put = [&](void* out, int64_t at, float v) {
    if (a.grad_f32) static_cast<float*>(out)[at] = v;
    else static_cast<T*>(out)[at] = from_float<T>(v);
  };
  if (a.first + blockIdx.y == 1) {
    if (blockIdx.z > 0) return;
    float g, b;
    walk(a.pre_sums + c, a.pre_sums + a.groups * cols + c, ly, a.groups, 32, g, b);
    add_all(g, b);
    if (ly == 0 && mine) {
      put(a.dpre_gamma, c, g);
      put(a.dpre_beta, c, b);
    }
    return;
  }
  const float pg = a.post_gamma && mine ? to_float(a.post_gamma[c]) : 1.f;
  const float pb = a.post_gamma && mine ? to_float(a.post_beta[c]) : 0.f;
  const int at_once = 32 / a.split;  // gate rows
  const int64_t second = a.gates * a.pieces * cols;
  float sg = 0.f, sb = 0.f;
  const int64_t gate_first = static_cast<int64_t>(blockIdx.z) * a.gates_per_block;
  const int64_t gate_last = min(gate_first + a.gates_per_block, a.gates);
  if (a.pieces == 1) {
    for (int64_t gate0 = gate_first + ly; mine && gate0 < gate_last; gate0 += 8 * 32) {
      float d[8], df[8], g[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {  // (past the last gate row the last one again, to no effect)
        const int64_t at = min(gate0 + 32 * k, gate_last - 1) * cols + c;
        d[k] = a.gate_sums[at];
        df[k] = a.gate_sums[second + at];
        g[k] = a.gate ? to_float(a.gate[at]) : 1.f;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (gate0 + 32 * k >= gate_last) continue;
        if (a.gate) put(a.dgate, (gate0 + 32 * k) * cols + c, pg * df[k] + pb * d[k]);
        sg += g[k] * df[k];
        sb += g[k] * d[k];
      }
    }
  } else {
    for (int64_t gate0 = gate_first; gate0 < gate_last; gate0 += at_once) {
      const int64_t gate_row = gate0 + ly / a.split;
      const bool here = gate_row < gate_last;
      float d, df;
      const float* const p = a.gate_sums + gate_row * a.pieces * cols + c;
      walk(p, p + second, ly % a.split, here ? a.pieces : 0, a.split, d, df);
      if (a.split == 32) add_all(d, df);  // (of the one gate row)
      else if (a.split > 1) add_lanes(a.split, d, df);
      if (here && mine && ly % a.split == 0) {
        float g = 1.f;
        if (a.gate) {
          put(a.dgate, gate_row * cols + c, pg * df + pb * d);
          g = to_float(a.gate[gate_row * cols + c]);
        }
        sg += g * df;
        sb += g * d;
      }
    }
  }
  if (!a.post_gamma) return;
  if (a.split < 32 || a.pieces == 1) add_all(sg, sb);
  if (ly != 0 || !mine) return;
  if (a.post_sums) {
    a.post_sums[blockIdx.z * cols + c] = sg;
    a.post_sums[(gridDim.z + blockIdx.z) * cols + c] = sb;
  } else {
    put(a.dpost_gamma, c, sg);
    put(a.dpost_beta, c, sb);
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
  // How a row of `chunks` chunks is laid over threads: as few chunks to a thread as there are threads for, which takes the fewest
  // instructions from a row's first to its last, since few rows, or few to a workgroup, is what a training step has; but
  //  - forward, from 8192 rows on, half the threads with two chunks each: at the rate of memory, what is on its way counts
  //    (bf16, us, one chunk | two: (2048, 2048) 9.1 | 11.0, (2048, 4096) 13.1 | 16.9, (8192, 4096) 56.8 | 52.8,
  //    (16384, 1024) 24.9 | 23.4, (16384, 2048) 53.4 | 51.5, (16384, 4096) 110 | 103)
  //  - backward, 65 to 128 chunks, one wave: no barriers, and a workgroup's rows share their column sums (bf16 1024 columns, two
  //    waves | one: 2048 rows 20.4 | 16.0, 16384 rows 51.0 | 50.1)
  //  - past 512 chunks two to a thread: 1024 threads have too few registers each (bf16 (2048, 8192) backward 58.0 | 54.8).
  // Past 1024 chunks nothing is left but two to each of 1024 threads, whose 128 registers do not hold a row of the backward with both
  // norms: bf16 spills 320 to 364 bytes a lane (off the chunks 472 to 532), fp32 none to 44 (172 to 192), the bf16 forward 52 to 168.
  // bf16 (2048, 12288) forward 52 us, with f8 and x8 95, backward 273, of 41, 51 and 61 by its bytes; fp32 (2048, 6144) backward 70 of 61.
  static bool pick_shape(bool forward, int64_t rows, int64_t chunks, Shape* s) {
    const bool two = forward ? rows >= 8192 : false;
    if (chunks <= 16) *s = {16, 1};
    else if (chunks <= 32) *s = {32, 1};
    else if (chunks <= 64) *s = {64, 1};
    else if (chunks <= 128) *s = two || !forward ? Shape{64, 2} : Shape{128, 1};
    else if (chunks <= 256) *s = two ? Shape{128, 2} : Shape{256, 1};
    else if (chunks <= 512) *s = two ? Shape{256, 2} : Shape{512, 1};
    else if (chunks <= 1024) *s = {512, 2};
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

  template <int TPR, int VPT, bool ANY, bool KEEP>
  static int launch_fwd(const ResidualNormFwd<T>& a, hipStream_t stream) {
    constexpr int WG = TPR <= 64 ? 256 : TPR;
    constexpr int RPW = WG / TPR;
    const int64_t want = ceil_div(a.rows, RPW);
    const int64_t cap = static_cast<int64_t>(device_info().cu_count) * (2048 / WG);
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(std::min(want, cap))), dim3(WG), 0, stream, a);
    };
    if (a.post_gamma && a.pre_gamma) launch(residual_norm_fwd_kernel<T, TPR, VPT, WG, ANY, true, true, KEEP>);
    else if (a.post_gamma) launch(residual_norm_fwd_kernel<T, TPR, VPT, WG, ANY, true, false, KEEP>);
    else if (a.pre_gamma) launch(residual_norm_fwd_kernel<T, TPR, VPT, WG, ANY, false, true, KEEP>);
    else launch(residual_norm_fwd_kernel<T, TPR, VPT, WG, ANY, false, false, KEEP>);
    MG_LAUNCH_CHECK();
    return MG_OK;
  }

#define MG_RESIDUAL_NORM_FWD_SHAPES(CALL) \
  CALL(16, 1);                            \
  CALL(32, 1);                            \
  CALL(64, 1);                            \
  CALL(64, 2);                            \
  CALL(128, 1);                           \
  CALL(128, 2);                           \
  CALL(256, 1);                           \
  CALL(256, 2);                           \
  CALL(512, 1);                           \
  CALL(512, 2);                           \
  CALL(1024, 2)
#define MG_RESIDUAL_NORM_BWD_SHAPES(CALL) \
  CALL(16, 1);                            \
  CALL(32, 1);                            \
  CALL(64, 1);                            \
  CALL(64, 2);                            \
  CALL(256, 1);                           \
  CALL(512, 1);                           \
  CALL(512, 2);                           \
  CALL(1024, 2)

  template <bool ANY>
  static int dispatch_fwd(Shape s, const ResidualNormFwd<T>& a, hipStream_t stream) {
#define MG_CASE(TPR_, VPT_)           \
  if (s.tpr == TPR_ && s.vpt == VPT_) \
  return a.f8 || a.x8 ? launch_fwd<TPR_, VPT_, ANY, true>(a, stream) : launch_fwd<TPR_, VPT_, ANY, false>(a, stream)
    MG_RESIDUAL_NORM_FWD_SHAPES(MG_CASE);
#undef MG_CASE
    return fail(MG_ERR_UNSUPPORTED, "residual_norm_fwd: no kernel for row shape (%d, %d)", s.tpr, s.vpt);
  }

  static int fwd(const ResidualNormFwd<T>& a, int dtype, hipStream_t stream) {
    Shape s;
    if (a.cols >= VEC && pick_shape(true, a.rows, ceil_div(a.cols, VEC), &s)) {
      if (aligned(a.cols, {a.f, a.h, a.gate, a.post_gamma, a.post_beta, a.pre_gamma, a.pre_beta, a.h_out, a.x}))
        return dispatch_fwd<false>(s, a, stream);
      return dispatch_fwd<true>(s, a, stream);
    }
    if (a.f8) MG_TRY(act8_store(a.f, a.f8, a.rows, a.cols, false, dtype, stream));
    hipLaunchKernelGGL((residual_norm_fwd_wide_kernel<T, 1024>), dim3(static_cast<unsigned>(std::min(a.rows, kWideGroups))), dim3(1024), 0,
                       stream, a);
    MG_LAUNCH_CHECK();
    if (a.x8) MG_TRY(act8_store(a.x, a.x8, a.rows, a.cols, false, dtype, stream));
    return MG_OK;
  }

  // Splits the rows over at most `most` workgroups of `rows_at_once` rows: fewer gate rows than workgroups are cut into
  // pieces, more are dealt out whole.  (Counts between do not fill the device: 129 to 255 gate rows are a workgroup each, 257 are
  // two to a workgroup.  us a million values, bf16 (gates 512, 384) with 128 | 129 | 200 | 256 | 257 | 300 gate rows 2.8 | 3.6 | 2.7 |
  // 2.7 | 3.4 | 3.1; pieces are whole multiples of rows_at_once, so (2587, 1001) with 13 gate rows of 199 is 169 workgroups.)
  static int64_t partition(ResidualNormBwd<T>& a, int64_t most, int rows_at_once, bool interleave) {
    a.own = 0;
    const int64_t per_gate = std::max<int64_t>(1, std::min(most / a.gates, ceil_div(a.gate_rows, rows_at_once)));
    a.gates_per_group = ceil_div(a.gates, most);
    if (a.gates_per_group > 1 || per_gate == 1) {
      a.pieces = 1;
      a.piece_start = 0;
      a.piece_span = a.gate_rows;
      // (us by workgroups | rows in flight, 384 columns of 16384 rows in bf16, a gate row for every 64 rows, which leaves seven of eight
      // with nothing, 22.9 | 58.4, for every 16, half of them, 28.3 | 27.6, for every 4 50.8 | 34.5, for each 161 | 61)
      a.own = rows_at_once > 1 && a.gates * (a.gate_rows < rows_at_once ? 8 : 2) >= most * rows_at_once;
      a.row_step = a.own ? 1 : rows_at_once;
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

  // Takes the column sums' scratch for `groups` workgroups.
  static int take_sums(ResidualNormBwd<T>& a, int64_t groups, Scratch& scratch) {
    const int64_t gate = a.post_gamma || a.gate ? 2 * a.gates * a.pieces * a.cols : 0;
    const int64_t pre = a.pre_gamma ? 2 * groups * a.cols : 0;
    const int64_t post = a.post_gamma && finish_blocks(a) > 1 ? 2 * finish_blocks(a) * a.cols : 0;
    // (the second array starts where float4s may)
    const int64_t at = ceil_div(gate, 4) * 4;
    MG_TRY(scratch.take(std::max<int64_t>(1, at + pre + post) * static_cast<int64_t>(sizeof(float))));
    a.gate_sums = gate ? scratch.as<float>() : nullptr;
    a.pre_sums = pre ? scratch.as<float>() + at : nullptr;
    a.post_sums = post ? scratch.as<float>() + at + pre : nullptr;
    return MG_OK;
  }

  // Blocks of gate rows that the second stage is dealt out in; pieces are summed in one.
  // (one block: 640 us of (16384, 384) with a gate a token instead of 61)
  static constexpr int64_t kGatesPerBlock = 256;
  static int64_t finish_blocks(const ResidualNormBwd<T>& a) {
    return a.pieces == 1 ? std::min<int64_t>(65535, ceil_div(a.gates, kGatesPerBlock)) : 1;
  }

  static int finish(const ResidualNormBwd<T>& a, int64_t groups, void* const (&out)[4], hipStream_t stream) {
    if (!a.gate_sums && !a.pre_sums) return MG_OK;
    ResidualNormFinish<T> f{};
    f.gate_sums = a.gate_sums;
    f.pre_sums = a.pre_sums;
    f.gate = a.gate;
    f.post_gamma = a.post_gamma;
    f.post_beta = a.post_beta;
    f.dgate = a.dgate;
    f.dpost_gamma = out[0];
    f.dpost_beta = out[1];
    f.dpre_gamma = out[2];
    f.dpre_beta = out[3];
    f.cols = a.cols;
    f.groups = groups;
    f.gates = a.gates;
    f.gates_per_block = ceil_div(a.gates, finish_blocks(a));
    f.post_sums = a.post_sums;
    f.pieces = a.pieces;
    f.grad_f32 = a.grad_f32;
    f.split = 32;
    while (f.split > 1 && (32 / f.split) < a.gates) f.split /= 2;
    f.first = a.gate_sums ? 0 : 1;
    const unsigned jobs = (a.gate_sums ? 1u : 0u) + (a.pre_sums ? 1u : 0u), blocks = static_cast<unsigned>(finish_blocks(a));
    const dim3 both(1, jobs, a.gate_sums ? blocks : 1u);
    MG_TRY(launch_finish(f, both, stream));
    if (!a.post_sums) return MG_OK;
    // The post norm's gradients from the blocks', as the pre norm's come from the workgroups'.
    f.pre_sums = a.post_sums;
    f.groups = blocks;
    f.dpre_gamma = out[0];
    f.dpre_beta = out[1];
    f.first = 1;
    return launch_finish(f, dim3(1), stream);
  }
  // A workgroup of 1024 threads for 32 columns.  A launch counts its threads in 32 bits, so 2^25 columns a launch.
  static int launch_finish(ResidualNormFinish<T> f, dim3 grid, hipStream_t stream) {
    constexpr int64_t kColumns = 1 << 25;
    for (f.first_column = 0; f.first_column < f.cols; f.first_column += kColumns) {
      grid.x = static_cast<unsigned>(ceil_div(std::min(f.cols - f.first_column, kColumns), 32));
      hipLaunchKernelGGL((residual_norm_finish_kernel<T>), grid, dim3(1024), 0, stream, f);
      MG_LAUNCH_CHECK();
    }
    return MG_OK;
  }

  template <int TPR, int VPT, bool ANY, bool F8>
  static int launch_bwd(ResidualNormBwd<T> a, void* const (&out)[4], hipStream_t stream) {
    constexpr int WG = TPR <= 64 ? 512 : TPR;
    constexpr int RPW = WG / TPR;
    const bool interleave = a.rows * a.cols * static_cast<int64_t>(sizeof(T)) >= (int64_t{16} << 20);
    // Eight waves a CU: each workgroup has its parameters to load and its sums to write, and the next row is on its way anyway
    // (us with 4 | 8 | 16 waves: (4096, 768) fp16 31 | 26 | 34, (16384, 384) bf16 - | 22 | 26, (8192, 4096) bf16 - | 79 | 88).
    const int64_t most = static_cast<int64_t>(device_info().cu_count) * std::max(1, 8 * kWave / WG);
    const int64_t groups = partition(a, most, RPW, interleave);
    Scratch sums;
    MG_TRY(take_sums(a, groups, sums));
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(a.pieces, static_cast<unsigned>(groups / a.pieces)), dim3(WG), 0, stream, a);
    };
    if (a.post_gamma && a.pre_gamma) launch(residual_norm_bwd_kernel<T, TPR, VPT, WG, ANY, F8, true, true>);
    else if (a.post_gamma) launch(residual_norm_bwd_kernel<T, TPR, VPT, WG, ANY, F8, true, false>);
    else if (a.pre_gamma) launch(residual_norm_bwd_kernel<T, TPR, VPT, WG, ANY, F8, false, true>);
    else launch(residual_norm_bwd_kernel<T, TPR, VPT, WG, ANY, F8, false, false>);
    MG_LAUNCH_CHECK();
    return finish(a, groups, out, stream);
  }

  template <bool ANY>
  static int dispatch_bwd(Shape s, const ResidualNormBwd<T>& a, void* const (&out)[4], hipStream_t stream) {
#define MG_CASE(TPR_, VPT_)           \
  if (s.tpr == TPR_ && s.vpt == VPT_) \
  return a.f8 ? launch_bwd<TPR_, VPT_, ANY, true>(a, out, stream) : launch_bwd<TPR_, VPT_, ANY, false>(a, out, stream)
    MG_RESIDUAL_NORM_BWD_SHAPES(MG_CASE);
#undef MG_CASE
    return fail(MG_ERR_UNSUPPORTED, "residual_norm_bwd: no kernel for row shape (%d, %d)", s.tpr, s.vpt);
  }
#undef MG_RESIDUAL_NORM_FWD_SHAPES
#undef MG_RESIDUAL_NORM_BWD_SHAPES

  // out: dpost_gamma, dpost_beta, dpre_gamma, dpre_beta.
  static int bwd(ResidualNormBwd<T> a, void* const (&out)[4], int dtype, hipStream_t stream) {
    Shape s;
    if (a.cols >= VEC && pick_shape(false, a.rows, ceil_div(a.cols, VEC), &s)) {
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
    hipLaunchKernelGGL((residual_norm_bwd_wide_kernel<T, 1024>), dim3(static_cast<unsigned>(std::min(a.rows, kWideGroups))), dim3(1024), 0,
                       stream, a);
    MG_LAUNCH_CHECK();
    const int64_t blocks = ceil_div(a.cols, 256);
    const int64_t most = std::max<int64_t>(1, ceil_div(static_cast<int64_t>(device_info().cu_count) * 4, blocks));
    const int64_t groups = partition(a, std::min<int64_t>(most, 65535), 1, false);
    MG_TRY(take_sums(a, groups, part));
    hipLaunchKernelGGL((residual_norm_bwd_columns_kernel<T, 256>),
                       dim3(static_cast<unsigned>(blocks), a.pieces, static_cast<unsigned>(groups / a.pieces)), dim3(256), 0,
                       stream, a);
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
