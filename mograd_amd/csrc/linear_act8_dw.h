// dW = dY^T X' of a Linear layer whose input X' is kept in 8 bits (mg_act8.h), by 128 x 128 tiles of v_mfma_f32_32x32x16.
//
// Both operands lie along the rows of the batch, which the product sums over, and both are put into LDS as [row][column] of
// 16-bit values, from which the transposing reads take fragments (gemm16_pipe_frag).  X' goes from bytes to 16-bit values on its
// way through registers: q 2^k is a bf16 number, and an fp16 one of an fp16 tensor, so the product is that of the restored
// tensor to the bit, without the tensor: 33 / 32 bytes a value are read instead of one pass that writes two and another that
// reads them.  A conversion, a multiplication and half a packing a value, done once for the 128 columns of dY that meet it.
//
// fp32 dY is cut into three bf16 terms of 8 significant bits each, dY = a + b + c without a remainder from |dY| = 2^-110 on, and
// to bf16's least number, 2^-133, below (truncation, so that the largest finite values do not round to infinity; the matrix
// instructions multiply subnormal numbers as they are), and X' is exact in bf16, so three products accumulate in fp32 what one of fp32
// operands would, at 16 / 3 times the rate of the fp32 matrix instructions.
//
// Steps of 64 rows (fp32: 32), two copies in LDS, 64 KB: two workgroups a CU.  The rows of the step after next are requested
// into registers while the present step is multiplied, those of the next one converted and written.
#pragma once

#include "gemm_16bit_deep.h"
#include "linear_act8.h"
#include "mg_act8.h"
#include "mg_rows.h"

namespace mg {

template <typename T>
struct Act8DwShape {
  static constexpr bool kF32 = sizeof(T) == 4;
  using E = std::conditional_t<std::is_same_v<T, f16_t>, f16_t, bf16_t>;  // what is multiplied
  static constexpr int kTerms = kF32 ? 3 : 1, kRows = kF32 ? 32 : 64;     // rows of a step
  static constexpr int kImage = kRows * 256;                              // bytes of 128 columns
  static constexpr int kStep = (kTerms + 1) * kImage, kLds = 2 * kStep;
};

// The work of workgroup `bid`; `lds` is Act8DwShape<T>::kLds bytes on 1024.
template <typename T>
__device__ __forceinline__ void act8_dw_block(char* lds, int bid, const Act8Dw<T>& p) {
  using S = Act8DwShape<T>;
  using E = typename S::E;
  constexpr int VEC = 16 / sizeof(T), CPR = 128 / VEC;                  // 16-byte chunks of a row of dY
  constexpr int NA = S::kRows * CPR / 256, NB = S::kRows * 16 / 256;    // requests of a thread and step: 16 bytes of dY, 8 of q
  int tile, split = 0, batch;
  if (p.splits > 1) {
    if (!gemm_split_work(bid, p.tiles_n * p.tiles_k, p.splits, 1, tile, split, batch)) return;
  } else {
    tile = bid;
  }
  int tn, tk;
  gemm_tile_of_block(tile, p.tiles_n, p.tiles_k, tn, tk, p.splits <= 1);
  tn = __builtin_amdgcn_readfirstlane(tn), tk = __builtin_amdgcn_readfirstlane(tk);
  split = __builtin_amdgcn_readfirstlane(split);
  const int n0 = tn * 128, k0 = tk * 128;
  const int m_begin = split * p.rows_per_split, m_end = min(p.M, m_begin + p.rows_per_split);
  const int steps = (m_end - m_begin + S::kRows - 1) / S::kRows;
  const int t = threadIdx.x, wave = t / kWave, lane = t % kWave, wr = wave / 2, wc = wave % 2;
  const bool with_db = p.db_part != nullptr && tk == 0;

  struct Staged {
    uint4 a[NA];
    uint2 b[NB];
    uint32_t e[NB];
  };
  // Requests: byte offsets from a step's first row, which is a scalar.  Columns past an array are read from its last ones: those of
  // dY are put in their places in `put`, and what belongs to no column of the result is not stored.
  const int ac = t % CPR, acol = min(n0 + ac * VEC, p.N - VEC), past = n0 + ac * VEC - acol;
  const int bcol = min(k0 + t % 16 * 8, static_cast<int>(p.ldx) - 8);
  const uint32_t a_row = static_cast<uint32_t>(p.ldy * sizeof(T)), b_row = static_cast<uint32_t>(p.ldx), e_row = b_row / kAct8Block;
  const int ar = t / CPR, br = t / 16;  // the thread's first rows of a step
  uint32_t a_at[NA], b_at[NB], e_at[NB];
  auto places = [&](int last) {  // of a step whose last row is `last`: rows past the range repeat it, and become zeros in `put`
#pragma unroll
    for (int i = 0; i < NA; ++i)
      a_at[i] = static_cast<uint32_t>(min(ar + i * (256 / CPR), last)) * a_row + acol * static_cast<int>(sizeof(T));
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const uint32_t row = static_cast<uint32_t>(min(br + i * 16, last));
      b_at[i] = row * b_row + bcol;
      e_at[i] = row * e_row + bcol / kAct8Block;
    }
  };
  places(min(S::kRows, m_end - m_begin) - 1);
  auto request = [&](int step, Staged& r) {  // (in order: the short one comes last)
    if (step >= steps) return;
    const int64_t m0 = m_begin + step * S::kRows;
    if (m0 + S::kRows > m_end) places(m_end - 1 - static_cast<int>(m0));
    const char* const a0 = reinterpret_cast<const char*>(p.dy) + m0 * p.ldy * static_cast<int64_t>(sizeof(T));
    const uint8_t* const b0 = p.q + m0 * p.ldx;
    const uint8_t* const e0 = p.e + m0 * (p.ldx / kAct8Block);
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const gemm_u4_any v = *reinterpret_cast<const gemm_u4_any*>(a0 + a_at[i]);
      r.a[i] = make_uint4(v[0], v[1], v[2], v[3]);
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      r.b[i] = *reinterpret_cast<const uint2*>(b0 + b_at[i]);
      r.e[i] = e0[e_at[i]];
    }
  };
  // A chunk that was read `past` columns before its place, moved there, zeros behind (all of it, from VEC columns on).
  auto shifted = [&](uint4 v) {
    constexpr int PER_WORD = 4 / sizeof(T);
    uint32_t w[4] = {v.x, v.y, v.z, v.w};
    const int words = past / PER_WORD;
    if constexpr (PER_WORD == 2) {
#pragma unroll
      for (int i = 0; i < 4; ++i) w[i] = past & 1 ? w[i] >> 16 | (i < 3 ? w[i + 1] << 16 : 0u) : w[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = words & 2 ? (i < 2 ? w[i + 2] : 0u) : w[i];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = words & 1 ? (i < 3 ? w[i + 1] : 0u) : w[i];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = words >= 4 ? 0u : w[i];
    return make_uint4(w[0], w[1], w[2], w[3]);
  };
  float db[VEC];
#pragma unroll
  for (int v = 0; v < VEC; ++v) db[v] = 0.f;
  // What seldom is to be done to a staged step: zeros past the range's rows, dY's last columns to their places, the sums of dY.
  auto prepare = [&](Staged& r, int step) {
    const int left = m_end - m_begin - step * S::kRows;
    if (left < S::kRows) {
#pragma unroll
      for (int i = 0; i < NA; ++i)
        if (ar + i * (256 / CPR) >= left) r.a[i] = make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int i = 0; i < NB; ++i)
        if (br + i * 16 >= left) r.b[i] = make_uint2(0, 0), r.e[i] = 7;
    }
    if (n0 + 128 > p.N) {
#pragma unroll
      for (int i = 0; i < NA; ++i) r.a[i] = shifted(r.a[i]);
    }
    if (with_db) {
#pragma unroll
      for (int i = 0; i < NA; ++i) {
        const uint32_t w[4] = {r.a[i].x, r.a[i].y, r.a[i].z, r.a[i].w};
        float v[VEC];
        VecAny<T, VEC>::unpack(w, v);
#pragma unroll
        for (int k = 0; k < VEC; ++k) db[k] += v[k];
      }
    }
  };
  // Request i of dY, and of q, into copy `copy` of LDS.  Chunk c of row r stands at c ^ gemm16_tr_swizzle(r).
  auto put_a = [&](const Staged& r, int i, int copy) {
    char* const at = lds + copy * S::kStep;
    const int row = ar + i * (256 / CPR);
    if constexpr (!S::kF32) {
      *reinterpret_cast<uint4*>(at + row * 256 + (ac ^ gemm16_tr_swizzle<128>(row)) * 16) = r.a[i];
    } else {
      float v[4] = {__uint_as_float(r.a[i].x), __uint_as_float(r.a[i].y), __uint_as_float(r.a[i].z), __uint_as_float(r.a[i].w)};
      char* const to = at + row * 256 + (ac / 2 ^ gemm16_tr_swizzle<128>(row)) * 16 + ac % 2 * 8;
#pragma unroll
      for (int term = 0; term < 3; ++term) {
        uint32_t u[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          u[k] = __float_as_uint(v[k]);
          // (an infinity stays one: infinity - infinity would make it a NaN)
          if (term < 2) v[k] = (u[k] & 0x7fffffffu) == 0x7f800000u ? 0.f : v[k] - __uint_as_float(u[k] & 0xffff0000u);
        }
        *reinterpret_cast<uint2*>(to + term * S::kImage) =
            make_uint2(__builtin_amdgcn_perm(u[1], u[0], 0x07060302u), __builtin_amdgcn_perm(u[3], u[2], 0x07060302u));
      }
    }
  };
  auto put_b = [&](const Staged& r, int i, int copy) {
    const int row = br + i * 16, c = t % 16;
    const float scale = act8_scale(r.e[i]);
    const uint32_t q[2] = {r.b[i].x, r.b[i].y};
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      float x[4];
      act8_unpack4(q[j], scale, x);
      w[2 * j] = gemm16_pack2<E>(x[0], x[1]);
      w[2 * j + 1] = gemm16_pack2<E>(x[2], x[3]);
    }
    *reinterpret_cast<uint4*>(lds + copy * S::kStep + S::kTerms * S::kImage + row * 256 + (c ^ gemm16_tr_swizzle<128>(row)) * 16) =
        make_uint4(w[0], w[1], w[2], w[3]);
  };

  floatx16 acc[2][2];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  // Step in `copy` multiplied, the staged one put into the other copy meanwhile: between the matrix instructions of one group,
  // which occupy their pipe for 128 clocks, goes a part of the conversions, and the reads of the next group's fragments before.
  constexpr int GROUPS = S::kRows / 16 * S::kTerms;  // four matrix instructions each: (16 rows, term)
  static_assert(S::kF32 ? NA + NB <= GROUPS : NA <= GROUPS && NB <= GROUPS, "a part of the work to each group");
  auto multiply = [&](int copy, const Staged& r) {
    const char* const at = lds + copy * S::kStep;
    uint4 fa[2][2], fb[2][2];
    auto read = [&](int g) {
      const int ks = g / S::kTerms, term = g % S::kTerms;
#pragma unroll
      for (int i = 0; i < 2; ++i)
        fa[g % 2][i] = gemm16_pipe_frag<false, S::kRows, 128>(at + term * S::kImage, wr * 64 + i * 32, ks, lane);
      if (term == 0)
#pragma unroll
        for (int j = 0; j < 2; ++j)
          fb[ks % 2][j] = gemm16_pipe_frag<false, S::kRows, 128>(at + S::kTerms * S::kImage, wc * 64 + j * 32, ks, lane);
    };
    read(0);
#pragma unroll
    for (int g = 0; g < GROUPS; ++g) {
      if (g + 1 < GROUPS) read(g + 1);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) acc[i][j] = GemmMma16<E>::run(fa[g % 2][i], fb[g / S::kTerms % 2][j], acc[i][j]);
      if (g < NA) put_a(r, g, copy ^ 1);
      if constexpr (S::kF32) {
        if (g >= NA && g - NA < NB) put_b(r, g - NA, copy ^ 1);
      } else {
        if (g < NB) put_b(r, g, copy ^ 1);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  };

  Staged r0{}, r1{};
  request(0, r0);
  request(1, r1);
  prepare(r0, 0);
#pragma unroll
  for (int i = 0; i < NA; ++i) put_a(r0, i, 0);
#pragma unroll
  for (int h = 0; h < NB; ++h) put_b(r0, h, 0);
  request(2, r0);
  __syncthreads();
  // Step s is in copy s % 2; r1, r0 hold steps s + 1 and s + 2 before an even step.  (An odd number of steps ends on one of
  // zeros, as everything past the range is put.)
  for (int s = 0; s < steps; s += 2) {
    prepare(r1, s + 1);
    multiply(0, r1);
    request(s + 3, r1);
    __syncthreads();
    prepare(r0, s + 2);
    multiply(1, r0);
    request(s + 4, r0);
    __syncthreads();
  }
  __syncthreads();

  if (with_db) {
    float* const sums = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int v = 0; v < VEC; ++v) sums[t / CPR * 128 + ac * VEC + v] = db[v];
    __syncthreads();
    if (t < 128 && n0 + t < p.N) {
      float s = 0.f;
#pragma unroll
      for (int r = 0; r < 256 / CPR; ++r) s += sums[r * 128 + t];
      p.db_part[static_cast<int64_t>(split) * p.N + n0 + t] = s;
    }
    __syncthreads();
  }
  if (p.splits > 1) {
    floatx4* const dst = reinterpret_cast<floatx4*>(p.partial) +
                         ((static_cast<int64_t>(split) * p.tiles_n + tn) * p.tiles_k + tk) * (kG16PartialTile / 4) + wave * 1024 + lane;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const floatx4 v = {acc[i][j][4 * g], acc[i][j][4 * g + 1], acc[i][j][4 * g + 2], acc[i][j][4 * g + 3]};
          if (p.partial_stream) __builtin_nontemporal_store(v, dst + (i * 2 + j) * 256 + g * 64);
          else dst[(i * 2 + j) * 256 + g * 64] = v;
        }
    return;
  }
  if (S::kF32 || p.dw32) {
    float* out;
    if constexpr (S::kF32) out = p.dw;
    else out = p.dw32;
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        gemm16_write_f32(acc[i][j], out, p.N, p.K, p.K, n0 + wr * 64 + 32 * i, k0 + wc * 64 + 32 * j, lane);
    return;
  }
  if constexpr (!S::kF32) {
    const float no_bias[2] = {0.f, 0.f};
    uint16_t* const mine = reinterpret_cast<uint16_t*>(lds) + wave * 64 * kG16Stride;
    gemm16_write_tile<T, false, false>(acc, mine, no_bias, p.dw, nullptr, p.N, p.K, p.K, 0, 0, 0, 1, n0, k0, wr * 64, wc * 64, lane,
                                       GemmEpilogue<T>{nullptr, nullptr, 0});
  }
}

template <typename T>
__global__ __launch_bounds__(256, 2) void act8_dw_kernel(Act8Dw<T> p) {
  __shared__ __attribute__((aligned(1024))) char lds[Act8DwShape<T>::kLds];
  act8_dw_block<T>(lds, blockIdx.x, p);
}

// dW and dX = dY W of a 16-bit layer in one launch: the ranges of dW, which run longer, first, then the tiles of dX, which fill
// the CUs as those drain.  dX takes the tiles of gemm_16bit_deep.h, with the activation's bytes for its mask.
template <typename T, bool RELU>
__global__ __launch_bounds__(256, 2) void linear_act8_kernel(Act8Dw<T> dw, Gemm16Problem<T> dx, int n_dw) {
  using Plain = Gemm16Deep<1, 1, 1>;
  using S = std::conditional_t<RELU, Gemm16DeepMask8<Plain>, Plain>;
  constexpr int LDS = S::kLds > Act8DwShape<T>::kLds ? S::kLds : Act8DwShape<T>::kLds;
  __shared__ __attribute__((aligned(1024))) char lds[LDS];
  if (static_cast<int>(blockIdx.x) < n_dw) act8_dw_block<T>(lds, blockIdx.x, dw);
  else gemm16_deep_block<T, S, true, false, false, false>(lds, blockIdx.x - n_dw, dx);
}

// The same of an fp32 layer, dX by gemm32_pipe_work's TS x TS tiles.  These run longer and go first: a step of them waits for its
// copies more than it multiplies, and dW's workgroups use the pipe meanwhile.
template <int TS, bool RELU>
__global__ __launch_bounds__(256, 2) void linear_act8_f32_kernel(Act8Dw<float> dw, Gemm16Problem<float> dx, int n_dx) {
  constexpr int LDS = 4 * kGemm32PipeOperand<TS> > Act8DwShape<float>::kLds ? 4 * kGemm32PipeOperand<TS> : Act8DwShape<float>::kLds;
  __shared__ __attribute__((aligned(1024))) char lds[LDS];
  if (static_cast<int>(blockIdx.x) >= n_dx) act8_dw_block<float>(lds, blockIdx.x - n_dx, dw);
  else
    gemm32_pipe_work<true, false, false, false, TS, RELU>(lds, blockIdx.x, n_dx, dx.A, dx.B, nullptr, dx.C, nullptr, dx.M, dx.N, dx.K,
                                                          dx.lda, dx.ldb, dx.ldc, 0, 0, 0, dx.tiles_m, dx.tiles_n, 1, dx.K, n_dx, dx.ep,
                                                          dx.mask8, dx.mask8_ld);
}

// n_dx == 0: dW alone.
template <typename T>
int launch_linear_act8(const Act8Dw<T>& dw, const Gemm16Problem<T>* dx, int x_tile, int64_t n_dw, int64_t n_dx, hipStream_t stream) {
  if (n_dw + n_dx > 0xffffffffLL / 256) return fail(MG_ERR_INVALID, "linear_bwd_act8: too many output tiles");
  if (n_dx == 0) {
    hipLaunchKernelGGL((act8_dw_kernel<T>), dim3(static_cast<unsigned>(n_dw)), dim3(256), 0, stream, dw);
  } else {
    auto launch = [&](auto kernel, int64_t first) {
      hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(n_dw + n_dx)), dim3(256), 0, stream, dw, *dx, static_cast<int>(first));
    };
    if constexpr (sizeof(T) == 2) {
      if (dx->mask8) launch(linear_act8_kernel<T, true>, n_dw);
      else launch(linear_act8_kernel<T, false>, n_dw);
    } else if (x_tile == 128) {
      if (dx->mask8) launch(linear_act8_f32_kernel<128, true>, n_dx);
      else launch(linear_act8_f32_kernel<128, false>, n_dx);
    } else {
      if (dx->mask8) launch(linear_act8_f32_kernel<64, true>, n_dx);
      else launch(linear_act8_f32_kernel<64, false>, n_dx);
    }
  }
  MG_LAUNCH_CHECK();
  return MG_OK;
}

}  // namespace mg
