// fp32 products on the 16-bit matrix cores: each operand as the sum of three bf16 numbers.
//
//   a = a0 + a1 + a2,  a0 = bf16(a), a1 = bf16(a - a0), a2 = bf16(a - a0 - a1): 24 bits, what fp32 has
//   a b = a0 b0 + (a0 b1 + a1 b0) + (a0 b2 + a1 b1 + a2 b0) + what is below 2^-24 of |a b|, left out
//
// Six products at sixteen times the rate of an fp32 one.  Every partial sum is an fp32 accumulator's, as there, six additions for 16 k.
// a - a0 and a - a0 - a1 are exact.  2-norm of the error, of the result's, here | with the fp32 instructions' kernels: a gated layer of
// (2048, 4096 <- 4096) 1.0e-6 | 1.15e-6, its dX 1.3e-6 | 1.15e-6, dW 6.6e-7 | 5.7e-7; of (16384, 1024 <- 384) 2.9e-7 | 3.5e-7, 6.6e-7 | 5.7e-7,
// 7.0e-7 | 9.4e-7; of (2048, 512 <- 784) 4.3e-7 | 5.0e-7, 4.7e-7 | 4.1e-7, 4.7e-7 | 3.4e-7.  (Without the last three of the six 4.4e-6.)  What
// bf16 cannot hold changes: an infinity, or a number that it rounds to one, from 3.3962e38 on, becomes NaN in all products that it is in, and
// of numbers below 2^-110 the last digits are lost.
//
// A workgroup of eight waves has 128 AI x 128 of the result, a wave 32 AI rows x 64 columns, in steps of 32 k.  The operands come through
// registers, where they are split, to LDS, three images a step of either operand in the layouts of gemm16_pipe_frag, two steps in LDS; the
// step after next is on its way from memory meanwhile.  They may lie at any address: the memory pipeline takes 16 bytes anywhere.
// Bound by the matrix cores and their power: (2048, 2 x 4096) <- 4096 takes 718 us with AI = 2, 191 TFLOP/s of fp32 and six times that of
// bf16, the matrix pipe 68 % busy at 1.6 GHz (AI = 1: 818 us, 56 %: LDS serves as many reads for half the products), against 1052 us of
// fp32 instructions, whose peak is 157 TFLOP/s.  No LDS bank conflicts.
#pragma once

#include "gemm_impl.h"

namespace mg {

constexpr int kSplitT = 128, kSplitBK = 32, kSplitThreads = 512;     // columns of a tile; AI times as many rows
constexpr int kSplitImage = kSplitT * kSplitBK * 2;                  // bytes of one bf16 image of B's step, and of 128 rows of A
template <int AI>
constexpr int kSplitLds = 2 * 3 * (AI + 1) * kSplitImage;           // two steps of three images of both operands: 96 or 144 KB

constexpr int64_t kSplitMost = 0x7fff0000LL;  // rows, columns and k: they are counted in 32 bits, with room to round up

// One product's arguments.
struct SplitProblem {
  const float *a, *b;
  float* c;         // (M, N), rows ldc apart; or, split along K, partial results (range, M, N)
  int M, N, K;
  int64_t lda, ldb, ldc;
  int tiles_m, tiles_n, k_per_split, splits;
  bool accumulate;  // c += (not split)
};

typedef float split_f4 __attribute__((ext_vector_type(4), aligned(4)));

// What a thread carries of an operand's step: eight consecutive elements along the contiguous axis, KC: row r = slot / 4, k = slot % 4 * 8;
// otherwise k-row slot / 16, rows slot % 16 * 8.  `row_of` maps a tile's row to the array's (KC), which clamps what is past the edge.
struct SplitChunk {
  float v[8];
};
__device__ __forceinline__ void split_load8(const float* p, int valid, SplitChunk& c) {
  if (valid >= 8) {
    const split_f4 lo = *reinterpret_cast<const split_f4*>(p), hi = *reinterpret_cast<const split_f4*>(p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) c.v[e] = lo[e], c.v[4 + e] = hi[e];
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) c.v[e] = e < valid ? p[e] : 0.f;
}
// Into the three images at `at`, where the chunk has position `pos`.
template <int ROWS>
__device__ __forceinline__ void split_store8(const SplitChunk& c, char* at, int pos) {
  uint32_t w[3][4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    float x = c.v[2 * e], y = c.v[2 * e + 1];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
      w[i][e] = bf16_pack2_rne(x, y);
      x -= __uint_as_float(w[i][e] << 16);
      y -= __uint_as_float(w[i][e] & 0xffff0000u);
    }
  }
#pragma unroll
  for (int i = 0; i < 3; ++i) *reinterpret_cast<uint4*>(at + i * (ROWS * kSplitBK * 2) + pos * 16) = make_uint4(w[i][0], w[i][1], w[i][2], w[i][3]);
}

// k-contiguous images of 32 k: four chunks a row, chunk c of row r at c ^ (r / 4 % 4), so that sixteen consecutive rows of a fragment's
// read, 64 bytes apart, fall on all banks.
template <bool KC, int ROWS>
__device__ __forceinline__ int split_position(int slot) {
  constexpr int CPK = ROWS / 8;
  if constexpr (KC) return slot / 4 * 4 + ((slot % 4) ^ (slot / 16 % 4));
  else return slot / CPK * CPK + ((slot % CPK) ^ gemm16_tr_swizzle<ROWS>(slot / CPK));
}
template <bool KC, int ROWS>
__device__ __forceinline__ uint4 split_frag(const char* at, int o_base, int ks, int lane) {
  if constexpr (KC) {
    const int r = o_base + lane % 32, g = ks * 2 + lane / 32;
    return *reinterpret_cast<const uint4*>(at + r * 64 + ((g ^ (r / 4 % 4)) * 16));
  } else {
    return gemm16_pipe_frag<false, kSplitBK, ROWS>(at, o_base, ks, lane);
  }
}

// The accumulators of a wave's 32 AI x 64 of the tile at (m0, n0), over k in [k_begin, k_end): acc[i][j] has rows 32 i and columns 32 j on.
// b_row (KC): the row of B of a tile's column.
template <int AI, bool A_KC, bool B_KC, typename BRow>
__device__ __forceinline__ void split_product(char* lds, const SplitProblem& p, int m0, int n0, int k_begin, int k_end, BRow&& b_row,
                                              floatx16 (&acc)[AI][2]) {
  constexpr int ROWS = AI * kSplitT, IMAGE_A = AI * kSplitImage, STEP = 3 * (IMAGE_A + kSplitImage);
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const int wm = wave / 2 * 32 * AI, wn = wave % 2 * 64;
#pragma unroll
  for (int i = 0; i < AI; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.f;
  const int steps = (k_end - k_begin + kSplitBK - 1) / kSplitBK;
  // this thread's chunks of either operand: where they start in the first step, what a step adds, how many elements are there
  const float *pa[AI], *pb;
  SplitChunk ca[AI], cb;
  auto slot_a = [](int i) { return i * kSplitThreads + static_cast<int>(threadIdx.x); };
  const int slot_b = threadIdx.x;
  constexpr int CPA = ROWS / 8, CPB = kSplitT / 8;
#pragma unroll
  for (int i = 0; i < AI; ++i) {
    const int slot = slot_a(i);
    if constexpr (A_KC) pa[i] = p.a + static_cast<int64_t>(min(m0 + slot / 4, p.M - 1)) * p.lda + k_begin + slot % 4 * 8;
    else pa[i] = p.a + static_cast<int64_t>(k_begin + slot / CPA) * p.lda + m0 + slot % CPA * 8;
  }
  if constexpr (B_KC) pb = p.b + b_row(slot_b / 4) * p.ldb + k_begin + slot_b % 4 * 8;
  else pb = p.b + static_cast<int64_t>(k_begin + slot_b / CPB) * p.ldb + n0 + slot_b % CPB * 8;
  const bool inside = (A_KC || m0 + ROWS <= p.M) && (B_KC || n0 + kSplitT <= p.N);  // no chunk of a whole step is cut off
  const int64_t step_a = A_KC ? kSplitBK : kSplitBK * p.lda, step_b = B_KC ? kSplitBK : kSplitBK * p.ldb;
  auto load = [&](int step) {
    const int k0 = k_begin + step * kSplitBK;
    if (inside && k0 + kSplitBK <= k_end) {
#pragma unroll
      for (int i = 0; i < AI; ++i) split_load8(pa[i] + step * step_a, 8, ca[i]);
      split_load8(pb + step * step_b, 8, cb);
      return;
    }
#pragma unroll
    for (int i = 0; i < AI; ++i) {
      const int slot = slot_a(i);
      split_load8(pa[i] + step * step_a, A_KC ? k_end - (k0 + slot % 4 * 8) : k0 + slot / CPA < k_end ? p.M - (m0 + slot % CPA * 8) : 0, ca[i]);
    }
    split_load8(pb + step * step_b, B_KC ? k_end - (k0 + slot_b % 4 * 8) : k0 + slot_b / CPB < k_end ? p.N - (n0 + slot_b % CPB * 8) : 0, cb);
  };
  auto put = [&](int copy) {
    char* const at = lds + copy * STEP;
#pragma unroll
    for (int i = 0; i < AI; ++i) split_store8<ROWS>(ca[i], at, split_position<A_KC, ROWS>(slot_a(i)));
    split_store8<kSplitT>(cb, at + 3 * IMAGE_A, split_position<B_KC, kSplitT>(slot_b));
  };
  load(0);
  put(0);
  if (steps > 1) load(1);
  for (int it = 0; it < steps; ++it) {
    __syncthreads();  // step `it` is in LDS, and nobody reads the other copy any more
    const char* const la = lds + (it & 1) * STEP;
    const char* const lb = la + 3 * IMAGE_A;
#pragma unroll
    for (int ks = 0; ks < kSplitBK / 16; ++ks) {
      uint4 fa[AI][3], fb[2][3];
#pragma unroll
      for (int t = 0; t < 3; ++t) {
#pragma unroll
        for (int i = 0; i < AI; ++i) fa[i][t] = split_frag<A_KC, ROWS>(la + t * IMAGE_A, wm + 32 * i, ks, lane);
#pragma unroll
        for (int j = 0; j < 2; ++j) fb[j][t] = split_frag<B_KC, kSplitT>(lb + t * kSplitImage, wn + 32 * j, ks, lane);
      }
      constexpr int kA[6] = {2, 1, 0, 1, 0, 0}, kB[6] = {0, 1, 2, 0, 1, 0};  // the smallest products first
#pragma unroll
      for (int t = 0; t < 6; ++t)
#pragma unroll
        for (int i = 0; i < AI; ++i)
#pragma unroll
          for (int j = 0; j < 2; ++j) acc[i][j] = GemmMma16<bf16_t>::run(fa[i][kA[t]], fb[j][kB[t]], acc[i][j]);
      if (ks == 0 && it + 1 < steps) {
        put((it + 1) & 1);
        if (it + 2 < steps) load(it + 2);
      }
    }
  }
}

// The work of workgroup `bid`: a tile (of a range of K), written as it lies in the registers, two runs of 128 bytes a store.
template <int AI, bool A_KC, bool B_KC, bool SPLIT_K>
__device__ __forceinline__ void split_block(char* lds, int bid, const SplitProblem& p) {
  const int tiles = p.tiles_m * p.tiles_n;
  int tile = bid, split = 0, batch, tm, tn;
  if constexpr (SPLIT_K) {
    if (!gemm_split_work(bid, tiles, p.splits, 1, tile, split, batch)) return;
  }
  gemm_tile_of_block(tile, p.tiles_m, p.tiles_n, tm, tn, !SPLIT_K);
  const int m0 = tm * AI * kSplitT, n0 = tn * kSplitT;
  const int k_begin = SPLIT_K ? split * p.k_per_split : 0, k_end = SPLIT_K ? min(p.K, k_begin + p.k_per_split) : p.K;
  floatx16 acc[AI][2];
  split_product<AI, A_KC, B_KC>(lds, p, m0, n0, k_begin, k_end, [&](int r) { return static_cast<int64_t>(min(n0 + r, p.N - 1)); }, acc);
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  float* const c = p.c + (SPLIT_K ? static_cast<int64_t>(split) * p.M * p.N : 0);
#pragma unroll
  for (int i = 0; i < AI; ++i)
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int col = n0 + wave % 2 * 64 + 32 * j + lane % 32;
      if (col >= p.N) continue;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int row = m0 + wave / 2 * 32 * AI + 32 * i + (r / 4) * 8 + (lane / 32) * 4 + r % 4;
        if (row >= p.M) continue;
        float* const at = c + static_cast<int64_t>(row) * (SPLIT_K ? p.N : p.ldc) + col;
        *at = !SPLIT_K && p.accumulate ? acc[i][j][r] + *at : acc[i][j][r];
      }
    }
}

// dW = dY^T X (its ranges of rows) and dX = dY W in one launch: workgroups [0, n_dw) take dW, whose ranges are the longer, the rest dX.
template <int AI, bool SPLIT_K>
__global__ __launch_bounds__(kSplitThreads) void split_linear_bwd_kernel(SplitProblem dw, SplitProblem dx, int n_dw) {
  __shared__ __attribute__((aligned(1024))) char lds[kSplitLds<AI>];
  const int bid = blockIdx.x;
  if (bid < n_dw) split_block<AI, false, false, SPLIT_K>(lds, bid, dw);
  else split_block<AI, true, false, false>(lds, bid - n_dw, dx);
}

}  // namespace mg
