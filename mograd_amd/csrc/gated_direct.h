// A gated Linear layer of few rows (or few tiles), its operands read from memory straight into the matrix cores' registers.
//
// What bounds a few tokens' pass is the weights' way from memory, each read once: nothing of them can be shared, so nothing goes
// through LDS.  A workgroup takes 16 columns of y, that is 16 rows of either weight, and 16 MT rows of x; its four waves divide K
// between them in units of four runs of 64 bytes, neighbouring waves neighbouring units, and the waves' sums meet in LDS, in one order.
// A matrix instruction takes 16 rows of a weight, 16 of x and 64 bytes of k of each: sixteen bytes a lane, lane l holding row l % 16
// and bytes 16 (l / 16) on, so that a load instruction takes whole runs.  (fp32: four instructions of 4 k each, k = 4 (l / 16) + j for
// j = 0 .. 3; both operands alike, so the order in which k is added is all that it changes.)  The next unit is on its way while one is
// multiplied: 12 KB a wave, 8 to 16 waves a CU.  (8, 8192 <- 4096) bf16 29 us, 4.6 TB/s; in 128 x 128 tiles 40.  More waves to a
// workgroup are 7 % faster there and slower for shorter rows ((10, 10336 <- 120) 3.3 us, with 8 waves 4.6).
#pragma once

#include "gated_linear.h"
#include "mg_rows.h"

namespace mg {

template <typename T>
struct GatedDirect {
  const T *x, *w, *bias;
  T *y, *gu;
  int M, F, K, tiles_f;
  int gate;
};

typedef float gated_f4 __attribute__((ext_vector_type(4)));

template <typename T>
struct GatedMma;
template <>
struct GatedMma<bf16_t> {
  static __device__ __forceinline__ gated_f4 run(uint4 a, uint4 b, gated_f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(gemm_bf16x8, a), __builtin_bit_cast(gemm_bf16x8, b), c, 0, 0, 0);
  }
};
template <>
struct GatedMma<f16_t> {
  static __device__ __forceinline__ gated_f4 run(uint4 a, uint4 b, gated_f4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(gemm_f16x8, a), __builtin_bit_cast(gemm_f16x8, b), c, 0, 0, 0);
  }
};
template <>
struct GatedMma<float> {
  static __device__ __forceinline__ gated_f4 run(uint4 a, uint4 b, gated_f4 c) {
    const uint32_t av[4] = {a.x, a.y, a.z, a.w}, bv[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(av[j]), __uint_as_float(bv[j]), c, 0, 0, 0);
    return c;
  }
};

// `valid` of the elements at p, up to sixteen bytes of them, and zeros behind.
__device__ __forceinline__ uint4 gated_gather(const float* p, int valid) {
  const float v[4] = {p[0], valid > 1 ? p[1] : 0.f, valid > 2 ? p[2] : 0.f, valid > 3 ? p[3] : 0.f};
  return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}
template <typename T>
__device__ __forceinline__ uint4 gated_gather(const T* p, int valid) {
  return gemm16_gather8(p, valid);
}

constexpr int kGatedDirectWaves = 4, kGatedDirectSteps = 4;  // waves; 64-byte steps of a unit
template <typename T, int MT>
__global__ __launch_bounds__(kGatedDirectWaves * 64) void gated_direct_kernel(GatedDirect<T> p) {
  constexpr int NW = kGatedDirectWaves, U = kGatedDirectSteps;
  constexpr int VEC = WideVec<T>::value, KS = 4 * VEC;  // elements of a lane's chunk, and of an instruction's k
  constexpr int NB = 2 + MT;                            // tiles of a step: gate, up, x
  __shared__ gated_f4 sums[NW][2 * MT][kWave];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave;
  const int f0 = static_cast<int>(blockIdx.x % p.tiles_f) * 16, m0 = static_cast<int>(blockIdx.x / p.tiles_f) * 16 * MT;
  const int64_t K = p.K;
  const T* base[NB];  // this lane's row of each tile; rows past the edge are the last one, and never stored
  const int64_t row = min(f0 + lane % 16, p.F - 1);
  base[0] = p.w + row * K;
  base[1] = p.w + (p.F + row) * K;
#pragma unroll
  for (int i = 0; i < MT; ++i) base[2 + i] = p.x + static_cast<int64_t>(min(m0 + 16 * i + lane % 16, p.M - 1)) * K;

  gated_f4 acc[2][MT];
#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) acc[i][j] = gated_f4{0.f, 0.f, 0.f, 0.f};

  const int at = lane / 16 * VEC;
  const int whole = p.K / (U * KS);  // units inside the rows
  uint4 v[2][U][NB];
  auto fetch = [&](int buf, int unit) {
    const int64_t k = static_cast<int64_t>(unit) * (U * KS) + at;
#pragma unroll
    for (int s = 0; s < U; ++s)
#pragma unroll
      for (int i = 0; i < NB; ++i) {
        const gemm_u4_any r = *reinterpret_cast<const gemm_u4_any*>(base[i] + k + s * KS);
        v[buf][s][i] = make_uint4(r[0], r[1], r[2], r[3]);
      }
  };
  auto multiply = [&](int buf) {
#pragma unroll
    for (int s = 0; s < U; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int j = 0; j < MT; ++j) acc[i][j] = GatedMma<T>::run(v[buf][s][i], v[buf][s][2 + j], acc[i][j]);
  };
  // Two units a turn, so that the buffers have fixed names.
  int unit = wave;
  if (unit < whole) fetch(0, unit);
  for (; unit < whole; unit += 2 * NW) {
    if (unit + NW < whole) fetch(1, unit + NW);
    multiply(0);
    if (unit + 2 * NW < whole) fetch(0, unit + 2 * NW);
    if (unit + NW < whole) multiply(1);
  }
  // What is left of the rows, a step at a time; chunks over their end element by element, zeros behind.
  for (int64_t k0 = static_cast<int64_t>(whole) * (U * KS) + static_cast<int64_t>(wave) * KS; k0 < K; k0 += NW * KS) {
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int64_t k = k0 + at;
      v[0][0][i] = make_uint4(0, 0, 0, 0);
      if (k < K) v[0][0][i] = gated_gather(base[i] + k, static_cast<int>(min(K - k, static_cast<int64_t>(VEC))));
    }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < MT; ++j) acc[i][j] = GatedMma<T>::run(v[0][0][i], v[0][0][2 + j], acc[i][j]);
  }

#pragma unroll
  for (int i = 0; i < 2; ++i)
#pragma unroll
    for (int j = 0; j < MT; ++j) sums[wave][i * MT + j][lane] = acc[i][j];
  __syncthreads();
  // A lane has four neighbouring columns of one row.
  for (int t = wave; t < MT; t += NW) {
    const int f = f0 + lane / 16 * 4, m = m0 + 16 * t + lane % 16;
    if (m >= p.M || f >= p.F) continue;
    gated_f4 g = sums[0][t][lane], u = sums[0][MT + t][lane];
#pragma unroll
    for (int n = 1; n < NW; ++n) g += sums[n][t][lane], u += sums[n][MT + t][lane];
    const int n = min(4, p.F - f);
    if (p.bias)
      for (int e = 0; e < n; ++e) g[e] += to_float(p.bias[f + e]), u[e] += to_float(p.bias[p.F + f + e]);
    T* const y = p.y + static_cast<int64_t>(m) * p.F + f;
    float out[4];
    gated_with(p.gate, [&](auto gate) {
#pragma unroll
      for (int e = 0; e < 4; ++e) out[e] = gated_act<sizeof(T) == 2, decltype(gate)::value>(g[e]) * u[e];
    });
    for (int e = 0; e < n; ++e) y[e] = from_float<T>(out[e]);
    if (p.gu) {
      T* const gu = p.gu + static_cast<int64_t>(m) * 2 * p.F + f;
      for (int e = 0; e < n; ++e) gu[e] = from_float<T>(g[e]), gu[p.F + e] = from_float<T>(u[e]);
    }
  }
}

}  // namespace mg
