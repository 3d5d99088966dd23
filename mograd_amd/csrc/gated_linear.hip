// C ABI of the gated Linear layer: argument checks, the choice of kernels, the gradient of the gate.
#include "gated_linear.h"

#include <cmath>

#include "gated_direct.h"
#include "gemm_16bit_small.h"
#include "gemm_f32_split.h"
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

// fp32: both projections from three bf16 numbers a value (gemm_f32_split.h) and y in one launch.  A tile has 64 columns of y: columns 32 j of
// a wave's are the gate's for j = 0 and the other projection's for j = 1.
template <int AI>
__global__ __launch_bounds__(kSplitThreads) void gated_split_kernel(SplitProblem p, const float* __restrict__ bias, float* __restrict__ gu, int gate) {
  __shared__ __attribute__((aligned(1024))) char lds[kSplitLds<AI>];
  int tm, tn;
  gemm_tile_of_block(blockIdx.x, p.tiles_m, p.tiles_n, tm, tn);
  const int F = p.N, m0 = tm * AI * kSplitT, f0 = tn * (kSplitT / 2);
  floatx16 acc[AI][2];
  auto row = [&](int r) { return min(f0 + r / 64 * 32 + r % 32, F - 1) + (r % 64 < 32 ? 0 : static_cast<int64_t>(F)); };
  split_product<AI, true, true>(lds, p, m0, 0, 0, p.K, row, acc);
  const int wave = threadIdx.x / kWave, lane = threadIdx.x % kWave, col = f0 + wave % 2 * 32 + lane % 32;
  if (col >= F) return;
  const float bg = bias ? bias[col] : 0.f, bu = bias ? bias[F + col] : 0.f;
  gated_with(gate, [&](auto kind) {
#pragma unroll
    for (int n = 0; n < 16 * AI; ++n) {
      const int i = n / 16, r = n % 16, m = m0 + wave / 2 * 32 * AI + 32 * i + (r / 4) * 8 + (lane / 32) * 4 + r % 4;
      if (m >= p.M) continue;
      const float g = acc[i][0][r] + bg, u = acc[i][1][r] + bu;
      p.c[static_cast<int64_t>(m) * F + col] = gated_act<false, decltype(kind)::value>(g) * u;
      if (gu) {
        float* const at = gu + static_cast<int64_t>(m) * 2 * F + col;
        __builtin_nontemporal_store(g, at);
        __builtin_nontemporal_store(u, at + F);
      }
    }
  });
}

static int launch_gated_split(const void* x, const void* w, const void* bias, void* y, void* gu, int64_t M, int64_t F, int64_t K, int gate,
                              int ai, hipStream_t stream) {
  const int64_t tiles_m = ceil_div(M, ai * kSplitT), tiles_n = ceil_div(F, kSplitT / 2);
  if (tiles_m * tiles_n > 0xffffffffLL / kSplitThreads) return fail(MG_ERR_INVALID, "gated_linear_fwd: too many output tiles");
  SplitProblem p{};
  p.a = static_cast<const float*>(x), p.b = static_cast<const float*>(w), p.c = static_cast<float*>(y);
  p.M = static_cast<int>(M), p.N = static_cast<int>(F), p.K = static_cast<int>(K), p.lda = p.ldb = K;
  p.tiles_m = static_cast<int>(tiles_m), p.tiles_n = static_cast<int>(tiles_n);
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(tiles_m * tiles_n)), dim3(kSplitThreads), 0, stream, p,
                       static_cast<const float*>(bias), static_cast<float*>(gu), gate);
  };
  if (ai == 2) launch(gated_split_kernel<2>);
  else launch(gated_split_kernel<1>);
  MG_LAUNCH_CHECK();
  return MG_OK;
}

// [dg du] from dy, g and u, rounded to the tensors' type as the products take it.  Bound by its bytes, five values an output: (16384, 1024) bf16
// 27 us, 6.2 TB/s.  The projections were put away in the forward pass and are read for the last time here: past the caches, which keep
// what this writes for the products (with them gradients of (16384, 1024 <- 384) bf16 93.9 -> 89.8 us, (32768, 2048 <- 512) 432 -> 427).
template <typename T, int VEC, int GATE>
__global__ __launch_bounds__(kGatedThreads) void gate_bwd_kernel(const T* __restrict__ dy, const T* __restrict__ gu, T* __restrict__ dgu,
                                                                int64_t items, int F, uint32_t per_row, int64_t first_block) {
  const int64_t item = (first_block + blockIdx.x) * kGatedThreads + threadIdx.x;
  if (item >= items) return;
  const int64_t row = item / per_row;
  const int c = static_cast<int>(item - row * per_row) * VEC;
  float d[VEC], g[VEC], u[VEC];
  VecIO<T, VEC>::load(dy + row * F + c, d);
  VecIO<T, VEC>::load_stream(gu + row * 2 * F + c, g);
  VecIO<T, VEC>::load_stream(gu + row * 2 * F + F + c, u);
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

// The same, and the column sums of [dg du], before they are rounded, over each group of `rows` rows, (groups, 2 F): a workgroup takes 64
// chunks of columns of a group, four rows at a time, and adds up what its threads have of a column in LDS.  (The products' own column sums
// would be those of rounded values, 1.4 times as far from the exact ones as a rounding of db alone.)
constexpr int kGateRows = 32;
template <typename T, int VEC, int GATE>
__global__ __launch_bounds__(kGatedThreads) void gate_bwd_sums_kernel(const T* __restrict__ dy, const T* __restrict__ gu, T* __restrict__ dgu,
                                                                     float* __restrict__ sums, int M, int F, int blocks_f, int rows) {
  __shared__ float parts[4][2][64 * VEC];
  const int bf = blockIdx.x % blocks_f, group = blockIdx.x / blocks_f, tx = threadIdx.x % 64, ty = threadIdx.x / 64;
  const int c = (bf * 64 + tx) * VEC;
  const int64_t r0 = static_cast<int64_t>(group) * rows, r1 = min(r0 + rows, static_cast<int64_t>(M));
  float sg[VEC], su[VEC];
#pragma unroll
  for (int i = 0; i < VEC; ++i) sg[i] = su[i] = 0.f;
  if (c < F) {
#pragma unroll 2
    for (int64_t row = r0 + ty; row < r1; row += 4) {
      float d[VEC], g[VEC], u[VEC];
      VecIO<T, VEC>::load(dy + row * F + c, d);
      if constexpr (sizeof(T) == 2) {
        VecIO<T, VEC>::load_stream(gu + row * 2 * F + c, g);
        VecIO<T, VEC>::load_stream(gu + row * 2 * F + F + c, u);
      } else {
        VecIO<T, VEC>::load(gu + row * 2 * F + c, g);
        VecIO<T, VEC>::load(gu + row * 2 * F + F + c, u);
      }
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        float act, slope;
        gated_act_slope<sizeof(T) == 2, GATE>(g[i], act, slope);
        g[i] = d[i] * u[i] * slope;
        u[i] = d[i] * act;
        sg[i] += g[i], su[i] += u[i];
      }
      VecIO<T, VEC>::store(dgu + row * 2 * F + c, g);
      VecIO<T, VEC>::store(dgu + row * 2 * F + F + c, u);
    }
  }
#pragma unroll
  for (int i = 0; i < VEC; ++i) parts[ty][0][tx * VEC + i] = sg[i], parts[ty][1][tx * VEC + i] = su[i];
  __syncthreads();
  for (int i = threadIdx.x; i < 2 * 64 * VEC; i += kGatedThreads) {
    const int half = i / (64 * VEC), at = i % (64 * VEC), col = bf * 64 * VEC + at;
    if (col >= F) continue;
    sums[static_cast<int64_t>(group) * 2 * F + half * F + col] = (parts[0][half][at] + parts[1][half][at]) + (parts[2][half][at] + parts[3][half][at]);
  }
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

// Whether a thread takes 16 bytes, and how many workgroups lie side by side.
static bool gate_sums_wide(int64_t F, int dtype, const void* dy, const void* gu) {
  return F % (16 / dtype_size(dtype)) == 0 && aligned16(dy) && aligned16(gu);
}
static int64_t gate_sums_across(int64_t F, int dtype, bool wide) { return ceil_div(F, wide ? 64 * 16 / dtype_size(dtype) : 64); }

// Rows of a group in 16 bits: as few as leave four workgroups a CU, four rows at least.  Fewer leave more sums to add, more leave CUs without
// work: all gradients in bf16 with 4 | 8 | 16 | 32 | 64 rows, us: (512, 2048 <- 1024) 31.5 | 32.8 | 35.6 | 43.0 | 56.4,
// (4096, 1024 <- 1024) 60.9 | 58.1 | 59.8 | 65.9 | 79.8, (16384, 1024 <- 384) 108.9 | 100.5 | 100.3 | 97.0 | 108.5.
static int gate_group_rows(int64_t M, int64_t F, int dtype, const void* dy, const void* gu) {
  const int64_t across = gate_sums_across(F, dtype, gate_sums_wide(F, dtype, dy, gu)), most = 4 * device_info().cu_count;
  int rows = 4;
  while (rows < (1 << 24) && ceil_div(M, rows) * across > most && rows < M) rows *= 2;
  return rows;
}

// [dg du] and its sums over groups of `rows` rows, for which this takes scratch.
template <typename T>
static int gate_bwd_sums(const void* dy, const void* gu, void* dgu, Scratch& sums, int64_t M, int64_t F, int gate, int rows, hipStream_t stream) {
  constexpr int VEC = WideVec<T>::value;
  constexpr int kType = sizeof(T) == 4 ? MG_F32 : MG_F16;  // (by its size)
  const bool wide = gate_sums_wide(F, kType, dy, gu);
  const int64_t blocks_f = gate_sums_across(F, kType, wide), groups = ceil_div(M, rows);
  if (blocks_f * groups > 0xffffffffLL / kGatedThreads) return fail(MG_ERR_INVALID, "gated_linear_bwd: too many rows");
  MG_TRY(sums.take(groups * 2 * F * static_cast<int64_t>(sizeof(float))));
  gated_with(gate, [&](auto kind) {
    constexpr int GATE = decltype(kind)::value;
    auto launch = [&](auto kernel) {
      hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(blocks_f * groups)), dim3(kGatedThreads), 0, stream, static_cast<const T*>(dy),
                         static_cast<const T*>(gu), static_cast<T*>(dgu), sums.as<float>(), static_cast<int>(M), static_cast<int>(F),
                         static_cast<int>(blocks_f), rows);
    };
    if (wide) launch(gate_bwd_sums_kernel<T, VEC, GATE>);
    else launch(gate_bwd_sums_kernel<T, 1, GATE>);
  });
  MG_LAUNCH_CHECK();
  return MG_OK;
}

// Which kernel a forward pass takes: the least of these estimates, in us.  kGatedDirect: gated_direct.h; kGatedSmall: 64 x 64 tiles, K in
// ranges; kGatedDeep: 128 x 128 or 256 x 256 tiles, which copy ragged operands first (a launch, and two passes over them).  Fitted to 800 shapes of 1 to 20000 rows, 32 to 8192 inputs and 32 to 12000 outputs, weights from
// memory, each by every way: over them the way taken is 1.4 % slower than each one's best on 16-byte chunks, 2.6 % off them (64 x 64 tiles
// up to 64 rows and 128 x 128 above: 31 %).  Whether the projections are kept, which is one value
// stored or three, is not looked at, so that y is the same either way.  `values`: two an output.
enum GatedWay { kGatedDirect, kGatedSmall, kGatedDeep, kGatedApart, kGatedSplit };
struct GatedChoice {
  GatedWay way;
  int tile;  // kGatedDirect: 16 or 32 rows; kGatedDeep: a Gemm16Tile; kGatedSplit: 1 or 2 times 128 rows
  int splits;
  double us;
};
static double gated_direct_us(int64_t M, int64_t F, int64_t K, double values, bool f32, bool ragged, double cus) {
  const int rows = M <= 16 ? 16 : 32;
  const double size = f32 ? 4 : 2, wgs = static_cast<double>(ceil_div(F, 16) * ceil_div(M, rows)), per_cu = std::ceil(wgs / cus);
  const double wg_kb = static_cast<double>(K) * size * (32 + rows) / 1e3, weights_mb = 2.0 * F * K * size / 1e6;
  const double again = static_cast<double>(ceil_div(M, rows));  // the weights come once from memory, then from caches
  if (f32) {
    const double step = rows == 16 ? 0.0183 : 0.0245, read = rows == 16 ? 0.2204 : 0.2634;
    return (rows == 16 ? 3.6 : 4.0) + std::max(step * wg_kb * per_cu, read * weights_mb * again) + 1.1 * values * size / 1e6;
  }
  const double step = (rows == 16 ? 0.016 : 0.0193) * (ragged ? 3.0 : 1.0), read = rows == 16 ? 0.156 : 0.2137;
  return 2.9 + std::max(step * wg_kb * per_cu, read * weights_mb * std::pow(again, 0.89)) + 1.7 * values * size / 1e6;
}
static GatedChoice choose_gated_16bit(int64_t M, int64_t F, int64_t K, bool ragged) {
  const double cus = device_info().cu_count, values = 2.0 * M * F, out = values * 2 / 1e6;
  const double steps = static_cast<double>(ceil_div(K, 64)), weights_mb = 4.0 * F * K / 1e6;
  constexpr int64_t kTiles = 1 << 23;  // of a launch, which counts its threads in 32 bits
  GatedChoice best{kGatedDirect, M <= 16 ? 16 : 32, 1, gated_direct_us(M, F, K, values, false, ragged, cus)};
  if (ceil_div(F, 16) * ceil_div(M, M <= 16 ? 16 : 32) > kTiles) best.us = 1e30;
  auto offer = [&](GatedWay way, int tile, int splits, double us) {
    if (us < best.us) best = GatedChoice{way, tile, splits, us};
  };
  if (const int64_t tiles = ceil_div(M, 64) * ceil_div(F, 32); (!ragged || K >= 8) && tiles <= kTiles) {
    for (int s = 1; s <= 16 && (s == 1 || (K >= 256 * s && tiles * s <= 1024)); ++s) {
      const double per_cu = std::ceil(static_cast<double>(tiles) * s / cus), walk = std::ceil(steps / s), parts = static_cast<double>(tiles) * s * 4096 / 1e6;
      const double us = ragged ? 3.04 + walk * (per_cu > 1 ? 0.292 * per_cu : 0.382) + 0.252 * out + 0.588 * (per_cu - 1) + (s > 1 ? 2.96 + 1.97 * parts : 0.0)
                               : 2.97 + walk * (per_cu > 1 ? 0.238 * per_cu : 0.232) + 0.191 * out + 0.475 * (per_cu - 1) + (s > 1 ? 3.16 + 1.6 * parts : 0.0);
      offer(kGatedSmall, 64, s, std::max(us, 3.0 + (ragged ? 0.354 : 0.215) * weights_mb));
    }
  }
  const double copies = ragged ? 2.4 + (static_cast<double>(M) * K + 2.0 * F * K) / 1e6 : 0.0;
  if (const int64_t tiles = ceil_div(M, 128) * ceil_div(F, 64); tiles <= kTiles) {
    const double per_cu = std::ceil(tiles / cus), pairs = std::floor(per_cu / 2), odd = per_cu - 2 * pairs, lines = K % 64 != 0 && K >= 512 ? 1.256 : 1.0;
    offer(kGatedDeep, kTile128, 1, copies + 3.83 + std::max(2.0, steps) * lines * (0.936 * pairs + (pairs == 0 ? 0.366 : 0.315) * odd) + 0.288 * out + 0.295 * (pairs + odd));
  }
  const double tiles = static_cast<double>(ceil_div(M, 256) * ceil_div(F, 128));
  offer(kGatedDeep, kTile256, 1, copies + 5.92 + std::ceil(tiles / cus) * ((tiles < 0.75 * cus ? 1.096 : 1.367) * std::max(2.0, steps) + 3.66) + 0.328 * out);
  // MOGRAD_HIP_GATED_TILE = 16 (straight from memory) | 64 | 128 | 256 and MOGRAD_HIP_GATED_SPLITS override the choice.
  if (env_str("MOGRAD_HIP_GATED_TILE")) {
    const int only = env_int("MOGRAD_HIP_GATED_TILE", 0);
    if (only == 16) return GatedChoice{kGatedDirect, M <= 16 ? 16 : 32, 1, 0.0};
    if (only == 64 && (!ragged || K >= 8)) return GatedChoice{kGatedSmall, 64, std::max(1, env_int("MOGRAD_HIP_GATED_SPLITS", 1)), 0.0};
    return GatedChoice{kGatedDeep, only == 256 ? kTile256 : kTile128, 1, 0.0};
  }
  return best;
}
// fp32: a plain product and the gate, within an eighth for most; from three bf16 numbers a value (gemm_f32_split.h) in tiles of 128 or 256
// rows, within 5 %; straight from memory.  Over 516 shapes of 16 to 20000 rows the way taken is 2.1 % slower than each one's best; without
// the products of bf16 numbers 15 %.  us, plain product | those: (2048, 4096 <- 4096) 1052 | 718, (16384, 1024 <- 384) 250 | 170,
// (8192, 256 <- 256) 32 | 18, (256, 1024 <- 4096) 47 | 152, (300, 300 <- 300) 7 | 19.
static GatedChoice choose_gated_f32(int64_t M, int64_t F, int64_t K) {
  const double cus = device_info().cu_count, values = static_cast<double>(M) * F, weights_mb = 8.0 * F * K / 1e6;
  const int rows = M <= 16 ? 16 : 32;
  GatedChoice best{kGatedApart, 0, 1, 6.9 + 10.4 * 4e-9 * values * K + 0.448 * values * 8 / 1e6 + 0.21 * weights_mb + 1.6 * K / 1e3};
  auto offer = [&](GatedWay way, int tile, double us) {
    if (us < best.us) best = GatedChoice{way, tile, 1, us};
  };
  if (ceil_div(F, 16) * ceil_div(M, rows) <= 1 << 22) offer(kGatedDirect, rows, gated_direct_us(M, F, K, 2 * values, true, false, cus));
  const double steps = static_cast<double>(ceil_div(K, kSplitBK));
  for (int ai = 1; ai <= 2; ++ai) {
    const int64_t tiles = ceil_div(M, ai * kSplitT) * ceil_div(F, kSplitT / 2);
    if (tiles > 1 << 22 || std::max(M, K) > kSplitMost) continue;
    offer(kGatedSplit, ai, 4.34 + std::ceil(tiles / cus) * (ai == 1 ? 1.117 * steps + 2.8 : 1.845 * steps + 6.9) + 0.169 * values * 12 / 1e6);
  }
  // MOGRAD_HIP_GATED_TILE = 16 (straight from memory) | 64 (apart) | 128 | 256 overrides the choice.
  switch (env_int("MOGRAD_HIP_GATED_TILE", 0)) {
    case 16: return GatedChoice{kGatedDirect, rows, 1, 0.0};
    case 64: return GatedChoice{kGatedApart, 0, 1, 0.0};
    case 128: return GatedChoice{kGatedSplit, 1, 1, 0.0};
    case 256: return GatedChoice{kGatedSplit, 2, 1, 0.0};
    default: return best;
  }
}

// Which kernels fp32 gradients take: those of any Linear backward (kGatedApart), or the products of bf16 numbers, dW in ranges of rows.  Fitted
// to the same shapes, within an eighth and 7 %; the way taken is 2.6 % slower than each one's best, the first alone 8 %.  us, any Linear
// backward's | those: (2048, 512 <- 784) 99 | 68, (2048, 4096 <- 4096) 2052 | 1486, (16384, 1024 <- 384) 586 | 364, (512, 2048 <- 512)
// 60 | 162.
static GatedChoice choose_gated_bwd_f32(int64_t M, int64_t F, int64_t K, bool dx, bool db) {
  const double cus = device_info().cu_count, N = 2.0 * F, values = static_cast<double>(M) * F;
  GatedChoice best{kGatedApart, 0, 1, 7.4 + 8.87 * (dx ? 4e-9 : 2e-9) * M * K * N + 0.326 * values * 20 / 1e6 + 0.894 * N * K * 4 / 1e6 + 1.15 * M * K * 4 / 1e6 +
                                          (db ? 0.08 : 0.0) + 1.11 * M / 1e3 + 5.4 * N / 1e3};
  const double steps_x = static_cast<double>(ceil_div(2 * F, kSplitBK));
  for (int ai = 1; ai <= 2 && std::max({M, 2 * F, K}) <= kSplitMost; ++ai) {
    const int64_t tiles_k = ceil_div(K, kSplitT), tiles_w = ceil_div(2 * F, ai * kSplitT) * tiles_k, tiles_x = dx ? ceil_div(M, ai * kSplitT) * tiles_k : 0;
    if (tiles_w > 1 << 21 || tiles_x > 1 << 21) continue;
    const double step = ai == 1 ? 1.58 : 2.37, ends = ai == 1 ? 2.3 : 5.1;
    for (int s = 1; s <= 24 && (s == 1 || (M >= 64 * s && tiles_w * s <= 600)); ++s) {
      const double steps_w = static_cast<double>(ceil_div(ceil_div(M, s), kSplitBK));
      const double load = (tiles_w * s * (steps_w * step + ends) + tiles_x * (steps_x * step + ends)) / cus, chain = std::max(steps_w, dx ? steps_x : 0.0) * step + ends;
      const double us = 4.5 + std::max(load, chain) + 0.36 * std::min(load, chain) + 0.196 * values * 20 / 1e6 + (s > 1 ? 2.2 + 0.243 * s * N * K * 4 / 1e6 : 0.0) + (db ? 4.1 : 0.0);
      if (us < best.us) best = GatedChoice{kGatedSplit, ai, s, us};
    }
  }
  // MOGRAD_HIP_GATED_BWD_TILE = 64 (apart) | 128 | 256 and MOGRAD_HIP_GATED_SPLITS override the choice.
  if (env_str("MOGRAD_HIP_GATED_BWD_TILE")) {
    const int only = env_int("MOGRAD_HIP_GATED_BWD_TILE", 0);
    return only == 64 ? GatedChoice{kGatedApart, 0, 1, 0.0} : GatedChoice{kGatedSplit, only == 256 ? 2 : 1, std::max(1, env_int("MOGRAD_HIP_GATED_SPLITS", 1)), 0.0};
  }
  return best;
}

template <typename T>
static int launch_gated_direct(const void* x, const void* w, const void* bias, void* y, void* gu, int64_t M, int64_t F, int64_t K, int gate,
                               int rows, hipStream_t stream) {
  const int64_t tiles_f = ceil_div(F, 16), blocks = tiles_f * ceil_div(M, rows);
  constexpr int kThreads = 64 * kGatedDirectWaves;
  if (blocks > 0xffffffffLL / kThreads) return fail(MG_ERR_INVALID, "gated_linear_fwd: too many output tiles");
  const GatedDirect<T> p{static_cast<const T*>(x), static_cast<const T*>(w), static_cast<const T*>(bias), static_cast<T*>(y), static_cast<T*>(gu),
                         static_cast<int>(M), static_cast<int>(F), static_cast<int>(K), static_cast<int>(tiles_f), gate};
  const dim3 grid(static_cast<unsigned>(blocks));
  if (rows == 16) hipLaunchKernelGGL((gated_direct_kernel<T, 1>), grid, dim3(kThreads), 0, stream, p);
  else hipLaunchKernelGGL((gated_direct_kernel<T, 2>), grid, dim3(kThreads), 0, stream, p);
  MG_LAUNCH_CHECK();
  return MG_OK;
}

// 64 x 64 tiles (32 columns of y), K in `splits` ranges.  ANY: operands of any alignment, K at least 8.
template <typename T, bool ANY>
static int launch_gated_small(GatedProblem<T> pr, int splits, hipStream_t stream) {
  const int64_t tiles_m = ceil_div(pr.M, kSmallT), tiles_n = ceil_div(pr.N, kSmallT / 2), tiles = tiles_m * tiles_n;
  const int k_per_split = static_cast<int>(ceil_div(ceil_div(pr.K, splits), kSmallBK) * kSmallBK);
  splits = static_cast<int>(ceil_div(pr.K, k_per_split));
  const int64_t grid = splits > 1 ? gemm_split_grid(tiles, splits, 1) : tiles;
  if (grid > 0xffffffffLL / 256) return fail(MG_ERR_INVALID, "gated_linear_fwd: too many output tiles");
  Scratch partial;
  if (splits > 1) MG_TRY(partial.take(splits * tiles * kSmallT * kSmallT * static_cast<int64_t>(sizeof(float))));
  pr.partial = partial.as<float>(), pr.tiles_m = static_cast<int>(tiles_m), pr.tiles_n = static_cast<int>(tiles_n);
  pr.splits = splits, pr.k_per_split = k_per_split;
  const dim3 blocks(static_cast<unsigned>(grid));
  if (splits == 1) {
    hipLaunchKernelGGL((gated_small_kernel<T, false, ANY>), blocks, dim3(256), 0, stream, pr);
    MG_LAUNCH_CHECK();
    return MG_OK;
  }
  hipLaunchKernelGGL((gated_small_kernel<T, true, ANY>), blocks, dim3(256), 0, stream, pr);
  MG_LAUNCH_CHECK();
  hipLaunchKernelGGL((gated_small_sum_kernel<T>), dim3(static_cast<unsigned>(tiles)), dim3(256), 0, stream, pr);
  MG_LAUNCH_CHECK();
  return MG_OK;
}

// 16 bits: both projections and y in one launch (two where K is in ranges); y comes from the projections before they are rounded.
template <typename T>
static int gated_fwd_16bit(const void* x, const void* w, const void* bias, void* y, void* gu, int64_t M, int64_t F, int64_t K, int gate,
                           hipStream_t stream) {
  const bool ragged = K % 8 != 0 || !aligned16(x) || !aligned16(w);
  const GatedChoice choice = choose_gated_16bit(M, F, K, ragged);
  if (choice.way == kGatedDirect) return launch_gated_direct<T>(x, w, bias, y, gu, M, F, K, gate, choice.tile, stream);
  int64_t ldx = K, ldw = K, no_batch = 0;
  PadCopies<T> pads;
  if (choice.way == kGatedDeep) {
    if (K % 8 != 0 || !aligned16(x)) MG_TRY(pads.add(&x, 1, M, K, &ldx, &no_batch));
    if (K % 8 != 0 || !aligned16(w)) MG_TRY(pads.add(&w, 1, 2 * F, K, &ldw, &no_batch));
    MG_TRY(pads.launch(stream));
    K = ceil_div(K, 8) * 8;  // (zeros behind K in an image)
  }
  GatedProblem<T> pr{};
  pr.A = static_cast<const T*>(x), pr.B = static_cast<const T*>(w), pr.bias = static_cast<const T*>(bias), pr.C = static_cast<T*>(y);
  pr.M = static_cast<int>(M), pr.N = static_cast<int>(F), pr.K = static_cast<int>(K);
  pr.lda = ldx, pr.ldb = ldw, pr.ldc = F, pr.batches = pr.splits = 1, pr.k_per_split = pr.K;
  pr.gu = static_cast<T*>(gu), pr.gate = gate;
  if (choice.way == kGatedDeep) return launch_gated_deep<T>(pr, static_cast<Gemm16Tile>(choice.tile), stream);
  return ragged ? launch_gated_small<T, true>(pr, choice.splits, stream) : launch_gated_small<T, false>(pr, choice.splits, stream);
}

// The longest walk of a product, K of the forward, M and 2 F of the gradients: a split walk's ranges are whole steps, whose ends are counted in
// 32 bits, so that of (2^31 - 300) rows in 32 ranges the last one would end at 2^31 and be read as far as that.
constexpr int64_t kGatedLongest = kSplitMost;

static int gated_check(const char* who, int64_t M, int64_t F, int64_t K, int gate, int dtype) {
  if (!is_float_dtype(dtype)) return fail(MG_ERR_INVALID, "%s: unsupported dtype %s", who, dtype_name(dtype));
  if (gate < MG_GATE_SILU || gate > MG_GATE_RELU) return fail(MG_ERR_INVALID, "%s: no such gate: %d", who, gate);
  if (M < 0 || F <= 0 || K <= 0 || M > 0x7fffffffLL || F > 0x3fffffffLL || K > kGatedLongest)
    return fail(MG_ERR_INVALID, "%s: bad shape M=%lld F=%lld K=%lld", who, static_cast<long long>(M), static_cast<long long>(F),
                static_cast<long long>(K));
  if (dtype != MG_F32 && K + 64 > kGemmDeepMaxLd)
    return fail(MG_ERR_UNSUPPORTED, "%s: no kernel for 16-bit rows of %lld", who, static_cast<long long>(K));
  return MG_OK;
}

// fp32: the gate's gradient with its column sums, then dW and dX as products of three bf16 numbers a value in one launch, then the sums over
// dW's ranges of rows and over the groups of db in one launch, or left on `list`.
static int gated_bwd_split(const void* dy, const void* gu, const void* x, const void* w, void* dx, void* dw, void* db, int64_t M, int64_t F, int64_t K,
                           bool dx_accumulate, int gate, int ai, int splits, DeferredList* list, hipStream_t stream) {
  const int64_t N = 2 * F, groups = ceil_div(M, kGateRows), numel = N * K;
  Scratch dgu, db_part, partial;
  MG_TRY(dgu.take(M * N * static_cast<int64_t>(sizeof(float))));
  if (db) {
    MG_TRY(gate_bwd_sums<float>(dy, gu, dgu.as<char>(), db_part, M, F, gate, kGateRows, stream));
  } else {
    MG_TRY(gate_bwd<float>(dy, gu, dgu.as<char>(), M, F, gate, stream));
  }
  const int k_per_split = static_cast<int>(ceil_div(ceil_div(M, splits), kSplitBK) * kSplitBK);
  splits = static_cast<int>(ceil_div(M, k_per_split));
  if (splits > 1) MG_TRY(partial.take(splits * numel * static_cast<int64_t>(sizeof(float))));
  SplitProblem pw{}, px{};
  pw.a = px.a = dgu.as<float>(), pw.b = static_cast<const float*>(x), px.b = static_cast<const float*>(w);
  pw.c = splits > 1 ? partial.as<float>() : static_cast<float*>(dw), px.c = static_cast<float*>(dx);
  pw.M = px.K = static_cast<int>(N), pw.N = px.N = static_cast<int>(K), pw.K = px.M = static_cast<int>(M);
  pw.lda = px.lda = N, pw.ldb = px.ldb = pw.ldc = px.ldc = K;
  pw.tiles_m = static_cast<int>(ceil_div(N, ai * kSplitT)), px.tiles_m = static_cast<int>(ceil_div(M, ai * kSplitT));
  pw.tiles_n = px.tiles_n = static_cast<int>(ceil_div(K, kSplitT));
  pw.k_per_split = k_per_split, pw.splits = splits, px.splits = 1, px.accumulate = dx_accumulate;
  const int64_t tiles = static_cast<int64_t>(pw.tiles_m) * pw.tiles_n, n_dw = splits > 1 ? gemm_split_grid(tiles, splits, 1) : tiles;
  const int64_t n_dx = dx ? static_cast<int64_t>(px.tiles_m) * px.tiles_n : 0;
  if (n_dw + n_dx > 0xffffffffLL / kSplitThreads) return fail(MG_ERR_INVALID, "gated_linear_bwd: too many output tiles");
  const dim3 grid(static_cast<unsigned>(n_dw + n_dx));
  auto launch = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(kSplitThreads), 0, stream, pw, px, static_cast<int>(n_dw)); };
  if (ai == 2 && splits > 1) launch(split_linear_bwd_kernel<2, true>);
  else if (ai == 2) launch(split_linear_bwd_kernel<2, false>);
  else if (splits > 1) launch(split_linear_bwd_kernel<1, true>);
  else launch(split_linear_bwd_kernel<1, false>);
  MG_LAUNCH_CHECK();
  const int64_t dw_blocks = splits > 1 ? ceil_div(numel, 1024) : 0, db_blocks = db ? ceil_div(N, 64) : 0;
  if (list) {
    list->out_dtype = MG_F32;
    if (splits > 1) {
      list->push(kDeferSplitRows, partial.as<float>(), dw, numel, static_cast<int>(N), static_cast<int>(K), splits, ceil_div(ceil_div(numel, 4), 1024));
      list->hold(partial);
    }
    if (db) {
      list->push(kDeferBiasRows, db_part.as<float>(), db, 0, 0, static_cast<int>(N), static_cast<int>(groups), ceil_div(db_blocks, 4));
      list->hold(db_part);
    }
    return MG_OK;
  }
  if (dw_blocks + db_blocks == 0) return MG_OK;
  hipLaunchKernelGGL((linear_bwd_finish_kernel<float, false>), dim3(static_cast<unsigned>(dw_blocks + db_blocks)), dim3(256), 0, stream, partial.as<float>(),
                     static_cast<float*>(dw), static_cast<int>(N), numel, splits, static_cast<int>(K), static_cast<int>(dw_blocks), db_part.as<float>(),
                     static_cast<float*>(db), db ? static_cast<int>(groups) : 0, static_cast<int>(N));
  MG_LAUNCH_CHECK();
  return MG_OK;
}

// The three gradients; `list`: that of a `_deferred` call, or null.
static int gated_bwd(const char* who, const void* dy, const void* gu, const void* x, const void* w, void* dx, void* dw, void* db, int64_t M,
                     int64_t F, int64_t K, int dx_accumulate, int gate, int dtype, int grad_dtype, DeferredList* list, mg_stream stream) {
  MG_TRY(gated_check(who, M, F, K, gate, dtype));
  if (std::max(M, 2 * F) > kGatedLongest)
    return fail(MG_ERR_INVALID, "%s: bad shape M=%lld F=%lld", who, static_cast<long long>(M), static_cast<long long>(F));
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
    MG_TRY(hold.begin(s));
    if (dtype == MG_F32) {
      const GatedChoice choice = choose_gated_bwd_f32(M, F, K, dx != nullptr, db != nullptr);
      if (choice.way == kGatedSplit)
        return gated_bwd_split(dy, gu, x, w, dx, dw, db, M, F, K, dx_accumulate != 0, gate, choice.tile, choice.splits, list, s);
    }
    Scratch dgu, db_part;
    MG_TRY(dgu.take(M * 2 * F * dtype_size(dtype)));
    const bool sums = db && dtype != MG_F32;
    const int rows = sums ? gate_group_rows(M, F, dtype, dy, gu) : 0;
    switch (dtype) {
      case MG_F32: MG_TRY(gate_bwd<float>(dy, gu, dgu.as<char>(), M, F, gate, s)); break;
      case MG_F16:
        if (sums) MG_TRY(gate_bwd_sums<f16_t>(dy, gu, dgu.as<char>(), db_part, M, F, gate, rows, s));
        else MG_TRY(gate_bwd<f16_t>(dy, gu, dgu.as<char>(), M, F, gate, s));
        break;
      default:
        if (sums) MG_TRY(gate_bwd_sums<bf16_t>(dy, gu, dgu.as<char>(), db_part, M, F, gate, rows, s));
        else MG_TRY(gate_bwd<bf16_t>(dy, gu, dgu.as<char>(), M, F, gate, s));
        break;
    }
    auto products = [&]() -> int {
      MG_TRY(mg_linear_bwd_fused(dgu.as<char>(), x, w, dx, dw, sums ? nullptr : db, M, 2 * F, K, dx_accumulate, 0, dtype, stream));
      if (!sums) return MG_OK;
      const int64_t groups = ceil_div(M, rows);
      const int cus = device_info().cu_count;
      if (dtype == MG_F16) reduce_partials_or_defer<f16_t>(db_part, static_cast<f16_t*>(db), nullptr, nullptr, groups, 2 * F, cus, s);
      else reduce_partials_or_defer<bf16_t>(db_part, static_cast<bf16_t*>(db), nullptr, nullptr, groups, 2 * F, cus, s);
      MG_LAUNCH_CHECK();
      return MG_OK;
    };
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
    const mg::GatedChoice choice = mg::choose_gated_f32(M, F, K);
    if (choice.way == mg::kGatedSplit) return mg::launch_gated_split(x, w, bias, y, gu, M, F, K, gate, choice.tile, s);
    if (choice.way == mg::kGatedDirect) return mg::launch_gated_direct<float>(x, w, bias, y, gu, M, F, K, gate, choice.tile, s);
    // the projections as one product, whose values are not rounded on the way; 3 M F values of 2 (K + 1) M F products' time.
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
