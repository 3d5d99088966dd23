// Activations in 8 bits: putting a tensor away and bringing it back (format: mg_act8.h).
#include "mg_act8.h"

namespace mg {

// A thread takes chunks of 16 bytes of x, neighbouring threads neighbouring ones, so that every access of a wave is one run of
// memory: (s + 33 / 32) bytes a value in one pass, bound by HBM.  The 4 (16 bits) or 8 (fp32) lanes of a block exchange its maximum.
// COUNT chunks a thread, a workgroup's width apart, are on their way at once where there are enough to give every CU work.
// (16384, 1536) bf16 there and back 30.1 us, 5.1 TB/s; (2048, 4096) fp32 16.5 (half a block a thread, 32 or 64 bytes of x side by side:
// 31.4 and 25.6).

template <typename T, bool ANY, typename Index, int COUNT>
__global__ __launch_bounds__(kAct8Threads) void act8_store_kernel(const T* __restrict__ x, uint8_t* __restrict__ q,
                                                                  uint8_t* __restrict__ exponents, int64_t chunks, int cols,
                                                                  uint32_t chunks_per_row, int keep_sign, int64_t first_block) {
  constexpr int VEC = WideVec<T>::value, LANES = kAct8Block / VEC;
  const int64_t first = (first_block + blockIdx.x) * (kAct8Threads * COUNT) + threadIdx.x;
  float v[COUNT][VEC];
#pragma unroll
  for (int k = 0; k < COUNT; ++k) {
    const int64_t u = first + k * kAct8Threads;
#pragma unroll
    for (int i = 0; i < VEC; ++i) v[k][i] = 0.f;
    if (u >= chunks) continue;
    int64_t row;
    int c;
    act8_place<VEC, Index>(static_cast<Index>(u), chunks_per_row, row, c);
    const T* const p = x + row * cols + c;
    if (c + VEC <= cols) {
      if constexpr (ANY) VecAny<T, VEC>::load(p, v[k]);
      else VecIO<T, VEC>::load(p, v[k]);
    } else {  // the row's last values one by one, zeros behind them
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (c + i < cols) v[k][i] = to_float(p[i]);
    }
  }
#pragma unroll
  for (int k = 0; k < COUNT; ++k) {
    const int64_t u = first + k * kAct8Threads;
    if (u >= chunks) return;  // (chunks come in whole blocks, and so do lanes)
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < VEC; ++i) m = max(m, act8_abs_bits(v[k][i]));
    const uint32_t e = act8_exponent<T>(act8_lanes_max<LANES>(m));
    const float inverse = act8_inverse(e);
    uint32_t w[VEC / 4];
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      const float x4[4] = {v[k][4 * i], v[k][4 * i + 1], v[k][4 * i + 2], v[k][4 * i + 3]};
      w[i] = act8_pack4(x4, inverse, keep_sign != 0);
    }
    if constexpr (VEC == 8) *reinterpret_cast<uint2*>(q + u * VEC) = make_uint2(w[0], w[1]);
    else *reinterpret_cast<uint32_t*>(q + u * VEC) = w[0];
    if (u % LANES == 0) exponents[u / LANES] = static_cast<uint8_t>(e);
  }
}

template <typename T, bool ANY, typename Index, int COUNT>
__global__ __launch_bounds__(kAct8Threads) void act8_load_kernel(const uint8_t* __restrict__ q,
                                                                 const uint8_t* __restrict__ exponents, T* __restrict__ x,
                                                                 int64_t chunks, int cols, uint32_t chunks_per_row,
                                                                 int64_t first_block) {
  act8_load_chunks<T, ANY, Index, COUNT>(first_block + blockIdx.x, q, exponents, x, chunks, cols, chunks_per_row);
}

// Every 16-byte chunk of x lies on 16 bytes.
template <typename T>
static bool act8_aligned(const void* x, int64_t cols) {
  return cols % WideVec<T>::value == 0 && aligned16(x);
}

// Calls `launch(kernel choice, first workgroup, workgroups)` with what the sizes ask for: chunks at any address or on 16 bytes, 32- or
// 64-bit division, one chunk a thread or four.  A launch counts its threads in 32 bits: 2^23 workgroups of 256 each time.
template <typename T, typename F>
static int act8_launch(const void* x, int64_t chunks, int64_t cols, F&& launch) {
  auto counted = [&](auto any, auto index, auto count) -> int {
    constexpr int64_t kBlocks = 1 << 23;
    const int64_t blocks = ceil_div(chunks, decltype(count)::value * kAct8Threads);
    for (int64_t first = 0; first < blocks; first += kBlocks) {
      launch(any, index, count, first, std::min(blocks - first, kBlocks));
      MG_LAUNCH_CHECK();
    }
    return MG_OK;
  };
  auto indexed = [&](auto any, auto index) {
    if (chunks >= act8_many_chunks()) return counted(any, index, std::integral_constant<int, 4>{});
    return counted(any, index, std::integral_constant<int, 1>{});
  };
  auto aligned = [&](auto any) {
    if (chunks <= 0x7fffffffLL) return indexed(any, uint32_t{});
    return indexed(any, uint64_t{});
  };
  if (act8_aligned<T>(x, cols)) return aligned(std::false_type{});
  return aligned(std::true_type{});
}

template <typename T>
static int act8_store_typed(const void* x, void* act8, int64_t rows, int64_t cols, bool keep_sign, hipStream_t stream) {
  const int64_t ld = act8_ld(cols), per_row = ld / WideVec<T>::value, chunks = rows * per_row;
  uint8_t* const q = static_cast<uint8_t*>(act8);
  return act8_launch<T>(x, chunks, cols, [&](auto any, auto index, auto count, int64_t first, int64_t blocks) {
    hipLaunchKernelGGL((act8_store_kernel<T, decltype(any)::value, decltype(index), decltype(count)::value>),
                       dim3(static_cast<unsigned>(blocks)), dim3(kAct8Threads), 0, stream, static_cast<const T*>(x), q,
                       q + rows * ld, chunks, static_cast<int>(cols), static_cast<uint32_t>(per_row), keep_sign ? 1 : 0, first);
  });
}

template <typename T>
static int act8_load_typed(const void* act8, void* x, int64_t rows, int64_t cols, hipStream_t stream) {
  const int64_t ld = act8_ld(cols), per_row = ld / WideVec<T>::value, chunks = rows * per_row;
  const uint8_t* const q = static_cast<const uint8_t*>(act8);
  return act8_launch<T>(x, chunks, cols, [&](auto any, auto index, auto count, int64_t first, int64_t blocks) {
    hipLaunchKernelGGL((act8_load_kernel<T, decltype(any)::value, decltype(index), decltype(count)::value>),
                       dim3(static_cast<unsigned>(blocks)), dim3(kAct8Threads), 0, stream, q, q + rows * ld,
                       static_cast<T*>(x), chunks, static_cast<int>(cols), static_cast<uint32_t>(per_row), first);
  });
}

// Rows and columns that the index arithmetic takes: both in 32 bits, the bytes of q in 40.
int act8_check(const char* who, int64_t rows, int64_t cols, int dtype) {
  if (!is_float_dtype(dtype)) return fail(MG_ERR_INVALID, "%s: unsupported dtype %s", who, dtype_name(dtype));
  if (rows < 0 || cols <= 0 || cols > 0x3fffffffLL || rows > 0x7fffffffLL ||
      (rows > 0 && act8_ld(cols) > (int64_t{1} << 40) / rows))
    return fail(MG_ERR_INVALID, "%s: bad shape rows=%lld cols=%lld", who, static_cast<long long>(rows),
                static_cast<long long>(cols));
  return MG_OK;
}

int act8_pointer_check(const char* who, const void* act8) {
  if (!act8) return fail(MG_ERR_INVALID, "%s: null pointer argument", who);
  if (!aligned16(act8)) return fail(MG_ERR_INVALID, "%s: an activation in 8 bits starts on a 16-byte boundary", who);
  return MG_OK;
}

int act8_store(const void* x, void* act8, int64_t rows, int64_t cols, bool keep_sign, int dtype, hipStream_t stream) {
  switch (dtype) {
    case MG_F32: return act8_store_typed<float>(x, act8, rows, cols, keep_sign, stream);
    case MG_F16: return act8_store_typed<f16_t>(x, act8, rows, cols, keep_sign, stream);
    default: return act8_store_typed<bf16_t>(x, act8, rows, cols, keep_sign, stream);
  }
}

int act8_load(const void* act8, void* x, int64_t rows, int64_t cols, int dtype, hipStream_t stream) {
  switch (dtype) {
    case MG_F32: return act8_load_typed<float>(act8, x, rows, cols, stream);
    case MG_F16: return act8_load_typed<f16_t>(act8, x, rows, cols, stream);
    default: return act8_load_typed<bf16_t>(act8, x, rows, cols, stream);
  }
}

}  // namespace mg

extern "C" {

int64_t mg_act8_bytes(int64_t rows, int64_t cols) {
  if (rows <= 0 || cols <= 0 || mg::act8_check("act8_bytes", rows, cols, MG_F32) != MG_OK) return 0;
  return mg::act8_bytes(rows, cols);
}

int mg_act8_store(const void* x, void* act8, int64_t rows, int64_t cols, int keep_sign, int dtype, mg_stream stream) {
  MG_TRY(mg::act8_check("act8_store", rows, cols, dtype));
  if (rows == 0) return MG_OK;
  if (!x) return mg::fail(MG_ERR_INVALID, "act8_store: null pointer argument");
  MG_TRY(mg::act8_pointer_check("act8_store", act8));
  return mg::act8_store(x, act8, rows, cols, keep_sign != 0, dtype, mg::to_stream(stream));
}

int mg_act8_load(const void* act8, void* x, int64_t rows, int64_t cols, int dtype, mg_stream stream) {
  MG_TRY(mg::act8_check("act8_load", rows, cols, dtype));
  if (rows == 0) return MG_OK;
  if (!x) return mg::fail(MG_ERR_INVALID, "act8_load: null pointer argument");
  MG_TRY(mg::act8_pointer_check("act8_load", act8));
  return mg::act8_load(act8, x, rows, cols, dtype, mg::to_stream(stream));
}

}  // extern "C"
