// Activations in 8 bits: putting a tensor away and bringing it back (format: mg_act8.h).
#include "mg_act8.h"
#include "mg_rows.h"

namespace mg {

// A thread takes 16 columns, half a block: 16 bytes of q, and two (16 bits) or four (fp32) 16-byte chunks of x.  The other
// half is its neighbouring lane's, so a block's maximum takes one exchange.  One pass, bound by HBM: (s + 33 / 32) bytes a value.
constexpr int kAct8Unit = 16;

// Row and first column of a unit.
template <typename Index>
__device__ __forceinline__ void act8_place(Index unit, uint32_t units_per_row, int64_t& row, int& c) {
  const Index r = unit / units_per_row;
  row = r;
  c = static_cast<int>(unit - r * units_per_row) * kAct8Unit;
}

template <typename T, bool ANY, typename Index>
__global__ __launch_bounds__(256) void act8_store_kernel(const T* __restrict__ x, uint8_t* __restrict__ q,
                                                         uint8_t* __restrict__ exponents, int64_t units, int cols,
                                                         uint32_t units_per_row, int keep_sign) {
  constexpr int VEC = WideVec<T>::value;
  const int64_t u = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (u >= units) return;  // (units come in pairs, and so do lanes)
  int64_t row;
  int c;
  act8_place<Index>(static_cast<Index>(u), units_per_row, row, c);
  const T* p = x + row * cols + c;
  float v[kAct8Unit / VEC][VEC];
  if (c + kAct8Unit <= cols) {
#pragma unroll
    for (int i = 0; i < kAct8Unit / VEC; ++i) {
      if constexpr (ANY) VecAny<T, VEC>::load(p + i * VEC, v[i]);
      else VecIO<T, VEC>::load(p + i * VEC, v[i]);
    }
  } else {  // the row's last values one by one, zeros behind them
#pragma unroll
    for (int i = 0; i < kAct8Unit; ++i) v[i / VEC][i % VEC] = c + i < cols ? to_float(p[i]) : 0.f;
  }
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < kAct8Unit; ++i) m = max(m, act8_abs_bits(v[i / VEC][i % VEC]));
  const uint32_t e = act8_exponent<T>(act8_lanes_max<2>(m));
  const float inverse = act8_inverse(e);
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float x4[4] = {v[4 * i / VEC][4 * i % VEC], v[4 * i / VEC][4 * i % VEC + 1], v[4 * i / VEC][4 * i % VEC + 2],
                         v[4 * i / VEC][4 * i % VEC + 3]};
    w[i] = act8_pack4(x4, inverse, keep_sign != 0);
  }
  *reinterpret_cast<uint4*>(q + u * kAct8Unit) = make_uint4(w[0], w[1], w[2], w[3]);
  if ((u & 1) == 0) exponents[u / 2] = static_cast<uint8_t>(e);
}

template <typename T, bool ANY, typename Index>
__global__ __launch_bounds__(256) void act8_load_kernel(const uint8_t* __restrict__ q, const uint8_t* __restrict__ exponents,
                                                        T* __restrict__ x, int64_t units, int cols, uint32_t units_per_row) {
  constexpr int VEC = WideVec<T>::value;
  const int64_t u = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (u >= units) return;
  int64_t row;
  int c;
  act8_place<Index>(static_cast<Index>(u), units_per_row, row, c);
  const uint4 r = *reinterpret_cast<const uint4*>(q + u * kAct8Unit);
  const float scale = act8_scale(exponents[u / 2]);
  const uint32_t w[4] = {r.x, r.y, r.z, r.w};
  float v[kAct8Unit / VEC][VEC];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float x4[4];
    act8_unpack4(w[i], scale, x4);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[4 * i / VEC][4 * i % VEC + j] = x4[j];
  }
  T* p = x + row * cols + c;
  if (c + kAct8Unit <= cols) {
#pragma unroll
    for (int i = 0; i < kAct8Unit / VEC; ++i) {
      if constexpr (ANY) VecAny<T, VEC>::store(p + i * VEC, v[i]);
      else VecIO<T, VEC>::store(p + i * VEC, v[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kAct8Unit; ++i)
      if (c + i < cols) p[i] = from_float<T>(v[i / VEC][i % VEC]);
  }
}

// Every 16-byte chunk of x lies on 16 bytes.
template <typename T>
static bool act8_aligned(const void* x, int64_t cols) {
  return cols % WideVec<T>::value == 0 && aligned16(x);
}

template <typename T>
static int act8_store_typed(const void* x, void* act8, int64_t rows, int64_t cols, bool keep_sign, hipStream_t stream) {
  const int64_t ld = act8_ld(cols), units = rows * (ld / kAct8Unit);
  uint8_t* const q = static_cast<uint8_t*>(act8);
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(ceil_div(units, 256))), dim3(256), 0, stream,
                       static_cast<const T*>(x), q, q + rows * ld, units, static_cast<int>(cols),
                       static_cast<uint32_t>(ld / kAct8Unit), keep_sign ? 1 : 0);
  };
  const bool narrow = units <= 0x7fffffffLL;
  if (act8_aligned<T>(x, cols)) {
    if (narrow) launch(act8_store_kernel<T, false, uint32_t>);
    else launch(act8_store_kernel<T, false, uint64_t>);
  } else {
    if (narrow) launch(act8_store_kernel<T, true, uint32_t>);
    else launch(act8_store_kernel<T, true, uint64_t>);
  }
  MG_LAUNCH_CHECK();
  return MG_OK;
}

template <typename T>
static int act8_load_typed(const void* act8, void* x, int64_t rows, int64_t cols, hipStream_t stream) {
  const int64_t ld = act8_ld(cols), units = rows * (ld / kAct8Unit);
  const uint8_t* const q = static_cast<const uint8_t*>(act8);
  auto launch = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3(static_cast<unsigned>(ceil_div(units, 256))), dim3(256), 0, stream, q, q + rows * ld,
                       static_cast<T*>(x), units, static_cast<int>(cols), static_cast<uint32_t>(ld / kAct8Unit));
  };
  const bool narrow = units <= 0x7fffffffLL;
  if (act8_aligned<T>(x, cols)) {
    if (narrow) launch(act8_load_kernel<T, false, uint32_t>);
    else launch(act8_load_kernel<T, false, uint64_t>);
  } else {
    if (narrow) launch(act8_load_kernel<T, true, uint32_t>);
    else launch(act8_load_kernel<T, true, uint64_t>);
  }
  MG_LAUNCH_CHECK();
  return MG_OK;
}

// Rows and columns that the format's index arithmetic takes: 2^31 workgroups of 256 units.
int act8_check(const char* who, int64_t rows, int64_t cols, int dtype) {
  if (!is_float_dtype(dtype)) return fail(MG_ERR_INVALID, "%s: unsupported dtype %s", who, dtype_name(dtype));
  if (rows < 0 || cols <= 0 || cols > 0x3fffffffLL || rows > 0x7fffffffLL ||
      (rows > 0 && act8_ld(cols) / kAct8Unit > (int64_t{1} << 38) / rows))
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
