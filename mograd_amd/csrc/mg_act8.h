// Activations in 8 bits ("act8"): blocks of 32 consecutive columns of a row, the last of a row possibly shorter, share a
// power of two 2^k, and each value is kept as a whole number q of -127 .. 127:
//
//   k = the least k with rint(max|x| / 2^k) <= 127, kept between the type's bounds,   q = rint(x / 2^k),   value = q 2^k
//
// A power of two costs up to one of the eight bits against max / 127, and buys that nothing else rounds: x / 2^k is exact, so
// which q a value gets does not depend on the order or the width of the arithmetic, and q 2^k is a bf16, an fp16 (of an fp16
// tensor) and an fp32 number as it is, so a product of the restored values needs no second rounding.
//
// In memory, one run of bytes of rows (ld + ld / 32), ld = cols rounded up to 32: first q, `rows` rows of ld signed bytes
// (zeros past the columns, so that every row starts on 32 bytes and a consumer reads whole blocks), then one byte k + 133 a
// block, `rows` rows of ld / 32.  The byte 255 marks a block that held an infinity or a NaN: its values are restored as NaN,
// so that what overflowed in the forward pass is seen in the gradients.
#pragma once

#include <type_traits>

#include "mg_device.h"
#include "mg_internal.h"
#include "mg_rows.h"

namespace mg {

constexpr int kAct8Block = 32;
inline int64_t act8_ld(int64_t cols) { return ceil_div(cols, kAct8Block) * kAct8Block; }
inline int64_t act8_bytes(int64_t rows, int64_t cols) { return rows * (act8_ld(cols) / kAct8Block * (kAct8Block + 1)); }

// act8.hip
int act8_check(const char* who, int64_t rows, int64_t cols, int dtype);
int act8_pointer_check(const char* who, const void* act8);
int act8_store(const void* x, void* act8, int64_t rows, int64_t cols, bool keep_sign, int dtype, hipStream_t stream);
int act8_load(const void* act8, void* x, int64_t rows, int64_t cols, int dtype, hipStream_t stream);

// The exponent bytes' bounds.  fp32 and bf16: 2^k and 2^-k are normal numbers.  fp16: from 2^-24, of which every fp16 number is
// a multiple, to 2^9, where 127 steps are still a finite fp16 number (values past 65024 become 65024).
template <typename T>
struct Act8Range {
  static constexpr uint32_t lo = 7, hi = 254;
};
template <>
struct Act8Range<f16_t> {
  static constexpr uint32_t lo = 109, hi = 142;
};

// The exponent byte of a block whose largest |x| has these bits: with |x| = 1.f 2^E it is E - 6 for f < 127 / 128 (then
// |x| / 2^k < 127.5) and E - 5 otherwise, which the addition carries into the exponent.
template <typename T>
__device__ __forceinline__ uint32_t act8_exponent(uint32_t max_bits) {
  const uint32_t e = (max_bits + 0x10000u) >> 23;
  return max_bits >= 0x7f800000u ? 255u : min(max(e, Act8Range<T>::lo), Act8Range<T>::hi);
}
// 2^k, NaN for a marked block.
__device__ __forceinline__ float act8_scale(uint32_t e) { return __uint_as_float(e == 255u ? 0x7fc00000u : (e - 6u) << 23); }
// 2^-k, for storing; a marked block's values become zeros.
__device__ __forceinline__ float act8_inverse(uint32_t e) { return __uint_as_float(e == 255u ? 0u : (260u - e) << 23); }

// Four values as bytes of q.  x / 2^k + 1.5 2^23 has the whole number that x / 2^k rounds to (to even) in its low byte.
// keep_sign: what is not zero is at least one step, so that a ReLU's mask can be read off q.
__device__ __forceinline__ uint32_t act8_pack4(const float (&x)[4], float inverse, bool keep_sign) {
  uint32_t b[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    float t = x[i] * inverse;
    if (keep_sign) t = x[i] != 0.f ? copysignf(fmaxf(fabsf(t), 1.f), x[i]) : 0.f;
    t = fminf(fmaxf(t, -127.f), 127.f);  // (also where the exponent's upper bound held, and NaN -> a number)
    b[i] = __float_as_uint(t + 12582912.f);
  }
  const uint32_t lo = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u);
  const uint32_t hi = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
  return inverse != 0.f ? lo | hi : 0u;
}

__device__ __forceinline__ void act8_unpack4(uint32_t q, float scale, float (&x)[4]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) x[i] = static_cast<float>(static_cast<int32_t>(q << (24 - 8 * i)) >> 24) * scale;
}

__device__ __forceinline__ uint32_t act8_abs_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// Largest of v over 2, 4 or 8 neighbouring lanes.
template <int LANES>
__device__ __forceinline__ uint32_t act8_lanes_max(uint32_t v) {
  auto move = [](uint32_t u, auto ctrl) {
    return static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(u), decltype(ctrl)::value, 0xf, 0xf, false));
  };
  if constexpr (LANES >= 2) v = max(v, move(v, std::integral_constant<int, kDppQuadXor1>{}));
  if constexpr (LANES >= 4) v = max(v, move(v, std::integral_constant<int, kDppQuadXor2>{}));
  if constexpr (LANES >= 8) v = max(v, move(v, std::integral_constant<int, kDppRowHalfMirror>{}));
  return v;
}

constexpr int kAct8Threads = 256;
// From so many chunks on a thread takes four.
inline int64_t act8_many_chunks() { return static_cast<int64_t>(device_info().cu_count) * 4 * kAct8Threads * 4; }

// Row and first column of a chunk.
template <int VEC, typename Index>
__device__ __forceinline__ void act8_place(Index chunk, uint32_t chunks_per_row, int64_t& row, int& c) {
  const Index r = chunk / chunks_per_row;
  row = r;
  c = static_cast<int>(chunk - r * chunks_per_row) * VEC;
}

// The work of workgroup `block` of a restoring pass (act8.hip): COUNT chunks of 16 bytes a thread.  ANY: x at any address, rows of any
// length.
template <typename T, bool ANY, typename Index, int COUNT>
__device__ __forceinline__ void act8_load_chunks(int64_t block, const uint8_t* __restrict__ q, const uint8_t* __restrict__ exponents,
                                                 T* __restrict__ x, int64_t chunks, int cols, uint32_t chunks_per_row) {
  constexpr int VEC = WideVec<T>::value, LANES = kAct8Block / VEC;
  const int64_t first = block * (kAct8Threads * COUNT) + threadIdx.x;
  uint32_t w[COUNT][VEC / 4], e[COUNT];
#pragma unroll
  for (int k = 0; k < COUNT; ++k) {
    const int64_t u = min(first + k * kAct8Threads, chunks - 1);
    if constexpr (VEC == 8) {
      const uint2 r = *reinterpret_cast<const uint2*>(q + u * VEC);
      w[k][0] = r.x;
      w[k][1] = r.y;
    } else {
      w[k][0] = *reinterpret_cast<const uint32_t*>(q + u * VEC);
    }
    e[k] = exponents[u / LANES];
  }
#pragma unroll
  for (int k = 0; k < COUNT; ++k) {
    const int64_t u = first + k * kAct8Threads;
    if (u >= chunks) return;
    int64_t row;
    int c;
    act8_place<VEC, Index>(static_cast<Index>(u), chunks_per_row, row, c);
    const float scale = act8_scale(e[k]);
    float v[VEC];
#pragma unroll
    for (int i = 0; i < VEC / 4; ++i) {
      float x4[4];
      act8_unpack4(w[k][i], scale, x4);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[4 * i + j] = x4[j];
    }
    T* const p = x + row * cols + c;
    if (c + VEC <= cols) {
      if constexpr (ANY) VecAny<T, VEC>::store(p, v);
      else VecIO<T, VEC>::store_stream(p, v);  // (restored for one reader; plain stores 33.2 and 18.6 us)
    } else {
#pragma unroll
      for (int i = 0; i < VEC; ++i)
        if (c + i < cols) p[i] = from_float<T>(v[i]);
    }
  }
}

}  // namespace mg
