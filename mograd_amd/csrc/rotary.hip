// Rotary positions: pairs of a head's columns turned by angles that grow with the token's position.
//
//   (y_a, y_b) = (x_a cos t - x_b sin t, x_a sin t + x_b cos t),   t = position(axis of the pair) * inv_freq(pair)
//
// a, b = i, i + pairs ("halves") or 2 i, 2 i + 1 ("neighbours"); the gradient is the turn by -t.  A token may have several positions
// (time, height, width of a patch), each pair goes by one of them.
//
// The angle.  fp32 positions of a million times a frequency near 1 are off by 0.06 of a radian, so the product is taken in 64 bits,
// in turns, its whole part dropped there, then that of quarter turns, and only the rest, at most pi / 4, goes to fp32, where the Taylor
// series of sine and cosine up to t^9 and t^10 are within 2e-9 of them.  (Positions up to 2^31: 4e-7 of a radian, of the product's rounding.)
// An angle serves all heads of a token: a workgroup takes as many tokens as make a table of 256 pairs, or up to 1024 where its heads are
// few, and then walks the tokens' columns with the table in LDS.  Bound by its bytes: (1, 32768, 32, 128) bf16 99 us, 5.4 TB/s.  Heads whose
// columns are no whole chunks go by chunks at any address, and the few columns left over one by one: 66 columns 100 us, 2.8 TB/s.
#include <algorithm>

#include "mg_device.h"
#include "mg_internal.h"
#include "mg_rows.h"

namespace mg {

constexpr int kRotaryThreads = 256;
constexpr int kRotaryPairs = 256;  // the most that a head's columns may have
constexpr int kRotaryTable = 1024, kRotaryTokens = 256;  // the most that a workgroup has of them, and of tokens

template <typename T>
struct Rotary {
  const T* x;
  T* y;
  const void* positions;  // null: the token's place in its sequence
  const float* inv_freq;
  int64_t S, tokens;
  int64_t xs[3], ys[3], ps[3];  // element strides: batch, token, head; positions: axis, batch, token
  int heads, pairs, rest;       // rest: columns behind the pairs, to be copied
  int tokens_per_block;
  bool wide_positions, neighbours, inverse;
  uint8_t axis[kRotaryPairs];
};

// Sine and cosine of `turns` turns.
__device__ __forceinline__ float2 rotary_sincos(double turns) {
  const double quarters = 4.0 * (turns - rint(turns)), whole = rint(quarters);
  const float t = static_cast<float>((quarters - whole) * 1.5707963267948966);
  const float q = t * t;
  const float s = t + t * q * (-1.6666667e-1f + q * (8.3333333e-3f + q * (-1.9841270e-4f + q * 2.7557319e-6f)));
  const float c = 1.f + q * (-0.5f + q * (4.1666667e-2f + q * (-1.3888889e-3f + q * (2.4801587e-5f + q * -2.7557319e-7f))));
  const int n = static_cast<int>(whole) & 3;
  const float a = n & 1 ? c : s, b = n & 1 ? s : c;
  return make_float2(n & 2 ? -a : a, (n == 1 || n == 2) ? -b : b);
}

// ANY: chunks at any address, and what is left over of the pairs and of the rest goes a pair, or a column, at a time.
template <typename T, bool ANY>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(Rotary<T> r, int64_t first_block) {
  __shared__ float2 table[kRotaryTable];  // (sin, cos)
  __shared__ int64_t at_x[kRotaryTokens], at_y[kRotaryTokens];
  const int64_t token0 = (first_block + blockIdx.x) * r.tokens_per_block;
  const int here = static_cast<int>(min(static_cast<int64_t>(r.tokens_per_block), r.tokens - token0));
  const int tid = threadIdx.x;
  if (tid < here) {
    const int64_t token = token0 + tid, b = token / r.S, s = token - b * r.S;
    at_x[tid] = b * r.xs[0] + s * r.xs[1];
    at_y[tid] = b * r.ys[0] + s * r.ys[1];
  }
  for (int entry = tid; entry < here * r.pairs; entry += kRotaryThreads) {
    const int tk = entry / r.pairs, i = entry - tk * r.pairs;
    const int64_t token = token0 + tk, b = token / r.S, s = token - b * r.S;
    double position;
    if (!r.positions) {
      position = static_cast<double>(s);
    } else {
      const int64_t at = r.axis[i] * r.ps[0] + b * r.ps[1] + s * r.ps[2];
      position = r.wide_positions ? static_cast<double>(static_cast<const int64_t*>(r.positions)[at])
                                  : static_cast<double>(static_cast<const int32_t*>(r.positions)[at]);
    }
    float2 sc = rotary_sincos(position * (static_cast<double>(r.inv_freq[i]) * 0.15915494309189535));
    if (r.inverse) sc.x = -sc.x;
    table[entry] = sc;
  }
  __syncthreads();

  constexpr int VEC = WideVec<T>::value;
  auto load = [](const T* p, float (&v)[VEC]) {
    if constexpr (ANY) VecAny<T, VEC>::load(p, v);
    else VecIO<T, VEC>::load(p, v);
  };
  auto store = [](T* p, const float (&v)[VEC]) {
    if constexpr (ANY) VecAny<T, VEC>::store(p, v);
    else VecIO<T, VEC>::store(p, v);
  };
  // Items of a head: chunks of pairs (halves: a chunk of either half; neighbours: VEC / 2 pairs), chunks of the rest, and what is left over.
  const int a0 = r.neighbours ? 2 * r.pairs / VEC : r.pairs / VEC, a1 = a0 + r.rest / VEC;
  const int done = r.neighbours ? a0 * (VEC / 2) : a0 * VEC;  // pairs in chunks
  const int a2 = ANY ? a1 + r.pairs - done : a1, per_head = ANY ? a2 + r.rest % VEC : a2;
  const int items = here * r.heads * per_head;
  for (int item = tid; item < items; item += kRotaryThreads) {
    const int row = item / per_head, c = item - row * per_head, tk = row / r.heads, h = row - tk * r.heads;
    const T* const x = r.x + at_x[tk] + h * r.xs[2];
    T* const y = r.y + at_y[tk] + h * r.ys[2];
    const float2* const sc = table + tk * r.pairs;
    if (c >= a0 && c < a1) {
      const int at = 2 * r.pairs + (c - a0) * VEC;
      if (x == y) continue;
      float v[VEC];
      load(x + at, v);
      store(y + at, v);
    } else if (ANY && c >= a2) {
      const int at = 2 * r.pairs + r.rest / VEC * VEC + c - a2;
      if (x != y) y[at] = x[at];
    } else if (ANY && c >= a1) {
      const int i = done + c - a1, a = r.neighbours ? 2 * i : i, b = r.neighbours ? 2 * i + 1 : i + r.pairs;
      const float va = to_float(x[a]), vb = to_float(x[b]);
      y[a] = from_float<T>(va * sc[i].y - vb * sc[i].x);
      y[b] = from_float<T>(va * sc[i].x + vb * sc[i].y);
    } else if (r.neighbours) {
      float v[VEC];
      load(x + c * VEC, v);
#pragma unroll
      for (int i = 0; i < VEC; i += 2) {
        const float2 p = sc[c * (VEC / 2) + i / 2];
        const float va = v[i], vb = v[i + 1];
        v[i] = va * p.y - vb * p.x;
        v[i + 1] = va * p.x + vb * p.y;
      }
      store(y + c * VEC, v);
    } else {
      float va[VEC], vb[VEC];
      load(x + c * VEC, va);
      load(x + r.pairs + c * VEC, vb);
#pragma unroll
      for (int i = 0; i < VEC; ++i) {
        const float2 p = sc[c * VEC + i];
        const float a = va[i], b = vb[i];
        va[i] = a * p.y - b * p.x;
        vb[i] = a * p.x + b * p.y;
      }
      store(y + c * VEC, va);
      store(y + r.pairs + c * VEC, vb);
    }
  }
}

template <typename T>
static int launch_rotary(Rotary<T> r, hipStream_t stream) {
  constexpr int VEC = WideVec<T>::value;
  constexpr int64_t kBlocks = 1 << 23;  // of a launch, which counts its threads in 32 bits
  // A table of 256 entries, of more where the tokens' columns are few chunks for 256 threads, but a workgroup or two a CU first.
  const int64_t few = std::max<int64_t>(1, r.tokens / (2 * device_info().cu_count));
  const int64_t chunks_of_token = std::max<int64_t>(1, static_cast<int64_t>(r.heads) * (r.pairs + r.rest) / VEC);
  const int64_t full = std::max<int64_t>(256 / r.pairs, std::min<int64_t>(kRotaryTable / r.pairs, ceil_div(512, chunks_of_token)));
  r.tokens_per_block = static_cast<int>(std::min<int64_t>({full, few, kRotaryTokens}));
  const bool chunks = (r.neighbours ? 2 * r.pairs : r.pairs) % VEC == 0 && r.rest % VEC == 0;
  bool on_chunks = chunks && aligned16(r.x) && aligned16(r.y);
  for (int i = 0; i < 3; ++i) on_chunks = on_chunks && r.xs[i] % VEC == 0 && r.ys[i] % VEC == 0;
  const int64_t blocks = ceil_div(r.tokens, r.tokens_per_block);
  for (int64_t first = 0; first < blocks; first += kBlocks) {
    const dim3 grid(static_cast<unsigned>(std::min(blocks - first, kBlocks))), threads(kRotaryThreads);
    if (on_chunks) hipLaunchKernelGGL((rotary_kernel<T, false>), grid, threads, 0, stream, r, first);
    else hipLaunchKernelGGL((rotary_kernel<T, true>), grid, threads, 0, stream, r, first);
    MG_LAUNCH_CHECK();
  }
  return MG_OK;
}

}  // namespace mg

extern "C" {

int mg_rotary(const void* x, void* y, const void* positions, const float* inv_freq, const int32_t* pair_axis, int64_t B, int64_t S,
              int64_t H, int64_t D, int64_t rotated, const int64_t* x_strides, const int64_t* y_strides, const int64_t* pos_strides,
              int axes, int pos_dtype, int neighbours, int inverse, int dtype, mg_stream stream) {
  const char* const who = "rotary";
  if (!mg::is_float_dtype(dtype)) return mg::fail(MG_ERR_INVALID, "%s: unsupported dtype %s", who, mg::dtype_name(dtype));
  constexpr int64_t kMost = int64_t{1} << 40;  // tokens
  if (B < 0 || S < 0 || H < 0 || D <= 0 || H > 0xffffff || D > 0xffffff || B > kMost || S > kMost || (B > 0 && S > kMost / B))
    return mg::fail(MG_ERR_INVALID, "%s: bad shape B=%lld S=%lld H=%lld D=%lld", who, static_cast<long long>(B),
                    static_cast<long long>(S), static_cast<long long>(H), static_cast<long long>(D));
  if (rotated <= 0 || rotated > D || rotated % 2 != 0 || rotated > 2 * mg::kRotaryPairs)
    return mg::fail(MG_ERR_INVALID, "%s: rotated=%lld of %lld columns: an even number of at most %d", who, static_cast<long long>(rotated),
                    static_cast<long long>(D), 2 * mg::kRotaryPairs);
  // (a workgroup counts its tokens' columns in 32 bits)
  if (H * D > (int64_t{1} << 22)) return mg::fail(MG_ERR_UNSUPPORTED, "%s: no kernel for %lld columns a token", who, static_cast<long long>(H * D));
  if (!x_strides || !y_strides) return mg::fail(MG_ERR_INVALID, "%s: null strides", who);
  const int64_t extents[3] = {B, S, H};
  for (int i = 0; i < 3; ++i) {
    if (x_strides[i] < 0 || y_strides[i] < 0) return mg::fail(MG_ERR_INVALID, "%s: negative stride", who);
    if (extents[i] > 1 && y_strides[i] == 0) return mg::fail(MG_ERR_INVALID, "%s: y's rows lie on each other", who);
    if (extents[i] > 1 && x == y && x && x_strides[i] != y_strides[i]) return mg::fail(MG_ERR_INVALID, "%s: in place with other strides", who);
  }
  const int pairs = static_cast<int>(rotated / 2);
  if (positions) {
    if (pos_dtype != MG_I32 && pos_dtype != MG_I64)
      return mg::fail(MG_ERR_INVALID, "%s: positions are int32 or int64, got %s", who, mg::dtype_name(pos_dtype));
    if (axes < 1 || axes > 255) return mg::fail(MG_ERR_INVALID, "%s: axes=%d", who, axes);
    if (!pos_strides) return mg::fail(MG_ERR_INVALID, "%s: null strides", who);
    for (int i = 0; i < 3; ++i)
      if (pos_strides[i] < 0) return mg::fail(MG_ERR_INVALID, "%s: negative stride", who);
    if (!pair_axis && axes != 1) return mg::fail(MG_ERR_INVALID, "%s: pairs of several axes need pair_axis", who);
    for (int i = 0; pair_axis && i < pairs; ++i)
      if (pair_axis[i] < 0 || pair_axis[i] >= axes)
        return mg::fail(MG_ERR_INVALID, "%s: pair %d goes by axis %d of %d", who, i, static_cast<int>(pair_axis[i]), axes);
  }
  if (B == 0 || S == 0 || H == 0) return MG_OK;
  if (!x || !y || !inv_freq) return mg::fail(MG_ERR_INVALID, "%s: null pointer argument", who);
  auto run = [&](auto zero) {
    using T = decltype(zero);
    mg::Rotary<T> r{};
    r.x = static_cast<const T*>(x), r.y = static_cast<T*>(y), r.positions = positions, r.inv_freq = inv_freq;
    r.S = S, r.tokens = B * S;
    for (int i = 0; i < 3; ++i) r.xs[i] = x_strides[i], r.ys[i] = y_strides[i], r.ps[i] = positions ? pos_strides[i] : 0;
    r.heads = static_cast<int>(H), r.pairs = pairs, r.rest = static_cast<int>(D - rotated);
    r.wide_positions = pos_dtype == MG_I64, r.neighbours = neighbours != 0, r.inverse = inverse != 0;
    for (int i = 0; i < pairs; ++i) r.axis[i] = static_cast<uint8_t>(positions && pair_axis ? pair_axis[i] : 0);
    return mg::launch_rotary(r, mg::to_stream(stream));
  };
  switch (dtype) {
    case MG_F32: return run(float{});
    case MG_F16: return run(mg::f16_t{});
    default: return run(mg::bf16_t{});
  }
}

}  // extern "C"
