// The norm of all gradients together, and gradients scaled down to a largest norm.
//
//   norm = sqrt(sum over all tensors of g^2),   out = g min(1, max_norm / norm)
//
// Squares and sums are held in 64 bits: those of fp32 numbers from 1e-23 to 1e19 neither vanish nor overflow there, and a sum over
// billions of them loses nothing that a norm in fp32 could show.  The tensors are cut into pieces, a workgroup each, whose sums go to
// scratch; whoever needs the norm adds those up in one order, so every result is the same in every run, and there are no atomics.
#include <algorithm>
#include <vector>

#include "mg_device.h"
#include "mg_internal.h"
#include "mg_rows.h"

namespace mg {

constexpr int kNormThreads = 256;
constexpr int kNormTensors = 128;  // of a launch: their places go in its arguments
constexpr int64_t kNormPieces = 2048;  // of all launches, about: what 256 CUs hold at once

struct NormTensors {
  const void* in[kNormTensors];
  void* out[kNormTensors];
  int64_t numel[kNormTensors];
  int end[kNormTensors];  // one past the tensor's last piece, counted in this launch
  uint8_t dtype[kNormTensors];
  int count;
};

// Piece `b` of a launch: its tensor, and its elements [from, to).
__device__ __forceinline__ int norm_piece(const NormTensors& t, int b, int64_t piece, int64_t& from, int64_t& to) {
  int lo = 0, hi = t.count - 1;  // the first tensor whose end is past b
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (t.end[mid] > b) hi = mid;
    else lo = mid + 1;
  }
  const int begin = lo ? t.end[lo - 1] : 0;
  from = static_cast<int64_t>(b - begin) * piece;
  to = min(from + piece, t.numel[lo]);
  return lo;
}

// The sum of `v` over the workgroup, in every thread; always in the same order.
__device__ __forceinline__ double norm_block_sum(double v, double* slots) {
#pragma unroll
  for (int m = 32; m > 0; m /= 2) v += __shfl_xor(v, m);
  const int wave = threadIdx.x / kWave;
  if (threadIdx.x % kWave == 0) slots[wave] = v;
  __syncthreads();
  return (slots[0] + slots[1]) + (slots[2] + slots[3]);
}

// Elements before the first 16-byte boundary at or behind p, of n at most.
template <typename T>
__device__ __forceinline__ int norm_head(const T* p, int64_t n) {
  const int head = static_cast<int>((16 - reinterpret_cast<uintptr_t>(p) % 16) % 16 / sizeof(T));
  return head < n ? head : static_cast<int>(n);
}

// A thread's sum of squares of n elements at any address: those up to a 16-byte boundary one by one, then sixteen bytes at a time, then
// the last ones.
template <typename T>
__device__ __forceinline__ double norm_piece_sum(const T* __restrict__ p, int64_t n) {
  constexpr int VEC = WideVec<T>::value, AHEAD = 4;
  double sum[2] = {0.0, 0.0};
  auto one = [&](int64_t i) {
    const double d = static_cast<double>(to_float(p[i]));
    sum[0] = fma(d, d, sum[0]);
  };
  const int head = norm_head(p, n);
  if (threadIdx.x < head) one(threadIdx.x);
  const int64_t last = head + (n - head) / VEC * VEC + threadIdx.x;
  if (last < n) one(last);
  p += head;
  const int64_t whole = (n - head) / VEC;
  int64_t i = threadIdx.x;
  auto add = [&](const float (&v)[VEC]) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) {
      const double d = static_cast<double>(v[e]);
      sum[e % 2] = fma(d, d, sum[e % 2]);
    }
  };
  for (; i + (AHEAD - 1) * kNormThreads < whole; i += AHEAD * kNormThreads) {
    float v[AHEAD][VEC];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) VecIO<T, VEC>::load(p + (i + a * kNormThreads) * VEC, v[a]);
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) add(v[a]);
  }
  for (; i < whole; i += kNormThreads) {
    float v[VEC];
    VecIO<T, VEC>::load(p + i * VEC, v);
    add(v);
  }
  return sum[0] + sum[1];
}

__global__ __launch_bounds__(kNormThreads) void norm_sums_kernel(NormTensors t, int64_t piece, double* __restrict__ sums) {
  __shared__ double slots[kNormThreads / kWave];
  int64_t from, to;
  const int which = norm_piece(t, blockIdx.x, piece, from, to);
  double sum;
  switch (t.dtype[which]) {
    case MG_F32: sum = norm_piece_sum<float>(static_cast<const float*>(t.in[which]) + from, to - from); break;
    case MG_F16: sum = norm_piece_sum<f16_t>(static_cast<const f16_t*>(t.in[which]) + from, to - from); break;
    default: sum = norm_piece_sum<bf16_t>(static_cast<const bf16_t*>(t.in[which]) + from, to - from); break;
  }
  sum = norm_block_sum(sum, slots);
  if (threadIdx.x == 0) sums[blockIdx.x] = sum;
}

// The norm of `count` sums, in every thread of the workgroup.
__device__ __forceinline__ float norm_of_sums(const double* __restrict__ sums, int64_t count, double* slots) {
  double v = 0.0;
  for (int64_t i = threadIdx.x; i < count; i += kNormThreads) v += sums[i];
  return static_cast<float>(sqrt(norm_block_sum(v, slots)));
}

__global__ __launch_bounds__(kNormThreads) void norm_finish_kernel(const double* __restrict__ sums, int64_t count, float* __restrict__ norm) {
  __shared__ double slots[kNormThreads / kWave];
  const float v = norm_of_sums(sums, count, slots);
  if (threadIdx.x == 0) *norm = v;
}

// The sum of `count` sums, as norm_of_sums adds them, which finds one then.
__global__ __launch_bounds__(kNormThreads) void norm_total_kernel(const double* __restrict__ sums, int64_t count, double* __restrict__ total) {
  __shared__ double slots[kNormThreads / kWave];
  double v = 0.0;
  for (int64_t i = threadIdx.x; i < count; i += kNormThreads) v += sums[i];
  v = norm_block_sum(v, slots);
  if (threadIdx.x == 0) *total = v;
}

// SAME: in and out lie alike on their 16-byte chunks, as they do where out is in.
template <typename T, bool SAME>
__device__ __forceinline__ void clip_chunks(const T* in, T* out, int64_t n, float scale) {
  constexpr int VEC = WideVec<T>::value, AHEAD = 4;
  auto one = [&](int64_t i) { out[i] = from_float<T>(to_float(in[i]) * scale); };
  const int head = norm_head(in, n);
  if (threadIdx.x < head) one(threadIdx.x);
  const int64_t last = head + (n - head) / VEC * VEC + threadIdx.x;
  if (last < n) one(last);
  in += head, out += head;
  const int64_t whole = (n - head) / VEC;
  auto store = [&](T* p, float (&v)[VEC]) {
#pragma unroll
    for (int e = 0; e < VEC; ++e) v[e] *= scale;
    if constexpr (!SAME) VecAny<T, VEC>::store(p, v);
    else VecIO<T, VEC>::store_stream(p, v);
  };
  int64_t i = threadIdx.x;
  for (; i + (AHEAD - 1) * kNormThreads < whole; i += AHEAD * kNormThreads) {
    float v[AHEAD][VEC];
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) VecIO<T, VEC>::load_stream(in + (i + a * kNormThreads) * VEC, v[a]);
#pragma unroll
    for (int a = 0; a < AHEAD; ++a) store(out + (i + a * kNormThreads) * VEC, v[a]);
  }
  for (; i < whole; i += kNormThreads) {
    float v[VEC];
    VecIO<T, VEC>::load_stream(in + i * VEC, v);
    store(out + i * VEC, v);
  }
}
template <typename T>
__device__ __forceinline__ void clip_piece(const T* in, T* out, int64_t n, float scale) {
  if (reinterpret_cast<uintptr_t>(in) % 16 == reinterpret_cast<uintptr_t>(out) % 16) clip_chunks<T, true>(in, out, n, scale);
  else clip_chunks<T, false>(in, out, n, scale);
}

// Every workgroup adds up the sums for itself (16 KB from the second-level cache), then scales its piece.  A scale of 1 in place is
// nothing to do.  This second reading and the results go past the caches, the first one through them, so that it leaves there what this
// one finds: bf16, 100 tensors, 3e8 elements 315 us, 5.7 TB/s of reading twice and writing (through the caches 372, both readings past them
// 337); 290 tensors without gaps, whose chunks start where they like, 382; 68 fp32 tensors of 1.1e7 24.7.
__global__ __launch_bounds__(kNormThreads) void clip_kernel(NormTensors t, int64_t piece, const double* __restrict__ sums, int64_t count,
                                                            float max_norm, float* __restrict__ norm_out) {
  __shared__ double slots[kNormThreads / kWave];
  const float norm = norm_of_sums(sums, count, slots);
  if (norm_out && blockIdx.x == 0 && threadIdx.x == 0) *norm_out = norm;
  const float scale = clip_scale(norm, max_norm);
  int64_t from, to;
  const int which = norm_piece(t, blockIdx.x, piece, from, to);
  if (scale == 1.f && t.in[which] == t.out[which]) return;
  switch (t.dtype[which]) {
    case MG_F32: return clip_piece<float>(static_cast<const float*>(t.in[which]) + from, static_cast<float*>(t.out[which]) + from, to - from, scale);
    case MG_F16: return clip_piece<f16_t>(static_cast<const f16_t*>(t.in[which]) + from, static_cast<f16_t*>(t.out[which]) + from, to - from, scale);
    default: return clip_piece<bf16_t>(static_cast<const bf16_t*>(t.in[which]) + from, static_cast<bf16_t*>(t.out[which]) + from, to - from, scale);
  }
}

// The tensors' pieces, launch by launch: calls launch(tensors, pieces in the launch, pieces before it).
template <typename L>
static int norm_launches(const void* const* in, void* const* out, const int64_t* numels, const int* dtypes, int64_t count, int64_t piece,
                         L&& launch) {
  NormTensors t{};
  int64_t before = 0, pieces = 0;
  auto flush = [&]() -> int {
    if (t.count == 0) return MG_OK;
    launch(t, static_cast<unsigned>(pieces), before);
    MG_LAUNCH_CHECK();
    before += pieces, pieces = 0, t.count = 0;
    return MG_OK;
  };
  for (int64_t i = 0; i < count; ++i) {
    if (numels[i] == 0) continue;
    t.in[t.count] = in[i], t.out[t.count] = out ? out[i] : nullptr, t.numel[t.count] = numels[i];
    t.dtype[t.count] = static_cast<uint8_t>(dtypes[i]);
    pieces += ceil_div(numels[i], piece);
    t.end[t.count++] = static_cast<int>(pieces);
    if (t.count == kNormTensors) MG_TRY(flush());
  }
  return flush();
}

// Elements of a piece: of kNormPieces pieces over all tensors, but 2048 at least (half a pass of a workgroup over fp32).
static int64_t norm_piece_elements(int64_t total) {
  return std::max<int64_t>(2048, ceil_div(ceil_div(total, kNormPieces), 2048) * 2048);
}

static int grad_norm(const char* who, const void* const* grads, void* const* out, const int64_t* numels, const int* dtypes, int64_t count,
                     bool clip, float max_norm, float* norm, mg_stream stream) {
  if (count < 0 || count > 0xffffff) return fail(MG_ERR_INVALID, "%s: %lld tensors", who, static_cast<long long>(count));
  if (clip && !(max_norm >= 0.f)) return fail(MG_ERR_INVALID, "%s: max_norm=%g", who, static_cast<double>(max_norm));
  if (count > 0 && (!grads || !numels || !dtypes || (clip && !out))) return fail(MG_ERR_INVALID, "%s: null pointer argument", who);
  int64_t total = 0, pieces = 0;
  for (int64_t i = 0; i < count; ++i) {
    if (!is_float_dtype(dtypes[i])) return fail(MG_ERR_INVALID, "%s: tensor %lld: unsupported dtype %s", who, static_cast<long long>(i), dtype_name(dtypes[i]));
    if (numels[i] < 0 || numels[i] > (int64_t{1} << 40) || total > (int64_t{1} << 41))
      return fail(MG_ERR_INVALID, "%s: tensor %lld has %lld elements", who, static_cast<long long>(i), static_cast<long long>(numels[i]));
    if (numels[i] > 0 && (!grads[i] || (clip && !out[i]))) return fail(MG_ERR_INVALID, "%s: tensor %lld: null pointer argument", who, static_cast<long long>(i));
    total += numels[i];
  }
  if (!norm && !clip) return fail(MG_ERR_INVALID, "%s: null pointer argument", who);
  if (total == 0) return norm ? mg_fill(norm, 0.0, 1, MG_F32, stream) : MG_OK;
  const int64_t piece = norm_piece_elements(total);
  for (int64_t i = 0; i < count; ++i) pieces += ceil_div(numels[i], piece);
  hipStream_t s = to_stream(stream);
  return without_exceptions(who, [&]() -> int {
    if (clip) {  // (a tensor that is there twice would be scaled by two workgroups at once)
      std::vector<const void*> outs;
      for (int64_t i = 0; i < count; ++i)
        if (numels[i] > 0) outs.push_back(out[i]);
      std::sort(outs.begin(), outs.end());
      if (std::adjacent_find(outs.begin(), outs.end()) != outs.end()) return fail(MG_ERR_INVALID, "%s: two of the results are one tensor", who);
    }
    CaptureHold hold;
    MG_TRY(hold.begin(s));
    Scratch mem;
    MG_TRY(mem.take((pieces + 1) * static_cast<int64_t>(sizeof(double))));
    double* sums = mem.as<double>();
    MG_TRY(norm_launches(grads, nullptr, numels, dtypes, count, piece, [&](const NormTensors& t, unsigned blocks, int64_t before) {
      hipLaunchKernelGGL(norm_sums_kernel, dim3(blocks), dim3(kNormThreads), 0, s, t, piece, sums + before);
    }));
    if (!clip) {
      hipLaunchKernelGGL(norm_finish_kernel, dim3(1), dim3(kNormThreads), 0, s, sums, pieces, norm);
      MG_LAUNCH_CHECK();
      return MG_OK;
    }
    // Of thousands of tensors there are as many more pieces; then the sums are added up once, and not in each workgroup.
    if (pieces > 4 * kNormPieces) {
      hipLaunchKernelGGL(norm_total_kernel, dim3(1), dim3(kNormThreads), 0, s, sums, pieces, sums + pieces);
      MG_LAUNCH_CHECK();
      sums += pieces, pieces = 1;
    }
    return norm_launches(grads, out, numels, dtypes, count, piece, [&](const NormTensors& t, unsigned blocks, int64_t before) {
      hipLaunchKernelGGL(clip_kernel, dim3(blocks), dim3(kNormThreads), 0, s, t, piece, sums, pieces, max_norm, before == 0 ? norm : nullptr);
    });
  });
}

}  // namespace mg

extern "C" {

int mg_grad_norm(const void* const* grads, const int64_t* numels, const int* dtypes, int64_t count, float* norm, mg_stream stream) {
  return mg::grad_norm("grad_norm", grads, nullptr, numels, dtypes, count, false, 0.f, norm, stream);
}

int mg_clip_grads(const void* const* grads, void* const* out, const int64_t* numels, const int* dtypes, int64_t count, float max_norm,
                  float* norm, mg_stream stream) {
  return mg::grad_norm("clip_grads", grads, out, numels, dtypes, count, true, max_norm, norm, stream);
}

}  // extern "C"
