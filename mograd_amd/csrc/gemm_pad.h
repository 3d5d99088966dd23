// Images of operands on 16-byte chunks, for the products whose copies into LDS need them so.
#pragma once

#include "gemm_impl.h"
#include "linear_act8.h"
#include "mg_act8.h"

namespace mg {

// dst (batch, rows, cols_to) = src (batch, rows, cols) with zero columns appended: the image of an
// operand that the copying kernels can read 16 bytes at a time.  cols_to is a whole number of
// 16-byte chunks and dst aligned to them; src may lie anywhere.  One thread per chunk; up to three arrays
// per launch.  Bound by its bytes, or by the launch for small arrays.
template <typename T>
struct PadJob {
  const T* src;
  T* dst;
  int64_t ld, batch_stride, chunks;  // chunks: of the whole array
  int rows, cols, cols_to;
};
template <typename T>
struct PadJobs {
  PadJob<T> job[3];
  int block_end[3];
};
template <typename T>
__device__ __forceinline__ void pad_columns(int b, const PadJobs<T>& jobs) {
  const int which = b < jobs.block_end[0] ? 0 : b < jobs.block_end[1] ? 1 : 2;
  const PadJob<T>& j = jobs.job[which];
  const int64_t i = static_cast<int64_t>(b - (which ? jobs.block_end[which - 1] : 0)) * 256 + threadIdx.x;
  if (i >= j.chunks) return;
  constexpr int E = 16 / sizeof(T);
  const int per_row = j.cols_to / E;
  const int64_t row = i / per_row;
  const int c0 = static_cast<int>(i - row * per_row) * E;
  const T* src = j.src + row / j.rows * j.batch_stride + row % j.rows * j.ld + c0;
  reinterpret_cast<uint4*>(j.dst)[i] = gemm_gather_chunk(src, j.cols - c0);
}
template <typename T>
__global__ __launch_bounds__(256) void pad_columns_kernel(PadJobs<T> jobs, int first_block) {
  pad_columns(first_block + static_cast<int>(blockIdx.x), jobs);
}
// The same, and an activation in 8 bits restored by the first workgroups.
template <typename T>
__global__ __launch_bounds__(256) void pad_and_restore_kernel(PadJobs<T> jobs, const uint8_t* q, const uint8_t* e, T* x, int64_t chunks,
                                                              int cols, uint32_t chunks_per_row, int restoring) {
  static_assert(kAct8Threads == 256, "a workgroup of either");
  const int b = blockIdx.x;
  if (b < restoring) act8_load_chunks<T, false, uint32_t, 1>(b, q, e, x, chunks, cols, chunks_per_row);
  else pad_columns(b - restoring, jobs);
}

// Collects the operands of one product that need such an image and makes them in one launch.
template <typename T>
struct PadCopies {
  PadJobs<T> jobs{};
  Scratch mem[3];
  int count = 0;
  int64_t blocks = 0;
  // The image of `src`, whose rows then lie `*ld` apart and batches `*batch_stride`.
  int add(const void** src, int64_t batch, int64_t rows, int64_t cols, int64_t* ld, int64_t* batch_stride) {
    constexpr int E = 16 / sizeof(T);
    // (long rows: whole cache lines, see deep_16bit_us)
    const int64_t unit = sizeof(T) == 2 && cols >= 2048 ? 64 : E, to = ceil_div(cols, unit) * unit;
    const int64_t images = *batch_stride == 0 ? 1 : batch;
    MG_TRY(mem[count].take(images * rows * to * static_cast<int64_t>(sizeof(T))));
    PadJob<T>& j = jobs.job[count];
    j = PadJob<T>{static_cast<const T*>(*src), mem[count].template as<T>(), *ld, *batch_stride, images * rows * (to / E),
                  static_cast<int>(rows), static_cast<int>(cols), static_cast<int>(to)};
    blocks += ceil_div(j.chunks, 256);
    for (int i = count; i < 3; ++i) jobs.block_end[i] = static_cast<int>(blocks);
    ++count;
    *src = j.dst;
    *ld = to;
    *batch_stride = images == 1 ? 0 : rows * to;
    return MG_OK;
  }
  int launch(hipStream_t stream) {
    if (count == 0 || blocks == 0) return MG_OK;
    if (blocks > 0x7fffffffLL) return fail(MG_ERR_INVALID, "matmul: operand too large");
    constexpr int64_t kBlocks = 1 << 23;  // of a launch, which counts its threads in 32 bits
    for (int64_t first = 0; first < blocks; first += kBlocks) {
      hipLaunchKernelGGL((pad_columns_kernel<T>), dim3(static_cast<unsigned>(std::min(blocks - first, kBlocks))), dim3(256), 0, stream, jobs,
                         static_cast<int>(first));
      MG_LAUNCH_CHECK();
    }
    return MG_OK;
  }
  // The copies, and `in` restored to (rows, cols) of T, in one launch where there are copies, none of what is restored, and chunks
  // few enough for a launch to count: (1999, 768) fp16 and a copy of (1999, 1001) 8.2 us, in two launches 10.0.
  int launch(const Act8Restore& in, int64_t rows, int64_t cols, bool copies_it, int dtype, hipStream_t stream) {
    const int64_t ld = act8_ld(cols), per_row = ld / WideVec<T>::value, chunks = rows * per_row;
    const int64_t restoring = ceil_div(chunks, kAct8Threads);
    if (count == 0 || copies_it || cols % WideVec<T>::value != 0 || chunks >= act8_many_chunks() ||
        blocks + restoring > 0xffffffffLL / 256) {
      MG_TRY(act8_load(in.act8, in.x, rows, cols, dtype, stream));
      return launch(stream);
    }
    const uint8_t* const q = static_cast<const uint8_t*>(in.act8);
    hipLaunchKernelGGL((pad_and_restore_kernel<T>), dim3(static_cast<unsigned>(restoring + blocks)), dim3(256), 0, stream, jobs, q,
                       q + rows * ld, static_cast<T*>(in.x), chunks, static_cast<int>(cols), static_cast<uint32_t>(per_row),
                       static_cast<int>(restoring));
    MG_LAUNCH_CHECK();
    return MG_OK;
  }
};

}  // namespace mg
