// The HIP runtime's calls that libmograd_hip.so makes, without a GPU, for tests of what the library asks for (tests/test_launches.py):
// loaded before the library with its symbols global, it takes their place.  Memory is addresses that nobody follows; launches are
// written down, and refused past what the runtime takes: 2^32 - 1 threads along an axis of the grid.
#include <hip/hip_runtime_api.h>

#include <atomic>
#include <cstring>
#include <mutex>
#include <string>

namespace {

std::mutex g_lock;
std::string g_launches;  // "grid x y z block x y z stream" a line
std::atomic<int64_t> g_mallocs{0}, g_next{int64_t{1} << 32};
std::atomic<int> g_error{0}, g_exchange_rc{0};
std::atomic<int> g_capturing{0};
std::atomic<unsigned long long> g_capture_id{1};
thread_local hipStreamCaptureMode t_mode = hipStreamCaptureModeGlobal;

struct Call {
  dim3 grid, block;
  size_t shared;
  hipStream_t stream;
};
thread_local Call t_call;

hipError_t answer(hipError_t e) {
  if (e != hipSuccess) g_error = e;
  return e;
}

}  // namespace

extern "C" {

// For the tests.
int64_t stub_launches(char* out, int64_t size) {
  std::lock_guard<std::mutex> hold(g_lock);
  if (size > 0) std::strncpy(out, g_launches.c_str(), static_cast<size_t>(size));
  return static_cast<int64_t>(g_launches.size());
}
void stub_reset() {
  std::lock_guard<std::mutex> hold(g_lock);
  g_launches.clear();
}
int64_t stub_mallocs() { return g_mallocs; }
// Streams other than the default one are being captured (into capture `id`), or not (0).
void stub_capture(unsigned long long id) {
  g_capturing = id != 0;
  g_capture_id = id;
}
void stub_exchange_fails(int rc) { g_exchange_rc = rc; }
int stub_mode() { return t_mode; }

hipError_t __hipPushCallConfiguration(dim3 grid, dim3 block, size_t shared, hipStream_t stream) {
  t_call = {grid, block, shared, stream};
  return hipSuccess;
}
hipError_t __hipPopCallConfiguration(dim3* grid, dim3* block, size_t* shared, hipStream_t* stream) {
  *grid = t_call.grid, *block = t_call.block, *shared = t_call.shared, *stream = t_call.stream;
  return hipSuccess;
}
hipError_t hipLaunchKernel(const void*, dim3 grid, dim3 block, void**, size_t, hipStream_t stream) {
  const unsigned g[3] = {grid.x, grid.y, grid.z}, b[3] = {block.x, block.y, block.z};
  for (int i = 0; i < 3; ++i)
    if (g[i] == 0 || b[i] == 0 || static_cast<uint64_t>(g[i]) * b[i] > 0xffffffffull) return answer(hipErrorInvalidConfiguration);
  std::lock_guard<std::mutex> hold(g_lock);
  for (unsigned v : {g[0], g[1], g[2], b[0], b[1], b[2]}) g_launches += std::to_string(v) + " ";
  g_launches += std::to_string(reinterpret_cast<uintptr_t>(stream)) + "\n";
  return hipSuccess;
}
hipError_t hipGetLastError(void) { return static_cast<hipError_t>(g_error.exchange(0)); }
hipError_t hipGetDevice(int* device) {
  *device = 0;
  return hipSuccess;
}
hipError_t hipDeviceGetAttribute(int* value, hipDeviceAttribute_t attribute, int) {
  *value = attribute == hipDeviceAttributeMultiprocessorCount ? 256 : 1024;
  return hipSuccess;
}
hipError_t hipMalloc(void** p, size_t n) {
  ++g_mallocs;
  *p = reinterpret_cast<void*>(g_next.fetch_add(static_cast<int64_t>((n + 4095) / 4096 * 4096)));
  return hipSuccess;
}
hipError_t hipFree(void*) { return hipSuccess; }
hipError_t hipSetDevice(int) { return hipSuccess; }
hipError_t hipGetSymbolAddress(void** p, const void*) { return hipMalloc(p, 4096); }
hipError_t hipMemcpyAsync(void*, const void*, size_t, hipMemcpyKind, hipStream_t) { return hipSuccess; }
hipError_t hipStreamCreate(hipStream_t* stream) {
  *stream = reinterpret_cast<hipStream_t>(g_next.fetch_add(4096));
  return hipSuccess;
}
hipError_t hipStreamDestroy(hipStream_t) { return hipSuccess; }
hipError_t hipStreamSynchronize(hipStream_t) { return hipSuccess; }
hipError_t hipDeviceSynchronize(void) { return hipSuccess; }
hipError_t hipStreamIsCapturing(hipStream_t stream, hipStreamCaptureStatus* status) {
  *status = stream && g_capturing ? hipStreamCaptureStatusActive : hipStreamCaptureStatusNone;
  return hipSuccess;
}
hipError_t hipStreamGetCaptureInfo(hipStream_t stream, hipStreamCaptureStatus* status, unsigned long long* id) {
  if (id) *id = g_capture_id;
  return hipStreamIsCapturing(stream, status);
}
hipError_t hipThreadExchangeStreamCaptureMode(hipStreamCaptureMode* mode) {
  if (g_exchange_rc != 0) return answer(static_cast<hipError_t>(g_exchange_rc.load()));
  std::swap(t_mode, *mode);
  return hipSuccess;
}

}  // extern "C"
