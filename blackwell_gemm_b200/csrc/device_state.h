// What the launchers of one library share about a device: set up once by
// gemm_capi.cu, read by the mixture-of-experts launchers (moe_capi.cu).
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

namespace b200 {

struct DeviceView {
  int device = -1;
  int sms = 0;
  int* status = nullptr;             // device error word
  cudaMemPool_t pool = nullptr;      // stream-ordered workspaces
  unsigned long long timeout_ns = 0; // bound on any single pipeline wait
};

// While it lives, this thread's calls leave captures of other threads alone: in
// CUDA's default capture mode any allocation, also one in the order of a
// stream that nobody captures, is refused and ends every capture under way.
struct RelaxedCapture {
  cudaStreamCaptureMode mode = cudaStreamCaptureModeRelaxed;
  RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
  ~RelaxedCapture() { cudaThreadExchangeStreamCaptureMode(&mode); }
  RelaxedCapture(const RelaxedCapture&) = delete;
  RelaxedCapture& operator=(const RelaxedCapture&) = delete;
};

// Memory of a pool, taken and given back in the order of `stream`.
template <class T>
inline bool pool_take(T** p, size_t bytes, cudaMemPool_t pool, cudaStream_t stream) {
  const RelaxedCapture relaxed;
  void* got = nullptr;
  if (pool == nullptr || cudaMallocFromPoolAsync(&got, bytes, pool, stream) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  *p = static_cast<T*>(got);
  return true;
}
inline bool pool_give(void* p, cudaStream_t stream) {
  const RelaxedCapture relaxed;
  return cudaFreeAsync(p, stream) == cudaSuccess;
}

// The current device, set up on its first call.  Returns a status code.
int device_view(DeviceView* out);

// What names a stream among all that the program ever has: a handle may come
// back after its stream is destroyed, and cudaStreamPerThread is one handle
// for another stream in each thread.  False where the stream has none.
bool stream_id(cudaStream_t stream, unsigned long long* id);

// A tiled tensor map of rank 2 or 3 over 1-, 2- or 4-byte elements, 128-byte
// swizzle, zero fill out of bounds.  strides_bytes: rank - 1 strides of the
// outer dimensions.  Returns a status code.
int encode_tensor(CUtensorMap* map, CUtensorMapDataType type, int rank, const void* base,
                  const cuuint64_t* dims, const cuuint64_t* strides_bytes, const cuuint32_t* box);

}  // namespace b200
