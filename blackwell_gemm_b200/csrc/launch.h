// What the launchers of the operators share (moe_capi.cu, ffn_capi.cu): tensor
// maps of operands, workspaces in stream order, launches.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>

#include "b200_moe.h"
#include "device_state.h"
#include "gemm_layout.h"

namespace b200 {

constexpr int kMaxDevices = 64;
// The kernels index an extent in 32 bits and may look a tile, a block's step or
// a block's chunk of tokens past its end.
constexpr int kMaxExtent = 0x7FFFFFFF - (1 << 25) + 1;

inline long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

template <class F>
inline bool set_smem(F* fn, int bytes) {
  return cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) ==
         cudaSuccess;
}

// Arrival counts of the streaming kernels: one array per (device, stream),
// made on the stream's first call; every launch leaves it at zero.  Null when
// none can be made, as for streams after the first 256 (the caller then clears
// counts of its own).
constexpr size_t kCountBytes = 4096 * sizeof(unsigned int);
unsigned int* stream_counts(const DeviceView& v, cudaStream_t stream);

// Slots and counts of one streaming launch.  Counts are the stream's own
// array, except under capture (a graph may be replayed on another stream),
// where they come with the slots and are cleared in the graph.
struct Workspace {
  char* base = nullptr;
  cudaStream_t stream = nullptr;
  template <class Args>
  int take(const DeviceView& v, size_t slot_bytes, cudaStream_t s, Args* args) {
    stream = s;
    cudaStreamCaptureStatus cap = cudaStreamCaptureStatusNone;
    if (cudaStreamIsCapturing(s, &cap) != cudaSuccess) {
      cudaGetLastError();
      cap = cudaStreamCaptureStatusActive;
    }
    args->counts = cap == cudaStreamCaptureStatusNone ? stream_counts(v, s) : nullptr;
    if (!pool_take(&base, kCountBytes + slot_bytes, v.pool, s)) return B200_ERR_LAUNCH;
    args->slots = reinterpret_cast<float*>(base + kCountBytes);
    if (args->counts == nullptr) {
      args->counts = reinterpret_cast<unsigned int*>(base);
      if (cudaMemsetAsync(base, 0, kCountBytes, s) != cudaSuccess) {
        cudaGetLastError();
        return B200_ERR_LAUNCH;
      }
    }
    return B200_OK;
  }
  ~Workspace() {
    if (base) pool_give(base, stream);
  }
};

// A buffer of the device's pool for one call, freed in stream order.
struct PoolBuffer {
  char* p = nullptr;
  cudaStream_t stream = nullptr;
  int take(const DeviceView& v, size_t bytes, cudaStream_t s) {
    stream = s;
    return pool_take(&p, bytes, v.pool, s) ? B200_OK : B200_ERR_LAUNCH;
  }
  ~PoolBuffer() {
    if (p) pool_give(p, stream);
  }
};

inline CUtensorMapDataType map_type(int dtype) {
  return dtype == B200_FP16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
}

inline int map_rows(CUtensorMap* m, int dtype, const void* p, int cols, int rows, int ld,
                    int box_rows) {
  const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
  const cuuint64_t strides[1] = {(cuuint64_t)ld * 2};
  const cuuint32_t box[2] = {kSlabK, (cuuint32_t)box_rows};
  return encode_tensor(m, map_type(dtype), 2, p, dims, strides, box);
}

inline int map_bank(CUtensorMap* m, int dtype, const void* p, int K, int N, int experts, int ld,
                    long long expert_stride, int box_rows) {
  const cuuint64_t dims[3] = {(cuuint64_t)K, (cuuint64_t)N, (cuuint64_t)experts};
  // (the stride of a bank of one is never used; any valid one will do)
  const cuuint64_t far = experts > 1 ? (cuuint64_t)expert_stride * 2 : (cuuint64_t)N * ld * 2;
  const cuuint64_t strides[2] = {(cuuint64_t)ld * 2, far};
  const cuuint32_t box[3] = {kSlabK, (cuuint32_t)box_rows, 1};
  return encode_tensor(m, map_type(dtype), 3, p, dims, strides, box);
}

inline bool tma_rows(const void* p, long long ld) { return aligned16(p) && (ld & 7) == 0; }

inline int zero_rows(void* p, int ld, int width, int rows, cudaStream_t stream) {
  if (rows == 0 || width == 0) return B200_OK;
  return cudaMemset2DAsync(p, (size_t)ld * 2, 0, (size_t)width * 2, rows, stream) == cudaSuccess
             ? B200_OK
             : B200_ERR_LAUNCH;
}

// Launch with programmatic stream serialization: the kernel's set-up overlaps
// the end of the one before it (every kernel launched so waits, grid_wait,
// before it touches global memory).
template <class... P, class... A>
int launch_clusters(void (*fn)(P...), int blocks, int cluster, int threads, size_t smem,
                    cudaStream_t stream, A&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)cluster;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 0 ? 2 : 1;
  if (cudaLaunchKernelEx(&cfg, fn, static_cast<P>(args)...) == cudaSuccess) return B200_OK;
  cudaGetLastError();
  return B200_ERR_LAUNCH;
}

// (clusters as the kernel itself says)
template <class... P, class... A>
int launch(void (*fn)(P...), int blocks, int threads, size_t smem, cudaStream_t stream,
           A&&... args) {
  return launch_clusters(fn, blocks, 0, threads, smem, stream, static_cast<A&&>(args)...);
}

}  // namespace b200
