// llmq_serve.cuh - what the serving operators on device memory share: checks
// of descriptors on the host, element types, and launches with programmatic
// dependent launch.  Inline functions only.
#pragma once

#include <cstdint>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "llmq_internal.h"

namespace llmq {

// ------------------------------------------------------------- host checks
// The first check that fails sets the error; later ones do nothing.
struct ServeCheck {
  const char *fn;
  int rc = LLMQ_OK;
  int device = -1;
  explicit ServeCheck(const char *name) : fn(name) {}

  void require(bool ok, const char *what) {
    if (rc != LLMQ_OK || ok) return;
    rc = LLMQ_ERR_ARG;
    llmq_set_error(rc, "%s: %s", fn, what);
  }
  // Arrays of T start on one: the kernels load and store whole elements.
  template <typename T>
  void elements(const T *p, const char *what) {
    if (rc != LLMQ_OK || reinterpret_cast<uintptr_t>(p) % sizeof(T) == 0) return;
    rc = LLMQ_ERR_ARG;
    llmq_set_error(rc, "%s: %s does not start on an element", fn, what);
  }
  void on_device() {
    if (rc != LLMQ_OK) return;
    int major = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e == cudaSuccess) e = cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, device);
    if (e != cudaSuccess || major != 10) {
      cudaGetLastError();
      rc = LLMQ_ERR_NO_DEVICE;
      llmq_set_error(rc, "%s: needs an sm_100 GPU (%s)", fn,
                     e != cudaSuccess ? cudaGetErrorString(e) : "another GPU is current");
    }
  }
  // p (null: nothing to check) lies in memory of the current GPU.
  void memory(const void *p, const char *what) {
    if (rc != LLMQ_OK || !p) return;
    cudaPointerAttributes at{};
    const cudaError_t e = cudaPointerGetAttributes(&at, p);
    if (e == cudaSuccess && (at.type == cudaMemoryTypeDevice || at.type == cudaMemoryTypeManaged) &&
        at.device == device)
      return;
    cudaGetLastError();
    rc = LLMQ_ERR_ARG;
    llmq_set_error(rc, "%s: %s is not memory of the current GPU", fn, what);
  }
  void launched(cudaError_t e) {
    if (rc != LLMQ_OK || e == cudaSuccess) return;
    cudaGetLastError();
    rc = LLMQ_ERR_CUDA;
    llmq_set_error(rc, "%s: launch failed (%s)", fn, cudaGetErrorString(e));
  }
};

// Rows or requests of a call: kernels and launch loops step over them in ints, by blocks of
// at most 4096.
constexpr int kServeMaxRows = 0x7fffffff - 4096;

inline bool serve_dtype(int t) { return t == LLMQ_F32 || t == LLMQ_F16 || t == LLMQ_BF16; }
inline size_t serve_bytes(int t) { return t == LLMQ_F32 ? 4 : 2; }
inline bool aligned16(const void *p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
inline bool aligned_to(const void *p, size_t n) { return reinterpret_cast<uintptr_t>(p) % n == 0; }

// A launch whose kernel may start before the previous one on the stream has
// ended; it waits with griddepcontrol.wait before it reads or writes memory.
template <typename... KArgs, typename... Args>
inline cudaError_t serve_launch(void (*kern)(KArgs...), dim3 grid, dim3 block, size_t smem, cudaStream_t st,
                                Args... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  llmqd_count_launch();
  return cudaLaunchKernelEx(&cfg, kern, args...);
}

// ----------------------------------------------------------------- device
__device__ __forceinline__ void serve_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void serve_dependents() { asm volatile("griddepcontrol.launch_dependents;"); }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) {
  return __float2half_rn(v);
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}

// N adjacent elements as one aligned load or store.
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

}  // namespace llmq
