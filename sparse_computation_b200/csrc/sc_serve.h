// Host-side helpers shared by the serving operators (sc_serve.cu,
// sc_adapters.cu): status codes at the C boundary, device selection, the
// device status word, and element types.
#pragma once

#include <cstdint>
#include <new>
#include <string>

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include "sc_internal.h"

namespace sc {
namespace serve {

inline void require(bool cond, int code, const char *msg) {
  if (!cond) throw sc_error(code, msg);
}

inline void cuda_check(cudaError_t e, const char *what) {
  if (e != cudaSuccess) throw sc_error(SC_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

struct DeviceGuard {
  int prev = -1, dev;
  explicit DeviceGuard(int d) : dev(d) {
    cuda_check(cudaGetDevice(&prev), "cudaGetDevice");
    if (prev != dev) cuda_check(cudaSetDevice(dev), "cudaSetDevice");
  }
  ~DeviceGuard() {
    if (prev != dev && prev >= 0) cudaSetDevice(prev);
  }
};

// One cudaMalloc'd block, freed on its own device.
struct DeviceBlock {
  int device = 0;
  void *p = nullptr;
  void alloc(int dev, size_t bytes, const char *what) {
    device = dev;
    cuda_check(cudaMalloc(&p, bytes), what);
  }
  DeviceBlock() = default;
  DeviceBlock(const DeviceBlock &) = delete;
  DeviceBlock &operator=(const DeviceBlock &) = delete;
  ~DeviceBlock() {
    if (!p) return;
    int prev = -1;
    if (cudaGetDevice(&prev) != cudaSuccess) return;
    if (prev != device) cudaSetDevice(device);
    cudaFree(p);
    if (prev != device) cudaSetDevice(prev);
  }
};

// Zeros at p when this returns.  The wait matters: the memset is asynchronous on
// the legacy stream, and a kernel that a non-blocking stream starts next could
// set a status before it.
inline void clear_words(void *p, size_t bytes) {
  cuda_check(cudaMemset(p, 0, bytes), "clear status");
  cuda_check(cudaStreamSynchronize(nullptr), "stream synchronize");
}

// Reads and clears a device status word after all work on its device.
inline int take_status(int device, int *word) {
  DeviceGuard dg(device);
  cuda_check(cudaDeviceSynchronize(), "device synchronize");
  int v = 0;
  cuda_check(cudaMemcpy(&v, word, sizeof v, cudaMemcpyDeviceToHost), "read status");
  if (v) clear_words(word, sizeof v);
  return v;
}

// A cleared status word of its own, on the current device.
inline void make_status(DeviceBlock &block, int device) {
  block.alloc(device, 256, "allocate status word");
  clear_words(block.p, 256);
}

inline int64_t type_bytes(int64_t t) { return t == SC_TYPE_F32 ? 4 : 2; }
inline bool type_ok(int64_t t) { return t == SC_TYPE_F32 || t == SC_TYPE_F16 || t == SC_TYPE_BF16; }

}  // namespace serve
}  // namespace sc

struct sc_kv_cache {
  sc_kv_pool pool;
  int device = 0;
  sc::serve::DeviceBlock status;
};

#define SC_SERVE_BEGIN try {
#define SC_SERVE_END                        \
  }                                         \
  catch (const sc_error &e) {               \
    sc_set_error(e.what());                 \
    return e.code;                          \
  }                                         \
  catch (const std::bad_alloc &) {          \
    sc_set_error("host allocation failed"); \
    return SC_ERR_NOMEM;                    \
  }                                         \
  catch (const std::exception &e) {         \
    sc_set_error(e.what());                 \
    return SC_ERR_ARG;                      \
  }                                         \
  return SC_OK;

#ifdef __CUDACC__
namespace sc {
namespace serve {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// The first error of a call's kernels stays until the host reads it.
__device__ __forceinline__ void set_status(int *word, int code) { atomicCAS(word, 0, code); }

}  // namespace serve
}  // namespace sc
#endif
