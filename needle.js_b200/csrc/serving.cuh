// serving.cuh -- what the serving operators (rope.cu, prefix_attn.cu, logits.cu) share: element
// types, vector access, powers of two, argument checks and the guard of their C entries.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <exception>
#include <initializer_list>
#include <string>

#include "../../include/needle_cuda.h"
#include "engine.cuh"

namespace needle {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }

template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N consecutive elements in one access (sizeof(T) * N of 2, 4, 8 or 16 bytes, aligned to its size).
template <class T, int N>
struct alignas(sizeof(T) * N) Vec {
  T v[N];
};

constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float power2f(float v) {  // 2^v, relative error 2^-22, 0 below 2^-126
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ uint32_t shared_address(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void barrier_init(uint64_t* b, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(shared_address(b)), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_arrive(uint64_t* b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(shared_address(b)) : "memory");
}
__device__ __forceinline__ bool barrier_try(uint64_t* b, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
      : "=r"(ok)
      : "r"(shared_address(b)), "r"(parity)
      : "memory");
  return ok != 0;
}
constexpr uint64_t kServingWaitNs = 2000000000ull;
// Waits for the phase of the given parity; false once kServingWaitNs has passed without it.
__device__ __forceinline__ bool barrier_wait(uint64_t* b, uint32_t parity) {
  if (barrier_try(b, parity)) return true;
  uint64_t start, now;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(start));
  for (;;) {
    for (int i = 0; i < 64; i++)
      if (barrier_try(b, parity)) return true;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
    if (now - start > kServingWaitNs) return false;
  }
}

// The same for a converged warp, all lanes polling: a branch that one lane takes, and coming back from it,
// costs a waiting warp about 200 cycles.
__device__ __forceinline__ bool barrier_wait_warp(uint64_t* b, uint32_t parity) {
  if (__all_sync(0xffffffffu, barrier_try(b, parity))) return true;
  uint64_t start, now;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(start));
  for (;;) {
    for (int i = 0; i < 64; i++)
      if (__all_sync(0xffffffffu, barrier_try(b, parity))) return true;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
    if (__any_sync(0xffffffffu, now - start > kServingWaitNs)) return false;
  }
}

// Global -> shared bulk copy whose bytes are counted on `bar`.
__device__ __forceinline__ void copy_bulk(void* to, const void* from, uint32_t bytes, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(shared_address(to)),
      "l"(from), "r"(bytes), "r"(shared_address(bar))
      : "memory");
}

inline size_t type_bytes(int32_t type) { return type == NEEDLE_TYPE_F32 ? 4 : 2; }

inline bool aligned_to(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) & (bytes - 1)) == 0; }

// Calls f(T{}) with the element type of a needle_type.
template <class F>
cudaError_t with_type(int32_t type, F f) {
  if (type == NEEDLE_TYPE_F32) return f(float{});
  if (type == NEEDLE_TYPE_F16) return f(__half{});
  return f(__nv_bfloat16{});
}

inline int refuse(const std::string& msg) {
  set_last_error(msg);
  return NEEDLE_BACKEND_UNAVAILABLE;
}

inline int refuse_cuda(const char* op, cudaError_t e) { return refuse(std::string(op) + ": " + cudaGetErrorString(e)); }

// Whether `p` is memory that kernels of the current device `device` can use: a host pointer or a
// buffer of another GPU is refused before a launch, where it would fault or cross the link unseen.
inline int check_buffer(const void* p, const char* name, int device) {
  cudaPointerAttributes a{};
  const cudaError_t e = cudaPointerGetAttributes(&a, p);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return refuse(std::string(name) + ": " + cudaGetErrorString(e));
  }
  if (a.type != cudaMemoryTypeDevice && a.type != cudaMemoryTypeManaged)
    return refuse(std::string(name) + " is not device memory");
  if (a.type == cudaMemoryTypeDevice && a.device != device)
    return refuse(std::string(name) + " is on device " + std::to_string(a.device) + ", the current device is " +
                  std::to_string(device));
  return NEEDLE_OK;
}

// A device buffer of a call (NULL: not given) and the bytes its elements are aligned to.
struct Buffer {
  const void* p;
  const char* name;
  size_t element;
};
using Buffers = std::initializer_list<Buffer>;

inline int check_alignment(Buffers buffers) {
  for (const Buffer& b : buffers)
    if (!aligned_to(b.p, b.element)) return refuse(std::string(b.name) + " is not aligned to its element type");
  return NEEDLE_OK;
}

inline int check_buffers(Buffers buffers, int device) {
  for (const Buffer& b : buffers)
    if (b.p)
      if (int rc = check_buffer(b.p, b.name, device)) return rc;
  return NEEDLE_OK;
}

// Runs an entry's body; no C++ exception crosses the C boundary.
template <class F>
int entry(F f) noexcept {
  try {
    return f();
  } catch (const std::exception& e) {
    try {
      return refuse(e.what());
    } catch (...) {
      return NEEDLE_BACKEND_UNAVAILABLE;
    }
  } catch (...) {
    return NEEDLE_BACKEND_UNAVAILABLE;
  }
}

}  // namespace needle
