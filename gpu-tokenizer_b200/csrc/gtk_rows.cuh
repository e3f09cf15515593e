// gtk_rows.cuh -- what the operators on rows of numbers share (gtk_embed.cu, gtk_logprobs.cu, gtk_sample.cu, gtk_paged.cu): element types,
// vector loads and stores, and the frame of their entry points.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <algorithm>
#include <cstdint>
#include <mutex>
#include <new>
#include <string>

#include "../../include/gputok_b200.h"
#include "gtk_device.cuh"

namespace gtk {

// ------------------------------------------------------------------------------------------------ device side
__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }

template <class T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

// V neighbouring elements as they lie in memory, moved in accesses of up to 16 bytes
template <class T, int V>
struct alignas(sizeof(T) * V < 16 ? sizeof(T) * V : 16) Pack {
  T e[V];
};

template <class T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T* p) { return *reinterpret_cast<const Pack<T, V>*>(p); }
template <class T, int V>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, V>& v) { *reinterpret_cast<Pack<T, V>*>(p) = v; }

// Everything that the kernels in front of this one in the stream have written is there afterwards (gtk::launch_behind).  It is
// read with loads that the compiler leaves behind this one and that the first-level cache has no part in (__ldcg, not __ldg).
__device__ __forceinline__ void await_kernel() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

// Copies of 16 bytes to shared memory that a thread does not wait for: begun, closed as a chunk, and awaited until at most PENDING of
// its own chunks are under way.
__device__ __forceinline__ void copy16(uint32_t shared_at, const void* from)
{
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(shared_at), "l"(from) : "memory");
}
__device__ __forceinline__ void end_chunk() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void await_chunks() { asm volatile("cp.async.wait_group %0;" ::"n"(PENDING) : "memory"); }

// Two 32-bit floats that one instruction works on.
struct Two {
  uint64_t v;
  Two() = default;
  __device__ __forceinline__ Two(float lo, float hi) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(lo), "f"(hi)); }
  __device__ __forceinline__ void get(float& lo, float& hi) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
};
__device__ __forceinline__ Two operator+(Two a, Two b)
{
  Two d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}
__device__ __forceinline__ Two operator*(Two a, Two b)
{
  Two d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d.v) : "l"(a.v), "l"(b.v));
  return d;
}
__device__ __forceinline__ Two fma2(Two a, Two b, Two c)
{
  Two d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return d;
}

// a 32-bit word's one or two elements as 32-bit floats
__device__ __forceinline__ Two word_pair(uint32_t w, __nv_bfloat16) { return Two(__uint_as_float(w << 16), __uint_as_float(w & 0xFFFF0000u)); }
__device__ __forceinline__ Two word_pair(uint32_t w, __half)
{
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
  return Two(f.x, f.y);
}

// ------------------------------------------------------------------------------------------------ host side
inline int element_size(int type) { return type == GTK_F32 ? 4 : 2; }
inline bool known_type(int type) { return type == GTK_F32 || type == GTK_BF16 || type == GTK_F16; }
inline bool aligned_to(const void* p, size_t bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }
// whether all rows of an array start on a multiple of what `pack` elements take, 16 bytes at most
inline bool rows_aligned(const void* p, int64_t stride, int type, int pack)
{
  const int64_t bytes = std::min<int64_t>(16, int64_t(pack) * element_size(type));
  return aligned_to(p, size_t(bytes)) && stride * element_size(type) % bytes == 0;
}

// f(T{}) for the C++ type of an element type that known_type() has accepted
template <class F>
cudaError_t with_type(int type, F&& f)
{
  switch (type) {
    case GTK_F32: return f(float{});
    case GTK_BF16: return f(__nv_bfloat16{});
    default: return f(__half{});
  }
}

// A kernel whose calls want more than the usual 48 KiB of dynamic shared memory is allowed all that a CTA can have, whatever this
// call wants: the limit belongs to the kernel on the device, and another thread's call of another size, under another handle's lock,
// must not find it lowered between the two calls here.
constexpr int kSharedMost = 227 << 10;
template <class... Formal>
cudaError_t allow_shared(void (*kernel)(Formal...), size_t smem)
{
  return smem > (48 << 10) ? cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedMost) : cudaSuccess;
}

template <class... Formal, class... Args>
cudaError_t launch(void (*kernel)(Formal...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args&&... args)
{
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid, cfg.blockDim = block, cfg.dynamicSmemBytes = smem, cfg.stream = stream;
  const cudaError_t e = allow_shared(kernel, smem);
  return e != cudaSuccess ? e : cudaLaunchKernelEx(&cfg, kernel, static_cast<Formal>(args)...);
}

// the same for a kernel that begins with await_kernel(): its blocks may take their places while the kernel in front of it
// in the stream is still ending
template <class... Formal, class... Args>
cudaError_t launch_behind(void (*kernel)(Formal...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args&&... args)
{
  cudaLaunchAttribute attr{};
  attr.id                                         = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid, cfg.blockDim = block, cfg.dynamicSmemBytes = smem, cfg.stream = stream;
  cfg.attrs = &attr, cfg.numAttrs = 1;
  const cudaError_t e = allow_shared(kernel, smem);
  return e != cudaSuccess ? e : cudaLaunchKernelEx(&cfg, kernel, static_cast<Formal>(args)...);
}

// the same in clusters of `cluster` blocks next to each other
template <class... Formal, class... Args>
cudaError_t launch_clusters(void (*kernel)(Formal...), dim3 grid, dim3 block, int cluster, size_t smem, cudaStream_t stream, Args&&... args)
{
  cudaLaunchAttribute attr{};
  attr.id               = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = unsigned(cluster), attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid, cfg.blockDim = block, cfg.dynamicSmemBytes = smem, cfg.stream = stream;
  cfg.attrs = &attr, cfg.numAttrs = cluster > 1 ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<Formal>(args)...);
}

// What a refused argument is reported with: a message, or nullptr when there is nothing to refuse.
using Refusal = const char*;

// An operator's call: check() is asked first, on host-only handles too; then launches(view) runs with the handle's
// device current and the caller's put back afterwards.  Nothing is thrown past it.
template <class Check, class Launches>
int run_operator(gtk_tokenizer* h, Check&& check, Launches&& launches) noexcept
{
  if (!h) return GTK_ERR_INVALID_ARG;
  try {
    std::lock_guard<std::mutex> lock(*handle_mutex(h));
    HandleView v;
    handle_view(h, &v);
    if (const Refusal why = check()) {
      *v.last_error = why;
      return GTK_ERR_INVALID_ARG;
    }
    if (v.device < 0) {
      *v.last_error = "host-only handle: no GPU entry points";
      return GTK_ERR_NO_DEVICE;
    }
    int before    = -1;
    cudaError_t e = cudaGetDevice(&before);
    if (e == cudaSuccess && before != v.device) e = cudaSetDevice(v.device);
    if (e == cudaSuccess) e = launches(v);
    if (before >= 0 && before != v.device) cudaSetDevice(before);
    if (e != cudaSuccess) {
      cudaGetLastError();  // reported here: the thread's next call, which asks for the last error behind its launches, has its own
      *v.last_error = std::string("launch: ") + cudaGetErrorString(e);
      return GTK_ERR_CUDA;
    }
    return GTK_OK;
  } catch (...) {  // std::bad_alloc of a message, std::system_error of the lock
    return GTK_ERR_MEMORY;
  }
}

}  // namespace gtk
