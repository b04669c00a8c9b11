// Device helpers shared by the training operators (eb_backward.cu, eb_layer_norm.cu, eb_adamw.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>
#include <cstring>
#include <type_traits>

#include "eb_internal.h"
#include "fwd_eb_train.h"

namespace fwd_eb {

// Programmatic stream serialisation: where a kernel releases its dependents at its start, the next grid of the stream may
// start its blocks as soon as all of this one's are resident, and waits until this one has finished.  Every
// kernel of these operators waits before its first access to memory, on every path.  It releases its successor
// early only where that is the next kernel of the same call (`more`): what comes behind a call may read the call's
// results through the read-only path, as the pooling kernels do with a table that AdamW has just written, and data on
// that path may not change while the reader is resident.
__device__ __forceinline__ void pdl_enter(bool more) {
  if (more) asm volatile("griddepcontrol.launch_dependents;");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}

template <typename... KArgs, typename... Args>
inline cudaError_t launch_pdl(void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, cudaStream_t st,
                              Args&&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3((unsigned)threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
  count_launch();
  return e != cudaSuccess ? e : cudaGetLastError();
}

// Lets a kernel take up to BYTES of dynamic shared memory; more than the default 48 KB (what is static counts
// too) has to be allowed once a device.
template <auto KERNEL, int BYTES>
inline cudaError_t allow_shared() {
  if (BYTES <= 40 * 1024) return cudaSuccess;
  static std::atomic<uint64_t> allowed{0};   // a bit a device
  int device = 0;
  cudaError_t e = cudaGetDevice(&device);
  if (e != cudaSuccess) return e;
  const uint64_t bit = device < 64 ? 1ull << device : 0;
  if (allowed.load(std::memory_order_relaxed) & bit) return cudaSuccess;
  e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, BYTES);
  if (e == cudaSuccess) allowed.fetch_or(bit, std::memory_order_relaxed);
  return e;
}

inline int dtype_size(int dtype) { return dtype == FWD_EB_F32 ? 4 : 2; }
inline bool aligned_to(const void* p, size_t bytes) { return (reinterpret_cast<uintptr_t>(p) % bytes) == 0; }

__device__ __forceinline__ float to_float(float x) { return x; }
__device__ __forceinline__ float to_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float to_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// One rounding, to nearest even, from the fp32 result to the stored type.
template <typename T>
__device__ __forceinline__ T from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

// 16 bytes from global to shared memory without passing through registers; groups complete in order.
__device__ __forceinline__ void copy16_async(void* shared, const void* global) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
               :: "r"((unsigned)__cvta_generic_to_shared(shared)), "l"(global) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {   // until at most the N newest groups are under way
  asm volatile("cp.async.wait_group %0;" :: "n"(N) : "memory");
}

// Two fp32 operations in one instruction (sm_100's packed pipe); each half rounds on its own.
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{.reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n"
      " add.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{.reg .b64 x, y;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n"
      " mul.rn.f32x2 x, x, y;\n mov.b64 {%0, %1}, x;}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{.reg .b64 x, y, z;\n mov.b64 x, {%2, %3};\n mov.b64 y, {%4, %5};\n mov.b64 z, {%6, %7};\n"
      " fma.rn.f32x2 x, x, y, z;\n mov.b64 {%0, %1}, x;}"
      : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 both(float x) { return make_float2(x, x); }

// V consecutive elements as aligned accesses of up to 16 bytes.
template <int BYTES>
struct Word;
template <>
struct Word<1> { using type = unsigned char; };
template <>
struct Word<2> { using type = unsigned short; };
template <>
struct Word<4> { using type = unsigned; };
template <>
struct Word<8> { using type = uint2; };
template <>
struct Word<16> { using type = uint4; };

template <typename T, int V>
struct Pack {
  static constexpr int kBytes = V * (int)sizeof(T);
  static constexpr int kWord = kBytes < 16 ? kBytes : 16;   // bytes of one access, and its alignment
  static constexpr int kWords = kBytes / kWord;
  using W = typename Word<kWord>::type;
  W w[kWords];
  __device__ __forceinline__ void load(const void* p) {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = static_cast<const W*>(p)[i];
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = W{};
  }
  __device__ __forceinline__ void store(void* p) const {
#pragma unroll
    for (int i = 0; i < kWords; ++i) static_cast<W*>(p)[i] = w[i];
  }
  __device__ __forceinline__ void get(float (&f)[V]) const {
    if constexpr (sizeof(T) == 4) {
      memcpy(f, w, sizeof(f));
    } else if constexpr (V == 1) {
      T t;
      memcpy(&t, w, sizeof(t));
      f[0] = to_float(t);
    } else {
      unsigned u[V / 2];
      memcpy(u, w, sizeof(u));
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        float2 t;
        if constexpr (std::is_same<T, __half>::value) {
          __half2 h;
          memcpy(&h, &u[i], 4);
          t = __half22float2(h);
        } else {
          __nv_bfloat162 h;
          memcpy(&h, &u[i], 4);
          t = __bfloat1622float2(h);
        }
        f[2 * i] = t.x;
        f[2 * i + 1] = t.y;
      }
    }
  }
  __device__ __forceinline__ void set(const float (&f)[V]) {
    if constexpr (sizeof(T) == 4) {
      memcpy(w, f, sizeof(f));
    } else if constexpr (V == 1) {
      const T t = from_float<T>(f[0]);
      memcpy(w, &t, sizeof(t));
    } else {
      unsigned u[V / 2];
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        if constexpr (std::is_same<T, __half>::value) {
          const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
          memcpy(&u[i], &h, 4);
        } else {
          const __nv_bfloat162 h = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
          memcpy(&u[i], &h, 4);
        }
      }
      memcpy(w, u, sizeof(u));
    }
  }
};

// V elements at p, whose type is only known at run time (the same for every thread of the grid).
template <int V>
__device__ __forceinline__ void load_any(const void* p, int dtype, long long at, float (&f)[V]) {
  if (dtype == FWD_EB_F32) {
    Pack<float, V> r;
    r.load(static_cast<const float*>(p) + at);
    r.get(f);
  } else if (dtype == FWD_EB_F16) {
    Pack<__half, V> r;
    r.load(static_cast<const __half*>(p) + at);
    r.get(f);
  } else {
    Pack<__nv_bfloat16, V> r;
    r.load(static_cast<const __nv_bfloat16*>(p) + at);
    r.get(f);
  }
}

template <int V>
__device__ __forceinline__ void store_any(void* p, int dtype, long long at, const float (&f)[V]) {
  if (dtype == FWD_EB_F32) {
    Pack<float, V> r;
    r.set(f);
    r.store(static_cast<float*>(p) + at);
  } else if (dtype == FWD_EB_F16) {
    Pack<__half, V> r;
    r.set(f);
    r.store(static_cast<__half*>(p) + at);
  } else {
    Pack<__nv_bfloat16, V> r;
    r.set(f);
    r.store(static_cast<__nv_bfloat16*>(p) + at);
  }
}

}  // namespace fwd_eb
