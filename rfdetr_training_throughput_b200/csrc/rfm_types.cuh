// Element types of the layer operators (RFM_DTYPE_*): loads, stores and the
// one rounding on the way out.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "rfm_common.cuh"

namespace rfm {

// The layer operators' kernels are launched with programmatic stream
// serialization: their CTAs may start while the kernel before them drains, and
// wait in chain_start before they touch memory, until that kernel has completed
// (and so, as it waited in its turn, everything before it).  About 2 us a launch
// where kernels are short (300 x 256 -> 91: 8.2 us a call without, 6.0 with).
// Every kernel that launch_chained starts calls chain_start first.
enum class Chain {
  kNext,   // behind another kernel of the same call
  kFirst,  // the call's first: an ordinary launch inside a stream capture, where the node before may be anything
  kNone,   // an ordinary launch
};

__device__ __forceinline__ void chain_start() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  grid_dependency_wait();
}

template <typename... Params, typename... Args>
int launch_chained(Chain chain, void (*kernel)(Params...), dim3 grid, int threads, int smem, int cluster,
                   cudaStream_t stream, const Args&... args) {
  cudaLaunchConfig_t config{};
  config.gridDim = grid;
  config.blockDim = dim3(static_cast<unsigned>(threads));
  config.dynamicSmemBytes = static_cast<size_t>(smem);
  config.stream = stream;
  cudaLaunchAttribute attrs[2];
  unsigned n = 0;
  if (cluster > 1) {
    attrs[n].id = cudaLaunchAttributeClusterDimension;
    attrs[n].val.clusterDim.x = static_cast<unsigned>(cluster);
    attrs[n].val.clusterDim.y = attrs[n].val.clusterDim.z = 1;
    ++n;
  }
  cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
  if (chain == Chain::kFirst && cudaStreamIsCapturing(stream, &capture) != cudaSuccess) {
    cudaGetLastError();
    capture = cudaStreamCaptureStatusInvalidated;  // an ordinary launch, which reports the stream's error
  }
  if (chain != Chain::kNone && capture == cudaStreamCaptureStatusNone) {
    attrs[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attrs[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  config.attrs = attrs;
  config.numAttrs = n;
  if (cudaLaunchKernelEx(&config, kernel, static_cast<Params>(args)...) != cudaSuccess) {
    cudaGetLastError();
    return RFM_ERR_LAUNCH;
  }
  return RFM_OK;
}

inline int dtype_bytes(int dtype) { return dtype == RFM_DTYPE_F32 ? 4 : 2; }
inline bool dtype_known(int dtype) {
  return dtype == RFM_DTYPE_F32 || dtype == RFM_DTYPE_BF16 || dtype == RFM_DTYPE_F16;
}

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_float(__half v) { return __half2float(v); }

template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) {
  return __float2bfloat16_rn(v);
}
template <>
__device__ __forceinline__ __half from_float<__half>(float v) {
  return __float2half_rn(v);
}

// VEC consecutive elements moved as one access (16 bytes for the full vectors).
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

// Two fp32 values in one register pair and one instruction (the sm_100 f32x2
// operations; each half is rounded by itself).
struct Pair {
  uint64_t v;
};
__device__ __forceinline__ Pair pair(float x, float y) {
  Pair r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ float2 split(Pair p) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p.v));
  return r;
}
__device__ __forceinline__ Pair operator+(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair fma(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

__device__ __forceinline__ Pair both(float x) { return pair(x, x); }

// Elements 2 i and 2 i + 1 of a pack.
template <typename T, int VEC>
__device__ __forceinline__ Pair load_pair(const Pack<T, VEC>& p, int i) {
  return pair(to_float(p.v[2 * i]), to_float(p.v[2 * i + 1]));
}
template <typename T, int VEC>
__device__ __forceinline__ void store_pair(Pack<T, VEC>& p, int i, Pair v) {
  const float2 f = split(v);
  p.v[2 * i] = from_float<T>(f.x);
  p.v[2 * i + 1] = from_float<T>(f.y);
}
template <>
__device__ __forceinline__ void store_pair<__nv_bfloat16, 8>(Pack<__nv_bfloat16, 8>& p, int i, Pair v) {
  reinterpret_cast<__nv_bfloat162*>(p.v)[i] = __float22bfloat162_rn(split(v));
}
template <>
__device__ __forceinline__ void store_pair<__half, 8>(Pack<__half, 8>& p, int i, Pair v) {
  reinterpret_cast<__half2*>(p.v)[i] = __float22half2_rn(split(v));
}

// Element i of a parameter array whose type is known at run time only (read
// once per thread, outside the row loops).
__device__ __forceinline__ float load_param(const void* p, int dtype, int64_t i) {
  if (dtype == RFM_DTYPE_F32) return static_cast<const float*>(p)[i];
  if (dtype == RFM_DTYPE_BF16) return to_float(static_cast<const __nv_bfloat16*>(p)[i]);
  return to_float(static_cast<const __half*>(p)[i]);
}

__device__ __forceinline__ void store_param(void* p, int dtype, int64_t i, float v) {
  if (dtype == RFM_DTYPE_F32) {
    static_cast<float*>(p)[i] = v;
  } else if (dtype == RFM_DTYPE_BF16) {
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
  } else {
    static_cast<__half*>(p)[i] = __float2half_rn(v);
  }
}

}  // namespace rfm
