// Shared helpers of the selective-state-space kernels (convolution, scan, single-token step).
#pragma once

#include "gdn_common.cuh"

namespace gdn {
namespace ssm {

inline int elem_size(int dt) { return dt == GDN_DTYPE_F32 ? 4 : dt == GDN_DTYPE_BF16 ? 2 : 0; }

// The library carries sm_100a code only; the answer is cached per device.
inline bool device_ok() {
  static std::atomic<int> cached[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  if (dev >= 0 && dev < 64) {
    const int c = cached[dev].load(std::memory_order_relaxed);
    if (c) return c > 0;
  }
  int major = 0, minor = 0;
  if (cudaDeviceGetAttribute(&major, cudaDevAttrComputeCapabilityMajor, dev) != cudaSuccess ||
      cudaDeviceGetAttribute(&minor, cudaDevAttrComputeCapabilityMinor, dev) != cudaSuccess)
    return false;
  const bool ok = major == 10 && minor == 0;
  if (dev >= 0 && dev < 64) cached[dev].store(ok ? 1 : -1, std::memory_order_relaxed);
  return ok;
}

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

inline int launched() { return cudaGetLastError() == cudaSuccess ? GDN_OK : GDN_ERR_LAUNCH; }

// Store N consecutive values, as one 16-byte vector where they fill one.
template <int N, typename T>
__device__ __forceinline__ void store_vec(T* p, const float (&v)[N]) {
  if constexpr (sizeof(T) * N == 16) {
    uint4 raw;
    T* e = reinterpret_cast<T*>(&raw);
#pragma unroll
    for (int i = 0; i < N; ++i) store_as(e + i, v[i]);
    *reinterpret_cast<uint4*>(p) = raw;
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) store_as(p + i, v[i]);
  }
}

// A parameter stored as fp32 or bf16.
__device__ __forceinline__ float load_param(const void* p, int64_t i, int dtype) {
  return dtype == GDN_DTYPE_F32 ? static_cast<const float*>(p)[i] : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_param(void* p, int64_t i, int dtype, float v) {
  if (dtype == GDN_DTYPE_F32)
    static_cast<float*>(p)[i] = v;
  else
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

__device__ __forceinline__ float sigmoid(float x) { return __fdividef(1.f, 1.f + __expf(-x)); }
__device__ __forceinline__ float silu(float x) { return x * sigmoid(x); }
// d silu(x) / dx
__device__ __forceinline__ float dsilu(float x) {
  const float g = sigmoid(x);
  return g * fmaf(x, 1.f - g, 1.f);
}
// log(1 + e^v) without cancellation for negative v; e^-|v| lies in (0, 1].
__device__ __forceinline__ float softplus(float v) { return fmaxf(v, 0.f) + log1pf(expf(-fabsf(v))); }

// Tokens of row b.
__device__ __forceinline__ int row_tokens(const int32_t* lengths, int b, int T) {
  return lengths ? min(max(lengths[b], 0), T) : T;
}

}  // namespace ssm
}  // namespace gdn
