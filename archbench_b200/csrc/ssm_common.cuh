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

// Hardware 2^x (about 2 units in the last place; 0 below 2^-126) and reciprocal (1 unit).
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
constexpr float LOG2E = 1.44269504088896340736f;

__device__ __forceinline__ float sigmoid(float x) { return rcp(1.f + ex2(-LOG2E * x)); }
__device__ __forceinline__ float silu(float x) { return x * sigmoid(x); }
// d silu(x) / dx
__device__ __forceinline__ float dsilu(float x) {
  const float g = sigmoid(x);
  return g * fmaf(x, 1.f - g, 1.f);
}
// log(1 + e^v) = max(v, 0) + log(1 + e) with e = e^-|v| in (0, 1]; log(1 + e) = 2 artanh(w), w = e / (2 + e) <= 1/3, by a
// polynomial in w^2 of relative error 8e-9 (a least-maximum fit), so small e keeps its relative precision.
__device__ __forceinline__ float softplus(float v) {
  const float e = ex2(-LOG2E * fabsf(v)), w = e * rcp(2.f + e), q = w * w;
  float r = fmaf(q, 0.2817838788032532f, 0.2796059250831604f);
  r = fmaf(q, r, 0.4002491235733032f);
  r = fmaf(q, r, 0.6666631698608398f);
  r = fmaf(q, r, 2.0f);
  return fmaf(w, r, fmaxf(v, 0.f));
}

// Two fp32 values in one 64-bit register: Blackwell multiplies and adds both with one instruction.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pack2(float lo, float hi) {
  f32x2 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(lo), "f"(hi));
  return r;
}
__device__ __forceinline__ float2 unpack2(f32x2 v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 r;
  asm("fma.rn.ftz.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("mul.rn.ftz.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 exp2_2(f32x2 x) {
  const float2 v = unpack2(x);
  return pack2(ex2(v.x), ex2(v.y));
}
__device__ __forceinline__ float sum2(f32x2 v) {
  const float2 e = unpack2(v);
  return e.x + e.y;
}

__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 r;
  asm("add.rn.ftz.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ f32x2 both(float v) { return pack2(v, v); }
// softplus and the sigmoid of two values (see above for the formulas).
__device__ __forceinline__ f32x2 sigmoid2(f32x2 x) {
  const float2 e = unpack2(add2(exp2_2(mul2(x, both(-LOG2E))), both(1.f)));
  return pack2(rcp(e.x), rcp(e.y));
}
__device__ __forceinline__ f32x2 softplus2(f32x2 v) {
  const float2 a = unpack2(v);
  const f32x2 e = exp2_2(mul2(pack2(fabsf(a.x), fabsf(a.y)), both(-LOG2E)));
  const float2 n = unpack2(add2(e, both(2.f)));
  const f32x2 w = mul2(e, pack2(rcp(n.x), rcp(n.y))), q = mul2(w, w);
  f32x2 r = fma2(q, both(0.2817838788032532f), both(0.2796059250831604f));
  r = fma2(q, r, both(0.4002491235733032f));
  r = fma2(q, r, both(0.6666631698608398f));
  r = fma2(q, r, both(2.0f));
  return fma2(w, r, pack2(fmaxf(a.x, 0.f), fmaxf(a.y, 0.f)));
}
// Two neighbouring token values in shared memory.
__device__ __forceinline__ f32x2 load_pair(const __nv_bfloat16* p) {
  const uint32_t r = *reinterpret_cast<const uint32_t*>(p);
  return pack2(__uint_as_float(r << 16), __uint_as_float(r & 0xffff0000u));
}
__device__ __forceinline__ f32x2 load_pair(const float* p) { return *reinterpret_cast<const f32x2*>(p); }

// 16 bytes into shared memory without a register; zeros where `on` is false (the address is then not read).
__device__ __forceinline__ void copy16(uint32_t dst, const void* src, bool on) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT>
__device__ __forceinline__ void copies_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory");
}
// 4, 8 or 16 bytes, always copied.
template <int BYTES>
__device__ __forceinline__ void copy_bytes(uint32_t dst, const void* src) {
  if (BYTES == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(dst), "l"(src), "n"(BYTES < 4 ? 4 : BYTES) : "memory");
}

// Tokens of row b.
__device__ __forceinline__ int row_tokens(const int32_t* lengths, int b, int T) {
  return lengths ? min(max(lengths[b], 0), T) : T;
}

}  // namespace ssm
}  // namespace gdn
