// Device helpers of the 8-bit linear path: element loads and stores, e4m3
// conversions and the scale of a block.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <atomic>
#include <type_traits>

#include "blocks.h"

namespace ob2 {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// max that keeps a NaN of either side (fmaxf drops it): a block that holds one
// must not get a finite scale.
__device__ __forceinline__ float max_nan(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// max_nan(m, |v|)
__device__ __forceinline__ float max_abs_nan(float m, float v) {
  float r;
  asm("{\n\t.reg .f32 t;\n\tabs.f32 t, %2;\n\tmax.NaN.f32 %0, %1, t;\n\t}" : "=f"(r) : "f"(m), "f"(v));
  return r;
}

// Two values rounded to a 16-bit type in one register.
template <typename T>
__device__ __forceinline__ uint32_t pack_rounded(float lo, float hi) {
  uint32_t r;
  if constexpr (std::is_same_v<T, __half>)
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Scale of a block and the factor its elements are multiplied with, from its
// largest magnitude.  The floor keeps the factor finite for an all-zero block;
// the comparison is false for NaN, which therefore reaches both.
__device__ __forceinline__ void block_scale(float amax, float& scale, float& inv) {
  const float a = amax < kAmaxFloor ? kAmaxFloor : amax;
  scale = __fdiv_rn(a, kE4m3Max);
  inv = __fdiv_rn(kE4m3Max, a);
}

// fp32 -> e4m3, nearest even, saturating at 448; NaN stays NaN.
__device__ __forceinline__ uint8_t to_e4m3(float v) {
  return (uint8_t)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d) {
  uint16_t lo, hi;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
  return (uint32_t)lo | ((uint32_t)hi << 16);
}
__device__ __forceinline__ float from_e4m3(uint8_t v) {
  return __half2float(__half(__nv_cvt_fp8_to_halfraw(v, __NV_E4M3)));
}

// The shared-memory opt-in is a per-device attribute of a kernel, set once: to the
// most that any call asks for, so that calls on several threads agree.
template <auto KERNEL>
int opt_in(int bytes) {
  constexpr int kMaxDevices = 64;
  static std::atomic<bool> done[kMaxDevices] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return (int)cudaErrorInvalidDevice;
  if (done[dev].load(std::memory_order_relaxed)) return 0;
  const cudaError_t e = cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e == cudaSuccess) done[dev].store(true, std::memory_order_relaxed);
  return (int)e;
}

// Programmatic dependent launch: the kernel's blocks may start while the previous
// kernel on the stream ends, and wait here before they touch global memory; the
// next kernel's may start once all of this one's have.
__device__ __forceinline__ void pdl_begin() {
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  asm volatile("griddepcontrol.wait;" ::: "memory");
}
template <typename... P, typename... A>
int launch_pdl(void (*kernel)(P...), unsigned grid, unsigned threads, size_t smem, cudaStream_t st, const A&... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(grid);
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return (int)cudaLaunchKernelEx(&cfg, kernel, P(args)...);
}

// The low two bytes of q as two fp16 (exact; NaN stays NaN).
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t q) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"((uint16_t)q));
  return r;
}
// c + a.lo * b.lo + a.hi * b.hi of two fp16 pairs, each step one fp32 rounding.
__device__ __forceinline__ float fma_f16x2(uint32_t a, uint32_t b, float c) {
  float d;
  asm("{\n\t.reg .b16 al, ah, bl, bh;\n\t"
      "mov.b32 {al, ah}, %1;\n\t"
      "mov.b32 {bl, bh}, %2;\n\t"
      "fma.rn.f32.f16 %0, al, bl, %3;\n\t"
      "fma.rn.f32.f16 %0, ah, bh, %0;\n\t}"
      : "=&f"(d)
      : "r"(a), "r"(b), "f"(c));
  return d;
}

// Calls f with a null pointer of the element type `t` (F32, F16 or BF16).
template <typename F>
auto with_type(int t, F f) {
  if (t == kF32) return f((float*)nullptr);
  if (t == kF16) return f((__half*)nullptr);
  return f((__nv_bfloat16*)nullptr);
}

}  // namespace ob2
