// Element types of the transformer operators (fp32, fp16, bf16): loads and stores of a few
// consecutive elements as fp32 values, one access where alignment allows it.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace modiff {

inline int dtype_bytes(int dtype) { return dtype == MODIFF_FP32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype == MODIFF_FP32 || dtype == MODIFF_FP16 || dtype == MODIFF_BF16; }

#ifdef __CUDACC__
template <typename T> __device__ inline float to_f32(T v);
template <> __device__ inline float to_f32<float>(float v) { return v; }
template <> __device__ inline float to_f32<__half>(__half v) { return __half2float(v); }
template <> __device__ inline float to_f32<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ inline T from_f32(float v);
template <> __device__ inline float from_f32<float>(float v) { return v; }
template <> __device__ inline __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <> __device__ inline __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// N consecutive elements as one (or, above 16 bytes, several) memory accesses; the address is
// aligned to min(16, N * sizeof(T)) bytes.
template <typename T, int N> struct alignas(sizeof(T) * N < 16 ? sizeof(T) * N : 16) Pack { T v[N]; };

template <typename T, int N>
__device__ inline void load_f32(const T* src, float (&out)[N]) {
  const Pack<T, N> p = *reinterpret_cast<const Pack<T, N>*>(src);
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = to_f32<T>(p.v[i]);
}
template <typename T, int N>
__device__ inline void store_f32(T* dst, const float (&in)[N]) {
  Pack<T, N> p;
#pragma unroll
  for (int i = 0; i < N; ++i) p.v[i] = from_f32<T>(in[i]);
  *reinterpret_cast<Pack<T, N>*>(dst) = p;
}

// (x, y) / s, correctly rounded, from r = 1 / s correctly rounded: two steps of Markstein's refinement (IBM
// J. Res. Dev. 34, 1990): with q within one ulp the remainder x - q s is exact in a fused multiply-add, and
// q + remainder * r rounds to the quotient.  Valid while nothing under- or overflows on the way.  Five
// instructions for two elements; the compiler's division alone was most of the
// quantisers' time.
__device__ inline float2 divide_pair(float x, float y, uint64_t r, uint64_t minus_s) {
  uint64_t v, q, e;
  float2 out;
  asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(x), "f"(y));
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(q) : "l"(v), "l"(r));
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(e) : "l"(q), "l"(minus_s), "l"(v));
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(q) : "l"(e), "l"(r));
  }
  asm("mov.b64 {%0, %1}, %2;" : "=f"(out.x), "=f"(out.y) : "l"(q));
  return out;
}
#endif

// Calls `fn` with a value of the element type that `dtype` names.
template <typename F>
inline int with_dtype(int dtype, F&& fn) {
  if (dtype == MODIFF_FP32) return fn(float());
  if (dtype == MODIFF_FP16) return fn(__half());
  return fn(__nv_bfloat16());
}

}  // namespace modiff
