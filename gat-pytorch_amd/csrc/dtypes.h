// Element types of the graph-transformer operators (fp32, bf16, fp16) and their dispatch.
#pragma once

#include "gatx_common.h"

namespace gatx {

inline int dtype_size(int dtype) { return dtype == GATX_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype >= GATX_F32 && dtype <= GATX_F16; }

// Calls f with a value of the element type (f is a generic lambda).
template <typename F>
inline int with_dtype(int dtype, F&& f) {
  if (dtype == GATX_F32) return f(float());
  if (dtype == GATX_BF16) return f(__bf16());
  return f(_Float16());
}

// N consecutive elements, moved as one access of up to 16 bytes.
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};
template <typename T, int N>
__device__ inline void load_f32(const T* p, float (&out)[N]) {
  const Pack<T, N> x = *reinterpret_cast<const Pack<T, N>*>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = (float)x.v[i];
}
template <typename T, int N>
__device__ inline void store_f32(T* p, const float (&in)[N]) {
  Pack<T, N> x;
#pragma unroll
  for (int i = 0; i < N; ++i) x.v[i] = (T)in[i];
  *reinterpret_cast<Pack<T, N>*>(p) = x;
}

inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// 1 / (1 + exp(-x)): exp overflows to inf below -88, and the quotient is the right 0.
__device__ inline float sigmoid(float x) { return 1.f / (1.f + __expf(-x)); }

}  // namespace gatx
