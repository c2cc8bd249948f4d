// Typed 4- and 8-wide access for kernels that compute in fp32 whatever the
// tensors' type: bf16, fp16 and fp32 share one spelling.
#pragma once

#include <hip/hip_runtime.h>

using bf16_t = __bf16;
using fp16_t = _Float16;

// N values of T that move as one access of N * sizeof(T) bytes.
template <typename T, int N>
struct alignas(sizeof(T) * N) Pack {
  T v[N];
};

template <typename T, int N>
__device__ inline void load_f32(const T* p, float (&out)[N]) {
  const Pack<T, N> a = *reinterpret_cast<const Pack<T, N>*>(p);
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = static_cast<float>(a.v[i]);
}

// One rounding, to nearest even, from the fp32 result to the tensor's type.
template <typename T, int N>
__device__ inline void store_f32(T* p, const float (&in)[N]) {
  Pack<T, N> a;
#pragma unroll
  for (int i = 0; i < N; ++i) a.v[i] = static_cast<T>(in[i]);
  *reinterpret_cast<Pack<T, N>*>(p) = a;
}

// Types as the launchers take them.
enum ElemType : int { kElemF32 = 0, kElemBF16 = 1, kElemF16 = 2 };
