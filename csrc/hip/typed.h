// Typed 4- and 8-wide access for kernels that compute in fp32 whatever the
// tensors' type: bf16, fp16 and fp32 share one spelling.
#pragma once

#include <hip/hip_runtime.h>

using bf16_t = __bf16;
using fp16_t = _Float16;

// N consecutive values of T that move as one access (two of 16 bytes above
// that), at any address that is T's own: global memory takes wide accesses
// unaligned, for a little more time where one crosses a line.
template <typename T, int N>
__device__ inline void load_f32(const T* p, float (&out)[N]) {
  typedef T Vec __attribute__((ext_vector_type(N)));
  Vec a;
  __builtin_memcpy(&a, p, sizeof(T) * N);
#pragma unroll
  for (int i = 0; i < N; ++i) out[i] = static_cast<float>(a[i]);
}

// One rounding, to nearest even, from the fp32 result to the tensor's type.
template <typename T, int N>
__device__ inline void store_f32(T* p, const float (&in)[N]) {
  typedef T Vec __attribute__((ext_vector_type(N)));
  Vec a;
#pragma unroll
  for (int i = 0; i < N; ++i) a[i] = static_cast<T>(in[i]);
  __builtin_memcpy(p, &a, sizeof(T) * N);
}

// The same past the caches: data that nobody reads again soon leaves them to
// what is.
template <typename T, int N>
__device__ inline void stream_in(const T* p, long left, float (&out)[N]) {
  if (left >= N && ((unsigned long)p & (sizeof(T) * N - 1)) == 0) {
    typedef T Vec __attribute__((ext_vector_type(N)));
    const Vec a = __builtin_nontemporal_load((const Vec*)p);
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = static_cast<float>(a[i]);
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    out[i] = i < left ? static_cast<float>(p[i]) : 0.0f;
}

template <typename T, int N>
__device__ inline void stream_out(T* p, long left, const float (&in)[N]) {
  if (left >= N && ((unsigned long)p & (sizeof(T) * N - 1)) == 0) {
    typedef T Vec __attribute__((ext_vector_type(N)));
    Vec a;
#pragma unroll
    for (int i = 0; i < N; ++i) a[i] = static_cast<T>(in[i]);
    __builtin_nontemporal_store(a, (Vec*)p);
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < left) p[i] = static_cast<T>(in[i]);
}

// The same where only the first `left` values are there; the others are 0.
template <typename T, int N>
__device__ inline void load_some(const T* p, long left, float (&out)[N]) {
  if (left >= N) {
    load_f32<T, N>(p, out);
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    out[i] = i < left ? static_cast<float>(p[i]) : 0.0f;
}

template <typename T, int N>
__device__ inline void store_some(T* p, long left, const float (&in)[N]) {
  if (left >= N) {
    store_f32<T, N>(p, in);
    return;
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    if (i < left) p[i] = static_cast<T>(in[i]);
}

// Types as the launchers take them.
enum ElemType : int { kElemF32 = 0, kElemBF16 = 1, kElemF16 = 2 };
