// omr_elem.h — what the operators that make a model's gradients share (omr_embed.hip, omr_norm.hip, omr_loss.hip):
// element types, vector loads and stores with conversion to and from fp32, and error reporting through
// omr_last_error().
#ifndef OMR_ELEM_H
#define OMR_ELEM_H

#include <hip/hip_runtime.h>

#include <cstdarg>
#include <cstdint>
#include <cstdio>

#include "omr.h"

namespace omr_detail {
int set_error(int code, const char* msg);
}  // namespace omr_detail

namespace omr_elem {

typedef float v4f __attribute__((ext_vector_type(4)));

inline int efail(const char* fmt, ...) __attribute__((format(printf, 1, 2)));
inline int efail(const char* fmt, ...) {
  char buf[256];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  return omr_detail::set_error(OMR_EINVAL, buf);
}

inline int elaunch(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return 0;
  char buf[256];
  snprintf(buf, sizeof(buf), "%s: %s", what, hipGetErrorString(e));
  return omr_detail::set_error(static_cast<int>(e), buf);
}

inline hipStream_t S(omr_stream_t s) { return static_cast<hipStream_t>(s); }

inline size_t elem_bytes(int dtype) { return dtype == OMR_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype == OMR_F32 || dtype == OMR_BF16 || dtype == OMR_F16; }
inline bool aligned(const void* p, size_t to) { return reinterpret_cast<uintptr_t>(p) % to == 0; }
inline uint64_t ceil_div(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

// fn is called with a value of the element type that dtype names
template <class F>
inline auto with_dtype(int dtype, F&& fn) {
  if (dtype == OMR_F32) return fn(float{});
  if (dtype == OMR_BF16) return fn(__bf16{});
  return fn(_Float16{});
}

template <class T, int N>
using vec_t = T __attribute__((ext_vector_type(N)));

// N consecutive elements as fp32 (exact for every element type), and back with one round-to-nearest-even.  Rows may
// begin at any element: whole vectors are loaded and stored at any alignment (one instruction up to 16 bytes, as fast as
// an aligned one where the address happens to be).
template <class T, int N>
using any_vec = vec_t<T, N> __attribute__((aligned(sizeof(T)), may_alias));

template <class T, int N>
__device__ __forceinline__ void load_f32(const T* p, float (&v)[N]) {
  if constexpr (N * sizeof(T) > 16) {
    load_f32<T, N / 2>(p, reinterpret_cast<float(&)[N / 2]>(v[0]));
    load_f32<T, N / 2>(p + N / 2, reinterpret_cast<float(&)[N / 2]>(v[N / 2]));
  } else {
    const vec_t<T, N> x = *reinterpret_cast<const any_vec<T, N>*>(p);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = static_cast<float>(x[i]);
  }
}

template <class T, int N>
__device__ __forceinline__ void store_f32(T* p, const float (&v)[N]) {
  if constexpr (N * sizeof(T) > 16) {
    store_f32<T, N / 2>(p, reinterpret_cast<const float(&)[N / 2]>(v[0]));
    store_f32<T, N / 2>(p + N / 2, reinterpret_cast<const float(&)[N / 2]>(v[N / 2]));
  } else {
    vec_t<T, N> x;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = static_cast<T>(v[i]);
    *reinterpret_cast<any_vec<T, N>*>(p) = x;
  }
}

// store_f32 of rows that are written once and not read here again: whole 16-byte pieces go out non-temporally
template <class T, int N>
__device__ __forceinline__ void stream_f32(T* p, const float (&v)[N]) {
  if constexpr (N * sizeof(T) > 16) {
    stream_f32<T, N / 2>(p, reinterpret_cast<const float(&)[N / 2]>(v[0]));
    stream_f32<T, N / 2>(p + N / 2, reinterpret_cast<const float(&)[N / 2]>(v[N / 2]));
  } else {
    vec_t<T, N> x;
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = static_cast<T>(v[i]);
    __builtin_nontemporal_store(x, reinterpret_cast<any_vec<T, N>*>(p));
  }
}

// The same for a piece at the end of a row, of which the first `n` elements exist (the others are read as 0)
template <class T, int N>
__device__ __forceinline__ void load_some(const T* p, uint32_t n, float (&v)[N]) {
  if (n >= N) {
    load_f32<T, N>(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = static_cast<uint32_t>(i) < n ? static_cast<float>(p[i]) : 0.0f;
  }
}

template <class T, int N>
__device__ __forceinline__ void store_some(T* p, uint32_t n, const float (&v)[N]) {
  if (n >= N) {
    store_f32<T, N>(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (static_cast<uint32_t>(i) < n) p[i] = static_cast<T>(v[i]);
  }
}

template <class T, int N>
__device__ __forceinline__ void stream_some(T* p, uint32_t n, const float (&v)[N]) {
  if (n >= N)
    stream_f32<T, N>(p, v);
  else
    store_some<T, N>(p, n, v);
}

// Sum over the 64 lanes of a wave, in every lane (fixed order: the same bits every run).
__device__ __forceinline__ float wave_sum(float v) {
#pragma unroll
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  return v;
}

}  // namespace omr_elem

#endif
