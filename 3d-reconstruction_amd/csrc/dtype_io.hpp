// Element types of the operators that take fp32, bf16 and fp16 tensors (GS_DTYPE_*): vector loads to fp32, stores that
// round to nearest even once.
#pragma once
#include "gs_common.hpp"

namespace gs {

using bf16_t = __bf16;
using f16_t = _Float16;

inline int dtype_size(int32_t dtype) { return dtype == GS_DTYPE_F32 ? 4 : (dtype == GS_DTYPE_BF16 || dtype == GS_DTYPE_F16) ? 2 : 0; }

template <int BYTES> struct RawVec;
template <> struct RawVec<16> { using type = uint4; };
template <> struct RawVec<8> { using type = uint2; };
template <> struct RawVec<4> { using type = uint32_t; };
template <> struct RawVec<2> { using type = uint16_t; };

// N consecutive elements at p (aligned to N * sizeof(T)) as fp32
template <typename T, int N> __device__ __forceinline__ void load_vec(const T* __restrict__ p, float (&f)[N]) {
  using R = typename RawVec<(int)sizeof(T) * N>::type;
  const R raw = *reinterpret_cast<const R*>(p);
  T e[N];
  __builtin_memcpy(e, &raw, sizeof(R));
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = (float)e[i];
}

template <typename T, int N> __device__ __forceinline__ void store_vec(T* __restrict__ p, const float (&f)[N]) {
  using R = typename RawVec<(int)sizeof(T) * N>::type;
  T e[N];
#pragma unroll
  for (int i = 0; i < N; ++i) e[i] = (T)f[i];
  R raw;
  __builtin_memcpy(&raw, e, sizeof(R));
  *reinterpret_cast<R*>(p) = raw;
}

// Calls f(T{}) with the element type of `dtype`; the caller has checked the code.
template <typename F> inline int with_dtype(int32_t dtype, F&& f) {
  switch (dtype) {
    case GS_DTYPE_F32: return f(float{});
    case GS_DTYPE_BF16: return f(bf16_t{});
    case GS_DTYPE_F16: return f(f16_t{});
    default: return GS_ERR_INVALID_ARG;
  }
}

}  // namespace gs
