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

// N consecutive elements in a register, as they were loaded
template <typename T, int N> using Raw = typename RawVec<(int)sizeof(T) * N>::type;

template <typename T, int N> __device__ __forceinline__ Raw<T, N> load_raw(const T* __restrict__ p) {
  return *reinterpret_cast<const Raw<T, N>*>(p);
}

template <typename T, int N> __device__ __forceinline__ void unpack(const Raw<T, N>& raw, float* __restrict__ f) {
  T e[N];
  __builtin_memcpy(e, &raw, sizeof(raw));
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = (float)e[i];
}

// N consecutive elements at p (aligned to N * sizeof(T)) as fp32
template <typename T, int N> __device__ __forceinline__ void load_vec(const T* __restrict__ p, float (&f)[N]) {
  using R = Raw<T, N>;
  const R raw = *reinterpret_cast<const R*>(p);
  T e[N];
  __builtin_memcpy(e, &raw, sizeof(R));
#pragma unroll
  for (int i = 0; i < N; ++i) f[i] = (float)e[i];
}

template <typename T, int N> __device__ __forceinline__ void store_vec(T* __restrict__ p, const float (&f)[N]) {
  using R = Raw<T, N>;
  T e[N];
#pragma unroll
  for (int i = 0; i < N; ++i) e[i] = (T)f[i];
  R raw;
  __builtin_memcpy(&raw, e, sizeof(R));
  *reinterpret_cast<R*>(p) = raw;
}

using word4 = __attribute__((ext_vector_type(4))) uint32_t;

// 16 bytes that are not kept in the caches on their way to memory
__device__ __forceinline__ void store16_nt(void* p, const word4& w) { __builtin_nontemporal_store(w, reinterpret_cast<word4*>(p)); }

template <typename T, int N> __device__ __forceinline__ void store_vec_nt(T* __restrict__ p, const float (&f)[N]) {
  if constexpr (sizeof(T) * N == 16) {
    T e[N];
#pragma unroll
    for (int i = 0; i < N; ++i) e[i] = (T)f[i];
    word4 w;
    __builtin_memcpy(&w, e, 16);
    store16_nt(p, w);
  } else {
    store_vec<T, N>(p, f);
  }
}

// Results from this size on, half of the Infinity Cache, are stored past the caches: whoever reads them next finds little of
// them there either way, and the inputs that are read meanwhile stay.  Measured with a pass over the result behind the
// operator: gradients of 67 MiB clipped into new tensors 72 us plain, 78 us past the caches; 135 MiB 179 / 167 us; 225 MiB
// 299 / 284 us; the label loss's gradient of 97 MiB 86 / 91 us, 195 MiB 191 / 189 us (122 / 100 us without that pass).
constexpr int64_t PAST_CACHES_MIN_BYTES = (int64_t)128 << 20;

// Calls f(T{}) with the element type of `dtype`; the caller has checked the code.
template <typename F> inline int with_dtype(int32_t dtype, F&& f) {
  switch (dtype) {
    case GS_DTYPE_F32: return f(float{});
    case GS_DTYPE_BF16: return f(bf16_t{});
    case GS_DTYPE_F16: return f(f16_t{});
    default: return GS_ERR_INVALID_ARG;
  }
}

// ---- wave reductions over DPP: the sum (or maximum) of the lanes before in each row of 16, then over the rows; lane 63
// has all of it.  Registers only, and always in the same order.
template <int CTRL, int ROWS> __device__ __forceinline__ uint32_t dpp_word(uint32_t x, uint32_t none) {
  return (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)x, CTRL, ROWS, 0xf, false);
}

template <typename F> __device__ __forceinline__ float wave_reduce(float x, float none, F&& f) {
  const uint32_t n = __float_as_uint(none);
  x = f(x, __uint_as_float(dpp_word<0x111, 0xf>(__float_as_uint(x), n)));  // row_shr 1, 2, 4, 8
  x = f(x, __uint_as_float(dpp_word<0x112, 0xf>(__float_as_uint(x), n)));
  x = f(x, __uint_as_float(dpp_word<0x114, 0xf>(__float_as_uint(x), n)));
  x = f(x, __uint_as_float(dpp_word<0x118, 0xf>(__float_as_uint(x), n)));
  x = f(x, __uint_as_float(dpp_word<0x142, 0xa>(__float_as_uint(x), n)));  // lane 15 of rows 0, 2 to rows 1, 3
  x = f(x, __uint_as_float(dpp_word<0x143, 0xc>(__float_as_uint(x), n)));  // lane 31 to rows 2, 3
  return __uint_as_float((uint32_t)__builtin_amdgcn_readlane((int)__float_as_uint(x), 63));
}
__device__ __forceinline__ float wave_sum_all(float x) { return wave_reduce(x, 0.f, [](float a, float b) { return a + b; }); }
__device__ __forceinline__ float wave_max_all(float x) {
  return wave_reduce(x, -INFINITY, [](float a, float b) { return fmaxf(a, b); });
}

template <int CTRL, int ROWS> __device__ __forceinline__ uint64_t dpp_max(uint64_t x) {
  const uint64_t y = ((uint64_t)dpp_word<CTRL, ROWS>((uint32_t)(x >> 32), 0u) << 32) | dpp_word<CTRL, ROWS>((uint32_t)x, 0u);
  return y > x ? y : x;
}
__device__ __forceinline__ uint64_t wave_max_all(uint64_t x) {
  x = dpp_max<0x111, 0xf>(x);
  x = dpp_max<0x112, 0xf>(x);
  x = dpp_max<0x114, 0xf>(x);
  x = dpp_max<0x118, 0xf>(x);
  x = dpp_max<0x142, 0xa>(x);
  x = dpp_max<0x143, 0xc>(x);
  return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(x >> 32), 63) << 32) |
         (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, 63);
}

}  // namespace gs
