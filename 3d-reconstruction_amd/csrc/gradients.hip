// Global norm of many gradient tensors and their scaling to a largest norm, in two launches.
//   norm = sqrt(sum_t sum_i g_t[i]^2),  c = min(1, max_norm / (norm + eps)),  out_t = c g_t
// Bound by HBM: one read of everything for the norm and, where something has to change, one read and one write more.
// The table of tensors (pointers, sizes, types) travels in the kernel arguments: nothing is copied to the device, so a
// call can be captured, and nothing outlives it.  A launch carries 128 tensors; more take further launches.
// The squares are summed in 64 bits (a square leaves the range of fp32 from 1.8e19 up and from 1e-19 down) in an order
// that the sizes, the order in memory and the distance from a 16-byte boundary fix: ranks that lay equal gradients out alike get
// equal bits.  The 64-bit sums cost nothing that shows: 708 MB of
// fp32 are read in 113 us (6.3 TB/s), 537 MB of bf16 in 83 us (6.4).  The second pass takes 183 us for those 537 MB, read and
// written (5.9 TB/s), and 5 us when nothing has to change.
#include <algorithm>
#include <vector>

#include "dtype_io.hpp"

namespace gs {

constexpr int GR_MAX_TENSORS = 128;  // 29 bytes each: the table stays within the 4 KiB of kernel arguments
constexpr int GR_THREADS = 256;
constexpr int GR_FLIGHT = 8;         // 16-byte vectors a thread has in flight
constexpr int GR_CHUNK_VECS = GR_FLIGHT * GR_THREADS;  // vectors of one chunk (32 KiB)
constexpr int GR_MAX_BLOCKS = 1024;  // four workgroups on each of 256 CUs; each of the second pass adds up all partial sums
constexpr int GR_MAX_PARTIALS = 4096;

struct GradTable {
  const void* src[GR_MAX_TENSORS];
  void* dst[GR_MAX_TENSORS];
  int64_t numel[GR_MAX_TENSORS];
  int32_t first_chunk[GR_MAX_TENSORS];  // first chunk of the tensor in this launch
  int8_t dtype[GR_MAX_TENSORS];
  int32_t tensors, chunks;
};
static_assert(sizeof(GradTable) <= 3840, "kernel arguments are 4 KiB");

__host__ __device__ inline int64_t gr_chunks(int64_t numel, int size) {
  const int64_t per = (int64_t)GR_CHUNK_VECS * (16 / size);
  const int64_t c = (numel + per - 1) / per;
  return c < 1 ? 1 : c;
}

// the tensor of chunk c: the last one whose first chunk is not behind it (every wave does this for itself)
__device__ __forceinline__ int gr_tensor(const GradTable& t, int c) {
  const int lane = threadIdx.x & 63;
  const bool a = lane < t.tensors && t.first_chunk[lane] <= c;
  const bool b = lane + 64 < t.tensors && t.first_chunk[lane + 64] <= c;
  const int n = __popcll(__ballot(a)) + __popcll(__ballot(b));
  return __builtin_amdgcn_readfirstlane(n - 1);
}

// sum over the workgroup in a fixed order; all threads get it
__device__ __forceinline__ double gr_block_sum(double v, double* lds) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < GR_THREADS / 64; ++w) s += lds[w];
  __syncthreads();
  return s;
}

// a tensor's values: a head up to the first 16-byte boundary, whole vectors, a tail
template <typename T> struct GradSpan {
  static constexpr int VE = 16 / (int)sizeof(T);
  int64_t head, vecs, numel;
  __device__ GradSpan(const void* p, int64_t n) : numel(n) {
    const int64_t h = (int64_t)(((16u - ((uintptr_t)p & 15u)) & 15u) / sizeof(T));
    head = h < n ? h : n;
    vecs = (n - head) / VE;
  }
};

template <typename T> __device__ __forceinline__ double gr_chunk_squares(const T* __restrict__ src, int64_t numel, int64_t chunk) {
  constexpr int VE = GradSpan<T>::VE;
  const GradSpan<T> s(src, numel);
  double acc = 0.0;
  const int64_t v0 = chunk * GR_CHUNK_VECS;
  const T* body = src + (s.head + v0 * VE);
  auto add = [&](const Raw<T, VE>& raw) {
    float f[VE];
    unpack<T, VE>(raw, f);
#pragma unroll
    for (int k = 0; k < VE; ++k) acc += (double)f[k] * (double)f[k];
  };
  if (v0 + GR_CHUNK_VECS <= s.vecs) {  // a whole chunk: all of a thread's vectors in flight
    Raw<T, VE> raw[GR_FLIGHT];
#pragma unroll
    for (int u = 0; u < GR_FLIGHT; ++u) raw[u] = load_raw<T, VE>(body + (int64_t)(u * GR_THREADS + threadIdx.x) * VE);
#pragma unroll
    for (int u = 0; u < GR_FLIGHT; ++u) add(raw[u]);
  } else {
    for (int64_t v = threadIdx.x; v < s.vecs - v0; v += GR_THREADS) add(load_raw<T, VE>(body + v * VE));
  }
  if (chunk == 0) {
    const int64_t tail0 = s.head + s.vecs * VE;
    const int64_t i = threadIdx.x < s.head ? threadIdx.x : tail0 + (threadIdx.x - s.head);
    if (i < numel) {
      const double x = (double)(float)src[i];
      acc += x * x;
    }
  }
  return acc;
}

__global__ __launch_bounds__(GR_THREADS) void grad_squares_kernel(GradTable t, double* __restrict__ partials) {
  __shared__ double lds[GR_THREADS / 64];
  double acc = 0.0;
  for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
    const int i = gr_tensor(t, c);
    const int64_t k = c - t.first_chunk[i];
    switch (t.dtype[i]) {
      case GS_DTYPE_F32: acc += gr_chunk_squares((const float*)t.src[i], t.numel[i], k); break;
      case GS_DTYPE_BF16: acc += gr_chunk_squares((const bf16_t*)t.src[i], t.numel[i], k); break;
      default: acc += gr_chunk_squares((const f16_t*)t.src[i], t.numel[i], k); break;
    }
  }
  const double s = gr_block_sum(acc, lds);
  if (threadIdx.x == 0) partials[blockIdx.x] = s;
}

// every workgroup adds up the partial sums by itself, in the same order: it saves a launch between the two passes
__device__ __forceinline__ float gr_norm(const double* __restrict__ partials, int n, double* lds) {
  double acc = 0.0;
  for (int i = threadIdx.x; i < n; i += GR_THREADS) acc += partials[i];
  return (float)sqrt(gr_block_sum(acc, lds));
}

__global__ __launch_bounds__(GR_THREADS) void grad_norm_kernel(const double* __restrict__ partials, int n, float* __restrict__ norm) {
  __shared__ double lds[GR_THREADS / 64];
  const float v = gr_norm(partials, n, lds);
  if (threadIdx.x == 0) *norm = v;
}

template <bool PAST, typename T>
__device__ __forceinline__ void gr_chunk_scale(const T* src, T* dst, int64_t numel, int64_t chunk, float c) {
  constexpr int VE = GradSpan<T>::VE;
  const GradSpan<T> s(src, numel);
  const int64_t v0 = chunk * GR_CHUNK_VECS;
  const T* body = src + (s.head + v0 * VE);
  T* out = dst + (s.head + v0 * VE);
  const bool wide = ((((uintptr_t)src) ^ ((uintptr_t)dst)) & 15u) == 0;
  auto put = [&](int64_t v, const Raw<T, VE>& raw) {
    float f[VE];
    unpack<T, VE>(raw, f);
#pragma unroll
    for (int k = 0; k < VE; ++k) f[k] *= c;
    if (wide) {
      if constexpr (PAST) store_vec_nt<T, VE>(out + v * VE, f); else store_vec<T, VE>(out + v * VE, f);
    } else {
#pragma unroll
      for (int k = 0; k < VE; ++k) out[v * VE + k] = (T)f[k];
    }
  };
  if (v0 + GR_CHUNK_VECS <= s.vecs) {
    Raw<T, VE> raw[GR_FLIGHT];
#pragma unroll
    for (int u = 0; u < GR_FLIGHT; ++u) raw[u] = load_raw<T, VE>(body + (int64_t)(u * GR_THREADS + threadIdx.x) * VE);
#pragma unroll
    for (int u = 0; u < GR_FLIGHT; ++u) put(u * GR_THREADS + threadIdx.x, raw[u]);
  } else {
    for (int64_t v = threadIdx.x; v < s.vecs - v0; v += GR_THREADS) put(v, load_raw<T, VE>(body + v * VE));
  }
  if (chunk == 0) {
    const int64_t tail0 = s.head + s.vecs * VE;
    const int64_t i = threadIdx.x < s.head ? threadIdx.x : tail0 + (threadIdx.x - s.head);
    if (i < numel) dst[i] = (T)((float)src[i] * c);
  }
}

template <bool PAST>
__global__ __launch_bounds__(GR_THREADS) void grad_scale_kernel(GradTable t, const double* __restrict__ partials, int n_partials,
                                                                float max_norm, float eps, int in_place, int write_norm,
                                                                float* __restrict__ norm) {
  __shared__ double lds[GR_THREADS / 64];
  const float v = gr_norm(partials, n_partials, lds);
  if (write_norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = v;
  const float q = max_norm / (v + eps);
  const float c = q > 1.0f ? 1.0f : q;  // a NaN norm stays one
  if (in_place && c == 1.0f) return;    // nothing changes
  // from the end: what was read last for the norm is still in the caches (268 MB and more of them read twice: 196 -> 182 us)
  for (int k = t.chunks - 1 - (int)blockIdx.x; k >= 0; k -= (int)gridDim.x) {
    const int i = gr_tensor(t, k);
    const int64_t at = k - t.first_chunk[i];
    switch (t.dtype[i]) {
      case GS_DTYPE_F32: gr_chunk_scale<PAST>((const float*)t.src[i], (float*)t.dst[i], t.numel[i], at, c); break;
      case GS_DTYPE_BF16: gr_chunk_scale<PAST>((const bf16_t*)t.src[i], (bf16_t*)t.dst[i], t.numel[i], at, c); break;
      default: gr_chunk_scale<PAST>((const f16_t*)t.src[i], (f16_t*)t.dst[i], t.numel[i], at, c); break;
    }
  }
}

// chunks of the tensors [t0, t1) of one launch, or -1 where a count leaves 32 bits
static int64_t gr_launch_chunks(int32_t t0, int32_t t1, const int64_t* numel, const int32_t* dtype) {
  int64_t c = 0;
  for (int32_t t = t0; t < t1; ++t) c += gr_chunks(numel[t], dtype_size(dtype[t]));
  return c < ((int64_t)1 << 31) - GR_MAX_BLOCKS ? c : -1;
}

static int gr_launch_blocks(int64_t chunks, int launches) {
  const int most = std::max(256, std::min(GR_MAX_BLOCKS, GR_MAX_PARTIALS / launches));
  return (int)std::min<int64_t>(chunks, most);
}

static int gr_check(int32_t n, const void* const* src, void* const* dst, const int64_t* numel, const int32_t* dtype) {
  if (n < 0 || (n > 0 && (!src || !numel || !dtype))) return GS_ERR_INVALID_ARG;
  for (int32_t t = 0; t < n; ++t) {
    const int size = dtype_size(dtype[t]);
    if (!size || numel[t] < 0) return GS_ERR_INVALID_ARG;
    if (numel[t] > 0 && (!src[t] || (dst && !dst[t]))) return GS_ERR_INVALID_ARG;
    if (((uintptr_t)src[t] | (dst ? (uintptr_t)dst[t] : 0)) & (uintptr_t)(size - 1)) return GS_ERR_INVALID_ARG;
  }
  return GS_OK;
}

// What is written may overlap nothing but its own source: two tensors on one memory would be scaled twice, in a race.
static int gr_check_overlap(int32_t n, const void* const* src, void* const* dst, const int64_t* numel, const int32_t* dtype) {
  struct Range { uintptr_t a, b; int32_t t; };
  try {
    std::vector<Range> out;
    out.reserve((size_t)n);
    for (int32_t t = 0; t < n; ++t)
      if (numel[t] > 0) out.push_back({(uintptr_t)dst[t], (uintptr_t)dst[t] + (uintptr_t)numel[t] * dtype_size(dtype[t]), t});
    std::sort(out.begin(), out.end(), [](const Range& x, const Range& y) { return x.a < y.a; });
    for (size_t i = 1; i < out.size(); ++i)
      if (out[i].a < out[i - 1].b) return GS_ERR_INVALID_ARG;
    for (int32_t t = 0; t < n; ++t) {
      if (numel[t] == 0 || src[t] == dst[t]) continue;
      const uintptr_t a = (uintptr_t)src[t], b = a + (uintptr_t)numel[t] * dtype_size(dtype[t]);
      auto it = std::upper_bound(out.begin(), out.end(), a, [](uintptr_t x, const Range& r) { return x < r.b; });
      if (it != out.end() && it->a < b) return GS_ERR_INVALID_ARG;
    }
  } catch (...) {  // no memory for the list
    return GS_ERR_WORKSPACE;
  }
  return GS_OK;
}

}  // namespace gs

extern "C" int64_t gs_grad_norm_workspace_bytes(int32_t n_tensors) {
  const int64_t launches = n_tensors > 0 ? gs::ceil_div(n_tensors, gs::GR_MAX_TENSORS) : 1;
  return 8 * std::max<int64_t>(gs::GR_MAX_PARTIALS, 256 * launches);
}

// phase 1: partial sums of all launches; phase 2: `norm` alone, or the scaling (which writes `norm` too)
static int gr_run(int32_t n, const void* const* src, void* const* dst, const int64_t* numel, const int32_t* dtype,
                  float max_norm, float eps, void* workspace, int64_t workspace_bytes, float* norm, hipStream_t s) {
  using namespace gs;
  int st = gr_check(n, src, dst, numel, dtype);
  if (st != GS_OK) return st;
  if (!norm || !workspace) return GS_ERR_INVALID_ARG;
  if (dst && (st = gr_check_overlap(n, src, dst, numel, dtype)) != GS_OK) return st;
  if (workspace_bytes < gs_grad_norm_workspace_bytes(n)) return GS_ERR_WORKSPACE;
  const int launches = n > 0 ? (int)ceil_div(n, GR_MAX_TENSORS) : 0;
  bool in_place = dst != nullptr;
  int64_t elsewhere = 0;  // bytes that are written to another place than they come from
  for (int32_t t = 0; dst && t < n; ++t)
    if (numel[t] > 0 && src[t] != dst[t]) {
      in_place = false;
      elsewhere += numel[t] * dtype_size(dtype[t]);
    }
  const bool past = elsewhere >= PAST_CACHES_MIN_BYTES;
  double* partials = (double*)workspace;
  int n_partials = 0;
  for (int pass = 0; pass < 2; ++pass) {
    for (int l = 0; l < launches; ++l) {
      const int32_t t0 = l * GR_MAX_TENSORS, t1 = std::min(n, t0 + GR_MAX_TENSORS);
      const int64_t chunks = gr_launch_chunks(t0, t1, numel, dtype);
      if (chunks < 0) return GS_ERR_UNSUPPORTED;
      GradTable tab;
      int32_t at = 0;
      for (int32_t t = t0; t < t1; ++t) {
        tab.src[t - t0] = src[t];
        tab.dst[t - t0] = dst ? dst[t] : nullptr;
        tab.numel[t - t0] = numel[t];
        tab.dtype[t - t0] = (int8_t)dtype[t];
        tab.first_chunk[t - t0] = at;
        at += (int32_t)gr_chunks(numel[t], dtype_size(dtype[t]));
      }
      tab.tensors = t1 - t0;
      tab.chunks = at;
      const int blocks = gr_launch_blocks(chunks, launches);
      if (pass == 0) {
        hipLaunchKernelGGL(grad_squares_kernel, dim3(blocks), dim3(GR_THREADS), 0, s, tab, partials + n_partials);
        n_partials += blocks;
      } else {
        auto* kernel = past ? &grad_scale_kernel<true> : &grad_scale_kernel<false>;
        hipLaunchKernelGGL(kernel, dim3(blocks), dim3(GR_THREADS), 0, s, tab, partials, n_partials, max_norm, eps,
                           in_place ? 1 : 0, l == 0 ? 1 : 0, norm);
      }
      GS_CHECK_LAUNCH();
    }
    if (pass == 0 && (!dst || launches == 0)) {
      hipLaunchKernelGGL(grad_norm_kernel, dim3(1), dim3(GR_THREADS), 0, s, partials, n_partials, norm);
      GS_CHECK_LAUNCH();
      return GS_OK;
    }
  }
  return GS_OK;
}

extern "C" int gs_grad_norm(int32_t n_tensors, const void* const* src_host, const int64_t* numel_host,
                            const int32_t* dtype_host, void* workspace, int64_t workspace_bytes, float* norm, void* stream) {
  return gr_run(n_tensors, src_host, nullptr, numel_host, dtype_host, 0.f, 0.f, workspace, workspace_bytes, norm,
                (hipStream_t)stream);
}

extern "C" int gs_grad_clip(int32_t n_tensors, const void* const* src_host, void* const* dst_host, const int64_t* numel_host,
                            const int32_t* dtype_host, float max_norm, float eps, void* workspace, int64_t workspace_bytes,
                            float* norm, void* stream) {
  if (!(max_norm >= 0.f) || !(eps >= 0.f) || (n_tensors > 0 && !dst_host)) return GS_ERR_INVALID_ARG;
  return gr_run(n_tensors, src_host, n_tensors > 0 ? dst_host : nullptr, numel_host, dtype_host, max_norm, eps, workspace,
                workspace_bytes, norm, (hipStream_t)stream);
}
