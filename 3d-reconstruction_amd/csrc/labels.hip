// Log probabilities of given labels under softmax(logits), with each row's entropy and its best alternatives, and the
// gradient.  With x a row of K logits, m = max x, e_j = exp(x_j - m), S = sum e_j, p_j = e_j / S:
//   log p_j = (x_j - m) - log S,  log_prob = log p_y,  entropy H = log S - (sum e_j (x_j - m)) / S
//   v_x_j = g_lp ([j = y] - p_j) - g_H p_j (log p_j + H) + sum_k g_top_k ([j = t_k] - p_j)
// m and log S are kept apart for the gradient: their sum would lose log S next to logits far from zero.  An exponential
// below 2^-126 is 0 (the hardware's flushes there).  The statistics are taken in one pass, m growing as the row is read (what was summed is scaled down when it does); the
// gradient is one more read of the logits and one write, from m, log S and H.
// A label outside [0, K) has no term: log_prob 0 and no gradient through it.  Logits of -inf have p = 0 and add nothing;
// a row of nothing but -inf has log probabilities -inf, entropy 0 and no gradient.  NaN, or +inf, makes its row NaN.
// The top alternatives are the largest logits, NaN above all, equal ones by the lower index.
#include "dtype_io.hpp"

namespace gs {

constexpr int LP_THREADS = 256;
constexpr float LP_LOG2E = 1.44269504088896340736f;

__device__ __forceinline__ float lp_exp(float d) { return __builtin_amdgcn_exp2f(d * LP_LOG2E); }

// max, sum of exp(x - max) and sum of exp(x - max) (x - max) of a part of a row
struct LpStat {
  float m, s, w;
};

// the statistics of two parts; scaling m down to a new maximum shifts w by (m_old - m_new) s
__device__ __forceinline__ LpStat lp_join(const LpStat& a, const LpStat& b) {
  const float m = fmaxf(a.m, b.m);
  if (m == -INFINITY) return {m, a.s + b.s, a.w + b.w};  // nothing but -inf so far (or NaN, which s keeps)
  LpStat r{m, 0.f, 0.f};
  const float da = a.m - m, db = b.m - m;
  const float ea = a.m == -INFINITY ? 0.f : lp_exp(da), eb = b.m == -INFINITY ? 0.f : lp_exp(db);
  r.s = a.s * ea + b.s * eb;
  r.w = (ea == 0.f ? 0.f : ea * (a.w + da * a.s)) + (eb == 0.f ? 0.f : eb * (b.w + db * b.s));
  return r;
}

__device__ __forceinline__ void lp_add(LpStat& st, float x) {
  if (x > st.m) {
    const float d = st.m - x;
    const float e = st.m == -INFINITY ? 0.f : lp_exp(d);
    st.w = e == 0.f ? 0.f : e * (st.w + d * st.s);
    st.s *= e;
    st.m = x;
  }
  if (x != -INFINITY) {
    const float d = x - st.m;
    const float e = lp_exp(d);
    st.s += e;
    if (e != 0.f) st.w += e * d;
  }
}

// a total order of logits: larger first, NaN above all, equal values (and the two zeros) by the lower index
__device__ __forceinline__ uint32_t lp_order(float x) {
  if (x != x) return 0xfffffffeu;  // a key of all ones stays free: it starts the search for the largest below another
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 becomes +0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ uint64_t lp_key(float x, uint32_t j) { return ((uint64_t)lp_order(x) << 32) | (uint32_t)~j; }

__device__ __forceinline__ uint64_t lp_wave_max(uint64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    const uint64_t w = __shfl_xor((unsigned long long)v, o);
    v = w > v ? w : v;
  }
  return v;
}

__device__ __forceinline__ int64_t lp_label(const void* labels, int label_bytes, int64_t r) {
  return label_bytes == 8 ? ((const int64_t*)labels)[r] : (int64_t)((const int32_t*)labels)[r];
}

struct LpFwd {
  int64_t rows, stride;
  int32_t K, top, label_bytes;
  const void* labels;
  float *log_prob, *entropy, *stats, *top_lp;
  int64_t* top_idx;
};

// (x - m) - log S, and what it is in a row of nothing but -inf
__device__ __forceinline__ float lp_log_p(float x, float m, float ls) { return ls == -INFINITY ? -INFINITY : (x - m) - ls; }

template <typename T>
__device__ __forceinline__ void lp_write_row(const LpFwd& a, int64_t r, const LpStat& st, float ls, const T* x) {
  a.stats[2 * r] = st.m;
  a.stats[2 * r + 1] = ls;
  a.entropy[r] = ls == -INFINITY ? 0.f : ls - st.w / st.s;
  const int64_t y = lp_label(a.labels, a.label_bytes, r);
  a.log_prob[r] = y < 0 || y >= a.K ? 0.f : lp_log_p((float)x[y], st.m, ls);
}

// one wave per row
template <typename T>
__global__ __launch_bounds__(LP_THREADS) void label_wave_fwd_kernel(LpFwd a, const T* __restrict__ logits) {
  const int lane = threadIdx.x & 63;
  const int64_t waves = (int64_t)gridDim.x * (LP_THREADS / 64);
  for (int64_t r = (int64_t)blockIdx.x * (LP_THREADS / 64) + (threadIdx.x >> 6); r < a.rows; r += waves) {
    const T* x = logits + r * a.stride;
    LpStat st{-INFINITY, 0.f, 0.f};
    for (int64_t j = lane; j < a.K; j += 64) lp_add(st, (float)x[j]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      const LpStat b{__shfl_xor(st.m, o), __shfl_xor(st.s, o), __shfl_xor(st.w, o)};
      st = lp_join(st, b);
    }
    const float ls = logf(st.s);  // -inf for a row of nothing but -inf, as for no other
    if (lane == 0) lp_write_row(a, r, st, ls, x);
    uint64_t below = ~0ull;
    for (int t = 0; t < a.top; ++t) {
      uint64_t best = 0;
      for (int64_t j = lane; j < a.K; j += 64) {
        const uint64_t k = lp_key((float)x[j], (uint32_t)j);
        if (k < below && k > best) best = k;
      }
      best = lp_wave_max(best);
      below = best;
      if (lane == 0) {
        const int64_t j = (int64_t)(uint32_t)~(uint32_t)best;
        a.top_idx[r * a.top + t] = j;
        a.top_lp[r * a.top + t] = lp_log_p((float)x[j], st.m, ls);
      }
    }
  }
}

struct LpBwd {
  int64_t rows, stride;
  int32_t K, top, label_bytes;
  const void* labels;
  const float *stats, *entropy;
  const int64_t* top_idx;
  const float *g_lp, *g_ent, *g_top;  // each may be NULL
};

// what a row's gradient needs: v_x_j = p_j (c0 - c1 (log p_j + H)) + the terms at y and t_k
struct LpRow {
  float m, ls, H, c0, c1, g;
  int64_t y;
};

__device__ __forceinline__ LpRow lp_row(const LpBwd& a, int64_t r) {
  LpRow w;
  w.m = a.stats[2 * r];
  w.ls = a.stats[2 * r + 1];
  w.H = a.entropy[r];
  const int64_t y = lp_label(a.labels, a.label_bytes, r);
  const bool kept = y >= 0 && y < a.K;
  w.y = kept ? y : -1;
  w.g = kept && a.g_lp ? a.g_lp[r] : 0.f;
  w.c0 = -w.g;
  if (a.g_top)
    for (int t = 0; t < a.top; ++t) w.c0 -= a.g_top[r * a.top + t];
  w.c1 = a.g_ent ? a.g_ent[r] : 0.f;
  return w;
}

__device__ __forceinline__ float lp_grad(const LpRow& w, float x) {
  const float d = (x - w.m) - w.ls;
  const float p = lp_exp(d);
  return p == 0.f ? 0.f : p * (w.c0 - w.c1 * (d + w.H));
}

template <typename T>
__global__ __launch_bounds__(LP_THREADS) void label_wave_bwd_kernel(LpBwd a, const T* __restrict__ logits, T* __restrict__ v) {
  const int lane = threadIdx.x & 63;
  const int64_t waves = (int64_t)gridDim.x * (LP_THREADS / 64);
  for (int64_t r = (int64_t)blockIdx.x * (LP_THREADS / 64) + (threadIdx.x >> 6); r < a.rows; r += waves) {
    const T* x = logits + r * a.stride;
    T* o = v + r * a.K;
    const LpRow w = lp_row(a, r);
    const bool none = w.ls == -INFINITY;
    for (int64_t j = lane; j < a.K; j += 64) {
      float g = none ? 0.f : lp_grad(w, (float)x[j]);
      if (!none) {
        if (j == w.y) g += w.g;
        if (a.g_top)
          for (int t = 0; t < a.top; ++t)
            if (a.top_idx[r * a.top + t] == j) g += a.g_top[r * a.top + t];
      }
      o[j] = (T)g;
    }
  }
}

static int lp_check(int64_t rows, int32_t K, int32_t dtype, int32_t top_k, const void* logits, int64_t row_stride,
                    const void* labels, int32_t label_bytes) {
  if (rows < 0 || K < 1 || !dtype_size(dtype) || top_k < 0 || top_k > K || row_stride < 0) return GS_ERR_INVALID_ARG;
  if (top_k > GS_LABEL_TOP_MAX) return GS_ERR_UNSUPPORTED;
  if (label_bytes != 4 && label_bytes != 8) return GS_ERR_INVALID_ARG;
  if (rows == 0) return GS_OK;
  if (!logits || !labels) return GS_ERR_INVALID_ARG;
  if (((uintptr_t)logits & (uintptr_t)(dtype_size(dtype) - 1)) || ((uintptr_t)labels & (uintptr_t)(label_bytes - 1)))
    return GS_ERR_INVALID_ARG;
  return GS_OK;
}

static unsigned lp_wave_grid(int64_t rows) {
  const int64_t b = ceil_div(rows, LP_THREADS / 64);
  return (unsigned)(b < (1 << 20) ? b : (1 << 20));
}

}  // namespace gs

extern "C" int64_t gs_label_log_probs_workspace_bytes(int64_t rows, int32_t K, int32_t top_k) { return 0; }

extern "C" int gs_label_log_probs_fwd(int64_t rows, int32_t K, int32_t dtype, int32_t top_k, const void* logits,
                                      int64_t row_stride, const void* labels, int32_t label_bytes, void* workspace,
                                      int64_t workspace_bytes, float* log_prob, float* entropy, float* stats,
                                      float* top_log_probs, int64_t* top_labels, void* stream) {
  using namespace gs;
  const int st = lp_check(rows, K, dtype, top_k, logits, row_stride, labels, label_bytes);
  if (st != GS_OK || rows == 0) return st;
  if (!log_prob || !entropy || !stats || (top_k > 0 && (!top_log_probs || !top_labels))) return GS_ERR_INVALID_ARG;
  if (workspace_bytes < gs_label_log_probs_workspace_bytes(rows, K, top_k)) return GS_ERR_WORKSPACE;
  const LpFwd a{rows, row_stride, K, top_k, label_bytes, labels, log_prob, entropy, stats, top_log_probs, top_labels};
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL(label_wave_fwd_kernel<T>, dim3(lp_wave_grid(rows)), dim3(LP_THREADS), 0, (hipStream_t)stream, a,
                       (const T*)logits);
    GS_CHECK_LAUNCH();
    return GS_OK;
  });
}

extern "C" int gs_label_log_probs_bwd(int64_t rows, int32_t K, int32_t dtype, int32_t top_k, const void* logits,
                                      int64_t row_stride, const void* labels, int32_t label_bytes, const float* stats,
                                      const float* entropy, const int64_t* top_labels, const float* g_log_prob,
                                      const float* g_entropy, const float* g_top_log_probs, void* v_logits, void* stream) {
  using namespace gs;
  const int st = lp_check(rows, K, dtype, top_k, logits, row_stride, labels, label_bytes);
  if (st != GS_OK || rows == 0) return st;
  if (!stats || !entropy || !v_logits || (g_top_log_probs && (top_k < 1 || !top_labels))) return GS_ERR_INVALID_ARG;
  if ((uintptr_t)v_logits & (uintptr_t)(dtype_size(dtype) - 1)) return GS_ERR_INVALID_ARG;
  const LpBwd a{rows, row_stride, K, top_k, label_bytes, labels, stats, entropy, top_labels, g_log_prob, g_entropy, g_top_log_probs};
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    hipLaunchKernelGGL(label_wave_bwd_kernel<T>, dim3(lp_wave_grid(rows)), dim3(LP_THREADS), 0, (hipStream_t)stream, a,
                       (const T*)logits, (T*)v_logits);
    GS_CHECK_LAUNCH();
    return GS_OK;
  });
}
