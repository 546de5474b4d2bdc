// Log probabilities of given labels under softmax(logits), with each row's entropy and its best alternatives, and the
// gradient.  With x a row of K logits, m = max x, e_j = exp(x_j - m), S = sum e_j, p_j = e_j / S:
//   log p_j = (x_j - m) - log S,  log_prob = log p_y,  entropy H = log S - (sum e_j (x_j - m)) / S
//   v_x_j = g_lp ([j = y] - p_j) - g_H p_j (log p_j + H) + sum_k g_top_k ([j = t_k] - p_j)
// m and log S are kept apart for the gradient: their sum would lose log S next to logits far from zero.  An exponential
// below 2^-126 is 0 (the hardware's flushes there).  The statistics are taken in one pass, m growing as the row is read
// (what was summed is scaled down when it does); the gradient is one more read of the logits and one write, from m, log S
// and H.
// A label outside [0, K) has no term: log_prob 0 and no gradient through it.  Logits of -inf have p = 0 and add nothing;
// a row of nothing but -inf has log probabilities -inf, entropy 0 and no gradient.  NaN, or +inf, makes its row NaN.
// The top alternatives are the largest logits, NaN above all, equal ones by the lower index.
#include <algorithm>
#include <type_traits>

#include "dtype_io.hpp"

namespace gs {

constexpr int LP_THREADS = 256;
constexpr int LP_SMALL = 64;       // classes up to which a lane takes a whole row
constexpr int LP_WAVE = 2048;      // classes up to which a wave holds a row in registers
constexpr int LP_SEGMENTS = 64;    // parts a long row is cut into at most
constexpr int LP_BLOCKS_FWD = 1024;  // workgroups that the rows are cut into segments for: four a CU, as segments cost a join
constexpr int LP_BLOCKS_BWD = 8192;
constexpr int LP_FLIGHT = 4;       // vectors a thread of the gradient has in flight
constexpr int LP_ADD = 16;         // values added to the statistics at a time
constexpr int LP_WAVE_LIST = 128;  // ... and a wave
constexpr int LP_LIST = 1024;      // candidates for the top alternatives that a workgroup lists
constexpr float LP_LOG2E = 1.44269504088896340736f;
constexpr float LP_LOW = -1.0e4f;  // stands for -inf next to an exponential that is 0 there: 0 * LP_LOW is 0

// The hardware's 2^x of the rounded d log2 e: off by (2 |d| + 2) 2^-24 of itself at most, which grows with the distance from
// the maximum as the term's weight falls (465750 x 19, all results against 64 bits: 8.5e-8, elementary torch operations 6.0e-8).
__device__ __forceinline__ float lp_exp(float d) { return __builtin_amdgcn_exp2f(d * LP_LOG2E); }

// max, sum of exp(x - max) and sum of exp(x - max) (x - max) of a part of a row.  m ignores NaN, which s and w keep; with
// nothing but -inf (and NaN) m stays -inf.
struct LpStat {
  float m, s, w;
};

// adds N values; the sums are taken relative to the new maximum, by which w shifts by (m_old - m_new) s
template <int N> __device__ __forceinline__ void lp_add(LpStat& st, const float (&x)[N]) {
  float m = st.m;
#pragma unroll
  for (int k = 0; k < N; ++k) m = fmaxf(m, x[k]);
  const float ref = m == -INFINITY ? 0.f : m;
  const float d = st.m - ref, e = lp_exp(d);  // 0 while there is nothing
  float w = e * (st.w + fmaxf(d, LP_LOW) * st.s), s = e * st.s;
#pragma unroll
  for (int k = 0; k < N; ++k) {
    const float dk = x[k] - ref, ek = lp_exp(dk);
    s += ek;
    w += ek * fmaxf(dk, LP_LOW);
  }
  st = {m, s, w};
}

__device__ __forceinline__ LpStat lp_join(const LpStat& a, const LpStat& b) {
  const float m = fmaxf(a.m, b.m);
  const float ref = m == -INFINITY ? 0.f : m;
  const float da = a.m - ref, db = b.m - ref, ea = lp_exp(da), eb = lp_exp(db);
  return {m, ea * a.s + eb * b.s, ea * (a.w + fmaxf(da, LP_LOW) * a.s) + eb * (b.w + fmaxf(db, LP_LOW) * b.s)};
}

// all lanes scale to the wave's maximum once, then add up
__device__ __forceinline__ LpStat lp_wave_join(const LpStat& st) {
  const float m = wave_max_all(st.m), ref = m == -INFINITY ? 0.f : m;
  const float d = st.m - ref, e = lp_exp(d);
  return {m, wave_sum_all(e * st.s), wave_sum_all(e * (st.w + fmaxf(d, LP_LOW) * st.s))};
}

// a total order of logits: larger first, NaN above all, equal values (and the two zeros) by the lower index
__device__ __forceinline__ uint32_t lp_order(float x) {
  if (x != x) return 0xfffffffeu;  // a key of all ones stays free: it starts the search for the largest below another
  const uint32_t u = __float_as_uint(x + 0.f);  // -0 becomes +0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float lp_value(uint32_t order) {  // of an order that is not NaN's
  return __uint_as_float(order & 0x80000000u ? order & 0x7fffffffu : ~order);
}
// the largest value that no order from `order` on is below; -inf for those below that of -inf
__device__ __forceinline__ float lp_least(uint32_t order) { return lp_value(order > 0x007fffffu ? order : 0x007fffffu); }
__device__ __forceinline__ uint64_t lp_key(float x, uint32_t j) { return ((uint64_t)lp_order(x) << 32) | (uint32_t)~j; }
__device__ __forceinline__ uint32_t lp_key_index(uint64_t key) { return ~(uint32_t)key; }

// A value that at least k of the wave's values (M a lane) reach, `reach` of them, and that the k-th largest is not far
// above: its upper half, bit by bit, and no further once just k reach it (what is listed from it on is ranked anyway).
// EXACT: the k-th largest itself.
template <bool EXACT, int M> __device__ __forceinline__ uint32_t lp_wave_kth(const uint32_t (&v)[M], int k, int& reach) {
  uint32_t found = 0;
  reach = 64 * M;
  for (int b = 31; b >= (EXACT ? 0 : 16); --b) {
    const uint32_t want = found | (1u << b);
    int c = 0;
#pragma unroll
    for (int i = 0; i < M; ++i) c += __popcll(__ballot(v[i] >= want));
    if (c >= k) {
      found = want;
      reach = c;
    }
    if (!EXACT && c == k) break;
  }
  return found;
}

__device__ __forceinline__ int64_t lp_label(const void* labels, int label_bytes, int64_t r) {
  return label_bytes == 8 ? ((const int64_t*)labels)[r] : (int64_t)((const int32_t*)labels)[r];
}

// n values from x on, as a head up to the first 16-byte boundary, whole vectors and a tail: every row of an odd number of
// classes starts at another alignment.  The head and the tail (fewer than 16 values) are a lane's single extra value each.
template <typename T> struct LpSpan {
  static constexpr int VE = 16 / (int)sizeof(T);
  const T* x;
  int n, head, vecs;
  __device__ LpSpan(const T* p, int count) : x(p), n(count) {
    const int h = (int)(((16u - ((uintptr_t)p & 15u)) & 15u) / sizeof(T));
    head = h < n ? h : n;
    vecs = (n - head) / VE;
  }
  __device__ int at(int v) const { return head + v * VE; }  // index of vector v's first value
  __device__ int extra(int t) const {                       // index of thread t's extra value, -1: none
    const int i = t < head ? t : head + vecs * VE + (t - head);
    return i < n ? i : -1;
  }
  __device__ void load(int v, float (&f)[VE]) const { load_vec<T, VE>(x + at(v), f); }
};

struct LpFwd {
  int64_t rows, stride;
  int32_t K, top, label_bytes;
  const void* labels;
  float *log_prob, *entropy, *stats, *top_lp;
  int64_t* top_idx;
};

// (x - m) - log S, and what it is in a row of nothing but -inf
__device__ __forceinline__ float lp_log_p(float x, float m, float ls) { return ls == -INFINITY ? -INFINITY : (x - m) - ls; }

// `ls` = log S: -inf for a row of nothing but -inf, as for no other
__device__ __forceinline__ void lp_write_row(const LpFwd& a, int64_t r, const LpStat& st, float ls, int64_t y, float x_y) {
  *reinterpret_cast<float2*>(a.stats + 2 * r) = make_float2(st.m, ls);
  a.entropy[r] = ls == -INFINITY ? 0.f : ls - st.w / st.s;
  a.log_prob[r] = y < 0 || y >= a.K ? 0.f : lp_log_p(x_y, st.m, ls);
}

template <typename T>
__device__ __forceinline__ void lp_write_row(const LpFwd& a, int64_t r, const LpStat& st, float ls, const T* x) {
  const int64_t y = lp_label(a.labels, a.label_bytes, r);
  lp_write_row(a, r, st, ls, y, y < 0 || y >= a.K ? 0.f : (float)x[y]);
}

__device__ __forceinline__ void lp_write_top(const LpFwd& a, int64_t r, int rank, uint32_t j, float x, float m, float ls) {
  a.top_idx[r * a.top + rank] = (int64_t)j;
  a.top_lp[r * a.top + rank] = lp_log_p(x, m, ls);
}

// ------------------------------------------------------------------------------------------- up to LP_SMALL classes
// A wave takes 64 rows: it reads their logits as one stretch, lane after lane, into LDS (rows an odd number of words
// apart: lanes that each walk their own row hit different banks), and each lane works on one row without any exchange.
// f / K for f < 64 K by a multiplication: (2^22 / K + 1) f is off by less than f / 2^22 < 1 / K.
// 465750 x 19 fp32: 13 us (3.5 TB/s with labels and results) and 19 us for the gradient (3.7 TB/s of logits); bound by the
// exponentials and LDS words of one lane a row, so that 16-bit rows, staged and written value by value, take the same (13 and
// 18 us for half the bytes).  Each alternative of a row costs K comparisons: 465750 x 19 with the five best 26 us, 300000 x 60
// 28 us, with the ten best 102 us, with the twenty best 211 us; gradients 24, 44, 51 and 74 us.
template <typename T>
__device__ __forceinline__ void lp_small_load(const T* __restrict__ logits, int64_t stride, int64_t row0, int rows, int K,
                                              int P, uint32_t magic, int lane, float* __restrict__ tile) {
  const T* base = logits + row0 * stride;
  const int total = rows * K;
#pragma unroll 8
  for (int f = lane; f < total; f += 64) {
    const int r = (int)(((uint32_t)f * magic) >> 22);
    const int c = f - r * K;
    tile[r * P + c] = (float)base[r * stride + c];
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

template <typename T>
__global__ __launch_bounds__(64) void label_small_fwd_kernel(LpFwd a, uint32_t magic, const T* __restrict__ logits) {
  extern __shared__ float tile[];
  const int lane = threadIdx.x, K = a.K, P = K | 1;
  for (int64_t row0 = (int64_t)blockIdx.x * 64; row0 < a.rows; row0 += (int64_t)gridDim.x * 64) {
    const int rows = (int)(a.rows - row0 < 64 ? a.rows - row0 : 64);
    lp_small_load(logits, a.stride, row0, rows, K, P, magic, lane, tile);
    if (lane < rows) {
      float* x = tile + lane * P;
      const int64_t r = row0 + lane;
      LpStat st{-INFINITY, 0.f, 0.f};
      for (int j = 0; j < K; ++j) st.m = fmaxf(st.m, x[j]);
      const float ref = st.m == -INFINITY ? 0.f : st.m;
      for (int j = 0; j < K; ++j) {
        const float d = x[j] - ref, e = lp_exp(d);
        st.s += e;
        st.w += e * fmaxf(d, LP_LOW);
      }
      const float ls = logf(st.s);
      const int64_t y = lp_label(a.labels, a.label_bytes, r);
      lp_write_row(a, r, st, ls, y, y < 0 || y >= K ? 0.f : x[y]);
      if (st.s == st.s) {
        // One after another; what is taken becomes NaN, which is above nothing.
        for (int t = 0; t < a.top; ++t) {
          float best = -INFINITY;
          int at = -1;
          for (int j = 0; j < K; ++j)
            if (x[j] > best) {
              best = x[j];
              at = j;
            }
          for (int j = 0; at < 0; ++j)  // nothing but -inf is left: the first (K >= top: there is one)
            if (j == K - 1 || x[j] == -INFINITY) at = j;
          x[at] = __builtin_nanf("");
          lp_write_top(a, r, t, (uint32_t)at, best, st.m, ls);
        }
      } else {  // with NaN above all
        uint64_t below = ~0ull;
        for (int t = 0; t < a.top; ++t) {
          uint64_t best = 0;
          for (int j = 0; j < K; ++j) {
            const uint64_t k = lp_key(x[j], (uint32_t)j);
            if (k < below && k > best) best = k;
          }
          below = best;
          const uint32_t j = lp_key_index(best);
          lp_write_top(a, r, t, j, x[j], st.m, ls);
        }
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// -------------------------------------------------------------------------------------------- up to LP_WAVE classes
// A wave holds a row in registers: NV vectors a lane and one extra value.  Read once, whatever is asked for.
// 8191 x 1000 fp32 with the five best 11 us (3.0 TB/s), a quarter of it for the alternatives, and 19 us where just three
// classes are not ruled out; bound by the instructions that every row takes whatever its length (reductions, the search for
// the threshold, listing), so that short rows are far from the bytes: 300000 x 100 76 us (1.6 TB/s), 16-bit 95 us, 200000 x 500
// 87 us (4.6 TB/s).  With more alternatives than lanes that hold values the whole row is listed: 300000 x 100 bf16 with the
// twenty best 641 us, and 300000 x 160 with 21, where the list overflows and they are taken one by one, 1483 us (fp32, whose
// rows fill twice the lanes, 208 us).  Six waves on a SIMD (forced to eight, with values spilled, 16 us); four at least: 8191 x
// 2048 bf16 with the twenty best 20 us, three waves 25.
// f(value, index) over thread t's strip: every LANES-th vector
template <int LANES, typename T, typename F> __device__ __forceinline__ void lp_walk(const LpSpan<T>& sp, int t, F&& f) {
  constexpr int VE = LpSpan<T>::VE;
  for (int v = t; v < sp.vecs; v += LANES) {
    float x[VE];
    sp.load(v, x);
#pragma unroll
    for (int k = 0; k < VE; ++k) f(x[k], sp.at(v) + k);
  }
  const int ex = sp.extra(t);
  if (ex >= 0) f((float)sp.x[ex], ex);
}

// Rows of many equal values (classes ruled out): lists what is above `tie` and, in the order of their indices, the values
// that equal it until there are `top`.  Returns how many are listed; more than LP_WAVE_LIST: too many are above it.  The row
// is read again, out of the caches: the registers that would keep it until here are better spent on more waves.
template <typename T>
__device__ __forceinline__ int lp_wave_ties(const LpSpan<T>& sp, int lane, int top, float tie, uint64_t* __restrict__ list) {
  constexpr int VE = LpSpan<T>::VE;
  const unsigned long long lower = (1ull << lane) - 1ull;
  int listed = 0;
  auto one = [&](bool in, float x, int j) {
    const unsigned long long b = __ballot(in);
    const int at = listed + __popcll(b & lower);
    if (in && at < LP_WAVE_LIST) list[at] = lp_key(x, (uint32_t)j);
    listed += __popcll(b);
  };
  const int ex = sp.extra(lane);
  const float x_ex = ex >= 0 ? (float)sp.x[ex] : -INFINITY;
  one(x_ex > tie, x_ex, ex);
  for (int v0 = 0; v0 < sp.vecs; v0 += 64) {
    float x[VE];
#pragma unroll
    for (int k = 0; k < VE; ++k) x[k] = -INFINITY;
    if (v0 + lane < sp.vecs) sp.load(v0 + lane, x);
#pragma unroll
    for (int k = 0; k < VE; ++k) one(x[k] > tie, x[k], sp.at(v0 + lane) + k);
  }
  if (listed > LP_WAVE_LIST - GS_LABEL_TOP_MAX) return LP_WAVE_LIST + 1;
  if (listed >= top) return listed;
  one(ex >= 0 && ex < sp.head && x_ex == tie, tie, ex);  // (no more than LP_WAVE_LIST in all: the head is short)
  for (int v0 = 0; v0 < sp.vecs && listed < top; v0 += 64) {
    float x[VE];
    const bool there = v0 + lane < sp.vecs;
    if (there) sp.load(v0 + lane, x);
    unsigned long long b[VE];
    int at = listed;
#pragma unroll
    for (int k = 0; k < VE; ++k) {
      b[k] = __ballot(there && x[k] == tie);
      at += __popcll(b[k] & lower);
      listed += __popcll(b[k]);
    }
#pragma unroll
    for (int k = 0; k < VE; ++k)
      if ((b[k] >> lane) & 1ull) {
        if (at < top) list[at] = lp_key(tie, (uint32_t)(sp.at(v0 + lane) + k));
        ++at;
      }
  }
  if (listed < top) one(ex >= sp.head && x_ex == tie, tie, ex);
  return listed < top ? listed : top;
}

template <typename T, int NV>
__global__ __launch_bounds__(LP_THREADS, 4) void label_wave_fwd_kernel(LpFwd a, const T* __restrict__ logits) {
  using Span = LpSpan<T>;
  constexpr int VE = Span::VE, NX = NV * VE + 1;
  __shared__ uint64_t lists[LP_THREADS / 64][LP_WAVE_LIST];
  uint64_t* list = lists[threadIdx.x >> 6];
  const int lane = threadIdx.x & 63;
  const int64_t waves = (int64_t)gridDim.x * (LP_THREADS / 64);
  for (int64_t r = (int64_t)blockIdx.x * (LP_THREADS / 64) + (threadIdx.x >> 6); r < a.rows; r += waves) {
    const Span sp(logits + r * a.stride, a.K);
    float x[NX];
#pragma unroll
    for (int i = 0; i < NX; ++i) x[i] = -INFINITY;
#pragma unroll
    for (int u = 0; u < NV; ++u)
      if (u * 64 + lane < sp.vecs) sp.load(u * 64 + lane, *reinterpret_cast<float(*)[VE]>(&x[u * VE]));
    const int ex = sp.extra(lane);
    if (ex >= 0) x[NX - 1] = (float)sp.x[ex];
    float lane_max = x[0];
#pragma unroll
    for (int i = 1; i < NX; ++i) lane_max = fmaxf(lane_max, x[i]);
    LpStat st{wave_max_all(lane_max), 0.f, 0.f};
    const float ref = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
    for (int i = 0; i < NX; ++i) {
      const float d = x[i] - ref, e = lp_exp(d);
      st.s += e;
      st.w += e * fmaxf(d, LP_LOW);
    }
    st.s = wave_sum_all(st.s);
    st.w = wave_sum_all(st.w);
    const float ls = logf(st.s);
    if (lane == 0) lp_write_row(a, r, st, ls, sp.x);
    if (a.top == 0) continue;
    // the index of a lane's value, -1 where it has none
    auto index = [&](int i) {
      if (i == NX - 1) return ex;
      const int v = (i / VE) * 64 + lane;
      return v < sp.vecs ? sp.at(v) + i % VE : -1;
    };
    // The k-th largest of the lanes' maxima is no larger than the k-th largest value: what is not below it is listed.  For
    // more than half as many alternatives as lanes that is too much, and the search goes over all values.
    int listed = LP_WAVE_LIST + 1;
    if (st.s == st.s) {  // (NaN is above all, and no lane's maximum shows it: such rows go the long way)
      uint32_t order;
      int reach;
      if (a.top <= 32) {
        const uint32_t one[1] = {lp_order(lane_max)};
        order = lp_wave_kth<false>(one, a.top, reach);
      } else {
        uint32_t all[NX];
#pragma unroll
        for (int i = 0; i < NX; ++i) all[i] = index(i) >= 0 ? lp_order(x[i]) : 0u;
        order = lp_wave_kth<false>(all, a.top, reach);
      }
      const float least = lp_least(order);
      listed = 0;
#pragma unroll
      for (int i = 0; i < NX; ++i) {
        if (__ballot(x[i] >= least)) {
          const int j = index(i);
          const bool in = j >= 0 && x[i] >= least;
          const unsigned long long b = __ballot(in);
          const int at = listed + __popcll(b & ((1ull << lane) - 1ull));
          if (in && at < LP_WAVE_LIST) list[at] = lp_key(x[i], (uint32_t)j);
          listed += __popcll(b);
        }
      }
      if (listed > LP_WAVE_LIST) {
        const uint32_t one[1] = {lp_order(lane_max)};
        listed = lp_wave_ties(sp, lane, a.top, lp_least(lp_wave_kth<true>(one, a.top, reach)), list);
      }
    }
    if (listed <= LP_WAVE_LIST) {  // each lane ranks one or two of them
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      for (int at = lane; at < listed; at += 64) {
        const uint64_t mine = list[at];
        int rank = 0;
        for (int i = 0; i < listed; ++i) rank += list[i] > mine;
        if (rank < a.top) lp_write_top(a, r, rank, lp_key_index(mine), lp_value((uint32_t)(mine >> 32)), st.m, ls);
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
    } else {  // NaN, or too many values above many equal ones: one alternative after another
      uint64_t below = ~0ull;
      for (int t = 0; t < a.top; ++t) {
        uint64_t best = 0;
        lp_walk<64>(sp, lane, [&](float f, int j) {
          const uint64_t k = lp_key(f, (uint32_t)j);
          if (k < below && k > best) best = k;
        });
        best = wave_max_all(best);
        below = best;
        const uint32_t j = lp_key_index(best);
        if (lane == 0) lp_write_top(a, r, t, j, (float)sp.x[j], st.m, ls);
      }
    }
  }
}

// ------------------------------------------------------------------------------------------------------- long rows
// A workgroup reads a segment of a row (all of it when there are rows enough to fill the card), four vectors a thread in
// flight.  A thread's strip is every 256th vector; its maximum comes out of the statistics for nothing, and the k-th
// largest of a wave's strip maxima is no larger than the k-th largest value: only strips that reach it are read again,
// and what they hold from it on is listed and ranked.  Where many strips reach it (equal logits, classes ruled out) the
// list takes what is above the k-th largest maximum and the first values that equal it.  Rows whose list overflows all the
// same or that hold NaN take the alternatives one by one, each thread keeping its strip's best and reading the strip again
// when it won.
// 2048 x 100277 bf16 74 us (5.5 TB/s); one row of 131072 bf16 with its eight best 6.2 us in 64 segments and 3.5 us to join
// them; 2048 x 131072 130 us with the twenty best, 109 us where all logits are equal (2.5 ms one by one).
struct LpPart {  // of one segment
  float m, s, w, pad;
};

template <typename T> __device__ __forceinline__ LpStat lp_strip(const LpSpan<T>& sp) {
  constexpr int VE = LpSpan<T>::VE;
  LpStat st{-INFINITY, 0.f, 0.f};
  int v = threadIdx.x;
  for (; v + 3 * LP_THREADS < sp.vecs; v += 4 * LP_THREADS) {
    Raw<T, VE> raw[4];  // (as loaded: a third of the registers, and all workgroups of a CU at once)
#pragma unroll
    for (int u = 0; u < 4; ++u) raw[u] = load_raw<T, VE>(sp.x + sp.at(v + u * LP_THREADS));
#pragma unroll
    for (int u = 0; u < 4; u += LP_ADD / VE) {
      float f[LP_ADD];
#pragma unroll
      for (int k = 0; k < LP_ADD / VE; ++k) unpack<T, VE>(raw[u + k], f + k * VE);
      lp_add<LP_ADD>(st, f);
    }
  }
  for (; v < sp.vecs; v += LP_THREADS) {
    float f[VE];
    sp.load(v, f);
    lp_add<VE>(st, f);
  }
  const int ex = sp.extra(threadIdx.x);
  if (ex >= 0) {
    const float f[1] = {(float)sp.x[ex]};
    lp_add<1>(st, f);
  }
  return st;
}

struct LpShared {
  LpStat part[LP_THREADS / 64];
  uint32_t strips[LP_THREADS];
  uint64_t best[LP_THREADS / 64];
  uint8_t who[LP_THREADS];  // strips that are walked together, `found` of them
  int listed, found;
  uint64_t list[LP_LIST];
};

// out(rank, key) for the k largest of n distinct keys in LDS (zeros are no keys)
template <typename F> __device__ __forceinline__ void lp_rank_list(const uint64_t* list, int n, int k, F&& out) {
  for (int i = threadIdx.x; i < n; i += LP_THREADS) {
    const uint64_t mine = list[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += list[j] > mine;
    if (rank < k && mine) out(rank, mine);
  }
}

// Largest of the workgroup's values, for all threads; two barriers.
__device__ __forceinline__ uint64_t lp_block_max(uint64_t v, uint64_t* lds) {
  v = wave_max_all(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  uint64_t m = lds[0];
#pragma unroll
  for (int w = 1; w < LP_THREADS / 64; ++w) m = lds[w] > m ? lds[w] : m;
  return m;
}

// f(value, index) over the strips of the threads that want theirs walked, all threads at the same number of vectors: a few
// threads with a long strip each would keep the workgroup waiting (2048 x 131072 bf16 with the twenty best 181 us, so 130;
// 2048 x 100277 with the five best 117 and 80 us).  sh.found is 0 before.
template <typename T, typename F>
__device__ __forceinline__ void lp_walk_some(const LpSpan<T>& sp, bool mine, LpShared& sh, F&& f) {
  constexpr int VE = LpSpan<T>::VE;
  if (mine) {
    sh.who[atomicAdd(&sh.found, 1)] = (uint8_t)threadIdx.x;
    const int ex = sp.extra(threadIdx.x);
    if (ex >= 0) f((float)sp.x[ex], ex);
  }
  __syncthreads();
  const uint32_t strips = (uint32_t)sh.found, items = strips * (uint32_t)((sp.vecs + LP_THREADS - 1) / LP_THREADS);
  for (uint32_t q = threadIdx.x; q < items; q += LP_THREADS) {  // (four at a time: no faster)
    const uint32_t i = q / strips;
    const int v = (int)(i * LP_THREADS + sh.who[q - i * strips]);
    if (v < sp.vecs) {
      float x[VE];
      sp.load(v, x);
#pragma unroll
      for (int k = 0; k < VE; ++k) f(x[k], sp.at(v) + k);
    }
  }
  __syncthreads();
}

// Lists what is above `kth` and, in the order of their indices, the values that equal it until there are `top`.  Returns
// how many are listed; more than LP_LIST: too many are above it.
template <typename T>
__device__ __forceinline__ int lp_block_ties(const LpSpan<T>& sp, uint32_t j0, int top, uint32_t strip, uint32_t kth,
                                             LpShared& sh) {
  constexpr int VE = LpSpan<T>::VE, WAVES = LP_THREADS / 64;
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  __syncthreads();
  if (t == 0) sh.listed = sh.found = 0;
  __syncthreads();
  lp_walk_some(sp, strip > kth, sh, [&](float x, int j) {
    if (lp_order(x) > kth) {
      const int at = atomicAdd(&sh.listed, 1);
      if (at < LP_LIST) sh.list[at] = lp_key(x, j0 + (uint32_t)j);
    }
  });
  int have = sh.listed, round = 0;
  if (have > LP_LIST - GS_LABEL_TOP_MAX) return LP_LIST + 1;
  if (have >= top) return have;
  // bits: which of the thread's values from index j on equal it, the threads in the order of their values
  auto take = [&](uint32_t bits, int j) {
    uint32_t* sums = sh.strips + (round++ & 1) * WAVES;
    const int own = __popc(bits);
    int at = own;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const int before = __shfl_up(at, o);
      if (lane >= o) at += before;
    }
    if (lane == 63) sums[wave] = (uint32_t)at;
    __syncthreads();
    at += have - own;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      if (w < wave) at += (int)sums[w];
      have += (int)sums[w];
    }
    for (; bits && at < top; bits &= bits - 1) {
      const uint32_t index = j0 + (uint32_t)(j + __ffs((int)bits) - 1);
      sh.list[at++] = ((uint64_t)kth << 32) | (uint32_t)~index;
    }
  };
  take(t < sp.head && lp_order((float)sp.x[t]) == kth ? 1u : 0u, t);
  for (int v0 = 0; v0 < sp.vecs && have < top; v0 += LP_THREADS) {
    uint32_t bits = 0;
    if (v0 + t < sp.vecs) {
      float x[VE];
      sp.load(v0 + t, x);
#pragma unroll
      for (int k = 0; k < VE; ++k) bits |= lp_order(x[k]) == kth ? 1u << k : 0u;
    }
    take(bits, sp.at(v0 + t));
  }
  if (have < top) {
    const int j = sp.at(sp.vecs) + t;
    take(j < sp.n && lp_order((float)sp.x[j]) == kth ? 1u : 0u, j);
  }
  __syncthreads();
  return have < top ? have : top;
}

// out(rank, key) for the segment's largest `top` values, in any order of ranks; j0 = index of its first value
template <typename T, typename F>
__device__ __forceinline__ void lp_block_top(const LpSpan<T>& sp, uint32_t j0, int top, const LpStat& strip, bool nan,
                                             LpShared& sh, F&& out) {
  int listed = LP_LIST + 1;
  if (!nan) {
    sh.strips[threadIdx.x] = lp_order(strip.m);
    if (threadIdx.x == 0) sh.listed = sh.found = 0;
    __syncthreads();
    uint32_t all[LP_THREADS / 64];  // (every wave searches for itself)
#pragma unroll
    for (int w = 0; w < LP_THREADS / 64; ++w) all[w] = sh.strips[w * 64 + (threadIdx.x & 63)];
    int reach;
    const float least = lp_least(lp_wave_kth<false>(all, top, reach));
    // else the list would be long or overflow: 2048 x 131072 of one value with the twenty best 109 us, listed first 268; one
    // row of 131072 with four values and the eight best 12 us, listed first 93
    const bool ties = reach > 2 * top + 16;
    if (!ties) {
      lp_walk_some(sp, strip.m >= least, sh, [&](float x, int j) {
        if (x >= least) {
          const int at = atomicAdd(&sh.listed, 1);
          if (at < LP_LIST) sh.list[at] = lp_key(x, j0 + (uint32_t)j);
        }
      });
      listed = sh.listed;
    }
    if (ties || listed > LP_LIST)
      listed = lp_block_ties(sp, j0, top, lp_order(strip.m), lp_wave_kth<true>(all, top, reach), sh);
  }
  if (listed <= LP_LIST) {
    lp_rank_list(sh.list, listed, top, out);
    return;
  }
  uint64_t below = ~0ull, best = 0;
  auto search = [&]() {
    best = 0;
    lp_walk<LP_THREADS>(sp, threadIdx.x, [&](float x, int j) {
      const uint64_t k = lp_key(x, j0 + (uint32_t)j);
      if (k < below && k > best) best = k;
    });
  };
  search();
  for (int t = 0; t < top; ++t) {
    const uint64_t won = lp_block_max(best, sh.best);
    if (threadIdx.x == 0 && won) out(t, won);
    if (won == best && won) {
      below = won;
      search();
    }
  }
}

template <typename T, bool TOP>
__global__ __launch_bounds__(LP_THREADS) void label_long_fwd_kernel(LpFwd a, int segments, int seg_len,
                                                                    const T* __restrict__ logits,
                                                                    LpPart* __restrict__ parts, uint64_t* __restrict__ keys) {
  __shared__ typename std::conditional<TOP, LpShared, LpStat[LP_THREADS / 64]>::type sh;
  LpStat* stats;
  if constexpr (TOP) stats = sh.part; else stats = sh;
  const int64_t items = a.rows * segments;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t r = item / segments;
    const int j0 = (int)(item % segments) * seg_len;
    const T* row = logits + r * a.stride;
    const LpSpan<T> sp(row + j0, a.K - j0 < seg_len ? a.K - j0 : seg_len);
    const LpStat strip = lp_strip(sp);
    LpStat st = lp_wave_join(strip);
    if ((threadIdx.x & 63) == 0) stats[threadIdx.x >> 6] = st;
    __syncthreads();
    st = stats[0];
#pragma unroll
    for (int w = 1; w < LP_THREADS / 64; ++w) st = lp_join(st, stats[w]);
    const float ls = logf(st.s);
    if (threadIdx.x == 0) {
      if (segments == 1) lp_write_row(a, r, st, ls, row);
      else parts[item] = {st.m, st.s, st.w, 0.f};
    }
    if constexpr (TOP) {
      if (segments > 1)
        for (int t = sp.n + threadIdx.x; t < a.top; t += LP_THREADS) keys[item * a.top + t] = 0;  // it holds fewer
      lp_block_top(sp, (uint32_t)j0, a.top, strip, st.s != st.s, sh, [&](int rank, uint64_t key) {
        if (segments == 1) {
          const uint32_t j = lp_key_index(key);
          lp_write_top(a, r, rank, j, (float)row[j], st.m, ls);
        } else {
          keys[item * a.top + rank] = key;
        }
      });
    }
    __syncthreads();
  }
}

// Joins the segments of a row: a wave, a lane to each segment.  A segment's keys come in order, so that the best of the
// row is among the lanes' first ones: whichever lane gave it goes on to its next.
template <typename T, bool TOP>
__global__ __launch_bounds__(64) void label_join_kernel(LpFwd a, int segments, const T* __restrict__ logits,
                                                        const LpPart* __restrict__ parts, const uint64_t* __restrict__ keys) {
  const int64_t r = blockIdx.x;
  const T* row = logits + r * a.stride;
  const int lane = threadIdx.x;
  static_assert(LP_SEGMENTS <= 64, "a lane takes one segment");
  extern __shared__ uint64_t list[];  // [segments][top]
  if constexpr (TOP) {
    const uint64_t* mine = keys + r * segments * a.top;
#pragma unroll 8
    for (int i = lane; i < segments * a.top; i += 64) list[i] = mine[i];
  }
  LpStat st{-INFINITY, 0.f, 0.f};
  if (lane < segments) {
    const LpPart p = parts[r * segments + lane];
    st = {p.m, p.s, p.w};
  }
  st = lp_wave_join(st);
  const float ls = logf(st.s);
  if (lane == 0) lp_write_row(a, r, st, ls, row);
  if constexpr (TOP) {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    int at = 0;
    uint64_t head = lane < segments ? list[lane * a.top] : 0ull, won = 0;
    for (int t = 0; t < a.top; ++t) {
      const uint64_t best = wave_max_all(head);
      if (lane == t) won = best;
      if (head == best) head = ++at < a.top ? list[lane * a.top + at] : 0ull;  // (keys are distinct; zeros are none)
    }
    if (lane < a.top) {
      const uint32_t j = lp_key_index(won);
      lp_write_top(a, r, lane, j, (float)row[j], st.m, ls);
    }
  }
}

// -------------------------------------------------------------------------------------------------------- gradient
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
  int64_t y;  // -1: no label
  bool none;  // nothing but -inf
};

__device__ __forceinline__ LpRow lp_row(const LpBwd& a, int64_t r) {
  LpRow w;
  w.m = a.stats[2 * r];
  w.ls = a.stats[2 * r + 1];
  w.H = a.entropy[r];
  w.none = w.ls == -INFINITY;
  const int64_t y = lp_label(a.labels, a.label_bytes, r);
  const bool kept = y >= 0 && y < a.K && !w.none;
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
  return lp_exp(d) * (w.c0 - w.c1 * (fmaxf(d, LP_LOW) + w.H));  // NaN stays in the exponential
}

// v at the t-th alternative of row r, whole
template <typename T> __device__ __forceinline__ T lp_grad_top(const LpBwd& a, const LpRow& w, int64_t r, int t, float x) {
  const int64_t j = a.top_idx[r * a.top + t];
  return (T)(lp_grad(w, x) + (j == w.y ? w.g : 0.f) + a.g_top[r * a.top + t]);
}

template <typename T, bool PAST>
__global__ __launch_bounds__(64) void label_small_bwd_kernel(LpBwd a, uint32_t magic, const T* __restrict__ logits,
                                                             T* __restrict__ v) {
  extern __shared__ float tile[];
  const int lane = threadIdx.x, K = a.K, P = K | 1;
  for (int64_t row0 = (int64_t)blockIdx.x * 64; row0 < a.rows; row0 += (int64_t)gridDim.x * 64) {
    const int rows = (int)(a.rows - row0 < 64 ? a.rows - row0 : 64);
    lp_small_load(logits, a.stride, row0, rows, K, P, magic, lane, tile);
    if (lane < rows) {
      float* x = tile + lane * P;
      const int64_t r = row0 + lane;
      const LpRow w = lp_row(a, r);
      for (int j = 0; j < K; ++j) x[j] = w.none ? 0.f : lp_grad(w, x[j]);
      if (w.y >= 0) x[w.y] += w.g;
      if (a.g_top && !w.none)
        for (int t = 0; t < a.top; ++t) x[a.top_idx[r * a.top + t]] += a.g_top[r * a.top + t];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    T* out = v + row0 * K;
    const int total = rows * K;
#pragma unroll 8
    for (int f = lane; f < total; f += 64) {
      const int r = (int)(((uint32_t)f * magic) >> 22);
      const T g = (T)tile[r * P + f - r * K];
      if constexpr (PAST) __builtin_nontemporal_store(g, out + f); else out[f] = g;
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// LANES threads (a wave, or a workgroup) over a part of a row; the gradient's row is as far apart from a 16-byte boundary
// as the logits' (`wide`), or is written value by value (a slice of channels, whose rows are not K apart).  2048 x 100277 bf16
// in 8192 segments 163 us, 5.0 TB/s (one vector in flight and a workgroup a row: 203 us).  A wave a row is bound by the latency
// of a row at a time: 300000 x 100 fp32 89 us (2.7 TB/s), bf16 123 us (1.0), 200000 x 500 148 and 89 us (5.4 and 4.5); with
// alternatives, whose places are stored a second time behind a wait, 300000 x 100 with five 173 us, with twenty 292 us.
template <typename T, int LANES, bool PAST>
__device__ __forceinline__ void lp_grad_span(const LpSpan<T>& sp, const LpRow& w, int j0, int t, T* __restrict__ out) {
  constexpr int VE = LpSpan<T>::VE;
  const bool wide = (((uintptr_t)sp.x ^ (uintptr_t)out) & 15u) == 0;
  const int y = (int)(w.y - j0);  // the label's place in this part, if it is in it
  auto put = [&](int v, const Raw<T, VE>& raw) {
    float f[VE];
    unpack<T, VE>(raw, f);
#pragma unroll
    for (int k = 0; k < VE; ++k) f[k] = w.none ? 0.f : lp_grad(w, f[k]);
    const int j = sp.at(v);
    if (w.y >= 0 && (uint32_t)(y - j) < (uint32_t)VE) {
#pragma unroll
      for (int k = 0; k < VE; ++k) f[k] += y == j + k ? w.g : 0.f;
    }
    if (wide) {
      if constexpr (PAST) store_vec_nt<T, VE>(out + j, f); else store_vec<T, VE>(out + j, f);
    } else {
#pragma unroll
      for (int k = 0; k < VE; ++k) out[j + k] = (T)f[k];
    }
  };
  int v = t;
  for (; v + (LP_FLIGHT - 1) * LANES < sp.vecs; v += LP_FLIGHT * LANES) {
    Raw<T, VE> raw[LP_FLIGHT];
#pragma unroll
    for (int u = 0; u < LP_FLIGHT; ++u) raw[u] = load_raw<T, VE>(sp.x + sp.at(v + u * LANES));
#pragma unroll
    for (int u = 0; u < LP_FLIGHT; ++u) put(v + u * LANES, raw[u]);
  }
  for (; v < sp.vecs; v += LANES) put(v, load_raw<T, VE>(sp.x + sp.at(v)));
  const int ex = sp.extra(t);
  if (ex >= 0) out[ex] = (T)((w.none ? 0.f : lp_grad(w, (float)sp.x[ex])) + (w.y >= 0 && ex == y ? w.g : 0.f));
}

template <typename T, bool PAST>
__global__ __launch_bounds__(LP_THREADS) void label_wave_bwd_kernel(LpBwd a, const T* __restrict__ logits, T* __restrict__ v) {
  const int lane = threadIdx.x & 63;
  const int64_t waves = (int64_t)gridDim.x * (LP_THREADS / 64);
  for (int64_t r = (int64_t)blockIdx.x * (LP_THREADS / 64) + (threadIdx.x >> 6); r < a.rows; r += waves) {
    const LpSpan<T> sp(logits + r * a.stride, a.K);
    const LpRow w = lp_row(a, r);
    T* out = v + r * a.K;
    lp_grad_span<T, 64, PAST>(sp, w, 0, lane, out);
    if (a.g_top && !w.none) {
      __builtin_amdgcn_s_waitcnt(0);  // the row's stores are out before some of its values are stored again
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
      if (lane < a.top) {
        const int64_t j = a.top_idx[r * a.top + lane];
        out[j] = lp_grad_top<T>(a, w, r, lane, (float)sp.x[j]);
      }
    }
  }
}

template <typename T, bool PAST>
__global__ __launch_bounds__(LP_THREADS) void label_long_bwd_kernel(LpBwd a, int segments, int seg_len,
                                                                    const T* __restrict__ logits, T* __restrict__ v) {
  const int64_t items = a.rows * segments;
  for (int64_t item = blockIdx.x; item < items; item += gridDim.x) {
    const int64_t r = item / segments;
    const int j0 = (int)(item % segments) * seg_len;
    const LpSpan<T> sp(logits + r * a.stride + j0, a.K - j0 < seg_len ? a.K - j0 : seg_len);
    const LpRow w = lp_row(a, r);
    T* out = v + r * a.K + j0;
    lp_grad_span<T, LP_THREADS, PAST>(sp, w, j0, threadIdx.x, out);
    if (a.g_top && !w.none) {
      __builtin_amdgcn_s_waitcnt(0);
      __syncthreads();
      if ((int)threadIdx.x < a.top) {
        const int64_t j = a.top_idx[r * a.top + threadIdx.x] - j0;
        if (j >= 0 && j < sp.n) out[j] = lp_grad_top<T>(a, w, r, threadIdx.x, (float)sp.x[j]);
      }
      __syncthreads();
    }
  }
}

static int lp_check(int64_t rows, int32_t K, int32_t dtype, int32_t top_k, const void* logits, int64_t row_stride,
                    const void* labels, int32_t label_bytes) {
  if (rows < 0 || K < 1 || !dtype_size(dtype) || top_k < 0 || top_k > K || row_stride < 0) return GS_ERR_INVALID_ARG;
  if (top_k > GS_LABEL_TOP_MAX || K > GS_LABEL_CLASSES_MAX) return GS_ERR_UNSUPPORTED;
  if (label_bytes != 4 && label_bytes != 8) return GS_ERR_INVALID_ARG;
  if (rows == 0) return GS_OK;
  if (!logits || !labels) return GS_ERR_INVALID_ARG;
  if (((uintptr_t)logits & (uintptr_t)(dtype_size(dtype) - 1)) || ((uintptr_t)labels & (uintptr_t)(label_bytes - 1)))
    return GS_ERR_INVALID_ARG;
  return GS_OK;
}

static unsigned lp_grid(int64_t items, int per_block) {
  const int64_t b = ceil_div(items, per_block);
  return (unsigned)(b < (1 << 20) ? b : (1 << 20));  // (the kernels go on to further items)
}

// Segments of a long row: about `blocks` workgroups in all, none shorter than a vector for each thread.
static int lp_segments(int64_t rows, int32_t K, int64_t blocks, int32_t* seg_len) {
  int64_t n = rows >= blocks ? 1 : ceil_div(blocks, rows);
  n = std::min<int64_t>(n, std::min<int64_t>(LP_SEGMENTS, ceil_div(K, 2048)));
  *seg_len = (int32_t)(ceil_div(ceil_div(K, n), 64) * 64);
  return (int)ceil_div(K, *seg_len);
}

template <typename F> static int with_vectors(int n, F&& f) {
  if (n <= 1) return f(std::integral_constant<int, 1>{});
  if (n <= 2) return f(std::integral_constant<int, 2>{});
  if (n <= 4) return f(std::integral_constant<int, 4>{});
  return f(std::integral_constant<int, 8>{});
}

static uint32_t lp_magic(int32_t K) { return (1u << 22) / (uint32_t)K + 1u; }

static int64_t lp_parts_bytes(int64_t items) { return ceil_div(items * (int64_t)sizeof(LpPart), 256) * 256; }

}  // namespace gs

extern "C" int64_t gs_label_log_probs_workspace_bytes(int64_t rows, int32_t K, int32_t top_k) {
  if (rows <= 0 || K <= gs::LP_WAVE || top_k < 0) return 0;
  int32_t seg_len;
  const int64_t segments = gs::lp_segments(rows, K, gs::LP_BLOCKS_FWD, &seg_len);
  return segments == 1 ? 0 : gs::lp_parts_bytes(rows * segments) + 8 * rows * segments * top_k;
}

extern "C" int gs_label_log_probs_fwd(int64_t rows, int32_t K, int32_t dtype, int32_t top_k, const void* logits,
                                      int64_t row_stride, const void* labels, int32_t label_bytes, void* workspace,
                                      int64_t workspace_bytes, float* log_prob, float* entropy, float* stats,
                                      float* top_log_probs, int64_t* top_labels, void* stream) {
  using namespace gs;
  const int st = lp_check(rows, K, dtype, top_k, logits, row_stride, labels, label_bytes);
  if (st != GS_OK || rows == 0) return st;
  if (!log_prob || !entropy || !stats || (top_k > 0 && (!top_log_probs || !top_labels))) return GS_ERR_INVALID_ARG;
  if ((uintptr_t)stats & 7) return GS_ERR_INVALID_ARG;
  const int64_t need = gs_label_log_probs_workspace_bytes(rows, K, top_k);
  if (workspace_bytes < need) return GS_ERR_WORKSPACE;
  if (need > 0 && (!workspace || ((uintptr_t)workspace & 15))) return GS_ERR_INVALID_ARG;
  const LpFwd a{rows, row_stride, K, top_k, label_bytes, labels, log_prob, entropy, stats, top_log_probs, top_labels};
  hipStream_t s = (hipStream_t)stream;
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const T* x = (const T*)logits;
    if (K <= LP_SMALL) {
      hipLaunchKernelGGL(label_small_fwd_kernel<T>, dim3(lp_grid(rows, 64)), dim3(64), 64 * (K | 1) * sizeof(float), s, a,
                         lp_magic(K), x);
      GS_CHECK_LAUNCH();
      return GS_OK;
    }
    if (K <= LP_WAVE)
      return with_vectors((int)ceil_div(K, 64 * LpSpan<T>::VE), [&](auto nv) {
        constexpr int NV = decltype(nv)::value;
        if constexpr (NV * LpSpan<T>::VE * 64 <= LP_WAVE) {
          hipLaunchKernelGGL((label_wave_fwd_kernel<T, NV>), dim3(lp_grid(rows, LP_THREADS / 64)), dim3(LP_THREADS), 0, s, a, x);
          GS_CHECK_LAUNCH();
          return GS_OK;
        }
        return GS_ERR_INVALID_ARG;
      });
    int32_t seg_len;
    const int segments = lp_segments(rows, K, LP_BLOCKS_FWD, &seg_len);
    LpPart* parts = (LpPart*)workspace;
    uint64_t* keys = (uint64_t*)((char*)workspace + lp_parts_bytes(rows * segments));
    const dim3 grid(lp_grid(rows * segments, 1)), block(LP_THREADS);
    if (top_k > 0)
      hipLaunchKernelGGL((label_long_fwd_kernel<T, true>), grid, block, 0, s, a, segments, seg_len, x, parts, keys);
    else
      hipLaunchKernelGGL((label_long_fwd_kernel<T, false>), grid, block, 0, s, a, segments, seg_len, x, parts, keys);
    GS_CHECK_LAUNCH();
    if (segments == 1) return GS_OK;
    if (top_k > 0)
      hipLaunchKernelGGL((label_join_kernel<T, true>), dim3((unsigned)rows), dim3(64), 8 * segments * top_k, s, a, segments,
                         x, parts, keys);
    else
      hipLaunchKernelGGL((label_join_kernel<T, false>), dim3((unsigned)rows), dim3(64), 0, s, a, segments, x, parts, keys);
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
  const bool past = rows * K * dtype_size(dtype) >= PAST_CACHES_MIN_BYTES;
  hipStream_t s = (hipStream_t)stream;
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    const T* x = (const T*)logits;
    if (K <= LP_SMALL) {
      const dim3 grid(lp_grid(rows, 64)), block(64);
      const size_t tile = 64 * (K | 1) * sizeof(float);
      if (past)
        hipLaunchKernelGGL((label_small_bwd_kernel<T, true>), grid, block, tile, s, a, lp_magic(K), x, (T*)v_logits);
      else
        hipLaunchKernelGGL((label_small_bwd_kernel<T, false>), grid, block, tile, s, a, lp_magic(K), x, (T*)v_logits);
    } else if (K <= LP_WAVE) {
      const dim3 grid(lp_grid(rows, LP_THREADS / 64)), block(LP_THREADS);
      if (past)
        hipLaunchKernelGGL((label_wave_bwd_kernel<T, true>), grid, block, 0, s, a, x, (T*)v_logits);
      else
        hipLaunchKernelGGL((label_wave_bwd_kernel<T, false>), grid, block, 0, s, a, x, (T*)v_logits);
    } else {
      int32_t seg_len;
      const int segments = lp_segments(rows, K, LP_BLOCKS_BWD, &seg_len);
      const dim3 grid(lp_grid(rows * segments, 1)), block(LP_THREADS);
      if (past)
        hipLaunchKernelGGL((label_long_bwd_kernel<T, true>), grid, block, 0, s, a, segments, seg_len, x, (T*)v_logits);
      else
        hipLaunchKernelGGL((label_long_bwd_kernel<T, false>), grid, block, 0, s, a, segments, seg_len, x, (T*)v_logits);
    }
    GS_CHECK_LAUNCH();
    return GS_OK;
  });
}
