// Embedding lookup with scaling, and the gradient of the table by sorted ids.
//   out[i] = scale * table[ids[i]]                          (an id outside [0, V) selects nothing: a row of zeros)
//   v_table[v] = scale * sum over i with ids[i] = v of v_out[i]   (a row that no id selects: zeros, whatever the scale)
// Both are bound by HBM.  The lookup reads n rows and writes n rows in the widest vectors that the row size and the
// alignment allow.  The gradient reads every row of v_out once and writes the table:
//   1. the ids are sorted, stably, with their positions: by one workgroup in LDS up to EMB_SORT1 of them, else by a radix
//      sort of three launches a digit.  The sort leaves most of the card idle, so its launches carry the zeros of the
//      table along: workgroups behind those of the sort fill a share of it each.
//   2. embed_runs_kernel cuts the sorted ids into pieces, one to a group of lanes as wide as a row.  A short run of equal
//      ids is added up by the group in whose piece it starts, and stored; of a long one each group adds what lies in its
//      piece.
//   3. embed_join_kernel adds the pieces of each long run.
// Sums are held in fp32 and rounded once at the end.  Their order is fixed (no float atomics) by the ids, the sizes and the
// width of the vectors that strides and addresses allow: ascending i in a short run, groups and workgroups joined as trees in a
// long one, threads' shares in a table of few rows.
// Up to EMB_DIRECT ids need no sort (but on a very large table): each workgroup picks the ids that fall among its rows.
// Nor does a table of few and short rows, however many ids: it is added up in LDS.
#include <algorithm>
#include <cmath>
#include <type_traits>

#include "dtype_io.hpp"

namespace gs {

constexpr int EMB_THREADS = 256;
constexpr int EMB_FLIGHT = 4;         // rows a thread of the lookup has in flight
constexpr int EMB_DIRECT = 256;
constexpr int EMB_FEW = 64;           // rows of a table that LDS holds once for each row that a workgroup reads at a time
constexpr int EMB_ROWS_MAX = 256;     // rows of the table per workgroup of the direct form
constexpr int EMB_SORT1 = 16384;      // ids that one workgroup sorts in LDS
constexpr int EMB_SORT1_THREADS = 1024;
constexpr int EMB_RADIX_BITS = 9;
constexpr int EMB_RADIX = 1 << EMB_RADIX_BITS;
constexpr int EMB_ITEMS = 8;          // ids per thread and launch of the radix sort
constexpr int EMB_TILE = EMB_THREADS * EMB_ITEMS;
constexpr int EMB_JOIN_THREADS = 1024;
constexpr int EMB_JOIN_PIECES = 256;  // pieces that a workgroup of the join looks at, at most
constexpr int EMB_PIECE_MAX = 64;
constexpr int EMB_FLIGHT_RUNS = 8;    // rows a group has in flight there
constexpr int EMB_JOIN_FLIGHT = 8;    // pieces a group of the join has in flight

__device__ __forceinline__ int64_t emb_id(const void* ids, int id_bytes, int64_t i) {
  return id_bytes == 8 ? ((const int64_t*)ids)[i] : (int64_t)((const int32_t*)ids)[i];
}

// ---------------------------------------------------------------------------------------------------------- lookup
// vpr vectors of N elements per row; a workgroup takes `rows_per` rows at a time, their vectors numbered through.
// f / vpr by a multiplication: exact while f * vpr < 2^32 (f is below 2048, vpr too unless rows_per is 1).  Bound by the
// rows' way through the caches and out: 200003 x 512 fp16 on 32000 rows 60 us (6.8 TB/s read and written, 4.0 of it HBM),
// 1M x 16 fp32 on 64 rows 14 us (5.2 TB/s), 16384 x 1024 bf16 11 us; one id 2.1 us.  Plain stores: nontemporal ones save
// 2 us of 60 and cost the pass behind them 3.
template <typename T, int N>
__global__ __launch_bounds__(EMB_THREADS) void embed_lookup_kernel(int64_t n, int64_t V, int64_t vpr, int rows_per,
                                                                   uint32_t magic, const T* __restrict__ table,
                                                                   int64_t ts, const void* __restrict__ ids, int id_bytes,
                                                                   float scale, T* __restrict__ out) {
  for (int64_t r0 = (int64_t)blockIdx.x * rows_per; r0 < n; r0 += (int64_t)gridDim.x * rows_per) {
    const int64_t rows = n - r0 < rows_per ? n - r0 : rows_per;
    const int64_t total = rows * vpr;
    for (int64_t f0 = threadIdx.x; f0 < total; f0 += EMB_FLIGHT * EMB_THREADS) {
      float x[EMB_FLIGHT][N];
      int64_t id[EMB_FLIGHT], c[EMB_FLIGHT];
#pragma unroll
      for (int u = 0; u < EMB_FLIGHT; ++u) {
        const int64_t f = f0 + u * EMB_THREADS < total ? f0 + u * EMB_THREADS : total - 1;
        const int64_t r = rows_per == 1 ? 0 : vpr == 1 ? f : (int64_t)__umulhi((uint32_t)f, magic);
        c[u] = (f - r * vpr) * N;
        id[u] = emb_id(ids, id_bytes, r0 + r);
      }
#pragma unroll
      for (int u = 0; u < EMB_FLIGHT; ++u) {
        if (id[u] >= 0 && id[u] < V) {
          load_vec<T, N>(table + id[u] * ts + c[u], x[u]);
        } else {
#pragma unroll
          for (int k = 0; k < N; ++k) x[u][k] = 0.f;
        }
      }
#pragma unroll
      for (int u = 0; u < EMB_FLIGHT; ++u) {
        const int64_t f = f0 + u * EMB_THREADS;
        if (f < total) {
          const bool any = id[u] >= 0 && id[u] < V;  // (0 * scale is no zero for every scale)
#pragma unroll
          for (int k = 0; k < N; ++k) x[u][k] = any ? x[u][k] * scale : 0.f;
          store_vec<T, N>(out + (r0 * vpr + f) * N, x[u]);
        }
      }
    }
  }
}

// ---------------------------------------------------------------------------------------------------------- gradient
// A row of N-element vectors is taken by a group of G lanes (G a power of two, at most a wave); rows wider than 64
// vectors take several column tiles (blockIdx.y).
struct EmbShape {
  int64_t n, V, vpr;  // ids, rows of the table, vectors per row
  int64_t gs;         // row stride of v_out in elements
  int32_t G, rows_per;
  int32_t piece, longest;  // sorted ids of a group; of a run that one group adds up by itself (no fewer)
  int32_t join;            // pieces that a workgroup of the join looks at
  float scale;
};

// The sorted sums go past the caches: the rows of v_out that are still to be read stay there instead.  Lookup and gradient,
// plain and past the caches: 100000 ids on 50000 x 256 fp32 101 and 97 us, 16384 on 131072 x 1024 bf16 81 and 79, 200003 on
// 32000 x 512 bf16 174 and 174 (185 and 191 with a pass over the gradient behind it).
template <typename T, int N, bool NT = true>
__device__ __forceinline__ void emb_store(T* __restrict__ p, const float (&acc)[N], float scale) {
  float x[N];
#pragma unroll
  for (int k = 0; k < N; ++k) x[k] = acc[k] * scale;
  if constexpr (NT) store_vec_nt<T, N>(p, x); else store_vec<T, N>(p, x);
}

// ---- the table's zeros, in `shares` stretches of whole vectors (the first also has what lies before and behind them)
// With ids for an eighth of the rows and more they go past the caches, for the same reason as the sums; with fewer the
// plain stores are faster.  131072 x 1024 bf16, lookup and gradient, plain / past the caches: 4096 ids 63 / 73 us, 8192
// ids 73 / 74 us, 16384 ids 87 / 79 us, 65536 ids 190 / 180 us.
struct EmbFill {
  char* base;
  int64_t bytes;
  int32_t share, shares, past_caches;
};

__device__ __forceinline__ void emb_fill(const EmbFill& f, int64_t block, int64_t blocks) {
  const int64_t lead = (int64_t)((16u - ((uintptr_t)f.base & 15u)) & 15u), head = lead < f.bytes ? lead : f.bytes;
  const int64_t vecs = (f.bytes - head) / 16;
  const int64_t per = (vecs + f.shares - 1) / f.shares, v0 = f.share * per, v1 = v0 + per < vecs ? v0 + per : vecs;
  uint4* body = reinterpret_cast<uint4*>(f.base + head);
  const int64_t first = v0 + block * blockDim.x + threadIdx.x, step = blocks * blockDim.x;
  if (f.past_caches)
    for (int64_t v = first; v < v1; v += step) store16_nt(body + v, word4{0, 0, 0, 0});
  else
    for (int64_t v = first; v < v1; v += step) body[v] = make_uint4(0, 0, 0, 0);
  if (f.share == 0 && block == 0) {
    const int64_t tail = head + vecs * 16, i = (int64_t)threadIdx.x * 2;  // both are fewer than 8 pairs of bytes
    if (i < head) *reinterpret_cast<uint16_t*>(f.base + i) = 0;
    if (tail + i < f.bytes) *reinterpret_cast<uint16_t*>(f.base + tail + i) = 0;
  }
}

// ---- stable sort of the ids with their positions
// Not radix_sort.hip's: that one sorts 64-bit keys (tile and depth) from given pairs, with the count in device memory, and has
// no room for the table's zeros.  Here keys are one word and the first digit's come straight from the ids, and a tile scatters
// through LDS, which pays for the few digits that ids have: 1M items, a digit of 9 bits 14 us against 24 from registers.
__device__ __forceinline__ uint32_t emb_key(const void* ids, int id_bytes, int64_t i, int64_t V) {
  const int64_t id = emb_id(ids, id_bytes, i);
  return id >= 0 && id < V ? (uint32_t)id : (uint32_t)V;  // ids that select nothing sort behind all rows
}

// For each of a wave's items the lanes whose item has the same digit (of `bits` bits from `shift` on), lower and upper half.
// All items at once: ballots of one do not wait for those of another.
template <int ITEMS>
__device__ __forceinline__ void emb_peers(const uint32_t (&key)[ITEMS], int64_t wave_first, int64_t n, int shift, int bits,
                                          uint32_t (&lo)[ITEMS], uint32_t (&hi)[ITEMS]) {
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const unsigned long long valid = __ballot(wave_first + i * 64 + (threadIdx.x & 63) < n);
    lo[i] = (uint32_t)valid;
    hi[i] = (uint32_t)(valid >> 32);
  }
  for (int b = shift; b < shift + bits; ++b) {
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const uint32_t bit = (uint32_t)__builtin_amdgcn_sbfe((int)key[i], b, 1);  // all ones or none
      const unsigned long long m = __ballot(bit != 0);
      lo[i] &= ~((uint32_t)m ^ bit);
      hi[i] &= ~((uint32_t)(m >> 32) ^ bit);
    }
  }
}

// One digit of the items that a workgroup holds in registers, wave by wave in their order: cnt [waves][radix] gets each
// wave's counts, and each item its rank among its wave's items of the same digit.
template <int ITEMS>
__device__ __forceinline__ void emb_rank(const uint32_t (&key)[ITEMS], int64_t wave_first, int64_t n, int shift, int bits,
                                         uint32_t* __restrict__ cnt, uint32_t (&rank)[ITEMS]) {
  uint32_t lo[ITEMS], hi[ITEMS];
  emb_peers(key, wave_first, n, shift, bits, lo, hi);
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const bool valid = wave_first + i * 64 + (threadIdx.x & 63) < n;
    const uint32_t d = (key[i] >> shift) & ((1u << bits) - 1u);
    const uint32_t before = __builtin_amdgcn_mbcnt_hi(hi[i], __builtin_amdgcn_mbcnt_lo(lo[i], 0));
    const uint32_t prev = cnt[d];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    if (valid && before == 0) cnt[d] = prev + (uint32_t)(__popc(lo[i]) + __popc(hi[i]));
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    rank[i] = prev + before;
  }
}

// exclusive sum over the workgroup's threads; `lds` has a word for each wave
template <int THREADS> __device__ __forceinline__ uint32_t emb_scan(uint32_t v, uint32_t* lds) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  uint32_t incl = v;
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const uint32_t t = __shfl_up(incl, o);
    if (lane >= o) incl += t;
  }
  if (lane == 63) lds[wave] = incl;
  __syncthreads();
  uint32_t before = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 64; ++w)
    if (w < wave) before += lds[w];
  __syncthreads();
  return before + incl - v;
}

// Workgroup 0 sorts up to 1024 ITEMS ids in LDS, digits of at most 8 bits; the others fill.  16384 ids of 13 bits take 22 us
// (ballots and LDS words in one CU), 3000 8 us; the zeros of a 268 MB table hide it: 50 us together, 5.4 TB/s of stores.
template <int ITEMS>
__global__ __launch_bounds__(EMB_SORT1_THREADS) void embed_sort1_kernel(int n, int64_t V, int bits,
                                                                        const void* __restrict__ ids, int id_bytes,
                                                                        uint32_t* __restrict__ keys_out,
                                                                        uint32_t* __restrict__ pos_out, EmbFill fill) {
  if (blockIdx.x > 0) {
    emb_fill(fill, blockIdx.x - 1, gridDim.x - 1);
    return;
  }
  constexpr int WAVES = EMB_SORT1_THREADS / 64, RADIX = 256;
  __shared__ uint32_t cnt[WAVES][RADIX];
  __shared__ uint32_t keys[ITEMS * EMB_SORT1_THREADS];
  __shared__ uint16_t poss[ITEMS * EMB_SORT1_THREADS];
  __shared__ uint32_t wsum[WAVES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, first = wave * 64 * ITEMS;
  const int passes = (bits + 7) / 8, per = (bits + passes - 1) / passes;
  uint32_t key[ITEMS], rank[ITEMS];
  uint16_t pos[ITEMS];
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {
    const int at = first + i * 64 + lane;
    key[i] = at < n ? emb_key(ids, id_bytes, at, V) : 0;
    pos[i] = (uint16_t)at;
  }
  for (int p = 0; p < passes; ++p) {
    for (int d = threadIdx.x; d < WAVES * RADIX; d += EMB_SORT1_THREADS) (&cnt[0][0])[d] = 0;
    __syncthreads();
    const int shift = p * per, width = bits - shift < per ? bits - shift : per;
    emb_rank<ITEMS>(key, first, n, shift, width, cnt[wave], rank);
    __syncthreads();
    uint32_t total = 0;
    if (threadIdx.x < RADIX)
      for (int w = 0; w < WAVES; ++w) total += cnt[w][threadIdx.x];
    uint32_t run = emb_scan<EMB_SORT1_THREADS>(total, wsum);
    if (threadIdx.x < RADIX)
      for (int w = 0; w < WAVES; ++w) {
        const uint32_t c = cnt[w][threadIdx.x];
        cnt[w][threadIdx.x] = run;
        run += c;
      }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (first + i * 64 + lane < n) {
        const uint32_t to = cnt[wave][(key[i] >> shift) & ((1u << width) - 1u)] + rank[i];
        keys[to] = key[i];
        poss[to] = pos[i];
      }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const int at = first + i * 64 + lane;
      key[i] = at < n ? keys[at] : 0;
      pos[i] = at < n ? poss[at] : 0;
    }
  }
#pragma unroll
  for (int i = 0; i < ITEMS; ++i) {  // (out of LDS too: words scattered over the lists would go out one a cycle)
    const int at = first + i * 64 + lane;
    if (at < n) {
      keys_out[at] = key[i];
      pos_out[at] = pos[i];
    }
  }
}

// One digit of the radix sort: the digits' counts per workgroup (digit by digit), their sums over the workgroups before,
// and the scatter.  `keys` NULL: the first digit, straight from the ids.  Workgroups from `blocks` on fill.  1M ids of 7
// bits: 7 + 4 + 10 us, a digit of 9 bits 9 + 4 + 14; bound by latency.  The scatter goes through LDS, where a workgroup's
// items of a digit come to lie next to each other (9 bits straight from registers: 24 us; 4096 items a workgroup: 18 us).
struct EmbDigit {
  int64_t n, V;
  const void* ids;
  int32_t id_bytes, shift, bits, blocks;
  const uint32_t *keys, *pos;
  uint32_t *keys_out, *pos_out;
  uint32_t *table, *totals;  // [radix][blocks], [radix]
  EmbFill fill;
};

__device__ __forceinline__ void emb_load_items(const EmbDigit& s, int64_t first, uint32_t (&key)[EMB_ITEMS]) {
  const int lane = threadIdx.x & 63;
#pragma unroll
  for (int i = 0; i < EMB_ITEMS; ++i) {
    const int64_t at = first + i * 64 + lane;
    key[i] = at < s.n ? (s.keys ? s.keys[at] : emb_key(s.ids, s.id_bytes, at, s.V)) : 0;
  }
}

__global__ __launch_bounds__(EMB_THREADS) void embed_hist_kernel(EmbDigit s) {
  if ((int)blockIdx.x >= s.blocks) {
    emb_fill(s.fill, blockIdx.x - s.blocks, gridDim.x - s.blocks);
    return;
  }
  __shared__ uint32_t hist[EMB_RADIX];
  for (int d = threadIdx.x; d < EMB_RADIX; d += EMB_THREADS) hist[d] = 0;
  __syncthreads();
  const int lane = threadIdx.x & 63;
  const int64_t first = (int64_t)blockIdx.x * EMB_TILE + (threadIdx.x >> 6) * (64 * EMB_ITEMS);
  uint32_t key[EMB_ITEMS];
  emb_load_items(s, first, key);
  uint32_t lo[EMB_ITEMS], hi[EMB_ITEMS];
  emb_peers(key, first, s.n, s.shift, s.bits, lo, hi);
#pragma unroll
  for (int i = 0; i < EMB_ITEMS; ++i)  // one addition per digit that a wave holds: grouped ids would queue up
    if (first + i * 64 + lane < s.n && __builtin_amdgcn_mbcnt_hi(hi[i], __builtin_amdgcn_mbcnt_lo(lo[i], 0)) == 0)
      atomicAdd(&hist[(key[i] >> s.shift) & ((1u << s.bits) - 1u)], (uint32_t)(__popc(lo[i]) + __popc(hi[i])));
  __syncthreads();
  for (int d = threadIdx.x; d < 1 << s.bits; d += EMB_THREADS) s.table[(int64_t)d * s.blocks + blockIdx.x] = hist[d];
}

// a wave per digit
__global__ __launch_bounds__(EMB_THREADS) void embed_digit_sums_kernel(EmbDigit s) {
  const int own = (1 << s.bits) / (EMB_THREADS / 64) + ((1 << s.bits) % (EMB_THREADS / 64) ? 1 : 0);
  if ((int)blockIdx.x >= own) {
    emb_fill(s.fill, blockIdx.x - own, gridDim.x - own);
    return;
  }
  const int lane = threadIdx.x & 63, d = blockIdx.x * (EMB_THREADS / 64) + (threadIdx.x >> 6);
  if (d >= 1 << s.bits) return;
  constexpr int PER = 8;
  uint32_t* row = s.table + (int64_t)d * s.blocks;
  uint32_t run = 0;
  for (int c0 = 0; c0 < s.blocks; c0 += 64 * PER) {  // PER in succession to a lane: one scan for all of them
    const int c = c0 + lane * PER;
    uint32_t v[PER], sum = 0;
#pragma unroll
    for (int k = 0; k < PER; ++k) v[k] = c + k < s.blocks ? row[c + k] : 0u;
#pragma unroll
    for (int k = 0; k < PER; ++k) sum += v[k];
    uint32_t incl = sum;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      const uint32_t t = __shfl_up(incl, o);
      if (lane >= o) incl += t;
    }
    uint32_t before = run + incl - sum;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
      if (c + k < s.blocks) row[c + k] = before;
      before += v[k];
    }
    run += __shfl(incl, 63);
  }
  if (lane == 0) s.totals[d] = run;
}

__global__ __launch_bounds__(EMB_THREADS) void embed_scatter_kernel(EmbDigit s) {
  if ((int)blockIdx.x >= s.blocks) {
    emb_fill(s.fill, blockIdx.x - s.blocks, gridDim.x - s.blocks);
    return;
  }
  constexpr int WAVES = EMB_THREADS / 64, PER = EMB_RADIX / EMB_THREADS;
  __shared__ uint32_t cnt[WAVES][EMB_RADIX];
  __shared__ uint32_t start[EMB_RADIX];
  __shared__ uint32_t keys[EMB_TILE], poss[EMB_TILE];
  __shared__ uint32_t wsum[WAVES];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, radix = 1 << s.bits;
  const int64_t first = (int64_t)blockIdx.x * EMB_TILE + wave * (64 * EMB_ITEMS);
  for (int d = threadIdx.x; d < WAVES * EMB_RADIX; d += EMB_THREADS) (&cnt[0][0])[d] = 0;
  uint32_t key[EMB_ITEMS], pos[EMB_ITEMS], rank[EMB_ITEMS], t[PER], sum = 0;
  emb_load_items(s, first, key);
#pragma unroll
  for (int i = 0; i < EMB_ITEMS; ++i) {
    const int64_t at = first + i * 64 + lane;
    pos[i] = s.pos && at < s.n ? s.pos[at] : (uint32_t)at;
  }
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int d = threadIdx.x * PER + k;
    t[k] = d < radix ? s.totals[d] : 0u;
    sum += t[k];
  }
  uint32_t run = emb_scan<EMB_THREADS>(sum, wsum);  // (its barriers also stand behind the zeros of cnt)
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    start[threadIdx.x * PER + k] = run;
    run += t[k];
  }
  emb_rank<EMB_ITEMS>(key, first, s.n, s.shift, s.bits, cnt[wave], rank);
  __syncthreads();
  sum = 0;
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    t[k] = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) t[k] += cnt[w][threadIdx.x * PER + k];
    sum += t[k];
  }
  run = emb_scan<EMB_THREADS>(sum, wsum);
#pragma unroll
  for (int k = 0; k < PER; ++k) {
    const int d = threadIdx.x * PER + k;
    if (d < radix) start[d] += s.table[(int64_t)d * s.blocks + blockIdx.x] - run;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
      const uint32_t c = cnt[w][d];
      cnt[w][d] = run;
      run += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < EMB_ITEMS; ++i)
    if (first + i * 64 + lane < s.n) {
      const uint32_t to = cnt[wave][(key[i] >> s.shift) & (uint32_t)(radix - 1)] + rank[i];
      keys[to] = key[i];
      poss[to] = pos[i];
    }
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * EMB_TILE;
  const int n = (int)(s.n - base < EMB_TILE ? s.n - base : EMB_TILE);
#pragma unroll
  for (int i = 0; i < EMB_ITEMS; ++i) {
    const int at = i * EMB_THREADS + threadIdx.x;
    if (at < n) {
      const uint32_t k = keys[at], to = start[(k >> s.shift) & (uint32_t)(radix - 1)] + at;
      s.keys_out[to] = k;
      s.pos_out[to] = poss[at];
    }
  }
}

// ---- sums of the runs
// first index in [lo, hi) with keys >= v
__device__ __forceinline__ int64_t emb_lower(const uint32_t* keys, int64_t lo, int64_t hi, uint32_t v) {
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (keys[mid] < v) lo = mid + 1; else hi = mid;
  }
  return lo;
}

// adds up the groups' sums, in their order, in group 0; lds [N][THREADS]
template <int THREADS, int N>
__device__ __forceinline__ void emb_add_groups(float (&acc)[N], int g, int G, float* __restrict__ lds) {
  for (int half = THREADS / G / 2; half > 0; half /= 2) {
    if (g >= half && g < 2 * half)
#pragma unroll
      for (int k = 0; k < N; ++k) lds[k * THREADS + threadIdx.x] = acc[k];
    __syncthreads();
    if (g < half)
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] += lds[k * THREADS + half * G + threadIdx.x];
    __syncthreads();
  }
}

// A group of G lanes takes the P sorted entries [i0, i1); its workgroup has their keys in LDS, with `longest` more on both
// sides.  partial [pieces][2][D] fp32: what lies in the piece of the long run that started before it (slot 0), and of the
// long run that starts in it (slot 1; there is one at most, and it goes on behind the piece).  A workgroup that has nothing
// but entries of a run that started before it adds up all its pieces, in slot 0 of the first, and has zeros for the others.
// Bound by the latency of
// scattered rows, FLIGHT of them a group: 1M rows of 64 bytes 24 us in 65 runs and 31 us in 200000 (2.7 and 2.5 TB/s),
// 16384 rows of 2 KB 14 us (3.8 TB/s with the stored sums).
template <typename T, int N>
__global__ __launch_bounds__(EMB_THREADS) void embed_runs_kernel(EmbShape sh, const uint32_t* __restrict__ keys,
                                                                 const uint32_t* __restrict__ pos,
                                                                 const T* __restrict__ v_out, float* __restrict__ partial,
                                                                 T* __restrict__ v_table) {
  extern __shared__ uint32_t lds[];
  constexpr int FLIGHT = EMB_FLIGHT_RUNS;
  const int P = sh.piece, M = sh.longest, groups = EMB_THREADS / sh.G, span = groups * P;
  const int64_t w0 = (int64_t)blockIdx.x * span;
  uint32_t* lkey = lds;                     // entries [w0 - M, w0 + span + M]
  uint32_t* lpos = lds + span + 2 * M + 1;  // entries [w0, w0 + span + M)
  for (int l = threadIdx.x; l < span + 2 * M + 1; l += EMB_THREADS) {
    const int64_t e = w0 - M + l;
    lkey[l] = e < 0 ? 0xfffffffeu : e < sh.n ? keys[e] : 0xffffffffu;  // neither is a key
  }
  for (int l = threadIdx.x; l < span + M; l += EMB_THREADS) lpos[l] = w0 + l < sh.n ? pos[w0 + l] : 0u;
  __syncthreads();
  const int g = threadIdx.x / sh.G;
  const int64_t vec = (int64_t)blockIdx.y * sh.G + (threadIdx.x & (sh.G - 1));
  const uint32_t* key = lkey + M + g * P;  // key[0]: the piece's first entry
  const uint32_t* at = lpos + g * P;
  const int64_t i0 = w0 + (int64_t)g * P;
  const uint32_t V = (uint32_t)sh.V, one = lkey[M];
  if (w0 + span <= sh.n && lkey[M - 1] == one && lkey[M + span - 1] == one && one < V) {  // (span >= longest: a long run)
    float acc[N];
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = 0.f;
    if (vec < sh.vpr)
      for (int i = 0; i < P; i += FLIGHT) {
        Raw<T, N> raw[FLIGHT];
#pragma unroll
        for (int u = 0; u < FLIGHT; ++u)
          raw[u] = load_raw<T, N>(v_out + (int64_t)at[i + u < P ? i + u : P - 1] * sh.gs + vec * N);
#pragma unroll
        for (int u = 0; u < FLIGHT; ++u)
          if (i + u < P) {
            float x[N];
            unpack<T, N>(raw[u], x);
#pragma unroll
            for (int k = 0; k < N; ++k) acc[k] += x[k];
          }
      }
    __syncthreads();  // the keys and positions have been read
    emb_add_groups<EMB_THREADS, N>(acc, g, sh.G, (float*)lds);
    if (vec < sh.vpr) {
      float* to = partial + 2 * (i0 / P) * (sh.vpr * N) + vec * N;
#pragma unroll
      for (int k = 0; k < N; ++k) to[k] = g == 0 ? acc[k] : 0.f;
    }
    return;
  }
  if (i0 >= sh.n || vec >= sh.vpr) return;
  const int i1 = sh.n - i0 < P ? (int)(sh.n - i0) : P;

  int a = 0;            // first entry to add
  bool before = false;  // ... which belongs to a long run that started before the piece
  if (key[-1] == key[0]) {
    const uint32_t k = key[0];
    const int s = key[-M] == k ? -M : (int)emb_lower(key, i0 < M ? -i0 : 1 - M, 0, k);
    before = s == -M || key[s + M] == k;
    if (!before) a = (int)emb_lower(key, 0, i1, k + 1);  // a short run: the group where it starts has it
  }
  int b = i1;  // behind the last entry to add
  if (a < i1 && key[i1] == key[i1 - 1]) {
    const uint32_t k = key[i1 - 1];
    const int s = (int)emb_lower(key, a, i1, k);
    if (!(before && s == 0) && key[s + M] != k) b = (int)emb_lower(key, i1, s + M, k + 1);  // a short run that starts here
  }
  const int64_t D = sh.vpr * N, col = vec * N, p = i0 / P;
  float acc[N];
#pragma unroll
  for (int k = 0; k < N; ++k) acc[k] = 0.f;
  int s = a;  // start of the run that is being added
  for (int i = a; i < b; i += FLIGHT) {
    if (key[i] >= V) break;  // nothing but ids that select nothing from here on
    Raw<T, N> raw[FLIGHT];
#pragma unroll
    for (int u = 0; u < FLIGHT; ++u)
      raw[u] = load_raw<T, N>(v_out + (int64_t)at[i + u < b ? i + u : b - 1] * sh.gs + col);
#pragma unroll
    for (int u = 0; u < FLIGHT; ++u) {
      const int e = i + u;
      if (e < b && key[e] < V) {
        float x[N];
        unpack<T, N>(raw[u], x);
#pragma unroll
        for (int k = 0; k < N; ++k) acc[k] += x[k];
        if (e + 1 == b || key[e + 1] != key[e]) {
          if (before || key[s + M] == key[s]) {
            float* to = partial + (2 * p + (before ? 0 : 1)) * D + col;
#pragma unroll
            for (int k = 0; k < N; ++k) to[k] = acc[k];
          } else {
            emb_store<T, N>(v_table + (int64_t)key[e] * D + col, acc, sh.scale);
          }
#pragma unroll
          for (int k = 0; k < N; ++k) acc[k] = 0.f;
          before = false;
          s = e + 1;
        }
      }
    }
  }
}

// Adds the partial sums of the long run of `key` that starts in piece `start`.  A piece is the run's exactly where its first
// entry is.  EMB_JOIN_FLIGHT are read at a time, whether they are or not: asking first would cost a trip to memory for each.
template <int N>
__device__ __forceinline__ void emb_add_pieces(float (&acc)[N], const uint32_t* __restrict__ keys, int pieces, int P,
                                               uint32_t key, int start, const float* __restrict__ partial, int64_t D) {
  bool more = true;
  for (int r = start; more; r += EMB_JOIN_FLIGHT) {
    float x[EMB_JOIN_FLIGHT][N];
    bool in[EMB_JOIN_FLIGHT];
#pragma unroll
    for (int u = 0; u < EMB_JOIN_FLIGHT; ++u) {
      const int c = r + u, d = c < pieces ? c : pieces - 1;
      in[u] = c == start || (c < pieces && keys[d * P] == key);
      const float* src = partial + (2 * d + (c == start ? 1 : 0)) * D;
#pragma unroll
      for (int k = 0; k < N; ++k) x[u][k] = src[k];
    }
#pragma unroll
    for (int u = 0; u < EMB_JOIN_FLIGHT; ++u)
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] += in[u] ? x[u][k] : 0.f;
    more = in[EMB_JOIN_FLIGHT - 1];
  }
}

// A workgroup looks at some pieces for long runs that start in them.  One of its groups takes a run of few pieces; all take
// one of many: its pieces up to the first stretch of `per` pieces that a workgroup of embed_runs_kernel added up, the sums
// of those stretches, and the pieces behind the last; the groups are added up in LDS, in their order.  4 us where there are
// none of 1M ids, 9 us for 65 of 15000, 10 us for one of all of them (120 us by its pieces alone).
template <typename T, int N>
__global__ __launch_bounds__(EMB_JOIN_THREADS) void embed_join_kernel(EmbShape sh, const uint32_t* __restrict__ keys,
                                                                      const float* __restrict__ partial,
                                                                      T* __restrict__ v_table) {
  __shared__ float lds[EMB_JOIN_THREADS * N];
  __shared__ int found[2][EMB_JOIN_PIECES], count[2];  // [longer ones]: pieces in which such a run starts
  __shared__ int behind;  // stretch in which the run ends
  constexpr int FLIGHT = EMB_JOIN_FLIGHT / 2;  // stretches
  const int P = sh.piece;
  const int g = threadIdx.x / sh.G, groups = EMB_JOIN_THREADS / sh.G, few = groups / 2 > 32 ? groups / 2 : 32;
  const int per = EMB_THREADS / sh.G;  // pieces of a workgroup of embed_runs_kernel; `few` are two of them or more
  const int64_t p0 = (int64_t)blockIdx.x * sh.join, pieces = (sh.n + P - 1) / P;
  if (threadIdx.x < 2) count[threadIdx.x] = 0;
  __syncthreads();
  if ((int)threadIdx.x < sh.join) {
    const int64_t p = p0 + threadIdx.x, i0 = p * P, i1 = i0 + P;
    if (i1 < sh.n) {
      const uint32_t k = keys[i1 - 1];
      // it goes on behind the piece, did not start before it, and is a long one
      if (k < (uint32_t)sh.V && keys[i1] == k && !(i0 > 0 && keys[i0 - 1] == k)) {
        const int64_t s = emb_lower(keys, i0, i1, k), far = p + few;
        if (s + sh.longest < sh.n && keys[s + sh.longest] == k) {
          const int longer = far * P < sh.n && keys[far * P] == k ? 1 : 0;
          found[longer][atomicAdd(&count[longer], 1)] = threadIdx.x;  // (in any order: each run is added by itself)
        }
      }
    }
  }
  __syncthreads();
  const int64_t vec = (int64_t)blockIdx.y * sh.G + (threadIdx.x & (sh.G - 1));
  const int64_t D = sh.vpr * N, col = vec * N;
  if (vec < sh.vpr)
    for (int q = g; q < count[0]; q += groups) {
      const int64_t p = p0 + found[0][q];
      const uint32_t key = keys[p * P + P - 1];
      float acc[N];
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] = 0.f;
      emb_add_pieces<N>(acc, keys, (int)pieces, P, key, (int)p, partial + col, D);
      emb_store<T, N>(v_table + (int64_t)key * D + col, acc, sh.scale);
    }
  for (int q = 0; q < count[1]; ++q) {
    const int64_t p = p0 + found[1][q];
    const uint32_t key = keys[p * P + P - 1];
    float acc[N];
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = 0.f;
    auto add = [&](const float* src) {
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] += src[k];
    };
    const int n = (int)sh.n, s0 = (int)p / per + 1;  // first stretch behind the one where it starts
    const float* sums = partial + (vec < sh.vpr ? col : 0);
    if (threadIdx.x == 0) behind = 0x7fffffff;
    __syncthreads();
    if ((int)p + g < s0 * per) add(sums + (2 * (p + g) + (g == 0 ? 1 : 0)) * D);  // (all are the run's)
    bool more = true;
    int end_at = 0x7fffffff;
    for (int r = s0 + g; more; r += FLIGHT * groups) {
      float x[FLIGHT][N];
      bool in[FLIGHT];
#pragma unroll
      for (int u = 0; u < FLIGHT; ++u) {
        const int c = r + u * groups;
        const uint32_t end = (uint32_t)(c + 1) * (per * P);  // (n is below 2^30, what is added to it far below that)
        const bool there = end <= (uint32_t)n;
        in[u] = there && keys[(there ? end : n) - 1] == key;
        const float* src = sums + 2 * (there ? c * per : p) * D;
#pragma unroll
        for (int k = 0; k < N; ++k) x[u][k] = src[k];
      }
#pragma unroll
      for (int u = FLIGHT - 1; u >= 0; --u)
        if (!in[u]) end_at = r + u * groups;
#pragma unroll
      for (int u = 0; u < FLIGHT; ++u)
#pragma unroll
        for (int k = 0; k < N; ++k) acc[k] += in[u] ? x[u][k] : 0.f;
      more = in[FLIGHT - 1];
    }
    for (int o = 1; o < 64; o <<= 1) end_at = min(end_at, __shfl_xor(end_at, o));
    if ((threadIdx.x & 63) == 0) atomicMin(&behind, end_at);
    __syncthreads();
    const int c = behind * per + g;  // the rest of them, in the stretch where the run ends
    if (g < per && c < pieces) {
      const float* src = sums + 2 * (int64_t)c * D;
      float x[N];
#pragma unroll
      for (int k = 0; k < N; ++k) x[k] = src[k];
      const bool in = keys[c * P] == key;
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] += in ? x[k] : 0.f;
    }
    emb_add_groups<EMB_JOIN_THREADS, N>(acc, g, sh.G, lds);
    if (g == 0 && vec < sh.vpr) emb_store<T, N>(v_table + (int64_t)key * D + col, acc, sh.scale);
  }
}

// ---- few rows (V <= EMB_FEW, of D <= 128 columns): no sort.  256 threads read 256 values at a time, several rows, a column
// each, and add them to a table in LDS that belongs to the thread's place among those rows: no two threads meet in a word.
// Equal ids in succession, the rule where Gaussians lie instance by instance, add up in a register first.  The tables of a
// workgroup are added up, in their order, and embed_few_join_kernel adds the workgroups'.
// 1M x 16 fp32 on 64 rows: 23 + 4 us (3.0 TB/s; these tables, 64 KiB a workgroup, leave a CU eight waves), against 55 us by
// the sort; on 8 rows 20 + 4 us.  A thread adds up to n Dp / 131072 values of a row one after another: fp32 as all sums here, but
// with an error that grows with n.
struct EmbFew {
  int64_t n, per, gs;   // ids, ids of a workgroup, row stride of v_out
  int32_t V, D, Dp;     // Dp: D rounded up to a power of two
};

template <typename T>
__global__ __launch_bounds__(EMB_THREADS) void embed_few_kernel(EmbFew sh, const void* __restrict__ ids, int id_bytes,
                                                                const T* __restrict__ v_out, float* __restrict__ partial) {
  extern __shared__ float tables[];  // [256 / Dp][V][Dp]
  constexpr int U = 16;
  const int S = EMB_THREADS / sh.Dp, col = threadIdx.x & (sh.Dp - 1);
  for (int e = threadIdx.x; e < sh.V * EMB_THREADS; e += EMB_THREADS) tables[e] = 0.f;
  __syncthreads();
  if (col < sh.D) {
    float* mine = tables + threadIdx.x / sh.Dp * sh.V * sh.Dp + col;
    const int64_t r0 = blockIdx.x * sh.per, r1 = r0 + sh.per < sh.n ? r0 + sh.per : sh.n;
    int last = -1;  // -1: no row
    float acc = 0.f;
    auto add = [&](int id, float x) {
      if (id != last) {
        if (last >= 0) mine[last * sh.Dp] += acc;
        last = id;
        acc = 0.f;
      }
      acc += x;
    };
    auto row = [&](int64_t q) {
      const int64_t id = emb_id(ids, id_bytes, q);
      return id >= 0 && id < sh.V ? (int)id : -1;
    };
    int64_t r = r0 + threadIdx.x / sh.Dp;
    for (; r + (int64_t)(U - 1) * S < r1; r += (int64_t)U * S) {
      int id[U];
      float x[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        id[u] = row(r + u * S);
        x[u] = (float)v_out[(r + u * S) * sh.gs + col];
      }
#pragma unroll
      for (int u = 0; u < U; ++u) add(id[u], x[u]);
    }
    for (; r < r1; r += S) add(row(r), (float)v_out[r * sh.gs + col]);
    if (last >= 0) mine[last * sh.Dp] += acc;
  }
  __syncthreads();
  const int size = sh.V * sh.Dp;
  for (int e = threadIdx.x; e < size; e += EMB_THREADS) {
    const int to = e & (sh.Dp - 1);
    if (to >= sh.D) continue;
    float sum = tables[e];
    for (int k = 1; k < S; ++k) sum += tables[k * size + e];
    partial[((int64_t)blockIdx.x * sh.V + e / sh.Dp) * sh.D + to] = sum;
  }
}

// 32 words of the table at a time, 32 threads to each
template <typename T>
__global__ __launch_bounds__(1024) void embed_few_join_kernel(int words, int blocks, float scale,
                                                              const float* __restrict__ partial, T* __restrict__ v_table) {
  __shared__ float lds[32][33];
  const int e = blockIdx.x * 32 + (threadIdx.x & 31), slice = threadIdx.x >> 5;
  float acc = 0.f;
  if (e < words) {
#pragma unroll 8
    for (int b = slice; b < blocks; b += 32) acc += partial[(int64_t)b * words + e];
  }
  lds[slice][threadIdx.x & 31] = acc;
  __syncthreads();
  if (slice == 0 && e < words) {
    for (int k = 1; k < 32; ++k) acc += lds[k][threadIdx.x];
    v_table[e] = (T)(acc * scale + 0.f);  // (+0 for a sum of nothing, whatever the sign of the scale)
  }
}

// A row that no id selects is zeros; its sum alone does not tell it from a selected row whose values add up to zero, which
// differs only where 0 * scale is no zero.  With such a scale (infinite or NaN) this follows: a workgroup for each row looks
// for an id of its own.
template <typename T>
__global__ __launch_bounds__(EMB_THREADS) void embed_few_unselected_kernel(EmbFew sh, const void* __restrict__ ids, int id_bytes,
                                                                           T* __restrict__ v_table) {
  bool any = false;
  for (int64_t i = threadIdx.x; i < sh.n && !any; i += EMB_THREADS) any = emb_id(ids, id_bytes, i) == (int64_t)blockIdx.x;
  if (!__syncthreads_or(any ? 1 : 0) && (int)threadIdx.x < sh.D) v_table[(int64_t)blockIdx.x * sh.D + threadIdx.x] = (T)0.f;
}

// Few ids: one launch.  The workgroup lists, in order, the ids that fall among its rows; each group adds those of its row.
// One id on 600 x 48 fp32: 2.9 us; 200 on 65536 x 256: 12 us, 5.6 TB/s of stores.
template <typename T, int N>
__global__ __launch_bounds__(EMB_THREADS) void embed_direct_kernel(EmbShape sh, const void* __restrict__ ids, int id_bytes,
                                                                   const T* __restrict__ v_out, T* __restrict__ v_table) {
  static_assert(EMB_DIRECT <= EMB_THREADS, "a thread looks at one id");
  __shared__ int hit_row[EMB_DIRECT], row_of[EMB_DIRECT];
  __shared__ uint32_t hit_pos[EMB_DIRECT];
  __shared__ int wave_hits[EMB_THREADS / 64];
  __shared__ int start[EMB_ROWS_MAX + 1];
  const int64_t v0 = (int64_t)blockIdx.x * sh.rows_per;
  const int rows = (int)(sh.V - v0 < sh.rows_per ? sh.V - v0 : sh.rows_per);
  const int64_t id = (int64_t)threadIdx.x < sh.n ? emb_id(ids, id_bytes, threadIdx.x) : -1;
  const bool mine = id >= v0 && id < v0 + rows;
  const unsigned long long ballot = __ballot(mine);
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  if (lane == 0) wave_hits[wave] = __popcll(ballot);
  __syncthreads();
  int at = 0, hits = 0;
#pragma unroll
  for (int w = 0; w < EMB_THREADS / 64; ++w) {
    if (w < wave) at += wave_hits[w];
    hits += wave_hits[w];
  }
  const int g = threadIdx.x / sh.G, groups = EMB_THREADS / sh.G;
  const int64_t vec = (int64_t)blockIdx.y * sh.G + (threadIdx.x & (sh.G - 1));
  float acc[N];
  if (hits > 0) {  // sorted by row, ids of a row in their order: each ranks itself
    at += __popcll(ballot & ((1ull << lane) - 1ull));
    if (mine) hit_row[at] = (int)(id - v0);
    __syncthreads();
    if (mine) {
      const int r = (int)(id - v0);
      int rank = 0;
      for (int h = 0; h < hits; ++h) rank += hit_row[h] < r || (hit_row[h] == r && h < at);
      row_of[rank] = r;
      hit_pos[rank] = threadIdx.x;
    }
    __syncthreads();
    for (int r = threadIdx.x; r <= rows; r += EMB_THREADS) {
      int lo = 0, hi = hits;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (row_of[mid] < r) lo = mid + 1; else hi = mid;
      }
      start[r] = lo;
    }
    __syncthreads();
  }
  if (vec >= sh.vpr) return;
  for (int r = g; r < rows; r += groups) {
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = 0.f;
    const int s = hits > 0 ? start[r] : 0, e = hits > 0 ? start[r + 1] : 0;
    for (int h = s; h < e; h += 8) {
      float x[8][N];
#pragma unroll
      for (int u = 0; u < 8; ++u) load_vec<T, N>(v_out + (int64_t)hit_pos[h + u < e ? h + u : e - 1] * sh.gs + vec * N, x[u]);
#pragma unroll
      for (int u = 0; u < 8; ++u)
        if (h + u < e)
#pragma unroll
          for (int k = 0; k < N; ++k) acc[k] += x[u][k];
    }
    emb_store<T, N, false>(v_table + (v0 + r) * sh.vpr * N + vec * N, acc, s < e ? sh.scale : 0.f);  // (0 * scale may be NaN)
  }
}

// the widest vector, in elements, that a row of D elements and the given strides and addresses allow
static int emb_vec(int64_t D, int size, int64_t stride, const void* a, const void* b) {
  for (int bytes = 16; bytes > size; bytes >>= 1)
    if (D * size % bytes == 0 && stride * size % bytes == 0 && (((uintptr_t)a | (uintptr_t)b) & (uintptr_t)(bytes - 1)) == 0)
      return bytes / size;
  return 1;
}

template <typename F> static int with_vec(int size, int N, F&& f) {
  if (N == 1) return f(std::integral_constant<int, 1>{});
  if (N == 2) return f(std::integral_constant<int, 2>{});
  if (N == 4) return f(std::integral_constant<int, 4>{});
  return size == 2 ? f(std::integral_constant<int, 8>{}) : GS_ERR_INVALID_ARG;
}

static int emb_bits(int64_t V) {
  int b = 1;
  while (b < 63 && ((int64_t)1 << b) <= V) ++b;  // holds the key V too
  return b;
}

static int64_t emb_round(int64_t bytes) { return (bytes + 255) / 256 * 256; }

// Tables beyond the Infinity Cache are better zeroed in one sweep: 64 ids on 131072 x 512 fp32 take 37 us directly and 41 us
// sorted, on 131072 x 1024 141 and 116 us.
static bool emb_direct(int64_t n, int64_t V, int64_t D) { return n <= EMB_DIRECT && V * D <= (int64_t)1 << 26; }

struct EmbWorkspace {
  int64_t keys, pos, keys_b, pos_b, table, totals, partial, total;
};

// enough groups to fill the card first, then longer pieces: fewer partial sums of long runs (embed_runs_kernel with pieces of
// 4 and of 16: 16384 ids on 5000 x 16 fp32 8.2 and 13.8 us, 1000 ids 5.7 and 9.8 us)
static int emb_piece(int64_t n, int64_t D) {
  return n * D < ((int64_t)1 << 20) ? 4 : n * D < ((int64_t)1 << 26) ? 16 : EMB_PIECE_MAX;
}

// Runs that one group adds up by itself: longer ones keep it busy while the others wait (16 or 64 as the longest: 16384 ids
// of a skewed choice of 5000 x 64 fp32 43 and 49 us, 1M of 200000 x 16 120 and 124; 1M spread over 50000 x 16 80 and 77).
// No fewer than a piece, no more than what a workgroup of embed_runs_kernel has at once.
static int emb_longest(int64_t n, int64_t D) { return std::max(16, emb_piece(n, D)); }

// The form for few rows is taken where a workgroup reads two rows or more at a time: gradients alone, by it and by the sort,
// 1M ids on 64 x 16 fp32 32 and 59 us, 38358 on 6 x 36 10 and 28, 20000 on 64 x 64 17 and 31, 300 on 64 x 64 16 and 13; but
// 100000 on 64 x 256 55 and 46, on 64 x 1024 143 and 72.
static bool emb_few(int64_t V, int64_t D) { return V <= EMB_FEW && D <= EMB_THREADS / 2; }

// Its workgroups: two on each CU, each with twice as many ids as the table has rows or more, so that writing and adding up
// their tables costs no more than reading the rows.
static int64_t emb_few_blocks(int64_t n, int64_t V) { return std::max<int64_t>(1, std::min<int64_t>(512, n / (2 * V))); }

static EmbWorkspace emb_workspace(int64_t n, int64_t V, int64_t D) {
  EmbWorkspace w = {};
  if (V == 0 || D == 0 || emb_direct(n, V, D)) return w;  // (a table without rows or columns: nothing is launched)
  if (emb_few(V, D)) {
    w.total = 4 * V * D * emb_few_blocks(n, V);
    return w;
  }
  const int64_t list = emb_round(4 * n), blocks = ceil_div(n, EMB_TILE);
  w.pos = w.keys + list;
  w.keys_b = w.pos + list;
  w.pos_b = w.keys_b + list;
  w.table = w.pos_b + list;
  w.totals = w.table + emb_round(4 * EMB_RADIX * blocks);
  w.partial = w.totals + emb_round(4 * EMB_RADIX);
  w.total = w.partial + 8 * D * ceil_div(n, emb_piece(n, D));
  return w;
}

// workgroups that fill one share of the table: four vectors a thread, more in a large one
static unsigned emb_fill_blocks(const EmbFill& f, int threads) {
  const int64_t b = ceil_div(f.bytes / f.shares, (int64_t)threads * 64);
  return (unsigned)std::min<int64_t>(std::max<int64_t>(b, 1), 4096);
}

// sorts the ids and zeroes the table; `w` says which of the two pairs of lists has the result
static int emb_sort(int64_t n, int64_t V, const void* ids, int32_t id_bytes, char* ws, const EmbWorkspace& w, void* v_table,
                    int64_t table_bytes, const uint32_t** keys, const uint32_t** pos, hipStream_t s) {
  const int bits = emb_bits(V);
  EmbFill fill{(char*)v_table, table_bytes, 0, 1, n >= V / 8 ? 1 : 0};
  uint32_t *ka = (uint32_t*)(ws + w.keys), *pa = (uint32_t*)(ws + w.pos);
  uint32_t *kb = (uint32_t*)(ws + w.keys_b), *pb = (uint32_t*)(ws + w.pos_b);
  if (n <= EMB_SORT1) {
    const dim3 grid(1 + emb_fill_blocks(fill, EMB_SORT1_THREADS)), block(EMB_SORT1_THREADS);
    if (n <= 4 * EMB_SORT1_THREADS)
      hipLaunchKernelGGL(embed_sort1_kernel<4>, grid, block, 0, s, (int)n, V, bits, ids, id_bytes, ka, pa, fill);
    else if (n <= 8 * EMB_SORT1_THREADS)
      hipLaunchKernelGGL(embed_sort1_kernel<8>, grid, block, 0, s, (int)n, V, bits, ids, id_bytes, ka, pa, fill);
    else
      hipLaunchKernelGGL(embed_sort1_kernel<16>, grid, block, 0, s, (int)n, V, bits, ids, id_bytes, ka, pa, fill);
    GS_CHECK_LAUNCH();
    *keys = ka;
    *pos = pa;
    return GS_OK;
  }
  const int passes = (bits + EMB_RADIX_BITS - 1) / EMB_RADIX_BITS, per = (bits + passes - 1) / passes;
  EmbDigit d{};
  d.n = n; d.V = V; d.ids = ids; d.id_bytes = id_bytes;
  d.blocks = (int32_t)ceil_div(n, EMB_TILE);
  d.table = (uint32_t*)(ws + w.table);
  d.totals = (uint32_t*)(ws + w.totals);
  fill.shares = 3 * passes;
  const unsigned more = emb_fill_blocks(fill, EMB_THREADS);
  const dim3 block(EMB_THREADS);
  for (int p = 0; p < passes; ++p) {
    d.shift = p * per;
    d.bits = std::min(per, bits - d.shift);
    d.keys = p ? (p & 1 ? ka : kb) : nullptr;
    d.pos = p ? (p & 1 ? pa : pb) : nullptr;
    d.keys_out = p & 1 ? kb : ka;
    d.pos_out = p & 1 ? pb : pa;
    d.fill = fill;
    d.fill.share = 3 * p;
    hipLaunchKernelGGL(embed_hist_kernel, dim3(d.blocks + more), block, 0, s, d);
    d.fill.share = 3 * p + 1;
    hipLaunchKernelGGL(embed_digit_sums_kernel, dim3((unsigned)ceil_div(1 << d.bits, EMB_THREADS / 64) + more), block, 0, s, d);
    d.fill.share = 3 * p + 2;
    hipLaunchKernelGGL(embed_scatter_kernel, dim3(d.blocks + more), block, 0, s, d);
    GS_CHECK_LAUNCH();
  }
  *keys = d.keys_out;
  *pos = d.pos_out;
  return GS_OK;
}

}  // namespace gs

extern "C" int gs_embedding_fwd(int64_t n, int64_t V, int64_t D, int32_t dtype, const void* table, int64_t table_stride,
                                const void* ids, int32_t id_bytes, float scale, void* out, void* stream) {
  using namespace gs;
  const int size = dtype_size(dtype);
  if (n < 0 || V < 0 || D < 0 || !size || (id_bytes != 4 && id_bytes != 8) || table_stride < 0) return GS_ERR_INVALID_ARG;
  if (n == 0 || D == 0) return GS_OK;
  if (!ids || !out || (V > 0 && !table)) return GS_ERR_INVALID_ARG;
  if (((uintptr_t)table | (uintptr_t)out) & (uintptr_t)(size - 1)) return GS_ERR_INVALID_ARG;
  if ((uintptr_t)ids & (uintptr_t)(id_bytes - 1)) return GS_ERR_INVALID_ARG;
  const int N = emb_vec(D, size, table_stride, table, out);
  const int64_t vpr = D / N;
  const int rows_per = vpr >= 2048 ? 1 : (int)(2048 / vpr);
  const uint32_t magic = vpr > 1 && rows_per > 1 ? (uint32_t)(((uint64_t)1 << 32) / (uint64_t)vpr + 1) : 0;
  const int64_t blocks = ceil_div(n, rows_per);
  const dim3 grid((unsigned)(blocks < (1 << 20) ? blocks : (1 << 20)));
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    return with_vec(size, N, [&](auto nv) {
      constexpr int NV = decltype(nv)::value;
      if constexpr (NV * (int)sizeof(T) <= 16) {
        hipLaunchKernelGGL((embed_lookup_kernel<T, NV>), grid, dim3(EMB_THREADS), 0, (hipStream_t)stream, n, V, vpr, rows_per,
                           magic, (const T*)table, table_stride, ids, id_bytes, scale, (T*)out);
        GS_CHECK_LAUNCH();
        return GS_OK;
      }
      return GS_ERR_INVALID_ARG;
    });
  });
}

extern "C" int64_t gs_embedding_bwd_workspace_bytes(int64_t n, int64_t V, int64_t D) {
  if (n < 0 || V < 0 || D < 0) return 0;
  return gs::emb_workspace(n, V, D).total;
}

extern "C" int gs_embedding_bwd(int64_t n, int64_t V, int64_t D, int32_t dtype, const void* ids, int32_t id_bytes,
                                const void* v_out, int64_t v_out_stride, float scale, void* workspace,
                                int64_t workspace_bytes, void* v_table, void* stream) {
  using namespace gs;
  const int size = dtype_size(dtype);
  if (n < 0 || V < 0 || D < 0 || !size || (id_bytes != 4 && id_bytes != 8) || v_out_stride < 0) return GS_ERR_INVALID_ARG;
  if (V == 0 || D == 0) return GS_OK;
  if (n >= ((int64_t)1 << 30) || V >= ((int64_t)1 << 31)) return GS_ERR_UNSUPPORTED;  // 2^32 threads of a launch
  if (!v_table || (n > 0 && (!ids || !v_out))) return GS_ERR_INVALID_ARG;
  if (((uintptr_t)v_out | (uintptr_t)v_table) & (uintptr_t)(size - 1)) return GS_ERR_INVALID_ARG;
  if ((uintptr_t)ids & (uintptr_t)(id_bytes - 1)) return GS_ERR_INVALID_ARG;
  const EmbWorkspace w = emb_workspace(n, V, D);
  if (w.total > 0 && (!workspace || ((uintptr_t)workspace & 15))) return GS_ERR_INVALID_ARG;
  if (workspace_bytes < w.total) return GS_ERR_WORKSPACE;
  hipStream_t s = (hipStream_t)stream;
  const int N = !emb_direct(n, V, D) && emb_few(V, D) ? 1 : emb_vec(D, size, v_out_stride, v_out, v_table);
  EmbShape sh;
  sh.n = n; sh.V = V; sh.vpr = D / N; sh.gs = v_out_stride; sh.scale = scale;
  sh.G = 1;
  while (sh.G < 64 && sh.G < sh.vpr) sh.G <<= 1;
  const int64_t tiles = ceil_div(sh.vpr, sh.G);
  if (tiles > 65535) return GS_ERR_UNSUPPORTED;  // rows above 4M vectors
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    return with_vec(size, N, [&](auto nv) {
      constexpr int NV = decltype(nv)::value;
      if constexpr (NV * (int)sizeof(T) <= 16) {
        if (emb_direct(n, V, D)) {
          // enough workgroups for 256 CUs first, then more rows each
          const int64_t per = std::max<int64_t>(ceil_div(V * tiles, 2048), EMB_THREADS / sh.G);
          sh.rows_per = (int)std::min<int64_t>(per, EMB_ROWS_MAX);
          hipLaunchKernelGGL((embed_direct_kernel<T, NV>), dim3((unsigned)ceil_div(V, sh.rows_per), (unsigned)tiles),
                             dim3(EMB_THREADS), 0, s, sh, ids, id_bytes, (const T*)v_out, (T*)v_table);
          GS_CHECK_LAUNCH();
          return GS_OK;
        }
        if (emb_few(V, D)) {
          if constexpr (NV == 1) {
            EmbFew few{n, 0, v_out_stride, (int32_t)V, (int32_t)D, 1};
            while (few.Dp < D) few.Dp <<= 1;
            const int64_t blocks = emb_few_blocks(n, V);
            few.per = ceil_div(n, blocks);
            hipLaunchKernelGGL(embed_few_kernel<T>, dim3((unsigned)blocks), dim3(EMB_THREADS),
                               V * EMB_THREADS * sizeof(float), s, few, ids, id_bytes, (const T*)v_out, (float*)workspace);
            GS_CHECK_LAUNCH();
            const int words = (int)(V * D);
            hipLaunchKernelGGL(embed_few_join_kernel<T>, dim3((unsigned)ceil_div(words, 32)), dim3(1024), 0, s, words,
                               (int)blocks, scale, (const float*)workspace, (T*)v_table);
            GS_CHECK_LAUNCH();
            if (!std::isfinite(scale)) {
              hipLaunchKernelGGL(embed_few_unselected_kernel<T>, dim3((unsigned)V), dim3(EMB_THREADS), 0, s, few, ids, id_bytes,
                                 (T*)v_table);
              GS_CHECK_LAUNCH();
            }
            return GS_OK;
          }
          return GS_ERR_INVALID_ARG;
        }
        const uint32_t *keys, *pos;
        const int st = emb_sort(n, V, ids, id_bytes, (char*)workspace, w, v_table, V * D * size, &keys, &pos, s);
        if (st != GS_OK || n == 0) return st;  // (of no ids the zeros are all)
        sh.G = std::max(sh.G, 4);  // (keeps a workgroup's share of the sorted ids within 32 KiB of LDS)
        sh.piece = emb_piece(n, D);
        sh.longest = emb_longest(n, D);
        float* partial = (float*)((char*)workspace + w.partial);
        const int64_t pieces = ceil_div(n, sh.piece);
        sh.join = (int)std::min<int64_t>(std::max<int64_t>(pieces / 256, 16), EMB_JOIN_PIECES);
        const int span = EMB_THREADS / sh.G * sh.piece;
        hipLaunchKernelGGL((embed_runs_kernel<T, NV>), dim3((unsigned)ceil_div(n, span), (unsigned)tiles), dim3(EMB_THREADS),
                           std::max(2 * span + 3 * sh.longest + 1, EMB_THREADS * NV) * sizeof(uint32_t), s, sh, keys, pos,
                           (const T*)v_out, partial, (T*)v_table);
        GS_CHECK_LAUNCH();
        hipLaunchKernelGGL((embed_join_kernel<T, NV>), dim3((unsigned)ceil_div(pieces, sh.join), (unsigned)tiles),
                           dim3(EMB_JOIN_THREADS), 0, s, sh, keys, partial, (T*)v_table);
        GS_CHECK_LAUNCH();
        return GS_OK;
      }
      return GS_ERR_INVALID_ARG;
    });
  });
}
