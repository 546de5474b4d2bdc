// Embedding lookup with scaling, and the gradient of the table by sorted ids.
//   out[i] = scale * table[ids[i]]                          (an id outside [0, V) selects nothing: a row of zeros)
//   v_table[v] = scale * sum over i with ids[i] = v, in ascending i, of v_out[i]
// Both are bound by HBM.  The lookup reads n rows and writes n rows in the widest vectors that the row size and the
// alignment allow.  The gradient reads every row of v_out once and writes every row of the table once:
//   ids -> (id, position) pairs, stably sorted by id (gs_radix_sort_pairs_u64_u32_bits);
//   embed_rows_kernel   owns rows of the table: finds each row's run in the sorted ids, adds its rows of v_out (or
//                       writes zeros), leaves out the runs longer than EMB_LONG;
//   embed_pieces_kernel cuts the sorted ids into pieces of EMB_LONG and adds up what of a long run lies in each;
//   embed_join_kernel   adds the pieces of each long run.
// Sums are held in fp32, taken in an order that the ids alone fix (no float atomics), and rounded once at the end.
// Up to EMB_DIRECT ids need no sort: each workgroup picks the ids that fall among its rows of the table.
#include "dtype_io.hpp"

namespace gs {

constexpr int EMB_THREADS = 256;
constexpr int EMB_LONG = 64;
constexpr int EMB_DIRECT = 256;
constexpr int EMB_ROWS_MAX = 256;  // rows of the table per workgroup

__device__ __forceinline__ int64_t emb_id(const void* ids, int id_bytes, int64_t i) {
  return id_bytes == 8 ? ((const int64_t*)ids)[i] : (int64_t)((const int32_t*)ids)[i];
}

// ---------------------------------------------------------------------------------------------------------- lookup
// vpr vectors of N elements per row; a workgroup takes `rows_per` rows at a time, their vectors numbered through.
// f / vpr by a multiplication: exact while f * vpr < 2^32 (the host keeps rows_per * vpr at 4096, or rows_per at 1).
template <typename T, int N>
__global__ __launch_bounds__(EMB_THREADS) void embed_lookup_kernel(int64_t n, int64_t V, int64_t vpr, int rows_per,
                                                                   uint32_t magic, const T* __restrict__ table,
                                                                   int64_t ts, const void* __restrict__ ids, int id_bytes,
                                                                   float scale, T* __restrict__ out) {
  for (int64_t r0 = (int64_t)blockIdx.x * rows_per; r0 < n; r0 += (int64_t)gridDim.x * rows_per) {
    const int64_t rows = n - r0 < rows_per ? n - r0 : rows_per;
    const int64_t total = rows * vpr;
    for (int64_t f = threadIdx.x; f < total; f += EMB_THREADS) {
      int64_t r, c;
      if (rows_per == 1) {
        r = 0; c = f;
      } else {
        r = vpr == 1 ? f : (int64_t)__umulhi((uint32_t)f, magic);
        c = f - r * vpr;
      }
      const int64_t id = emb_id(ids, id_bytes, r0 + r);
      float x[N];
      if (id >= 0 && id < V) {
        load_vec<T, N>(table + id * ts + c * N, x);
#pragma unroll
        for (int k = 0; k < N; ++k) x[k] *= scale;
      } else {
#pragma unroll
        for (int k = 0; k < N; ++k) x[k] = 0.f;
      }
      store_vec<T, N>(out + ((r0 + r) * vpr + c) * N, x);
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
  float scale;
};

template <typename T, int N>
__device__ __forceinline__ void emb_add(float (&acc)[N], const T* __restrict__ v_out, int64_t gs, int64_t pos, int64_t col) {
  float x[N];
  load_vec<T, N>(v_out + pos * gs + col, x);
#pragma unroll
  for (int k = 0; k < N; ++k) acc[k] += x[k];
}

// sum of v_out over the sorted entries [s, e), in order, four rows in flight
template <typename T, int N>
__device__ __forceinline__ void emb_sum(float (&acc)[N], const uint32_t* __restrict__ pos, int64_t s, int64_t e,
                                        const T* __restrict__ v_out, int64_t gs, int64_t col) {
  int64_t i = s;
  for (; i + 4 <= e; i += 4) {
    float x[4][N];
#pragma unroll
    for (int u = 0; u < 4; ++u) load_vec<T, N>(v_out + (int64_t)pos[i + u] * gs + col, x[u]);
#pragma unroll
    for (int u = 0; u < 4; ++u)
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] += x[u][k];
  }
  for (; i < e; ++i) emb_add<T, N>(acc, v_out, gs, (int64_t)pos[i], col);
}

template <typename T, int N>
__device__ __forceinline__ void emb_store(T* __restrict__ p, const float (&acc)[N], float scale) {
  float x[N];
#pragma unroll
  for (int k = 0; k < N; ++k) x[k] = acc[k] * scale;
  store_vec<T, N>(p, x);
}

__global__ __launch_bounds__(EMB_THREADS) void embed_keys_kernel(int64_t n, int64_t V, const void* __restrict__ ids,
                                                                 int id_bytes, uint64_t* __restrict__ keys,
                                                                 uint32_t* __restrict__ pos) {
  const int64_t i = (int64_t)blockIdx.x * EMB_THREADS + threadIdx.x;
  if (i >= n) return;
  const int64_t id = emb_id(ids, id_bytes, i);
  keys[i] = id >= 0 && id < V ? (uint64_t)id : (uint64_t)V;  // ids that select nothing sort behind all rows
  pos[i] = (uint32_t)i;
}

// first index in [lo, hi) with keys >= v
__device__ __forceinline__ int64_t emb_lower(const uint64_t* __restrict__ keys, int64_t lo, int64_t hi, uint64_t v) {
  while (lo < hi) {
    const int64_t mid = (lo + hi) >> 1;
    if (keys[mid] < v) lo = mid + 1; else hi = mid;
  }
  return lo;
}

template <typename T, int N>
__global__ __launch_bounds__(EMB_THREADS) void embed_rows_kernel(EmbShape sh, const uint64_t* __restrict__ keys,
                                                                 const uint32_t* __restrict__ pos,
                                                                 const T* __restrict__ v_out, T* __restrict__ v_table) {
  __shared__ int64_t start[EMB_ROWS_MAX + 1];
  const int64_t v0 = (int64_t)blockIdx.x * sh.rows_per;
  const int rows = (int)(sh.V - v0 < sh.rows_per ? sh.V - v0 : sh.rows_per);
  for (int r = threadIdx.x; r <= rows; r += EMB_THREADS) start[r] = emb_lower(keys, 0, sh.n, (uint64_t)(v0 + r));
  __syncthreads();
  const int g = threadIdx.x / sh.G, groups = EMB_THREADS / sh.G;
  const int64_t vec = (int64_t)blockIdx.y * sh.G + (threadIdx.x & (sh.G - 1));
  if (vec >= sh.vpr) return;
  for (int r = g; r < rows; r += groups) {
    const int64_t s = start[r], e = start[r + 1];
    if (e - s > EMB_LONG) continue;
    float acc[N];
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = 0.f;
    emb_sum<T, N>(acc, pos, s, e, v_out, sh.gs, vec * N);
    emb_store<T, N>(v_table + (v0 + r) * sh.vpr * N + vec * N, acc, sh.scale);
  }
}

// The run of the key at `i`, known to start within EMB_LONG before it or to be long: true if it has more than EMB_LONG
// entries.  `s` gets its start where that lies in (i - EMB_LONG, i].
__device__ __forceinline__ bool emb_long(const uint64_t* __restrict__ keys, int64_t n, int64_t i, int64_t& s) {
  const uint64_t k = keys[i];
  if (i >= EMB_LONG && keys[i - EMB_LONG] == k) { s = -1; return true; }
  s = emb_lower(keys, i >= EMB_LONG ? i - EMB_LONG + 1 : 0, i, k);
  return s + EMB_LONG < n && keys[s + EMB_LONG] == k;
}

// partial [pieces][2][D] fp32: what of the long run that holds the piece's first entry (slot 0), and of the one that
// holds its last entry where that is another (slot 1), lies in the piece
template <typename T, int N>
__global__ __launch_bounds__(EMB_THREADS) void embed_pieces_kernel(EmbShape sh, const uint64_t* __restrict__ keys,
                                                                   const uint32_t* __restrict__ pos,
                                                                   const T* __restrict__ v_out, float* __restrict__ partial) {
  const int64_t p = (int64_t)blockIdx.x * (EMB_THREADS / sh.G) + threadIdx.x / sh.G;
  const int64_t i0 = p * EMB_LONG;
  const int64_t vec = (int64_t)blockIdx.y * sh.G + (threadIdx.x & (sh.G - 1));
  if (i0 >= sh.n || vec >= sh.vpr) return;
  const int64_t i1 = i0 + EMB_LONG < sh.n ? i0 + EMB_LONG : sh.n;
  const int64_t D = sh.vpr * N;
  const uint64_t k0 = keys[i0], k1 = keys[i1 - 1];
  int64_t s;
  if (k0 < (uint64_t)sh.V && emb_long(keys, sh.n, i0, s)) {
    const int64_t e = k1 == k0 ? i1 : emb_lower(keys, i0, i1, k0 + 1);
    float acc[N];
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = 0.f;
    emb_sum<T, N>(acc, pos, i0, e, v_out, sh.gs, vec * N);
    float* dst = partial + (2 * p) * D + vec * N;
#pragma unroll
    for (int k = 0; k < N; ++k) dst[k] = acc[k];
  }
  if (k1 != k0 && k1 < (uint64_t)sh.V && emb_long(keys, sh.n, i1 - 1, s)) {  // starts inside the piece: s is its start
    float acc[N];
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = 0.f;
    emb_sum<T, N>(acc, pos, s, i1, v_out, sh.gs, vec * N);
    float* dst = partial + (2 * p + 1) * D + vec * N;
#pragma unroll
    for (int k = 0; k < N; ++k) dst[k] = acc[k];
  }
}

// One workgroup per piece and column tile: the one in whose piece a long run starts adds the run's pieces, the groups of
// the workgroup in turn, and joins the groups in LDS.
template <typename T, int N>
__global__ __launch_bounds__(EMB_THREADS) void embed_join_kernel(EmbShape sh, const uint64_t* __restrict__ keys,
                                                                 const float* __restrict__ partial, T* __restrict__ v_table) {
  const int64_t p = blockIdx.x;
  const int64_t i0 = p * EMB_LONG;
  const int64_t i1 = i0 + EMB_LONG < sh.n ? i0 + EMB_LONG : sh.n;
  const uint64_t key = keys[i1 - 1];
  if (key >= (uint64_t)sh.V || i1 >= sh.n || keys[i1] != key) return;  // a long run that starts here goes on behind the piece
  if (i0 > 0 && keys[i0 - 1] == key) return;                           // started before
  const int64_t s = emb_lower(keys, i0, i1, key);
  if (s + EMB_LONG >= sh.n || keys[s + EMB_LONG] != key) return;
  const int64_t e = emb_lower(keys, s + EMB_LONG, sh.n, key + 1);
  const int64_t last = (e - 1) / EMB_LONG;  // the piece of its last entry
  const int g = threadIdx.x / sh.G, groups = EMB_THREADS / sh.G;
  const int64_t vec = (int64_t)blockIdx.y * sh.G + (threadIdx.x & (sh.G - 1));
  const int64_t D = sh.vpr * N;
  float acc[N];
#pragma unroll
  for (int k = 0; k < N; ++k) acc[k] = 0.f;
  if (vec < sh.vpr) {
    for (int64_t q = p + g; q <= last; q += groups) {
      const float* src = partial + (2 * q + (q == p && s != i0 ? 1 : 0)) * D + vec * N;
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] += src[k];
    }
  }
  __shared__ float lds[EMB_THREADS * N];
#pragma unroll
  for (int k = 0; k < N; ++k) lds[threadIdx.x * N + k] = acc[k];
  __syncthreads();
  if (g != 0 || vec >= sh.vpr) return;
  for (int h = 1; h < groups; ++h)
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] += lds[(h * sh.G + threadIdx.x) * N + k];
  emb_store<T, N>(v_table + (int64_t)key * D + vec * N, acc, sh.scale);
}

// Few ids: one launch.  The workgroup lists, in order, the ids that fall among its rows; each group adds those of its row.
template <typename T, int N>
__global__ __launch_bounds__(EMB_THREADS) void embed_direct_kernel(EmbShape sh, const void* __restrict__ ids, int id_bytes,
                                                                   const T* __restrict__ v_out, T* __restrict__ v_table) {
  static_assert(EMB_DIRECT <= EMB_THREADS, "a thread looks at one id");
  __shared__ int hit_row[EMB_DIRECT];
  __shared__ uint32_t hit_pos[EMB_DIRECT];
  __shared__ int wave_hits[EMB_THREADS / 64];
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
  if (mine) {
    at += __popcll(ballot & ((1ull << lane) - 1ull));
    hit_row[at] = (int)(id - v0);
    hit_pos[at] = threadIdx.x;
  }
  __syncthreads();
  const int g = threadIdx.x / sh.G, groups = EMB_THREADS / sh.G;
  const int64_t vec = (int64_t)blockIdx.y * sh.G + (threadIdx.x & (sh.G - 1));
  if (vec >= sh.vpr) return;
  for (int r = g; r < rows; r += groups) {
    float acc[N];
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = 0.f;
    for (int h = 0; h < hits; ++h)
      if (hit_row[h] == r) emb_add<T, N>(acc, v_out, sh.gs, (int64_t)hit_pos[h], vec * N);
    emb_store<T, N>(v_table + (v0 + r) * sh.vpr * N + vec * N, acc, sh.scale);
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

struct EmbWorkspace {
  int64_t keys, pos, keys_b, pos_b, sort, sort_bytes, partial, total;
};

static EmbWorkspace emb_workspace(int64_t n, int64_t V, int64_t D) {
  EmbWorkspace w = {};
  if (n <= EMB_DIRECT) return w;
  w.keys = 0;
  w.pos = w.keys + emb_round(8 * n);
  w.keys_b = w.pos + emb_round(4 * n);
  w.pos_b = w.keys_b + emb_round(8 * n);
  w.sort = w.pos_b + emb_round(4 * n);
  w.sort_bytes = gs_radix_sort_workspace_bytes(n);
  w.partial = w.sort + emb_round(w.sort_bytes);
  w.total = w.partial + 8 * D * ceil_div(n, EMB_LONG);
  return w;
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
  const int N = emb_vec(D, size, v_out_stride, v_out, v_table);
  EmbShape sh;
  sh.n = n; sh.V = V; sh.vpr = D / N; sh.gs = v_out_stride; sh.scale = scale;
  sh.G = 1;
  while (sh.G < 64 && sh.G < sh.vpr) sh.G <<= 1;
  const int64_t tiles = ceil_div(sh.vpr, sh.G);
  if (tiles > 65535) return GS_ERR_UNSUPPORTED;  // rows above 4M vectors
  // enough workgroups for 256 CUs first, then more rows each
  const int groups = EMB_THREADS / sh.G;
  int64_t per = ceil_div(V * tiles, 2048);
  per = per < groups ? groups : per;
  sh.rows_per = (int)(per < EMB_ROWS_MAX ? per : EMB_ROWS_MAX);
  const int64_t row_blocks = ceil_div(V, sh.rows_per);
  const dim3 row_grid((unsigned)row_blocks, (unsigned)tiles);
  return with_dtype(dtype, [&](auto t) {
    using T = decltype(t);
    return with_vec(size, N, [&](auto nv) {
      constexpr int NV = decltype(nv)::value;
      if constexpr (NV * (int)sizeof(T) <= 16) {
        if (n <= EMB_DIRECT) {
          hipLaunchKernelGGL((embed_direct_kernel<T, NV>), row_grid, dim3(EMB_THREADS), 0, s, sh, ids, id_bytes,
                             (const T*)v_out, (T*)v_table);
          GS_CHECK_LAUNCH();
          return GS_OK;
        }
        char* b = (char*)workspace;
        uint64_t* keys = (uint64_t*)(b + w.keys);
        uint32_t* pos = (uint32_t*)(b + w.pos);
        hipLaunchKernelGGL(embed_keys_kernel, dim3((unsigned)ceil_div(n, EMB_THREADS)), dim3(EMB_THREADS), 0, s, n, V, ids,
                           id_bytes, keys, pos);
        GS_CHECK_LAUNCH();
        int32_t in_b = 0;
        const int st = gs_radix_sort_pairs_u64_u32_bits(n, 0, emb_bits(V), keys, pos, (uint64_t*)(b + w.keys_b),
                                                        (uint32_t*)(b + w.pos_b), b + w.sort, w.sort_bytes, &in_b, stream);
        if (st != GS_OK) return st;
        if (in_b) { keys = (uint64_t*)(b + w.keys_b); pos = (uint32_t*)(b + w.pos_b); }
        hipLaunchKernelGGL((embed_rows_kernel<T, NV>), row_grid, dim3(EMB_THREADS), 0, s, sh, keys, pos, (const T*)v_out,
                           (T*)v_table);
        GS_CHECK_LAUNCH();
        float* partial = (float*)(b + w.partial);
        const int64_t pieces = ceil_div(n, EMB_LONG);
        hipLaunchKernelGGL((embed_pieces_kernel<T, NV>), dim3((unsigned)ceil_div(pieces, groups), (unsigned)tiles),
                           dim3(EMB_THREADS), 0, s, sh, keys, pos, (const T*)v_out, partial);
        GS_CHECK_LAUNCH();
        hipLaunchKernelGGL((embed_join_kernel<T, NV>), dim3((unsigned)pieces, (unsigned)tiles), dim3(EMB_THREADS), 0, s, sh,
                           keys, partial, (T*)v_table);
        GS_CHECK_LAUNCH();
        return GS_OK;
      }
      return GS_ERR_INVALID_ARG;
    });
  });
}
