// lg_edges.cu — squared distances along the edges of a graph and the gradient
// with respect to the vertices' features.
//
//   d2_e     = sum_c (x[i_e, c] - x[j_e, c])^2
//   dx[v, :] = 2 sum over the edges e at v of g_e (x[v, :] - x[other end, :])
//
// The gradient is a row sum: every vertex lists its edges (lg_edge_graph: one
// stable sort of both edge ends, so first the edges it begins, then those it
// ends, ascending), a group of lanes walks the list and writes the row once.
// No atomics: the result does not change from run to run.  Vertices with more
// than LG_EDGE_CHUNK edges are summed in chunks of that length, one group a
// chunk, and the chunks' sums added in order, so a hub does not hold up the
// rest.  Both directions are bound by the gathers of x rows (L2 as long as x
// fits).
#include "lg_feat.cuh"

#include "../../include/lanczos_b200.h"

namespace lg {
namespace feat {
namespace {

constexpr int kThreads = 256;

// ---------------------------------------------------------------------------
// Lists of the edges at every vertex
// ---------------------------------------------------------------------------
__global__ void __launch_bounds__(kThreads) edge_check_kernel(long long n, long long m, const long long* __restrict__ idx,
                                                              int* __restrict__ ends, int* __restrict__ bad) {
  for (long long p = (long long)blockIdx.x * blockDim.x + threadIdx.x; p < 2 * m; p += (long long)gridDim.x * blockDim.x) {
    const long long v = idx[p];
    const bool ok = v >= 0 && v < n;
    if (!ok) *bad = 1;
    ends[p] = ok ? (int)v : 0;
  }
}

__global__ void __launch_bounds__(kThreads) edge_lists_kernel(long long m, const int* __restrict__ ends,
                                                              const uint2* __restrict__ sorted, int* __restrict__ other,
                                                              int* __restrict__ eid) {
  for (long long q = (long long)blockIdx.x * blockDim.x + threadIdx.x; q < 2 * m; q += (long long)gridDim.x * blockDim.x) {
    const long long p = sorted[q].y;
    const bool second = p >= m;
    eid[q] = (int)(second ? p - m : p);
    other[q] = ends[second ? p - m : p + m];
  }
}

// rowptr[v] = first sorted position with a key >= v, by bisection.
__global__ void __launch_bounds__(kThreads) edge_rowptr_kernel(long long n, long long n2, const uint2* __restrict__ sorted,
                                                               int* __restrict__ rowptr) {
  for (long long v = (long long)blockIdx.x * blockDim.x + threadIdx.x; v <= n; v += (long long)gridDim.x * blockDim.x) {
    long long lo = 0, hi = n2;
    while (lo < hi) {
      const long long mid = (lo + hi) >> 1;
      if ((long long)sorted[mid].x < v) lo = mid + 1;
      else hi = mid;
    }
    rowptr[v] = (int)lo;
  }
}

// ---------------------------------------------------------------------------
// Distances: a group of 1 << lg lanes per edge
// ---------------------------------------------------------------------------
struct EdgeArgs {
  long long n, m, ld;
  int nv, lg;
};

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) edge_dist_kernel(EdgeArgs a, const int* __restrict__ ends,
                                                             const T* __restrict__ x, Acc<T>* __restrict__ d2) {
  typedef Acc<T> A;
  const int lane = threadIdx.x & ((1 << a.lg) - 1);
  const int ngrp = kThreads >> a.lg;
  const long long e = (long long)blockIdx.x * ngrp + (threadIdx.x >> a.lg);
  A s = 0;
  if (e < a.m) {
    const T* xi = x + ends[e] * a.ld;
    const T* xj = x + ends[a.m + e] * a.ld;
    for (int c = lane; c < a.nv; c += 1 << a.lg) {
      const Vec<T, V> u = load_vec<T, V>(xi + (long long)c * V), w = load_vec<T, V>(xj + (long long)c * V);
#pragma unroll
      for (int k = 0; k < V; ++k) {
        const A d = to_acc(u.v[k]) - to_acc(w.v[k]);
        s += d * d;
      }
    }
  }
  for (int o = 1 << a.lg >> 1; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0 && e < a.m) d2[e] = s;
}

// ---------------------------------------------------------------------------
// Gradient: a group of lanes per vertex (or per chunk of a long list) and per
// piece of 1 << lg vectors of the row (blockIdx.y)
// ---------------------------------------------------------------------------
constexpr int kBatch = 4;

template <typename T, int V>
__device__ __forceinline__ void edge_row_sum(const EdgeArgs& a, long long v, int b, int e, int c,
                                             const int* __restrict__ other, const int* __restrict__ eid,
                                             const T* __restrict__ x, const Acc<T>* __restrict__ g, Acc<T>* acc) {
  typedef Acc<T> A;
  const Vec<T, V> xv = load_vec<T, V>(x + v * a.ld + (long long)c * V);
  for (int q = b; q < e; q += kBatch) {
    int o[kBatch];
    A w[kBatch];
    Vec<T, V> y[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; ++u) {
      const int p = q + u < e ? q + u : e - 1;
      o[u] = other[p];
      w[u] = g[eid[p]];
    }
#pragma unroll
    for (int u = 0; u < kBatch; ++u) y[u] = load_vec<T, V>(x + o[u] * a.ld + (long long)c * V);
#pragma unroll
    for (int u = 0; u < kBatch; ++u)
      if (q + u < e) {
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] += w[u] * (to_acc(xv.v[k]) - to_acc(y[u].v[k]));
      }
  }
}

template <typename T, int V> __device__ __forceinline__ void edge_store(T* p, const Acc<T>* acc) {
  Vec<T, V> o;
#pragma unroll
  for (int k = 0; k < V; ++k) o.v[k] = from_acc<T>((Acc<T>)2 * acc[k]);
  store_vec<T, V>(p, o);
}

template <typename T, int V>
__global__ void __launch_bounds__(kThreads) edge_grad_kernel(EdgeArgs a, const int* __restrict__ rowptr,
                                                             const int* __restrict__ other, const int* __restrict__ eid,
                                                             const T* __restrict__ x, const Acc<T>* __restrict__ g,
                                                             T* __restrict__ dx) {
  const int lane = threadIdx.x & ((1 << a.lg) - 1);
  const int ngrp = kThreads >> a.lg;
  const long long v = (long long)blockIdx.x * ngrp + (threadIdx.x >> a.lg);
  const int c = (blockIdx.y << a.lg) + lane;
  if (v >= a.n || c >= a.nv) return;
  const int b = rowptr[v], e = rowptr[v + 1];
  if (e - b > LG_EDGE_CHUNK) return;   // summed by chunks
  Acc<T> acc[V];
#pragma unroll
  for (int k = 0; k < V; ++k) acc[k] = 0;
  edge_row_sum<T, V>(a, v, b, e, c, other, eid, x, g, acc);
  edge_store<T, V>(dx + v * a.nv * V + (long long)c * V, acc);
}

// Chunks of the long lists: chunk_row names the vertex, chunk_first the first
// position of its list entry in other / eid.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) edge_chunk_kernel(EdgeArgs a, int nchunks, const int* __restrict__ rowptr,
                                                              const int* __restrict__ other, const int* __restrict__ eid,
                                                              const int* __restrict__ chunk_row,
                                                              const int* __restrict__ chunk_first,
                                                              const T* __restrict__ x, const Acc<T>* __restrict__ g,
                                                              Acc<T>* __restrict__ part) {
  const int lane = threadIdx.x & ((1 << a.lg) - 1);
  const int ngrp = kThreads >> a.lg;
  const long long q = (long long)blockIdx.x * ngrp + (threadIdx.x >> a.lg);
  const int c = (blockIdx.y << a.lg) + lane;
  if (q >= nchunks || c >= a.nv) return;
  const int v = chunk_row[q], b = chunk_first[q];
  const int end = rowptr[v + 1], e = end - b > LG_EDGE_CHUNK ? b + LG_EDGE_CHUNK : end;
  Acc<T> acc[V];
#pragma unroll
  for (int k = 0; k < V; ++k) acc[k] = 0;
  edge_row_sum<T, V>(a, v, b, e, c, other, eid, x, g, acc);
  Acc<T>* o = part + q * a.nv * V + (long long)c * V;
#pragma unroll
  for (int k = 0; k < V; ++k) o[k] = acc[k];
}

// One block row per long vertex: its first chunk is long_first[r], the chunks
// follow one another.
template <typename T>
__global__ void __launch_bounds__(kThreads) edge_long_kernel(int dim, const int* __restrict__ rowptr,
                                                             const int* __restrict__ long_row,
                                                             const int* __restrict__ long_first,
                                                             const Acc<T>* __restrict__ part, T* __restrict__ dx) {
  const long long v = long_row[blockIdx.x];
  const long long q0 = long_first[blockIdx.x];
  const int count = (rowptr[v + 1] - rowptr[v] + LG_EDGE_CHUNK - 1) / LG_EDGE_CHUNK;
  for (int c = blockIdx.y * blockDim.x + threadIdx.x; c < dim; c += gridDim.y * blockDim.x) {
    Acc<T> s = 0;
#pragma unroll 8
    for (int k = 0; k < count; ++k) s += part[(q0 + k) * dim + c];
    dx[v * dim + c] = from_acc<T>((Acc<T>)2 * s);
  }
}

int group_log(int nv) {
  int l = 0;
  while (l < 5 && (1 << l) < nv) ++l;
  return l;
}

template <typename T, int V>
cudaError_t edge_dist(EdgeArgs a, int dim, const int* ends, const T* x, void* d2, cudaStream_t st) {
  a.nv = dim / V;
  a.lg = group_log(a.nv);
  const int ngrp = kThreads >> a.lg;
  edge_dist_kernel<T, V><<<(unsigned)((a.m + ngrp - 1) / ngrp), kThreads, 0, st>>>(a, ends, x, static_cast<Acc<T>*>(d2));
  return cudaGetLastError();
}

struct LongLists {
  int nlong, nchunks;
  const int *row, *first, *chunk_row, *chunk_first;
};

template <typename T, int V>
cudaError_t edge_grad(EdgeArgs a, int dim, const int* rowptr, const int* other, const int* eid, const T* x,
                      const void* g, T* dx, const LongLists& l, void* ws, cudaStream_t st) {
  typedef Acc<T> A;
  a.nv = dim / V;
  a.lg = group_log(a.nv);
  const int ngrp = kThreads >> a.lg;
  const unsigned cols = (unsigned)((a.nv + (1 << a.lg) - 1) >> a.lg);
  const A* gv = static_cast<const A*>(g);
  edge_grad_kernel<T, V><<<dim3((unsigned)((a.n + ngrp - 1) / ngrp), cols), kThreads, 0, st>>>(a, rowptr, other, eid, x,
                                                                                              gv, dx);
  if (l.nlong > 0) {
    A* part = static_cast<A*>(ws);
    edge_chunk_kernel<T, V><<<dim3((unsigned)((l.nchunks + ngrp - 1) / ngrp), cols), kThreads, 0, st>>>(
        a, l.nchunks, rowptr, other, eid, l.chunk_row, l.chunk_first, x, gv, part);
    const unsigned pieces = (unsigned)((dim + kThreads - 1) / kThreads);
    edge_long_kernel<T><<<dim3((unsigned)l.nlong, pieces < 65535u ? pieces : 65535u), kThreads, 0, st>>>(
        dim, rowptr, l.row, l.first, part, dx);
  }
  return cudaGetLastError();
}

bool edge_sizes_ok(long long n, long long m) {
  return n >= 1 && n < 2147483647LL && m >= 1 && 2 * m < 2147483647LL;
}

bool edge_args_ok(long long n, long long m, int dim, int dtype) {
  return edge_sizes_ok(n, m) && dim >= 1 && dim <= (1 << 20) && elem_size(dtype);
}

int wide_grid(long long n) {
  const long long need = (n + kThreads - 1) / kThreads, most = 16LL * (sm_count() > 0 ? sm_count() : 1);
  return (int)(need < most ? need : most);
}

}  // namespace
}  // namespace feat
}  // namespace lg

using namespace lg;
using namespace lg::feat;

#define LG_EDGE_DISPATCH(F)                                                              \
  switch (dtype) {                                                                       \
    case LG_F64: return vec >= 2 ? F(double, 2) : F(double, 1);                          \
    case LG_F32: return vec >= 4 ? F(float, 4) : vec == 2 ? F(float, 2) : F(float, 1);   \
    case LG_F16:                                                                         \
      return vec >= 8 ? F(__half, 8) : vec == 4 ? F(__half, 4) : vec == 2 ? F(__half, 2) : F(__half, 1); \
    default:                                                                             \
      return vec >= 8 ? F(__nv_bfloat16, 8) : vec == 4 ? F(__nv_bfloat16, 4)             \
             : vec == 2 ? F(__nv_bfloat16, 2) : F(__nv_bfloat16, 1);                     \
  }

extern "C" size_t lg_edge_graph_workspace_bytes(long long n, long long m) {
  return edge_sizes_ok(n, m) ? sort_ids_workspace(n, 2 * m) : 0;
}

extern "C" int lg_edge_graph(long long n, long long m, const long long* idx, int* ends, int* rowptr, int* other,
                             int* eid, int* bad, void* ws, size_t ws_bytes, void* stream) {
  if (!edge_sizes_ok(n, m) || !idx || !ends || !rowptr || !other || !eid || !bad || !ws ||
      ws_bytes < sort_ids_workspace(n, 2 * m))
    return bad_args("lg_edge_graph: invalid arguments");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = cudaMemsetAsync(bad, 0, sizeof(int), st);
  if (e != cudaSuccess) return cuda_status(e, "lg_edge_graph");
  edge_check_kernel<<<wide_grid(2 * m), kThreads, 0, st>>>(n, m, idx, ends, bad);
  uint2* sorted = nullptr;
  e = sort_ids(n, 2 * m, idx, 1, 0, 0, ws, nullptr, 0, SideFill{nullptr, 0}, &sorted, st);
  if (e != cudaSuccess) return cuda_status(e, "lg_edge_graph");
  edge_lists_kernel<<<wide_grid(2 * m), kThreads, 0, st>>>(m, ends, sorted, other, eid);
  edge_rowptr_kernel<<<wide_grid(n + 1), kThreads, 0, st>>>(n, 2 * m, sorted, rowptr);
  return cuda_status(cudaGetLastError(), "lg_edge_graph");
}

extern "C" int lg_edge_sqdist(long long n, long long m, int dim, int dtype, const int* ends, const void* x,
                              long long ld_x, void* d2, void* stream) {
  if (!edge_args_ok(n, m, dim, dtype) || !ends || !x || ld_x < dim || !d2)
    return bad_args("lg_edge_sqdist: invalid arguments");
  EdgeArgs a = {};
  a.n = n;
  a.m = m;
  a.ld = ld_x;
  Align al(elem_size(dtype));
  al.address(x);
  al.elements(ld_x);
  al.elements(dim);
  const int vec = al.vec();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto run = [&]() -> cudaError_t {
#define LG_F(T, V) edge_dist<T, V>(a, dim, ends, static_cast<const T*>(x), d2, st)
    LG_EDGE_DISPATCH(LG_F)
#undef LG_F
  };
  return cuda_status(run(), "lg_edge_sqdist");
}

extern "C" size_t lg_edge_sqdist_grad_workspace_bytes(int nchunks, int dim, int dtype) {
  return (size_t)(nchunks > 0 ? nchunks : 0) * (dim > 0 ? dim : 0) * acc_size(dtype);
}

extern "C" int lg_edge_sqdist_grad(long long n, long long m, int dim, int dtype, const int* rowptr, const int* other,
                                   const int* eid, int nlong, const int* long_row, const int* long_first, int nchunks,
                                   const int* chunk_row, const int* chunk_first, const void* x, long long ld_x,
                                   const void* g, void* dx, void* ws, size_t ws_bytes, void* stream) {
  if (!edge_args_ok(n, m, dim, dtype) || !rowptr || !other || !eid || !x || ld_x < dim || !g || !dx || nlong < 0 ||
      nchunks < nlong ||
      (nlong > 0 && (!long_row || !long_first || !chunk_row || !chunk_first || !ws ||
                     ws_bytes < lg_edge_sqdist_grad_workspace_bytes(nchunks, dim, dtype))))
    return bad_args("lg_edge_sqdist_grad: invalid arguments");
  EdgeArgs a = {};
  a.n = n;
  a.m = m;
  a.ld = ld_x;
  Align al(elem_size(dtype));
  al.address(x);
  al.address(dx);
  al.elements(ld_x);
  al.elements(dim);
  const int vec = al.vec();
  const LongLists l = {nlong, nchunks, long_row, long_first, chunk_row, chunk_first};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto run = [&]() -> cudaError_t {
#define LG_F(T, V) \
  edge_grad<T, V>(a, dim, rowptr, other, eid, static_cast<const T*>(x), g, static_cast<T*>(dx), l, ws, st)
    LG_EDGE_DISPATCH(LG_F)
#undef LG_F
  };
  return cuda_status(run(), "lg_edge_sqdist_grad");
}
