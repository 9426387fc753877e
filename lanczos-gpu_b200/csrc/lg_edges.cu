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
// rest.
//
// Both directions are bound by the gathers of x rows from L2: by their latency, so
// a group keeps several edges' rows in flight, and by the instructions around
// them, so a lane takes two vectors of a row where the row has them.
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
// Distances: a group of 1 << lg lanes takes kEdges edges
// ---------------------------------------------------------------------------
struct EdgeArgs {
  long long n, m;
  unsigned stride;       // bytes from one row of x to the next
  int nv, lg;
};

template <typename T> __device__ __forceinline__ const T* row_at(const T* x, int i, unsigned stride) {
  return reinterpret_cast<const T*>(reinterpret_cast<const char*>(x) + (unsigned long long)(unsigned)i * stride);
}

constexpr int kEdges = 4;

// K vectors a lane; LOOP: the row has more than K << lg.
template <typename T, int V, int K, bool LOOP>
__global__ void __launch_bounds__(kThreads) edge_dist_kernel(EdgeArgs a, const int* __restrict__ ends,
                                                             const T* __restrict__ x, Acc<T>* __restrict__ d2) {
  typedef Acc<T> A;
  typedef Lane<T, V> L;
  const int lane = threadIdx.x & ((1 << a.lg) - 1);
  const int ngrp = kThreads >> a.lg;
  const long long e0 = (long long)blockIdx.x * ngrp * kEdges + (threadIdx.x >> a.lg);
  const T *xi[kEdges], *xj[kEdges];
  L s[kEdges];
#pragma unroll
  for (int u = 0; u < kEdges; ++u) {
    const long long e = e0 + u * ngrp;
    const bool in = e < a.m;
    xi[u] = row_at(x, in ? ends[e] : 0, a.stride) + lane * V;
    xj[u] = row_at(x, in ? ends[a.m + e] : 0, a.stride) + lane * V;
    s[u] = spread<L>((A)0);
  }
  const L minus = spread<L>((A)-1);
  for (int c = lane; c < (LOOP ? a.nv : lane + 1); c += K << a.lg) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (c + (k << a.lg) >= a.nv) break;
      Vec<T, V> p[kEdges], q[kEdges];
      const int at = (c - lane + (k << a.lg)) * V;
#pragma unroll
      for (int u = 0; u < kEdges; ++u) {
        p[u] = load_vec<T, V>(xi[u] + at);
        q[u] = load_vec<T, V>(xj[u] + at);
      }
#pragma unroll
      for (int u = 0; u < kEdges; ++u) {
#pragma unroll
        for (int n = 0; n < lanes<V>; ++n) {
          const L d = fma(widen<T, V>(q[u].v, n), minus, widen<T, V>(p[u].v, n));
          s[u] = fma(d, d, s[u]);
        }
      }
    }
  }
#pragma unroll
  for (int u = 0; u < kEdges; ++u) {
    A t = sum(s[u]);
    for (int o = 1 << a.lg >> 1; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    const long long e = e0 + u * ngrp;
    if (lane == 0 && e < a.m) d2[e] = t;
  }
}

// ---------------------------------------------------------------------------
// Gradient: a group of lanes per vertex (or per chunk of a long list) and per
// piece of K << lg vectors of the row (blockIdx.y)
// ---------------------------------------------------------------------------
struct GradArgs {
  EdgeArgs e;
  int nchunks;
  const int *rowptr, *other, *eid, *chunk_row, *chunk_first;
};

// First the chunks, then the vertices.  A vertex row is written to dx, a chunk's
// sum to part.  The indices of a batch of list entries are fetched while the rows
// of the batch before are worked on.
template <typename T, int V, int K>
__global__ void __launch_bounds__(kThreads) edge_grad_kernel(GradArgs a, const T* __restrict__ x,
                                                             const Acc<T>* __restrict__ g, T* __restrict__ dx,
                                                             Acc<T>* __restrict__ part) {
  typedef Acc<T> A;
  typedef Lane<T, V> L;
  constexpr int N = lanes<V>, B = 4;   // list entries in flight
  const int lg = a.e.lg, lane = threadIdx.x & ((1 << lg) - 1);
  const long long unit = (long long)blockIdx.x * (kThreads >> lg) + (threadIdx.x >> lg);
  const bool chunk = unit < a.nchunks;
  if (unit >= a.nchunks + a.e.n) return;
  const long long v = chunk ? a.chunk_row[unit] : unit - a.nchunks;
  int b = a.rowptr[v], e = a.rowptr[v + 1];
  if (chunk) {
    b = a.chunk_first[unit];
    if (e - b > LG_EDGE_CHUNK) e = b + LG_EDGE_CHUNK;
  } else if (e - b > LG_EDGE_CHUNK) {
    return;   // summed by chunks
  }
  int at[K];
  bool on[K];
  Vec<T, V> own[K];
  L acc[K][N];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = (blockIdx.y * K + k) * (1 << lg) + lane;
    on[k] = c < a.e.nv;
    at[k] = on[k] ? c * V : 0;
    own[k] = load_vec<T, V>(row_at(x, (int)v, a.e.stride) + at[k]);
#pragma unroll
    for (int n = 0; n < N; ++n) acc[k][n] = spread<L>((A)0);
  }
  const L minus = spread<L>((A)-1);
  int next[B], edge[B];
#pragma unroll
  for (int u = 0; u < B; ++u) {
    next[u] = b + u < e ? a.other[b + u] : (int)v;
    edge[u] = b + u < e ? a.eid[b + u] : -1;
  }
  for (int q = b; q < e; q += B) {
    Vec<T, V> y[B][K];
    A w[B];
#pragma unroll
    for (int u = 0; u < B; ++u) {
      if (edge[u] >= 0) {
        const T* r = row_at(x, next[u], a.e.stride);
        w[u] = g[edge[u]];
#pragma unroll
        for (int k = 0; k < K; ++k) y[u][k] = load_vec<T, V>(r + at[k]);
      }
    }
    const int p = q + B;
#pragma unroll
    for (int u = 0; u < B; ++u) {
      next[u] = p + u < e ? a.other[p + u] : (int)v;
      edge[u] = p + u < e ? a.eid[p + u] : -1;
    }
#pragma unroll
    for (int u = 0; u < B; ++u) {
      if (q + u < e) {
        const L f = spread<L>(w[u]);
#pragma unroll
        for (int k = 0; k < K; ++k)
#pragma unroll
          for (int n = 0; n < N; ++n)
            acc[k][n] = fma(f, fma(widen<T, V>(y[u][k].v, n), minus, widen<T, V>(own[k].v, n)), acc[k][n]);
      }
    }
  }
  const long long dim = (long long)a.e.nv * V;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (!on[k]) continue;
    if (chunk) {
#pragma unroll
      for (int n = 0; n < N; ++n) narrow<A, V>(acc[k][n], part + unit * dim + at[k], n);
    } else {
      Vec<T, V> o;
      const L two = spread<L>((A)2);
#pragma unroll
      for (int n = 0; n < N; ++n) narrow<T, V>(mul(acc[k][n], two), o.v, n);
      store_vec<T, V>(dx + v * dim + at[k], o);
    }
  }
}

// The long vertices: a block adds 32 columns of a vertex's chunks (from
// long_first[r] on, one after the other), eight rows of threads taking every
// eighth chunk.
template <typename T>
__global__ void __launch_bounds__(kThreads) edge_long_kernel(int dim, const int* __restrict__ rowptr,
                                                             const int* __restrict__ long_row,
                                                             const int* __restrict__ long_first, const Acc<T>* part,
                                                             T* __restrict__ dx) {
  __shared__ Acc<T> red[kThreads / 32][33];
  griddep_wait();
  const long long v = long_row[blockIdx.x], q0 = long_first[blockIdx.x];
  const int count = (rowptr[v + 1] - rowptr[v] + LG_EDGE_CHUNK - 1) / LG_EDGE_CHUNK;
  const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5;
  for (int c0 = blockIdx.y * 32; c0 < dim; c0 += gridDim.y * 32) {
    const int c = c0 + lane;
    Acc<T> s = 0;
    if (c < dim) {
#pragma unroll 4
      for (int k = grp; k < count; k += kThreads / 32) s += part[(q0 + k) * dim + c];
    }
    __syncthreads();
    red[grp][lane] = s;
    __syncthreads();
    if (grp == 0 && c < dim) {
      Acc<T> t = 0;
#pragma unroll
      for (int k = 0; k < kThreads / 32; ++k) t += red[k][lane];
      dx[v * dim + c] = from_acc<T>((Acc<T>)2 * t);
    }
  }
}

// Lanes of a group, each with up to two vectors of the row.
int group_log(int nv) {
  int l = 0;
  while (l < 5 && (2 << l) < nv) ++l;
  return l;
}

template <typename T, int V>
cudaError_t edge_dist(EdgeArgs a, int dim, const int* ends, const T* x, void* d2, cudaStream_t st) {
  a.nv = dim / V;
  a.lg = group_log(a.nv);
  const int per = (kThreads >> a.lg) * kEdges;
  const unsigned grid = (unsigned)((a.m + per - 1) / per);
  Acc<T>* out = static_cast<Acc<T>*>(d2);
  if (a.nv > 64) edge_dist_kernel<T, V, 2, true><<<grid, kThreads, 0, st>>>(a, ends, x, out);
  else if (a.nv > 1) edge_dist_kernel<T, V, 2, false><<<grid, kThreads, 0, st>>>(a, ends, x, out);
  else edge_dist_kernel<T, V, 1, false><<<grid, kThreads, 0, st>>>(a, ends, x, out);
  return cudaGetLastError();
}

struct LongLists {
  int nlong;
  const int *row, *first;
};

template <typename T, int V>
cudaError_t edge_grad(GradArgs a, int dim, const T* x, const void* g, T* dx, const LongLists& l, void* ws,
                      cudaStream_t st) {
  typedef Acc<T> A;
  a.e.nv = dim / V;
  a.e.lg = group_log(a.e.nv);
  const int ngrp = kThreads >> a.e.lg;
  const unsigned cols = (unsigned)((a.e.nv + (2 << a.e.lg) - 1) / (2 << a.e.lg));
  A* part = static_cast<A*>(ws);
  const dim3 grid((unsigned)((a.e.n + a.nchunks + ngrp - 1) / ngrp), cols);
  const A* gv = static_cast<const A*>(g);
  if (a.e.nv > 1) edge_grad_kernel<T, V, 2><<<grid, kThreads, 0, st>>>(a, x, gv, dx, part);
  else edge_grad_kernel<T, V, 1><<<grid, kThreads, 0, st>>>(a, x, gv, dx, part);
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess && l.nlong > 0) {
    const unsigned pieces = (unsigned)((dim + 31) / 32);
    e = launch_pdl(edge_long_kernel<T>, dim3((unsigned)l.nlong, pieces < 65535u ? pieces : 65535u), dim3(kThreads), 0, st,
                   dim, a.rowptr, l.row, l.first, part, dx);
  }
  return e;
}

bool edge_sizes_ok(long long n, long long m) {
  return n >= 1 && n < 2147483647LL && m >= 1 && 2 * m < 2147483647LL;
}

bool edge_args_ok(long long n, long long m, int dim, int dtype, long long ld) {
  return edge_sizes_ok(n, m) && dim >= 1 && dim <= (1 << 20) && elem_size(dtype) && ld >= dim &&
         ld * elem_size(dtype) < (1LL << 32);
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
  if (!edge_args_ok(n, m, dim, dtype, ld_x) || !ends || !x || !d2)
    return bad_args("lg_edge_sqdist: invalid arguments");
  EdgeArgs a = {};
  a.n = n;
  a.m = m;
  a.stride = (unsigned)(ld_x * elem_size(dtype));
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
  if (!edge_args_ok(n, m, dim, dtype, ld_x) || !rowptr || !other || !eid || !x || !g || !dx || nlong < 0 ||
      nchunks < nlong ||
      (nlong > 0 && (!long_row || !long_first || !chunk_row || !chunk_first || !ws ||
                     ws_bytes < lg_edge_sqdist_grad_workspace_bytes(nchunks, dim, dtype))))
    return bad_args("lg_edge_sqdist_grad: invalid arguments");
  GradArgs a = {};
  a.e.n = n;
  a.e.m = m;
  a.e.stride = (unsigned)(ld_x * elem_size(dtype));
  a.nchunks = nlong > 0 ? nchunks : 0;
  a.rowptr = rowptr;
  a.other = other;
  a.eid = eid;
  a.chunk_row = chunk_row;
  a.chunk_first = chunk_first;
  Align al(elem_size(dtype));
  al.address(x);
  al.address(dx);
  al.elements(ld_x);
  al.elements(dim);
  const int vec = al.vec();
  const LongLists l = {nlong, long_row, long_first};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto run = [&]() -> cudaError_t {
#define LG_F(T, V) edge_grad<T, V>(a, dim, static_cast<const T*>(x), g, static_cast<T*>(dx), l, ws, st)
    LG_EDGE_DISPATCH(LG_F)
#undef LG_F
  };
  return cuda_status(run(), "lg_edge_sqdist_grad");
}
