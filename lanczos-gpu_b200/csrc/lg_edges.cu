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
// a group keeps several edges' rows in flight; by L1, which looks up every row a lane
// group touches; and by the instructions around them, so a lane takes two vectors of a
// row where the row has more than two.  10^6 vertices, 5 10^6 edges with far ends, 10
// fp32: forward 67 us (L1 71 % busy, 68 % of the issue slots), backward 138 us (80 %,
// 56 %); rows of 12 in 16-byte pieces take the same, and a lane a vector takes 20 us
// longer.  10^5 vertices, 10^6 edges, 64 fp32: 32 us and 53 us.
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

// The rows of x from 16-byte boundaries, filled up with zeros: a thread makes one
// vector.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) edge_pack_kernel(long long n, int dim, int nv, const T* __restrict__ x,
                                                             long long ld, T* __restrict__ out) {
  for (long long t = (long long)blockIdx.x * kThreads + threadIdx.x; t < n * nv; t += (long long)gridDim.x * kThreads) {
    const long long row = t / nv;
    const int c = (int)(t - row * nv) * V;
    Vec<T, V> o;
#pragma unroll
    for (int k = 0; k < V; ++k) o.v[k] = c + k < dim ? x[row * ld + c + k] : from_acc<T>((Acc<T>)0);
    store_vec<T, V>(out + t * V, o);
  }
}

template <typename T> __device__ __forceinline__ const T* row_at(const T* x, int i, unsigned stride) {
  return reinterpret_cast<const T*>(reinterpret_cast<const char*>(x) + (unsigned long long)(unsigned)i * stride);
}

constexpr int kEdges = 4;

// Blocks that an SM is to hold, which sets the registers: the most that do not spill
// them.  10^6 vertices, 5 10^6 edges, 10 fp32 in pairs: 67 us with 6, 70 us with 5,
// 80 us without a bound; 50,000 vertices, 500,000 edges, 1024 fp32: 250 us with 4,
// 262 us with 3, 316 us without.
template <typename T, int V, int K, bool LOOP>
constexpr int dist_blocks = K == 1 ? 4 : sizeof(T) * V <= 8 ? 6 : sizeof(T) == 8 && LOOP ? 3 : 4;

// K vectors a lane; LOOP: the row has more than K << lg.  All vectors of a turn are on
// their way before the first is used (64 fp32, 10^6 edges: 35 us, 40 us one vector
// after the other).
template <typename T, int V, int K, bool LOOP>
__global__ void __launch_bounds__(kThreads, dist_blocks<T, V, K, LOOP>)
    edge_dist_kernel(EdgeArgs a, const int* __restrict__ ends, const T* __restrict__ x, Acc<T>* __restrict__ d2) {
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
    Vec<T, V> p[K][kEdges], q[K][kEdges];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int at = (c - lane + (k << a.lg)) * V;
#pragma unroll
      for (int u = 0; u < kEdges; ++u) {
        typename Word<sizeof(T) * V>::type zero = {};
        memcpy(&p[k][u], &zero, sizeof(zero));
        memcpy(&q[k][u], &zero, sizeof(zero));
        if (c + (k << a.lg) < a.nv) {
          p[k][u] = load_vec<T, V>(xi[u] + at);
          q[k][u] = load_vec<T, V>(xj[u] + at);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int u = 0; u < kEdges; ++u) {
#pragma unroll
        for (int n = 0; n < lanes<V>; ++n) {
          const L d = fma(widen<T, V>(q[k][u].v, n), minus, widen<T, V>(p[k][u].v, n));
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
  int dim;               // columns of dx; at most e.nv vectors
  int nchunks;
  const int *rowptr, *other, *eid, *chunk_row, *chunk_first;
};

// First the chunks, then the vertices.  A vertex row is written to dx, a chunk's
// sum to part.  The indices of a batch of list entries are fetched while the rows
// of the batch before are worked on.
// WHOLE: whole vectors of dx can be stored.
template <typename T, int V, int K, bool WHOLE>
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
#pragma unroll
  for (int k = 0; k < K; ++k) {
    if (!on[k]) continue;
    if (chunk) {
#pragma unroll
      for (int n = 0; n < N; ++n) narrow<A, V>(acc[k][n], part + unit * a.e.nv * V + at[k], n);
    } else {
      Vec<T, V> o;
      const L two = spread<L>((A)2);
#pragma unroll
      for (int n = 0; n < N; ++n) narrow<T, V>(mul(acc[k][n], two), o.v, n);
      if (WHOLE) {
        store_vec<T, V>(dx + v * ((long long)a.e.nv * V) + at[k], o);
      } else {
#pragma unroll
        for (int n = 0; n < V; ++n)
          if (at[k] + n < a.dim) dx[v * a.dim + at[k] + n] = o.v[n];
      }
    }
  }
}

// The long vertices: a block adds 32 columns of a vertex's chunks (from
// long_first[r] on, one after the other, pitch columns each), eight rows of
// threads taking every eighth chunk.
template <typename T>
__global__ void __launch_bounds__(kThreads) edge_long_kernel(int dim, long long pitch, const int* __restrict__ rowptr,
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
      for (int k = grp; k < count; k += kThreads / 32) s += part[(q0 + k) * pitch + c];
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
  a.nv = (dim + V - 1) / V;
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
  a.e.nv = (dim + V - 1) / V;
  a.e.lg = a.e.nv == 2 ? 1 : group_log(a.e.nv);
  const int ngrp = kThreads >> a.e.lg;
  const unsigned cols = (unsigned)((a.e.nv + (2 << a.e.lg) - 1) / (2 << a.e.lg));
  A* part = static_cast<A*>(ws);
  const dim3 grid((unsigned)((a.e.n + a.nchunks + ngrp - 1) / ngrp), cols);
  const A* gv = static_cast<const A*>(g);
  const bool whole = dim % V == 0 && reinterpret_cast<uintptr_t>(dx) % (V * sizeof(T)) == 0;
  if (a.e.nv > 2 && whole) edge_grad_kernel<T, V, 2, true><<<grid, kThreads, 0, st>>>(a, x, gv, dx, part);
  else if (a.e.nv > 2) edge_grad_kernel<T, V, 2, false><<<grid, kThreads, 0, st>>>(a, x, gv, dx, part);
  else if (whole) edge_grad_kernel<T, V, 1, true><<<grid, kThreads, 0, st>>>(a, x, gv, dx, part);
  else edge_grad_kernel<T, V, 1, false><<<grid, kThreads, 0, st>>>(a, x, gv, dx, part);
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess && l.nlong > 0) {
    const unsigned pieces = (unsigned)((dim + 31) / 32);
    e = launch_pdl(edge_long_kernel<T>, dim3((unsigned)l.nlong, pieces < 65535u ? pieces : 65535u), dim3(kThreads), 0, st,
                   dim, (long long)a.e.nv * V, a.rowptr, l.row, l.first, part, dx);
  }
  return e;
}

// The gradient forms list positions a few beyond a list's end, and a list's length
// rounded up to chunks, in 32 bits.
bool edge_sizes_ok(long long n, long long m) {
  return n >= 1 && n < 2147483647LL && m >= 1 && m <= (2147483647LL - LG_EDGE_CHUNK) / 2;
}

bool edge_args_ok(long long n, long long m, int dim, int dtype, long long ld) {
  return edge_sizes_ok(n, m) && dim >= 1 && dim <= (1 << 20) && elem_size(dtype) && ld >= dim &&
         ld * elem_size(dtype) < (1LL << 32);
}

// An x whose rows can be read only in narrow pieces is copied to aligned rows
// first, where its 2 m gathers then take at least a piece less for every 3 bytes
// copied.  Measured forward + backward, us, without and with the copy: 10^5 vertices,
// 10^6 edges, 333 fp16 909 and 571, 33 fp32 201 and 122; 500,000 vertices, 10^6 edges,
// 33 fp32 331 and 293; at a piece for 4 bytes (10^6 vertices, 5 10^6 edges, 7 fp64) 282
// both.  Under 16 MB of gathers the second launch costs more than it saves; above
// 8 GB the copy would burden the device's memory.
size_t packed_bytes(const EdgeArgs& a, int dim, int dtype, const void* x, long long ld) {
  const long long es = elem_size(dtype), v16 = (dim * es + 15) / 16;
  Align al((int)es);
  al.address(x);
  al.elements(ld);
  al.elements(dim);
  const bool pays = 6.0 * (double)a.m * (double)(dim / al.vec() - v16) >= (double)a.n * (double)(dim * es + 16 * v16) &&
                    a.m * dim * es >= (16LL << 20) && a.n <= (8LL << 30) / (16 * v16);
  return pays ? (size_t)(a.n * v16 * 16) : 0;
}

template <typename T>
cudaError_t pack(EdgeArgs& a, int dim, const void* x, long long ld, void* out, cudaStream_t st) {
  constexpr int V = 16 / sizeof(T);
  const int nv = (dim + V - 1) / V;
  const long long blocks = (a.n * nv + kThreads - 1) / kThreads;
  a.stride = (unsigned)nv * 16;
  edge_pack_kernel<T, V><<<(unsigned)(blocks < (1 << 30) ? blocks : (1 << 30)), kThreads, 0, st>>>(
      a.n, dim, nv, static_cast<const T*>(x), ld, static_cast<T*>(out));
  return cudaGetLastError();
}

cudaError_t pack_any(EdgeArgs& a, int dim, int dtype, const void* x, long long ld, void* out, cudaStream_t st) {
  switch (dtype) {
    case LG_F64: return pack<double>(a, dim, x, ld, out, st);
    case LG_F32: return pack<float>(a, dim, x, ld, out, st);
    case LG_F16: return pack<__half>(a, dim, x, ld, out, st);
    default: return pack<__nv_bfloat16>(a, dim, x, ld, out, st);
  }
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
      ws_bytes < sort_ids_workspace(n, 2 * m) || !aligned(8, idx) || !aligned(4, ends, rowptr, other, eid, bad) ||
      !aligned(kWsAlign, ws))
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

extern "C" size_t lg_edge_sqdist_workspace_bytes(long long n, long long m, int dim, int dtype, const void* x,
                                                long long ld_x) {
  if (!edge_args_ok(n, m, dim, dtype, ld_x)) return 0;
  EdgeArgs a = {};
  a.n = n;
  a.m = m;
  return packed_bytes(a, dim, dtype, x, ld_x);
}

extern "C" int lg_edge_sqdist(long long n, long long m, int dim, int dtype, const int* ends, const void* x,
                              long long ld_x, void* d2, void* ws, size_t ws_bytes, void* stream) {
  const size_t nb = lg_edge_sqdist_workspace_bytes(n, m, dim, dtype, x, ld_x);
  if (!edge_args_ok(n, m, dim, dtype, ld_x) || !ends || !x || !d2 || (nb && (!ws || ws_bytes < nb)) ||
      !aligned(4, ends) || !aligned(elem_size(dtype), x) || !aligned(acc_size(dtype), d2) || !aligned(kWsAlign, ws))
    return bad_args("lg_edge_sqdist: invalid arguments");
  EdgeArgs a = {};
  a.n = n;
  a.m = m;
  a.stride = (unsigned)(ld_x * elem_size(dtype));
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  Align al(elem_size(dtype));
  al.address(x);
  al.elements(ld_x);
  al.elements(dim);
  const int vec = nb ? 16 / elem_size(dtype) : al.vec();
  if (nb) {
    const cudaError_t e = pack_any(a, dim, dtype, x, ld_x, ws, st);
    if (e != cudaSuccess) return cuda_status(e, "lg_edge_sqdist");
    x = ws;
  }
  auto run = [&]() -> cudaError_t {
#define LG_F(T, V) edge_dist<T, V>(a, dim, ends, static_cast<const T*>(x), d2, st)
    LG_EDGE_DISPATCH(LG_F)
#undef LG_F
  };
  return cuda_status(run(), "lg_edge_sqdist");
}

namespace {
size_t part_bytes(int nchunks, int dim, int dtype) {
  const size_t es = elem_size(dtype), wide = (dim * es + 15) / 16 * 16 / es;   // columns of packed rows
  return align_up((size_t)nchunks * wide * acc_size(dtype));
}
}  // namespace

extern "C" size_t lg_edge_sqdist_grad_workspace_bytes(long long n, long long m, int dim, int dtype, const void* x,
                                                     long long ld_x, int nchunks) {
  if (!edge_args_ok(n, m, dim, dtype, ld_x) || nchunks < 0) return 0;
  return part_bytes(nchunks, dim, dtype) + lg_edge_sqdist_workspace_bytes(n, m, dim, dtype, x, ld_x);
}

extern "C" int lg_edge_sqdist_grad(long long n, long long m, int dim, int dtype, const int* rowptr, const int* other,
                                   const int* eid, int nlong, const int* long_row, const int* long_first, int nchunks,
                                   const int* chunk_row, const int* chunk_first, const void* x, long long ld_x,
                                   const void* g, void* dx, void* ws, size_t ws_bytes, void* stream) {
  if (!edge_args_ok(n, m, dim, dtype, ld_x) || !rowptr || !other || !eid || !x || !g || !dx || nlong < 0 ||
      nchunks < nlong || (nlong > 0 && (!long_row || !long_first || !chunk_row || !chunk_first)) ||
      !aligned(4, rowptr, other, eid, long_row, long_first, chunk_row, chunk_first) ||
      !aligned(elem_size(dtype), x, dx) || !aligned(acc_size(dtype), g) || !aligned(kWsAlign, ws))
    return bad_args("lg_edge_sqdist_grad: invalid arguments");
  if (nlong == 0) nchunks = 0;
  const size_t nb = lg_edge_sqdist_grad_workspace_bytes(n, m, dim, dtype, x, ld_x, nchunks);
  if (nb && (!ws || ws_bytes < nb)) return bad_args("lg_edge_sqdist_grad: the workspace is too small");
  GradArgs a = {};
  a.e.n = n;
  a.e.m = m;
  a.e.stride = (unsigned)(ld_x * elem_size(dtype));
  a.dim = dim;
  a.nchunks = nchunks;
  a.rowptr = rowptr;
  a.other = other;
  a.eid = eid;
  a.chunk_row = chunk_row;
  a.chunk_first = chunk_first;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  Align al(elem_size(dtype));
  al.address(x);
  al.elements(ld_x);
  al.elements(dim);
  int vec = al.vec();
  if (nb > part_bytes(nchunks, dim, dtype)) {
    void* packed = static_cast<char*>(ws) + part_bytes(nchunks, dim, dtype);
    const cudaError_t e = pack_any(a.e, dim, dtype, x, ld_x, packed, st);
    if (e != cudaSuccess) return cuda_status(e, "lg_edge_sqdist_grad");
    x = packed;
    vec = 16 / elem_size(dtype);
  }
  const LongLists l = {nlong, long_row, long_first};
  auto run = [&]() -> cudaError_t {
#define LG_F(T, V) edge_grad<T, V>(a, dim, static_cast<const T*>(x), g, static_cast<T*>(dx), l, ws, st)
    LG_EDGE_DISPATCH(LG_F)
#undef LG_F
  };
  return cuda_status(run(), "lg_edge_sqdist_grad");
}
