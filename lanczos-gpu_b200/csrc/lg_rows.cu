// lg_rows.cu — rows of a table by id (embedding lookup) and the table's
// gradient by sorted ids.
//
//   out[t, :]  = s * W[id_t, :]           s: none, a number, one value a column
//   dW[v, :]   = s * G[v, :],   G[v, :] = sum over t with id_t = v, ascending t, of g[t, :]
//   ds[c]      = sum_v W[v, c] G[v, c]
//
// ds is written over the table's rows instead of over the tokens: the sum over
// the tokens of one id is G, which the gradient forms anyway, so W is read
// once for every different id.
//
// An id equal to the padding id gives a row of zeros and takes no gradient; an
// id outside [0, rows) reads nothing, gives a row of NaN and takes no gradient.
//
// Lookup: one access per lane, the loads of four rows (short rows) or four
// pieces of a row (long rows) in flight before the first store; short rows of an
// awkward length lie in one line over the lanes.  Bound by memory: nothing is reused
// but rows named twice.  10^6 x 64 fp32 by a permutation: 86 us, 6.0 TB/s.
//
// Gradient: the ids are sorted (stable, with their positions) and the sorted
// positions cut into tiles of equal length; a group of lanes sums the rows of one
// tile, one vector of columns per lane.  Equal tiles keep the work even whatever
// the distribution of the ids.  A run of equal ids inside a tile is finished and
// written at once.  One that crosses tiles leaves partial sums (Acc<T>): in shared
// memory for the tiles of one block, which are added up there, and in memory for
// runs that cross blocks, which the last of their blocks to finish adds up in
// block order.  No sum depends on which block that is, so the result does not
// change from run to run.  Rows that no id names are set to zero by the SMs that
// have no part in the sort and, for the rest of them, by further blocks of the sum's
// launch.  What bounds it: memory, the whole of dW being written (131072 x 2048 bf16,
// 16384 ids: 122 us at 4.9 TB/s), and below some 100 MB the sort.
#include "lg_feat.cuh"

#include "../../include/lanczos_b200.h"

#include <cooperative_groups.h>

namespace lg {
namespace feat {
namespace {

constexpr int kThreads = 256;

__device__ __forceinline__ long long load_id(const void* ids, int ids64, long long t) {
  return ids64 ? static_cast<const long long*>(ids)[t] : (long long)static_cast<const int*>(ids)[t];
}

// ---------------------------------------------------------------------------
// Lookup
// ---------------------------------------------------------------------------
struct GatherArgs {
  long long rows, n, ld;
  int nv, lg;              // vectors per row; log2 of the lanes per row
  const void* ids;
  int ids64, has_pad;
  long long pad;
  const void* scale;       // Acc<T>, one per column
  double value;            // one for all
};

constexpr int kNone = 0, kValue = 1, kColumn = 2;

template <typename T, int V, int MODE>
__device__ __forceinline__ Vec<T, V> gather_value(const Vec<T, V>& x, long long id, bool ok, const GatherArgs& a,
                                                  int c) {
  Vec<T, V> y = x;
  if (MODE == kValue) {
    const Acc<T> s = (Acc<T>)a.value;
#pragma unroll
    for (int k = 0; k < V; ++k) y.v[k] = from_acc<T>(to_acc(x.v[k]) * s);
  } else if (MODE == kColumn) {
    const Acc<T>* s = static_cast<const Acc<T>*>(a.scale) + (long long)c * V;
#pragma unroll
    for (int k = 0; k < V; ++k) y.v[k] = from_acc<T>(to_acc(x.v[k]) * s[k]);
  }
  if (!ok) {
    const bool zero = a.has_pad && id == a.pad;
#pragma unroll
    for (int k = 0; k < V; ++k) y.v[k] = from_acc<T>(zero ? (Acc<T>)0 : (Acc<T>)NAN);
  }
  return y;
}

// WIDE: a warp takes 128 vectors of one row (blockIdx.y: which 128); else a
// group of 1 << lg lanes takes four rows.
template <typename T, int V, int MODE, bool WIDE>
__global__ void __launch_bounds__(kThreads) gather_kernel(GatherArgs a, const T* __restrict__ table,
                                                          T* __restrict__ out) {
  const int lane = threadIdx.x & ((1 << a.lg) - 1);
  const int grp = threadIdx.x >> a.lg, ngrp = kThreads >> a.lg;
  const long long dim = (long long)a.nv * V;
  if (WIDE) {
    const long long t = (long long)blockIdx.x * ngrp + grp;
    if (t >= a.n) return;
    const long long id = load_id(a.ids, a.ids64, t);
    const bool ok = id >= 0 && id < a.rows && !(a.has_pad && id == a.pad);
    const T* src = table + (ok ? id : 0) * a.ld;
    const int c0 = blockIdx.y * 128 + lane;
    Vec<T, V> x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (ok && c0 + 32 * u < a.nv) x[u] = load_vec<T, V>(src + (long long)(c0 + 32 * u) * V);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int c = c0 + 32 * u;
      if (c < a.nv) store_vec<T, V>(out + t * dim + (long long)c * V, gather_value<T, V, MODE>(x[u], id, ok, a, c));
    }
  } else {
    const long long t0 = (long long)blockIdx.x * ngrp * 4 + grp;
    if (lane >= a.nv) return;
    long long id[4];
    bool ok[4];
    Vec<T, V> x[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const long long t = t0 + (long long)u * ngrp;
      id[u] = t < a.n ? load_id(a.ids, a.ids64, t) : -1;
      ok[u] = id[u] >= 0 && id[u] < a.rows && !(a.has_pad && id[u] == a.pad);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (ok[u]) x[u] = load_vec<T, V>(table + id[u] * a.ld + (long long)lane * V);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const long long t = t0 + (long long)u * ngrp;
      if (t < a.n)
        store_vec<T, V>(out + t * dim + (long long)lane * V, gather_value<T, V, MODE>(x[u], id[u], ok[u], a, lane));
    }
  }
}

// The vectors of all rows in one line, four a thread: for rows of up to 48 vectors
// that would leave a sixth of the lanes above idle or more.  Of a table of 20,000 rows,
// which L2 holds: 10^6 ids x 17 fp32: 32 us instead of 59, 10^6 x 10 fp64 20 instead of
// 24, 606,060 x 33 fp32 38 instead of 60; the division by the row length costs more where
// few lanes are idle (198,019 x 101 fp32: 37 instead of 24).
template <typename T, int V, int MODE>
__global__ void __launch_bounds__(kThreads) gather_flat_kernel(GatherArgs a, const T* __restrict__ table,
                                                               T* __restrict__ out) {
  const unsigned total = (unsigned)a.n * (unsigned)a.nv;
  const unsigned p0 = blockIdx.x * (4u * kThreads) + threadIdx.x;
  long long id[4];
  int c[4];
  bool ok[4];
  Vec<T, V> x[4];
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const unsigned p = p0 + u * kThreads, t = p / (unsigned)a.nv;
    c[u] = (int)(p - t * (unsigned)a.nv);
    id[u] = p < total ? load_id(a.ids, a.ids64, t) : -1;
    ok[u] = id[u] >= 0 && id[u] < a.rows && !(a.has_pad && id[u] == a.pad);
  }
#pragma unroll
  for (int u = 0; u < 4; ++u)
    if (ok[u]) x[u] = load_vec<T, V>(table + id[u] * a.ld + (long long)c[u] * V);
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const unsigned p = p0 + u * kThreads;
    if (p < total) store_vec<T, V>(out + (long long)p * V, gather_value<T, V, MODE>(x[u], id[u], ok[u], a, c[u]));
  }
}

template <typename T, int V>
cudaError_t gather_launch(GatherArgs a, int mode, const T* table, T* out, cudaStream_t st) {
  int slots = 1;   // lanes that a row's vectors would get
  while (slots < a.nv) slots *= 2;
  if (a.nv <= 48 && 5 * slots > 6 * a.nv && a.n * a.nv < (1LL << 32) - 4 * kThreads) {
    const unsigned blocks = (unsigned)((a.n * a.nv + 4 * kThreads - 1) / (4 * kThreads));
    if (mode == kNone) gather_flat_kernel<T, V, kNone><<<blocks, kThreads, 0, st>>>(a, table, out);
    else if (mode == kValue) gather_flat_kernel<T, V, kValue><<<blocks, kThreads, 0, st>>>(a, table, out);
    else gather_flat_kernel<T, V, kColumn><<<blocks, kThreads, 0, st>>>(a, table, out);
    return cudaGetLastError();
  }
  const bool wide = a.nv > 32;
  a.lg = 5;
  if (!wide) {
    a.lg = 0;
    while ((1 << a.lg) < a.nv) ++a.lg;
  }
  const long long per = (long long)(kThreads >> a.lg) * (wide ? 1 : 4);
  const dim3 grid((unsigned)((a.n + per - 1) / per), wide ? (unsigned)((a.nv + 127) / 128) : 1u);
  if (wide) {
    if (mode == kNone) gather_kernel<T, V, kNone, true><<<grid, kThreads, 0, st>>>(a, table, out);
    else if (mode == kValue) gather_kernel<T, V, kValue, true><<<grid, kThreads, 0, st>>>(a, table, out);
    else gather_kernel<T, V, kColumn, true><<<grid, kThreads, 0, st>>>(a, table, out);
  } else {
    if (mode == kNone) gather_kernel<T, V, kNone, false><<<grid, kThreads, 0, st>>>(a, table, out);
    else if (mode == kValue) gather_kernel<T, V, kValue, false><<<grid, kThreads, 0, st>>>(a, table, out);
    else gather_kernel<T, V, kColumn, false><<<grid, kThreads, 0, st>>>(a, table, out);
  }
  return cudaGetLastError();
}

// ---------------------------------------------------------------------------
// Stable sort of the ids: least significant digit first, at most 8 bits a
// pass, three kernels a pass.  Every block owns a contiguous span of the
// input, every warp of it a contiguous part; a warp ranks 32 keys at a time by
// matching lanes of equal digit, so equal digits keep their order.
// ---------------------------------------------------------------------------
constexpr int kSortWarps = 8;
constexpr int kSortThreads = kSortWarps * 32;
constexpr int kDigits = 256;
constexpr int kMaxTiles = 296;

struct SortArgs {
  long long n, span;       // span: keys of one block, a multiple of kSortThreads
  unsigned rows;
  int shift, mask, width, tiles;
  const void* ids;         // first pass: the ids themselves
  int ids64, has_pad;
  long long pad;
  const uint2* in;
  uint2* out;
  unsigned* counts;        // [digit][tile], then the totals [digit]
};

__device__ __forceinline__ uint2 sort_pair(const SortArgs& a, long long p) {
  if (a.in) return a.in[p];
  const long long id = load_id(a.ids, a.ids64, p);
  const bool ok = id >= 0 && id < (long long)a.rows && !(a.has_pad && id == a.pad);
  return make_uint2(ok ? (unsigned)id : a.rows, (unsigned)p);
}

// The lanes whose digit (width bits) equals this lane's, among those that are
// `in`; by one vote a bit.  All lanes of the warp vote, always: votes and
// __syncwarps of some of them took 88 us for a sort of 131,072 ids in one cluster,
// these 74 us.
__device__ __forceinline__ unsigned equal_lanes(bool in, unsigned digit, int width) {
  unsigned same = __ballot_sync(0xffffffffu, in);
#pragma unroll
  for (int b = 0; b < 10; ++b) {
    if (b < width) {
      const bool bit = digit >> b & 1u;
      const unsigned vote = __ballot_sync(0xffffffffu, bit);
      same &= bit ? vote : ~vote;
    }
  }
  return same;
}

// Digit counts of the block's span, per warp, in shared memory.
__device__ __forceinline__ void sort_count(const SortArgs& a, unsigned (*cnt)[kDigits]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kSortWarps * kDigits; i += kSortThreads) (&cnt[0][0])[i] = 0;
  __syncthreads();
  const long long part = a.span / kSortWarps;
  const long long p0 = blockIdx.x * a.span + warp * part;
  for (long long i = 0; i < part; i += 128) {
    unsigned key[4];
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const long long p = p0 + i + 32 * u + lane;
      key[u] = i + 32 * u < part && p < a.n ? sort_pair(a, p).x : 0xffffffffu;
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const long long p = p0 + i + 32 * u + lane;
      if (i + 32 * u < part && p < a.n) atomicAdd(&cnt[warp][(key[u] >> a.shift) & a.mask], 1u);
    }
  }
  __syncthreads();
}

__global__ void __launch_bounds__(kSortThreads) sort_count_kernel(SortArgs a) {
  __shared__ unsigned cnt[kSortWarps][kDigits];
  sort_count(a, cnt);
  const int d = threadIdx.x;
  if (d <= a.mask) {
    unsigned s = 0;
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) s += cnt[w][d];
    a.counts[(size_t)d * a.tiles + blockIdx.x] = s;
  }
}

// One warp per digit: exclusive prefix over the tiles, and the digit's total.
__global__ void __launch_bounds__(32) sort_scan_kernel(SortArgs a) {
  unsigned* c = a.counts + (size_t)blockIdx.x * a.tiles;
  unsigned run = 0;
  for (int t0 = 0; t0 < a.tiles; t0 += 32) {
    const int t = t0 + threadIdx.x;
    const unsigned v = t < a.tiles ? c[t] : 0;
    unsigned s = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const unsigned u = __shfl_up_sync(0xffffffffu, s, o);
      if ((int)threadIdx.x >= o) s += u;
    }
    if (t < a.tiles) c[t] = run + s - v;
    run += __shfl_sync(0xffffffffu, s, 31);
  }
  if (threadIdx.x == 0) a.counts[(size_t)kDigits * a.tiles + blockIdx.x] = run;
}

// Exclusive prefix over the values of the block's threads.
__device__ __forceinline__ unsigned digit_prefix(unsigned v, unsigned* scratch) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned s = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned u = __shfl_up_sync(0xffffffffu, s, o);
    if (lane >= o) s += u;
  }
  if (lane == 31) scratch[warp] = s;
  __syncthreads();
  unsigned t = lane < (int)(blockDim.x >> 5) ? scratch[lane] : 0;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned u = __shfl_up_sync(0xffffffffu, t, o);
    if (lane >= o) t += u;
  }
  return (warp ? __shfl_sync(0xffffffffu, t, warp - 1) : 0) + s - v;
}

__global__ void __launch_bounds__(kSortThreads) sort_scatter_kernel(SortArgs a) {
  __shared__ unsigned cnt[kSortWarps][kDigits];
  __shared__ unsigned scratch[kSortWarps];
  sort_count(a, cnt);
  const int d = threadIdx.x;
  const bool used = d <= a.mask;
  unsigned base = digit_prefix(used ? a.counts[(size_t)kDigits * a.tiles + d] : 0, scratch);
  if (used) {
    base += a.counts[(size_t)d * a.tiles + blockIdx.x];
#pragma unroll
    for (int w = 0; w < kSortWarps; ++w) {
      const unsigned c = cnt[w][d];
      cnt[w][d] = base;
      base += c;
    }
  }
  __syncthreads();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long part = a.span / kSortWarps;
  const long long p0 = blockIdx.x * a.span + warp * part;
  for (long long i = 0; i < part; i += 32) {
    const long long p = p0 + i + lane;
    const bool in = p < a.n;
    const uint2 kv = in ? sort_pair(a, p) : make_uint2(0, 0);
    const unsigned dg = (kv.x >> a.shift) & a.mask;
    const unsigned peers = equal_lanes(in, dg, a.width);
    const unsigned rank = __popc(peers & ((1u << lane) - 1));
    const unsigned at = cnt[warp][dg];
    __syncwarp();
    if (in && rank == 0) cnt[warp][dg] = at + __popc(peers);
    __syncwarp();
    if (in) a.out[at + rank] = kv;
  }
}

// ---------------------------------------------------------------------------
// The same sort in one launch, by one cluster of 1, 4 or 8 blocks, for up to
// kClusterMost ids.  The blocks exchange their digit counts through distributed
// shared memory and the pairs through L2; a cluster barrier stands where the other
// form has a launch.  Digits of up to 10 bits, so two passes for up to 2^20 rows.
// Every thread keeps its ITEMS pairs and their places among the equal digits of its
// warp from the counting on.  16384 ids over 131072 rows: 23 us, half of it waiting
// at the barriers for the exchanged counts and the scattered pairs.  (Pairs that stay
// in the shared memory of one block: 35 us, since one SM ranks them all.)
// ---------------------------------------------------------------------------
constexpr int kClusterThreads = 1024;
constexpr int kClusterWarps = kClusterThreads / 32;
constexpr int kClusterCtas = 8;
constexpr int kClusterMost = 16 * kClusterThreads * kClusterCtas;

struct ClusterSortArgs {
  SortArgs s;              // n, rows, ids; in / out as below
  uint2* buf[2];
  int passes, width;
  unsigned* zero;          // words to clear for the kernels that follow
  int nzero;
  SideFill fill;           // bytes to clear by the blocks behind those that sort
};

// The share of block `me` of `all` of the bytes to clear.
__device__ __forceinline__ void side_fill(const SideFill& f, int me, int all) {
  char* p = static_cast<char*>(f.p);
  char* const end = p + f.bytes;
  const long long at = (long long)me * blockDim.x + threadIdx.x, step = (long long)all * blockDim.x;
  const long long skip = (16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15;
  if (at < skip && p + at < end) p[at] = 0;
  p += skip;
  const long long vecs = end > p ? (end - p) / 16 : 0;
  for (long long i = at; i < vecs; i += step) reinterpret_cast<uint4*>(p)[i] = make_uint4(0, 0, 0, 0);
  p += vecs * 16;
  if (p + at < end) p[at] = 0;
}

template <int ITEMS>
__global__ void __launch_bounds__(kClusterThreads, 1) sort_cluster_kernel(ClusterSortArgs c) {
  extern __shared__ __align__(16) unsigned smem[];
  cooperative_groups::cluster_group cluster = cooperative_groups::this_cluster();
  const int ctas = (int)cluster.num_blocks(), me = (int)cluster.block_rank();
  if ((int)blockIdx.x >= ctas) {   // not the first cluster
    side_fill(c.fill, blockIdx.x - ctas, gridDim.x - ctas);
    return;
  }
  const int digits = 1 << c.width, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  unsigned* own = smem + (size_t)warp * digits;                  // counts of this warp, then its places
  unsigned* all = smem + (size_t)kClusterWarps * digits;         // [block][digit] counts
  __shared__ unsigned scratch[kClusterWarps];
  for (int i = me * kClusterThreads + threadIdx.x; i < c.nzero; i += ctas * kClusterThreads) c.zero[i] = 0;
  const long long p0 = ((long long)(me * kClusterWarps + warp) * ITEMS) * 32 + lane;
  cluster.sync();   // every block runs before its shared memory is written
  for (int pass = 0; pass < c.passes; ++pass) {
    SortArgs a = c.s;
    a.in = pass ? c.buf[(pass - 1) & 1] : nullptr;
    const int shift = pass * c.width, mask = digits - 1;
    uint2 kv[ITEMS];
    unsigned place[ITEMS];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const long long p = p0 + 32 * i;
      kv[i] = make_uint2(0, 0);
      if (p < a.n) kv[i] = pass ? __ldcg(a.in + p) : sort_pair(a, p);
    }
    // a warp's counts are its own until the block adds them up
    for (int i = lane * 4; i < digits; i += 128) *reinterpret_cast<uint4*>(own + i) = make_uint4(0, 0, 0, 0);
    __syncwarp();
#pragma unroll
    for (int i = 0; i < ITEMS; ++i) {
      const bool in = p0 + 32 * i < a.n;
      const unsigned d = (kv[i].x >> shift) & mask;
      const unsigned peers = equal_lanes(in, d, c.width);
      const unsigned rank = __popc(peers & ((1u << lane) - 1));
      const unsigned at = own[d];
      __syncwarp();
      if (in && rank == 0) own[d] = at + __popc(peers);
      __syncwarp();
      place[i] = at + rank;
    }
    __syncthreads();
    const int d = threadIdx.x;
    unsigned total = 0;
    if (d < digits) {
#pragma unroll
      for (int w = 0; w < kClusterWarps; ++w) total += smem[w * digits + d];
      for (int q = 0; q < ctas; ++q) cluster.map_shared_rank(all, q)[me * digits + d] = total;
    }
    cluster.sync();
    unsigned below = 0;
    total = 0;
    if (d < digits) {
      for (int q = 0; q < ctas; ++q) {
        const unsigned v = all[q * digits + d];
        if (q < me) below += v;
        total += v;
      }
    }
    unsigned base = digit_prefix(total, scratch) + below;
    if (d < digits) {
#pragma unroll
      for (int w0 = 0; w0 < kClusterWarps; w0 += 8) {
        unsigned v[8];
#pragma unroll
        for (int w = 0; w < 8; ++w) v[w] = smem[(w0 + w) * digits + d];
#pragma unroll
        for (int w = 0; w < 8; ++w) {
          smem[(w0 + w) * digits + d] = base;
          base += v[w];
        }
      }
    }
    __syncthreads();
    uint2* out = c.buf[pass & 1];
#pragma unroll
    for (int i = 0; i < ITEMS; ++i)
      if (p0 + 32 * i < a.n) out[own[(kv[i].x >> shift) & mask] + place[i]] = kv[i];
    cluster.sync();   // the pairs are in memory, and `all` may be written again
  }
}

// Up to kSmallMost ids: every thread counts the pairs before its own, which is the
// place of its pair.  One read of shared memory serves four comparisons of a warp.
constexpr int kSmallMost = 512;

__global__ void __launch_bounds__(kSmallMost) sort_small_kernel(ClusterSortArgs c) {
  __shared__ __align__(16) unsigned key[kSmallMost];
  if (blockIdx.x > 0) {
    side_fill(c.fill, blockIdx.x - 1, gridDim.x - 1);
    return;
  }
  for (int i = threadIdx.x; i < c.nzero; i += kSmallMost) c.zero[i] = 0;
  const int p = threadIdx.x, n = (int)c.s.n;
  uint2 kv = make_uint2(0xffffffffu, 0);
  if (p < n) kv = sort_pair(c.s, p);
  key[p] = kv.x;
  __syncthreads();
  if (p >= n) return;
  int place = 0;
  for (int i = 0; i < n; i += 4) {
    const uint4 k = *reinterpret_cast<const uint4*>(key + i);
    place += (k.x < kv.x || (k.x == kv.x && i < p)) + (k.y < kv.x || (k.y == kv.x && i + 1 < p)) +
             (k.z < kv.x || (k.z == kv.x && i + 2 < p)) + (k.w < kv.x || (k.w == kv.x && i + 3 < p));
  }
  c.buf[0][place] = kv;
}

// Blocks of a sort with clearing.  Clusters of 4 find room on nearly all SMs, which
// clears 128 MB beside the sort of 16384 ids in 26 us; clusters of 8 took 41 us, and
// the sort alone takes 23 us with either.
constexpr int kFillCtas = 144;

template <int ITEMS> cudaError_t launch_cluster_sort(const ClusterSortArgs& c, int ctas, cudaStream_t st) {
  const int smem = (int)sizeof(unsigned) * ((kClusterWarps + kClusterCtas) << c.width);
  static std::atomic<unsigned long long> done{0};
  cudaError_t e = smem_attr_once(done, reinterpret_cast<const void*>(sort_cluster_kernel<ITEMS>),
                                 (int)sizeof(unsigned) * ((kClusterWarps + kClusterCtas) << 10));
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(c.fill.bytes ? kFillCtas : ctas);   // the first cluster sorts
  cfg.blockDim = dim3(kClusterThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = (unsigned)ctas;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, sort_cluster_kernel<ITEMS>, c);
}

int key_bits(long long rows) {   // keys are 0 .. rows
  int b = 1;
  while ((rows >> b) != 0) ++b;
  return b;
}

int sort_tiles(long long n) {
  const long long t = (n + 2047) / 2048;
  return (int)(t < kMaxTiles ? t : kMaxTiles);
}

}  // namespace

size_t sort_ids_workspace(long long rows, long long n) {
  (void)rows;
  return 2 * align_up(sizeof(uint2) * (size_t)n) +
         align_up(sizeof(unsigned) * kDigits * (size_t)(sort_tiles(n) + 1));
}

cudaError_t sort_ids(long long rows, long long n, const void* ids, int ids64, long long pad, int has_pad, void* ws,
                     unsigned* zero, int nzero, SideFill fill, uint2** sorted, cudaStream_t st) {
  uint2* buf[2] = {static_cast<uint2*>(ws),
                   reinterpret_cast<uint2*>(static_cast<char*>(ws) + align_up(sizeof(uint2) * (size_t)n))};
  SortArgs a = {};
  a.n = n;
  a.rows = (unsigned)rows;
  a.ids = ids;
  a.ids64 = ids64;
  a.pad = pad;
  a.has_pad = has_pad;
  const int bits = key_bits(rows);
  if (n <= kClusterMost) {
    ClusterSortArgs c = {};
    c.s = a;
    c.buf[0] = buf[0];
    c.buf[1] = buf[1];
    c.passes = (bits + 9) / 10;
    c.width = (bits + c.passes - 1) / c.passes;
    if (c.width < 2) c.width = 2;   // a row of counts is a multiple of 16 bytes
    c.zero = zero;
    c.nzero = nzero;
    c.fill = fill;
    if (n <= kSmallMost) {
      *sorted = buf[0];
      sort_small_kernel<<<fill.bytes ? 1 + 2 * kFillCtas : 1, kSmallMost, 0, st>>>(c);
      return cudaGetLastError();
    }
    *sorted = buf[(c.passes - 1) & 1];
    constexpr long long four = 4 * kClusterThreads;   // ids of a block
    if (n <= four && !fill.bytes) return launch_cluster_sort<4>(c, 1, st);
    if (n <= 4 * four) return launch_cluster_sort<4>(c, 4, st);
    if (n <= 8 * four) return launch_cluster_sort<4>(c, 8, st);
    return launch_cluster_sort<16>(c, 8, st);
  }
  if (nzero) {
    const cudaError_t e = cudaMemsetAsync(zero, 0, sizeof(unsigned) * (size_t)nzero, st);
    if (e != cudaSuccess) return e;
  }
  if (fill.bytes) {
    const cudaError_t e = cudaMemsetAsync(fill.p, 0, fill.bytes, st);
    if (e != cudaSuccess) return e;
  }
  a.tiles = sort_tiles(n);
  const long long per = (n + a.tiles - 1) / a.tiles;
  a.span = (per + kSortThreads - 1) / kSortThreads * kSortThreads;
  a.counts = reinterpret_cast<unsigned*>(static_cast<char*>(ws) + 2 * align_up(sizeof(uint2) * (size_t)n));
  const int passes = (bits + 7) / 8, width = (bits + passes - 1) / passes;
  for (int k = 0; k < passes; ++k) {
    a.shift = k * width;
    a.mask = (1 << width) - 1;
    a.width = width;
    a.in = k ? buf[(k - 1) & 1] : nullptr;
    a.out = buf[k & 1];
    sort_count_kernel<<<a.tiles, kSortThreads, 0, st>>>(a);
    sort_scan_kernel<<<a.mask + 1, 32, 0, st>>>(a);
    sort_scatter_kernel<<<a.tiles, kSortThreads, 0, st>>>(a);
  }
  *sorted = buf[(passes - 1) & 1];
  return cudaGetLastError();
}

namespace {

// ---------------------------------------------------------------------------
// Sums over the runs of equal ids
// ---------------------------------------------------------------------------
struct SumArgs {
  long long n, ld_g, ld_w;   // ids; row strides of g and of the table
  unsigned rows;
  int nv, lg, tile;          // vectors per row, lanes of a group, positions per group
  int blocks;                // blocks along the positions; those behind them set rows to zero
  int fill;                  // rows per warp of those
  unsigned to_clear;         // the first rows, of which they clear the ones that no id names
  const uint2* sorted;
  unsigned* arrived;         // [column piece][block]: blocks of the run that starts there; [column piece]: blocks done
  int mode;                  // scale
  const void* scale;
  double value;
  void* ds;                  // where the last block to finish writes ds (null: column_sum does)
};

constexpr int kBatch = 4;

// Stores one finished row; adds its part of ds.
template <typename T, int V, bool DS>
__device__ __forceinline__ void finish_row(const SumArgs& a, unsigned v, int c, const Lane<T, V>* acc, const T* W,
                                           T* dW, Lane<T, V>* ds) {
  typedef Lane<T, V> L;
  const long long dim = (long long)a.nv * V, col = (long long)c * V;
  if (DS) {
    const Vec<T, V> w = load_vec<T, V>(W + v * a.ld_w + col);
#pragma unroll
    for (int k = 0; k < lanes<V>; ++k) ds[k] = fma(widen<T, V>(w.v, k), acc[k], ds[k]);
  }
  if (dW) {
    const Acc<T>* s = static_cast<const Acc<T>*>(a.scale) + col;
    Vec<T, V> y;
#pragma unroll
    for (int k = 0; k < lanes<V>; ++k) {
      L f = spread<L>((Acc<T>)a.value);
      if (a.mode == kColumn) f = widen<Acc<T>, V>(s, k);
      narrow<T, V>(a.mode == kNone ? acc[k] : mul(acc[k], f), y.v, k);
    }
    store_vec<T, V>(dW + v * dim + col, y);
  }
}

// Sets the rows that no id names to zero: a warp takes a.fill rows, finds which
// of them the sorted ids hold (one bisection a lane), and clears the others, each
// run of consecutive ones as one range of bytes, so that the row length does not
// matter to the width of the stores.
template <typename T> __device__ __forceinline__ void fill_rows(const SumArgs& a, long long dim, long long block, T* dW) {
  const int lane = threadIdx.x & 31;
  const long long v0 = (block * (kThreads / 32) + (threadIdx.x >> 5)) * a.fill;
  if (v0 >= a.to_clear) return;
  const long long v = v0 + lane;
  bool empty = lane < a.fill && v < a.to_clear;
  if (empty) {
    unsigned lo = 0, hi = (unsigned)a.n;
    while (lo < hi) {
      const unsigned mid = (lo + hi) >> 1;
      if (a.sorted[mid].x < v) lo = mid + 1;
      else hi = mid;
    }
    empty = lo >= a.n || a.sorted[lo].x != v;
  }
  unsigned todo = __ballot_sync(0xffffffffu, empty);
  while (todo) {
    const int first = __ffs(todo) - 1;
    const unsigned rest = ~(todo >> first);
    const int count = rest ? __ffs(rest) - 1 : 32;   // of consecutive rows (a shift by 32 - first fills with zeros)
    todo &= count + first >= 32 ? (1u << first) - 1u : ~(((1u << count) - 1u) << first);
    T* p = dW + (v0 + first) * dim;
    T* const end = p + count * dim;
    const T zero = from_acc<T>((Acc<T>)0);
    // up to the next multiple of 16 bytes, whole vectors, the rest
    const int skip = (int)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / (int)sizeof(T);
    if (lane < skip && p + lane < end) p[lane] = zero;
    p += skip;
    const long long vecs = end > p ? (end - p) / (16 / (long long)sizeof(T)) : 0;
    uint4* q = reinterpret_cast<uint4*>(p);
    for (long long i = lane; i < vecs; i += 32) q[i] = make_uint4(0, 0, 0, 0);
    p += vecs * (16 / sizeof(T));
    if (p + lane < end) p[lane] = zero;
  }
}

// The block in which the run of `key` that enters block b starts, and the one in
// which the run that leaves block b (or is in it) ends; by one warp.  `span` is a
// block's positions.
__device__ __forceinline__ int run_first(const SumArgs& a, unsigned key, long long span, int b) {
  const int lane = threadIdx.x & 31;
  for (int s0 = b - 1;; s0 -= 32) {
    const int s = s0 - lane;
    const bool starts = s <= 0 || a.sorted[s * span - 1].x != key;
    const unsigned m = __ballot_sync(0xffffffffu, starts);
    if (m) return s0 - (__ffs(m) - 1) > 0 ? s0 - (__ffs(m) - 1) : 0;
  }
}
__device__ __forceinline__ int run_last(const SumArgs& a, unsigned key, long long span, int b) {
  const int lane = threadIdx.x & 31;
  for (int e0 = b;; e0 += 32) {
    const int e = e0 + lane;
    const bool ends = (e + 1) * span >= a.n || a.sorted[(e + 1) * span].x != key;
    const unsigned m = __ballot_sync(0xffffffffu, ends);
    if (m) return e0 + __ffs(m) - 1;
  }
}

// part: two rows of sums per block: [0] the run that came in over its left border,
// [1] the run that starts in it and leaves over the right one.  ds_part: two rows
// per block (DS: with the column scale's gradient): the rows that it finished by itself,
// and the run that starts in it and crosses blocks (whichever block adds that up).
//
// Four blocks a SM where 16-byte vectors of fp32 or fp64 would take a few registers too
// many (10^6 ids of 10^6 x 16 fp32: 138 us instead of 154); eight 16-bit values would
// spill (200,000 ids of 1000 x 128 bf16: 57 us instead of 50).
template <typename T, int V, bool DS>
__global__ void __launch_bounds__(kThreads, sizeof(T) >= 4 && sizeof(T) * V == 16 ? 4 : 0)
    sum_kernel(SumArgs a, const T* __restrict__ g, const T* __restrict__ W, T* __restrict__ dW, Acc<T>* part,
               Acc<T>* ds_part) {
  typedef Acc<T> A;
  typedef Lane<T, V> L;
  constexpr int N = lanes<V>;
  __shared__ __align__(16) A head[kThreads * V], tail[kThreads * V];
  __shared__ int flags[kThreads];      // per group
  __shared__ int cross[6];             // first and last block of the two crossing runs; whether to add them up
  griddep_wait();
  // The blocks that sum and those that clear rows alternate, so that the ones'
  // waits for loads run beside the others' stores.
  const long long most = gridDim.x;
  const int block = (int)((long long)blockIdx.x * a.blocks / most);
  if ((int)(((long long)blockIdx.x + 1) * a.blocks / most) == block) {
    fill_rows<T>(a, (long long)a.nv * V, ((long long)blockIdx.x - block) * gridDim.y + blockIdx.y, dW);
    return;
  }
  enum { kCameIn = 1, kGoesOn = 2, kSingle = 4 };
  const int lane = threadIdx.x & ((1 << a.lg) - 1);
  const int grp = threadIdx.x >> a.lg, ngrp = kThreads >> a.lg;
  const int c = (blockIdx.y << a.lg) + lane;
  const long long dim = (long long)a.nv * V, col = (long long)c * V;
  const long long span = (long long)ngrp * a.tile;
  const long long b0 = block * span, b1 = b0 + span < a.n ? b0 + span : a.n;
  const long long p0 = b0 + (long long)grp * a.tile, p1 = p0 + a.tile < a.n ? p0 + a.tile : a.n;
  const bool there = p0 < a.n, on = there && c < a.nv;
  const L zero = spread<L>((A)0);
  L ds[N];
#pragma unroll
  for (int k = 0; k < N; ++k) ds[k] = zero;
  unsigned first = a.rows, last = a.rows;
  int mine = 0;
  if (there) {
    first = a.sorted[p0].x;
    last = a.sorted[p1 - 1].x;
    mine = (first < a.rows && p0 > 0 && a.sorted[p0 - 1].x == first ? kCameIn : 0) |
           (last < a.rows && p1 < a.n && a.sorted[p1].x == last ? kGoesOn : 0) | (first == last ? kSingle : 0);
  }
  if (on && first < a.rows) {
    L acc[N];
#pragma unroll
    for (int k = 0; k < N; ++k) acc[k] = zero;
    unsigned cur = first;
    bool came_in = mine & kCameIn;
    uint2 next[kBatch];   // the pairs of the next batch come while the rows of this one do
#pragma unroll
    for (int u = 0; u < kBatch; ++u) next[u] = p0 + u < p1 ? a.sorted[p0 + u] : make_uint2(a.rows, 0);
    for (long long p = p0; p < p1 && cur < a.rows; p += kBatch) {
      uint2 kv[kBatch];
      Vec<T, V> x[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) kv[u] = next[u];
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (kv[u].x < a.rows) x[u] = load_vec<T, V>(g + kv[u].y * a.ld_g + col);
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        next[u] = p + kBatch + u < p1 ? a.sorted[p + kBatch + u] : make_uint2(a.rows, 0);
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        if (kv[u].x != cur && p + u < p1) {   // the run of `cur` ends inside the tile
          if (came_in) {
#pragma unroll
            for (int k = 0; k < N; ++k) narrow<A, V>(acc[k], head + threadIdx.x * V, k);
          } else if (cur < a.rows) {
            finish_row<T, V, DS>(a, cur, c, acc, W, dW, ds);
          }
          came_in = false;
          cur = kv[u].x;
#pragma unroll
          for (int k = 0; k < N; ++k) acc[k] = zero;
        }
        if (kv[u].x < a.rows) {
#pragma unroll
          for (int k = 0; k < N; ++k) acc[k] = add(acc[k], widen<T, V>(x[u].v, k));
        }
      }
    }
    if (cur < a.rows) {   // the tile's last run
      if (came_in) {
#pragma unroll
        for (int k = 0; k < N; ++k) narrow<A, V>(acc[k], head + threadIdx.x * V, k);
      } else if (mine & kGoesOn) {
#pragma unroll
        for (int k = 0; k < N; ++k) narrow<A, V>(acc[k], tail + threadIdx.x * V, k);
      } else {
        finish_row<T, V, DS>(a, cur, c, acc, W, dW, ds);
      }
    }
  }
  if (lane == 0) flags[grp] = mine;
  __syncthreads();

  // Runs that cross the block's tiles: the group in which one starts adds up the
  // heads of those behind it; the run that came into the block is group 0's too.
  A* mine_part = part + (long long)block * 2 * dim;
  const bool through = (mine & (kCameIn | kSingle | kGoesOn)) == (kCameIn | kSingle | kGoesOn);
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    const bool starts = which == 0 ? grp == 0 && (mine & kCameIn) : (mine & kGoesOn) && !((mine & kCameIn) && (mine & kSingle));
    if (on && starts) {
      L acc[N];
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] = widen<A, V>((which ? tail : head) + threadIdx.x * V, k);
      bool more = which ? true : through;
      int q = grp + 1;
      for (; more && q < ngrp && b0 + (long long)q * a.tile < a.n; ++q) {
#pragma unroll
        for (int k = 0; k < N; ++k) acc[k] = add(acc[k], widen<A, V>(head + ((q << a.lg) + lane) * V, k));
        more = (flags[q] & (kSingle | kGoesOn)) == (kSingle | kGoesOn);
      }
      if (which == 0 || more) {
#pragma unroll
        for (int k = 0; k < N; ++k) narrow<A, V>(acc[k], mine_part + which * dim + col, k);
      } else {
        finish_row<T, V, DS>(a, last, c, acc, W, dW, ds);
      }
    }
  }

  // Runs that cross blocks
  const unsigned key_in = a.sorted[b0].x, key_out = a.sorted[b1 - 1].x;
  const bool enters = b0 > 0 && key_in < a.rows && a.sorted[b0 - 1].x == key_in;
  const bool leaves = b1 < a.n && key_out < a.rows && a.sorted[b1].x == key_out;
  const bool starts_here = leaves && !(enters && key_in == key_out);
  if (enters || starts_here) {
    __threadfence();
    __syncthreads();
    if (threadIdx.x < 32) {
      const int f = enters ? run_first(a, key_in, span, block) : 0, e = enters ? run_last(a, key_in, span, block) : 0;
      const int e2 = starts_here ? run_last(a, key_out, span, block) : 0;
      if (threadIdx.x == 0) {
        unsigned* n = a.arrived + (size_t)blockIdx.y * a.blocks;
        cross[0] = f;
        cross[1] = e;
        cross[2] = enters && atomicAdd(n + f, 1u) == (unsigned)(e - f);
        cross[3] = block;
        cross[4] = e2;
        cross[5] = starts_here && atomicAdd(n + block, 1u) == (unsigned)(e2 - (int)block);
      }
    }
    __syncthreads();
    __threadfence();
#pragma unroll 1
    for (int which = 0; which < 2; ++which) {
      if (!cross[3 * which + 2]) continue;
      const int f = cross[3 * which], count = cross[3 * which + 1] - f + 1, each = (count + ngrp - 1) / ngrp;
      L acc[N], join[N];
#pragma unroll
      for (int k = 0; k < N; ++k) acc[k] = join[k] = zero;
      if (c < a.nv) {
        const int to = (grp + 1) * each < count ? (grp + 1) * each : count;
#pragma unroll 4
        for (int i = grp * each; i < to; ++i) {
          const A* o = part + ((long long)(f + i) * 2 + (i == 0 ? 1 : 0)) * dim + col;
          A v[V];
#pragma unroll
          for (int k = 0; k < V; ++k) v[k] = __ldcg(o + k);
#pragma unroll
          for (int k = 0; k < N; ++k) acc[k] = add(acc[k], widen<A, V>(v, k));
        }
      }
      __syncthreads();
#pragma unroll
      for (int k = 0; k < N; ++k) narrow<A, V>(acc[k], head + threadIdx.x * V, k);
      __syncthreads();
      if (grp == 0 && c < a.nv) {
        for (int q = 1; q < ngrp; ++q) {
#pragma unroll
          for (int k = 0; k < N; ++k) acc[k] = add(acc[k], widen<A, V>(head + ((q << a.lg) + lane) * V, k));
        }
        finish_row<T, V, DS>(a, which ? key_out : key_in, c, acc, W, dW, join);
        if (DS) {
#pragma unroll
          for (int k = 0; k < N; ++k) narrow<A, V>(join[k], ds_part + ((long long)f * 2 + 1) * dim + col, k);
        }
      }
    }
  }
  if (DS) {
    __syncthreads();
#pragma unroll
    for (int k = 0; k < N; ++k) narrow<A, V>(ds[k], head + threadIdx.x * V, k);
    __syncthreads();
    if (grp == 0 && c < a.nv) {
      for (int q = 1; q < ngrp; ++q) {
#pragma unroll
        for (int k = 0; k < N; ++k) ds[k] = add(ds[k], widen<A, V>(head + ((q << a.lg) + lane) * V, k));
      }
      A* o = ds_part + (long long)block * 2 * dim + col;
#pragma unroll
      for (int k = 0; k < N; ++k) {
        narrow<A, V>(ds[k], o, k);
        if (!starts_here) narrow<A, V>(zero, o + dim, k);
      }
    }
    if (a.ds) {
      __threadfence();
      __syncthreads();
      if (threadIdx.x == 0)
        cross[0] = atomicAdd(a.arrived + (size_t)gridDim.y * a.blocks + blockIdx.y, 1u) == (unsigned)a.blocks - 1;
      __syncthreads();
      if (!cross[0]) return;
      __threadfence();
      L all[N];
#pragma unroll
      for (int k = 0; k < N; ++k) all[k] = zero;
      if (c < a.nv) {
#pragma unroll 8
        for (int r = grp; r < 2 * a.blocks; r += ngrp) {
          A v[V];
#pragma unroll
          for (int k = 0; k < V; ++k) v[k] = __ldcg(ds_part + r * dim + col + k);
#pragma unroll
          for (int k = 0; k < N; ++k) all[k] = add(all[k], widen<A, V>(v, k));
        }
      }
#pragma unroll
      for (int k = 0; k < N; ++k) narrow<A, V>(all[k], head + threadIdx.x * V, k);
      __syncthreads();
      if (grp == 0 && c < a.nv) {
        for (int q = 1; q < ngrp; ++q) {
#pragma unroll
          for (int k = 0; k < N; ++k) all[k] = add(all[k], widen<A, V>(head + ((q << a.lg) + lane) * V, k));
        }
#pragma unroll
        for (int k = 0; k < N; ++k) narrow<A, V>(all[k], static_cast<A*>(a.ds) + col, k);
      }
    }
  }
}

struct SumPlan {
  int lg, cols, tile, blocks, fill;
};

// Tiles of 4 to 32 positions (more where that would leave over 2^16 blocks): as
// long as they leave four blocks a SM.
constexpr int kSms = 148;   // of a B200

// Bytes cleared beside the sort: about what the SMs that do not sort write in the time of
// one of 16384 ids (23 us).  131072 x 2048 bf16 with 16384 ids: 122 us, 146 us with none,
// 130 us with all 537 MB cleared there.  Sorts of fewer ids end before the clearing, those
// of up to 131,072 (74 us) after it; what is not cleared here is by the sum's launch.
constexpr long long kSideFillMost = 128LL << 20;

SumPlan sum_plan(long long n, int nv, long long row_bytes) {
  SumPlan p;
  p.lg = 0;
  while (p.lg < 5 && (1 << p.lg) < nv) ++p.lg;
  p.cols = (nv + (1 << p.lg) - 1) >> p.lg;
  const int ngrp = kThreads >> p.lg;
  p.tile = 4;
  while ((p.tile < 32 && n * p.cols > 2LL * p.tile * ngrp * 4 * kSms) || n / ((long long)p.tile * ngrp) > 65536) p.tile *= 2;
  p.blocks = (int)((n + (long long)p.tile * ngrp - 1) / ((long long)p.tile * ngrp));
  p.fill = row_bytes >= 32768 ? 1 : 32768 / (int)row_bytes < 32 ? 32768 / (int)row_bytes : 32;   // 32 KB a warp
  return p;
}

// Up to this many blocks for each group of lanes the last block of the sum to finish
// adds up ds itself, 32 partial rows a group, which saves a launch (100,000 x 20 fp64,
// 8192 ids: 58.6 us instead of 63.5 with the call's host time); beyond, column_sum with its wider grid.
constexpr int kLastBlockRows = 16;

struct ScatterLayout {
  size_t sort, arrived, part, ds, total;
};

// Room for any vector width that the addresses allow.
ScatterLayout scatter_layout(long long rows, int dim, int dtype, long long n, int want_ds) {
  const int es = acc_size(dtype), widest = 16 / elem_size(dtype);
  size_t blocks = 0, pieces = 0;
  for (int v = 1; v <= widest; v *= 2) {
    if (dim % v) break;
    const SumPlan p = sum_plan(n, dim / v, (long long)dim * elem_size(dtype));
    if ((size_t)p.blocks > blocks) blocks = p.blocks;
    if ((size_t)(p.blocks + 1) * p.cols > pieces) pieces = (size_t)(p.blocks + 1) * p.cols;
  }
  ScatterLayout l;
  l.sort = align_up(sort_ids_workspace(rows, n));
  l.arrived = align_up(sizeof(unsigned) * pieces);
  l.part = align_up(blocks * 2 * dim * es);
  l.ds = want_ds ? align_up(blocks * 2 * dim * es) : 0;
  l.total = l.sort + l.arrived + l.part + l.ds;
  return l;
}

template <typename T, int V>
cudaError_t scatter_launch(SumArgs a, int dim, const T* g, const T* W, T* dW, void* d_scale, char* part, char* ds,
                           const SumPlan& p, int fill, cudaStream_t st) {
  a.nv = dim / V;
  a.lg = p.lg;
  a.tile = p.tile;
  a.blocks = p.blocks;
  a.fill = p.fill;
  Acc<T>* pt = reinterpret_cast<Acc<T>*>(part);
  Acc<T>* dp = reinterpret_cast<Acc<T>*>(ds);
  a.ds = p.blocks <= kLastBlockRows * (kThreads >> p.lg) ? d_scale : nullptr;
  const dim3 grid(p.blocks + fill, p.cols);
  const cudaError_t e =
      d_scale ? launch_pdl(sum_kernel<T, V, true>, grid, dim3(kThreads), 0, st, a, g, W, dW, pt, dp)
              : launch_pdl(sum_kernel<T, V, false>, grid, dim3(kThreads), 0, st, a, g, W, dW, pt, dp);
  if (e != cudaSuccess || !d_scale || a.ds) return e;
  return column_sum(dp, 2 * p.blocks, dim, dim, static_cast<Acc<T>*>(d_scale), st);
}

bool rows_args_ok(long long rows, int dim, int dtype, long long n, const void* ids, int mode, const void* scale) {
  return rows >= 1 && rows < 2147483647LL && dim >= 1 && dim <= (1 << 20) && n >= 1 && n < 2147483647LL && ids &&
         elem_size(dtype) && mode >= 0 && mode <= 2 && (mode != kColumn || scale);
}

}  // namespace
}  // namespace feat
}  // namespace lg

using namespace lg;
using namespace lg::feat;

// Calls F<T, V>(...) for the element type and the vector width.
#define LG_ROWS_DISPATCH(F)                                                              \
  switch (dtype) {                                                                       \
    case LG_F64: return vec >= 2 ? F(double, 2) : F(double, 1);                          \
    case LG_F32: return vec >= 4 ? F(float, 4) : vec == 2 ? F(float, 2) : F(float, 1);   \
    case LG_F16:                                                                         \
      return vec >= 8 ? F(__half, 8) : vec == 4 ? F(__half, 4) : vec == 2 ? F(__half, 2) : F(__half, 1); \
    default:                                                                             \
      return vec >= 8 ? F(__nv_bfloat16, 8) : vec == 4 ? F(__nv_bfloat16, 4)             \
             : vec == 2 ? F(__nv_bfloat16, 2) : F(__nv_bfloat16, 1);                     \
  }

extern "C" int lg_rows_gather(long long rows, int dim, int dtype, const void* table, long long ld_table, long long n,
                              const void* ids, int ids64, int scale_mode, const void* scale, double scale_value,
                              int has_padding, long long padding, void* out, void* stream) {
  if (!rows_args_ok(rows, dim, dtype, n, ids, scale_mode, scale) || !table || !out || ld_table < dim ||
      !aligned(elem_size(dtype), table, out) || !aligned(ids64 ? 8 : 4, ids) || !aligned(acc_size(dtype), scale))
    return bad_args("lg_rows_gather: invalid arguments");
  GatherArgs a = {};
  a.rows = rows;
  a.n = n;
  a.ld = ld_table;
  a.ids = ids;
  a.ids64 = ids64;
  a.has_pad = has_padding;
  a.pad = padding;
  a.scale = scale;
  a.value = scale_value;
  Align al(elem_size(dtype));
  al.address(table);
  al.address(out);
  al.elements(ld_table);
  al.elements(dim);
  const int vec = al.vec();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto run = [&]() -> cudaError_t {
#define LG_F(T, V) (a.nv = dim / V, gather_launch<T, V>(a, scale_mode, static_cast<const T*>(table), static_cast<T*>(out), st))
    LG_ROWS_DISPATCH(LG_F)
#undef LG_F
  };
  return cuda_status(run(), "lg_rows_gather");
}

extern "C" size_t lg_rows_scatter_workspace_bytes(long long rows, int dim, int dtype, long long n, int want_scale) {
  if (!rows_args_ok(rows, dim, dtype, n, &rows, 0, nullptr)) return 0;
  return scatter_layout(rows, dim, dtype, n, want_scale).total;
}

extern "C" int lg_rows_scatter(long long rows, int dim, int dtype, const void* table, long long ld_table, long long n,
                               const void* ids, int ids64, int scale_mode, const void* scale, double scale_value,
                               int has_padding, long long padding, const void* g, long long ld_g, void* d_table,
                               void* d_scale, void* ws, size_t ws_bytes, void* stream) {
  if (!rows_args_ok(rows, dim, dtype, n, ids, scale_mode, scale) || !g || ld_g < dim || !ws || (!d_table && !d_scale) ||
      (d_scale && (!table || ld_table < dim || scale_mode != kColumn)) || !aligned(elem_size(dtype), table, g, d_table) ||
      !aligned(acc_size(dtype), scale, d_scale) || !aligned(ids64 ? 8 : 4, ids) || !aligned(kWsAlign, ws))
    return bad_args("lg_rows_scatter: invalid arguments");
  const ScatterLayout l = scatter_layout(rows, dim, dtype, n, d_scale != nullptr);
  if (ws_bytes < l.total) return bad_args("lg_rows_scatter: workspace too small");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  char* w = static_cast<char*>(ws);
  Align al(elem_size(dtype));
  al.address(g);
  al.elements(ld_g);
  al.elements(dim);
  if (d_table) al.address(d_table);
  if (d_scale) {
    al.address(table);
    al.elements(ld_table);
  }
  const int vec = al.vec();
  const SumPlan p = sum_plan(n, dim / vec, (long long)dim * elem_size(dtype));
  SumArgs a = {};
  a.n = n;
  a.ld_g = ld_g;
  a.ld_w = ld_table;
  a.rows = (unsigned)rows;
  a.mode = scale_mode;
  a.scale = scale;
  a.value = scale_value;
  a.arrived = reinterpret_cast<unsigned*>(w + l.sort);
  uint2* sorted = nullptr;
  // The sort keeps a few SMs busy for 10 to 30 us.  The others clear the last rows of
  // the gradient meanwhile, of which those that ids name are then written twice; the
  // sum's launch clears what is left of the rows that no id names.
  const long long row_bytes = (long long)dim * elem_size(dtype);
  long long cleared = 0;
  if (d_table && n <= kClusterMost && n < rows) {
    cleared = kSideFillMost / row_bytes;
    if (cleared > rows) cleared = rows;
  }
  SideFill side = {nullptr, 0};
  if (cleared) side = {static_cast<char*>(d_table) + (rows - cleared) * row_bytes, (size_t)(cleared * row_bytes)};
  a.to_clear = (unsigned)(d_table ? rows - cleared : 0);
  const cudaError_t e =
      sort_ids(rows, n, ids, ids64, padding, has_padding, w, a.arrived, (p.blocks + 1) * p.cols, side, &sorted, st);
  if (e != cudaSuccess) return cuda_status(e, "lg_rows_scatter");
  a.sorted = sorted;
  const long long per = (long long)p.fill * (kThreads / 32) * p.cols;
  const int fill_blocks = (int)((a.to_clear + per - 1) / per);
  auto run = [&]() -> cudaError_t {
#define LG_F(T, V)                                                                                                  \
  scatter_launch<T, V>(a, dim, static_cast<const T*>(g), static_cast<const T*>(table), static_cast<T*>(d_table), \
                       d_scale, w + l.sort + l.arrived, w + l.sort + l.arrived + l.part, p, fill_blocks, st)
    LG_ROWS_DISPATCH(LG_F)
#undef LG_F
  };
  return cuda_status(run(), "lg_rows_scatter");
}
