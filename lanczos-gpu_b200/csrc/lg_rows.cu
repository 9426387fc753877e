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
// pieces of a row (long rows) in flight before the first store.  Bound by
// memory: nothing is reused but rows named twice.
//
// Gradient: the ids are sorted (stable, with their positions), the sorted
// positions are cut into tiles of equal length, and a group of lanes sums the
// rows of one tile, one vector of columns per lane.  Equal tiles keep the work
// even whatever the distribution of the ids.  A run of equal ids inside a tile
// is finished and written at once; one that crosses a tile's border leaves
// partial sums (Acc<T>) that the join kernel adds in tile order.  No atomics:
// the result does not change from run to run.
#include "lg_feat.cuh"

#include "../../include/lanczos_b200.h"

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

template <typename T, int V>
cudaError_t gather_launch(GatherArgs a, int mode, const T* table, T* out, cudaStream_t st) {
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
  int shift, mask, tiles;
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

// Digit counts of the block's span, per warp, in shared memory.
__device__ __forceinline__ void sort_count(const SortArgs& a, unsigned (*cnt)[kDigits]) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kSortWarps * kDigits; i += kSortThreads) (&cnt[0][0])[i] = 0;
  __syncthreads();
  const long long part = a.span / kSortWarps;
  const long long p0 = blockIdx.x * a.span + warp * part;
  for (long long i = 0; i < part; i += 32) {
    const long long p = p0 + i + lane;
    if (p < a.n) atomicAdd(&cnt[warp][(sort_pair(a, p).x >> a.shift) & a.mask], 1u);
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

// Exclusive prefix over kDigits values, one per thread (256 threads).
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
  unsigned base = 0;
  for (int w = 0; w < warp; ++w) base += scratch[w];
  return base + s - v;
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
    const unsigned act = __ballot_sync(0xffffffffu, in);
    if (!act) break;
    if (in) {
      const uint2 kv = sort_pair(a, p);
      const unsigned dg = (kv.x >> a.shift) & a.mask;
      const unsigned peers = __match_any_sync(act, dg);
      const unsigned rank = __popc(peers & ((1u << lane) - 1));
      const unsigned at = cnt[warp][dg];
      __syncwarp(act);
      if (rank == 0) cnt[warp][dg] = at + __popc(peers);
      __syncwarp(act);
      a.out[at + rank] = kv;
    }
  }
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
                     uint2** sorted, cudaStream_t st) {
  uint2* buf[2] = {static_cast<uint2*>(ws),
                   reinterpret_cast<uint2*>(static_cast<char*>(ws) + align_up(sizeof(uint2) * (size_t)n))};
  SortArgs a = {};
  a.n = n;
  a.rows = (unsigned)rows;
  a.tiles = sort_tiles(n);
  const long long per = (n + a.tiles - 1) / a.tiles;
  a.span = (per + kSortThreads - 1) / kSortThreads * kSortThreads;
  a.ids = ids;
  a.ids64 = ids64;
  a.pad = pad;
  a.has_pad = has_pad;
  a.counts = reinterpret_cast<unsigned*>(static_cast<char*>(ws) + 2 * align_up(sizeof(uint2) * (size_t)n));
  const int bits = key_bits(rows), passes = (bits + 7) / 8, width = (bits + passes - 1) / passes;
  for (int k = 0; k < passes; ++k) {
    a.shift = k * width;
    a.mask = (1 << width) - 1;
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
  int nv, lg, tile, tiles;   // vectors per row, lanes, positions per tile, tiles
  const uint2* sorted;
  int mode;                  // scale
  const void* scale;
  double value;
  int want_ds;
};

constexpr int kBatch = 8;

// Stores one finished row; adds its part of ds.
template <typename T, int V>
__device__ __forceinline__ void finish_row(const SumArgs& a, unsigned v, int c, const Acc<T>* acc, const T* W, T* dW,
                                           Acc<T>* ds) {
  const long long dim = (long long)a.nv * V, col = (long long)c * V;
  if (a.want_ds) {
    const Vec<T, V> w = load_vec<T, V>(W + v * a.ld_w + col);
#pragma unroll
    for (int k = 0; k < V; ++k) ds[k] += to_acc(w.v[k]) * acc[k];
  }
  if (dW) {
    const Acc<T>* s = static_cast<const Acc<T>*>(a.scale) + col;
    Vec<T, V> y;
#pragma unroll
    for (int k = 0; k < V; ++k)
      y.v[k] = from_acc<T>(a.mode == kNone ? acc[k] : acc[k] * (a.mode == kValue ? (Acc<T>)a.value : s[k]));
    store_vec<T, V>(dW + v * dim + col, y);
  }
}

// Sum of the block's ds over its groups, written as one partial row.
template <typename T, int V>
__device__ __forceinline__ void block_ds(const SumArgs& a, int lane, int grp, int ngrp, int c, const Acc<T>* ds,
                                         Acc<T>* row) {
  __shared__ Acc<T> red[kThreads];
#pragma unroll
  for (int k = 0; k < V; ++k) {
    __syncthreads();
    red[threadIdx.x] = ds[k];
    __syncthreads();
    if (grp == 0 && c < a.nv) {
      Acc<T> s = 0;
      for (int g = 0; g < ngrp; ++g) s += red[(g << a.lg) + lane];
      row[(long long)c * V + k] = s;
    }
  }
}

// part: two rows of nv * V sums per tile: [0] the run that came in over the
// tile's left border, [1] the run that starts here and leaves over the right.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) sum_kernel(SumArgs a, const T* __restrict__ g, const T* __restrict__ W,
                                                       T* __restrict__ dW, Acc<T>* __restrict__ part,
                                                       Acc<T>* __restrict__ ds_part) {
  const int lane = threadIdx.x & ((1 << a.lg) - 1);
  const int grp = threadIdx.x >> a.lg, ngrp = kThreads >> a.lg;
  const int c = (blockIdx.y << a.lg) + lane;
  const long long t = (long long)blockIdx.x * ngrp + grp;
  const long long dim = (long long)a.nv * V;
  Acc<T> ds[V];
#pragma unroll
  for (int k = 0; k < V; ++k) ds[k] = 0;
  const bool on = t < a.tiles && c < a.nv;
  const long long p0 = t * a.tile;
  const long long p1 = p0 + a.tile < a.n ? p0 + a.tile : a.n;
  if (on) {
    const unsigned before = p0 > 0 ? a.sorted[p0 - 1].x : 0xffffffffu;
    const unsigned after = p1 < a.n ? a.sorted[p1].x : 0xffffffffu;
    Acc<T> acc[V];
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] = 0;
    unsigned cur = a.sorted[p0].x;
    bool came_in = cur == before;
    for (long long p = p0; p < p1 && cur < a.rows; p += kBatch) {
      uint2 kv[kBatch];
      Vec<T, V> x[kBatch];
#pragma unroll
      for (int u = 0; u < kBatch; ++u) kv[u] = p + u < p1 ? a.sorted[p + u] : make_uint2(a.rows, 0);
#pragma unroll
      for (int u = 0; u < kBatch; ++u)
        if (kv[u].x < a.rows) x[u] = load_vec<T, V>(g + kv[u].y * a.ld_g + (long long)c * V);
#pragma unroll
      for (int u = 0; u < kBatch; ++u) {
        if (kv[u].x != cur) {
          if (p + u < p1) {   // the run of `cur` ends inside the tile
            if (came_in) {
              Acc<T>* o = part + 2 * t * dim + (long long)c * V;
#pragma unroll
              for (int k = 0; k < V; ++k) o[k] = acc[k];
            } else if (cur < a.rows) {
              finish_row<T, V>(a, cur, c, acc, W, dW, ds);
            }
            came_in = false;
            cur = kv[u].x;
#pragma unroll
            for (int k = 0; k < V; ++k) acc[k] = 0;
          }
        }
        if (kv[u].x < a.rows) {
#pragma unroll
          for (int k = 0; k < V; ++k) acc[k] += to_acc(x[u].v[k]);
        }
      }
    }
    if (cur < a.rows) {   // the last run of the tile
      if (came_in || cur == after) {
        Acc<T>* o = part + (2 * t + (came_in ? 0 : 1)) * dim + (long long)c * V;
#pragma unroll
        for (int k = 0; k < V; ++k) o[k] = acc[k];
      } else {
        finish_row<T, V>(a, cur, c, acc, W, dW, ds);
      }
    }
  }
  if (a.want_ds) block_ds<T, V>(a, lane, grp, ngrp, c, ds, ds_part + blockIdx.x * dim);
}

// First position of the sorted pairs with a key above `key`, in [lo, n).
__device__ __forceinline__ long long run_end(const uint2* sorted, long long lo, long long n, unsigned key) {
  long long hi = n;
  while (lo < hi) {
    const long long mid = (lo + hi) >> 1;
    if (sorted[mid].x <= key) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

// The runs that cross tile borders: a block takes the run that starts in tile
// t and leaves it, its groups sum contiguous parts of the list of partial
// rows, and the groups' sums are added in order.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) join_kernel(SumArgs a, const T* __restrict__ W, T* __restrict__ dW,
                                                        const Acc<T>* __restrict__ part,
                                                        Acc<T>* __restrict__ ds_part) {
  __shared__ Acc<T> red[kThreads * V];
  const int lane = threadIdx.x & ((1 << a.lg) - 1);
  const int grp = threadIdx.x >> a.lg, ngrp = kThreads >> a.lg;
  const int c = (blockIdx.y << a.lg) + lane;
  const long long dim = (long long)a.nv * V;
  Acc<T> ds[V];
#pragma unroll
  for (int k = 0; k < V; ++k) ds[k] = 0;
  for (long long t = blockIdx.x; t + 1 < a.tiles; t += gridDim.x) {
    const long long p0 = t * a.tile, p1 = p0 + a.tile;
    const unsigned key = a.sorted[p1].x;
    if (key >= a.rows || a.sorted[p1 - 1].x != key) continue;            // no run leaves tile t
    if (p0 > 0 && a.sorted[p0 - 1].x == key) continue;                   // it started in an earlier tile
    const long long end = run_end(a.sorted, p1, a.n, key);
    const long long last = (end - 1) / a.tile;                           // partial rows t, t + 1 .. last
    const long long count = last - t + 1, each = (count + ngrp - 1) / ngrp;
    Acc<T> acc[V];
#pragma unroll
    for (int k = 0; k < V; ++k) acc[k] = 0;
    if (c < a.nv) {
      const long long e = (grp + 1) * each < count ? (grp + 1) * each : count;
#pragma unroll 4
      for (long long i = grp * each; i < e; ++i) {
        const Acc<T>* o = part + (2 * (t + i) + (i == 0 ? 1 : 0)) * dim + (long long)c * V;
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] += o[k];
      }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < V; ++k) red[threadIdx.x * V + k] = acc[k];
    __syncthreads();
    if (grp == 0 && c < a.nv) {
      for (int q = 1; q < ngrp; ++q) {
#pragma unroll
        for (int k = 0; k < V; ++k) acc[k] += red[((q << a.lg) + lane) * V + k];
      }
      finish_row<T, V>(a, key, c, acc, W, dW, ds);
    }
  }
  if (a.want_ds) block_ds<T, V>(a, lane, grp, ngrp, c, ds, ds_part + blockIdx.x * dim);
}

// How the sorted positions are cut: 32 to a tile, a power of two more when
// that would leave over 2^16 tiles.
int sum_tile(long long n) {
  int t = 32;
  while (n / t > 65536) t *= 2;
  return t;
}

struct SumPlan {
  int tile, tiles, lg, cols, blocks, join;   // cols: column pieces; blocks, join: blocks along the tiles
};

SumPlan sum_plan(long long n, int nv) {
  SumPlan p;
  p.tile = sum_tile(n);
  p.tiles = (int)((n + p.tile - 1) / p.tile);
  p.lg = 0;
  while (p.lg < 5 && (1 << p.lg) < nv) ++p.lg;
  p.cols = (nv + (1 << p.lg) - 1) >> p.lg;
  const int ngrp = kThreads >> p.lg;
  p.blocks = (p.tiles + ngrp - 1) / ngrp;
  p.join = p.tiles < 1024 ? p.tiles : 1024;
  return p;
}

struct ScatterLayout {
  size_t sort, part, ds, total;
};

// Sizes do not depend on the addresses: the vector may be as narrow as one
// element, which has the most column pieces and the same rows.
ScatterLayout scatter_layout(long long rows, int dim, int dtype, long long n, int want_ds) {
  const SumPlan p1 = sum_plan(n, dim);
  const int es = acc_size(dtype);
  ScatterLayout l;
  l.sort = align_up(sort_ids_workspace(rows, n));
  l.part = align_up((size_t)2 * p1.tiles * dim * es);
  // partial rows of ds: the fewest groups per block (32 lanes) give the most blocks
  const size_t blocks = (size_t)(p1.tiles + 7) / 8 + 1024;
  l.ds = want_ds ? align_up(blocks * dim * es) : 0;
  l.total = l.sort + l.part + l.ds;
  return l;
}

template <typename T, int V>
cudaError_t scatter_launch(SumArgs a, int dim, const T* g, const T* W, T* dW, void* d_scale, char* part, char* ds,
                           cudaStream_t st) {
  const SumPlan p = sum_plan(a.n, dim / V);
  a.nv = dim / V;
  a.lg = p.lg;
  a.tile = p.tile;
  a.tiles = p.tiles;
  Acc<T>* pt = reinterpret_cast<Acc<T>*>(part);
  Acc<T>* dp = reinterpret_cast<Acc<T>*>(ds);
  sum_kernel<T, V><<<dim3(p.blocks, p.cols), kThreads, 0, st>>>(a, g, W, dW, pt, dp);
  int rows = p.blocks;
  if (p.tiles > 1) {
    join_kernel<T, V><<<dim3(p.join, p.cols), kThreads, 0, st>>>(a, W, dW, pt, dp + (size_t)rows * dim);
    rows += p.join;
  }
  cudaError_t e = cudaGetLastError();
  if (e == cudaSuccess && a.want_ds) e = column_sum(dp, rows, dim, dim, static_cast<Acc<T>*>(d_scale), st);
  return e;
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
  if (!rows_args_ok(rows, dim, dtype, n, ids, scale_mode, scale) || !table || !out || ld_table < dim)
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
      (d_scale && (!table || ld_table < dim || scale_mode != kColumn)))
    return bad_args("lg_rows_scatter: invalid arguments");
  const ScatterLayout l = scatter_layout(rows, dim, dtype, n, d_scale != nullptr);
  if (ws_bytes < l.total) return bad_args("lg_rows_scatter: workspace too small");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  char* w = static_cast<char*>(ws);
  SumArgs a = {};
  a.n = n;
  a.ld_g = ld_g;
  a.ld_w = ld_table;
  a.rows = (unsigned)rows;
  a.mode = scale_mode;
  a.scale = scale;
  a.value = scale_value;
  a.want_ds = d_scale != nullptr;
  uint2* sorted = nullptr;
  cudaError_t e = sort_ids(rows, n, ids, ids64, padding, has_padding, w, &sorted, st);
  if (e == cudaSuccess && d_table)
    e = cudaMemsetAsync(d_table, 0, (size_t)rows * dim * elem_size(dtype), st);
  if (e != cudaSuccess) return cuda_status(e, "lg_rows_scatter");
  a.sorted = sorted;
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
  auto run = [&]() -> cudaError_t {
#define LG_F(T, V)                                                                                                  \
  scatter_launch<T, V>(a, dim, static_cast<const T*>(g), static_cast<const T*>(table), static_cast<T*>(d_table), \
                       d_scale, w + l.sort, w + l.sort + l.part, st)
    LG_ROWS_DISPATCH(LG_F)
#undef LG_F
  };
  return cuda_status(run(), "lg_rows_scatter");
}
