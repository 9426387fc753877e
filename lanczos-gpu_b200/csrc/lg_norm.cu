// lg_norm.cu — layer norm over the last dimension, forward and backward.
//
//   mu = mean(x),  r = 1 / sqrt(mean((x - mu)^2) + eps),  h = (x - mu) r
//   y  = h w + b
//   dx = r (wg - mean(wg) - h mean(wg h)),   wg = w g
//   dw = sum over rows of g h,   db = sum over rows of g
//
// A row is held in registers by a team of threads (a power of two: part of a
// warp for short rows, a whole block for long ones), so x is read once and the
// variance is the second pass over registers, about the row's own mean.  The
// backward pass reads x and g once each; every thread keeps the same columns
// for all rows of its block, so dw and db grow in registers and leave as one
// partial row per block, summed by column_sum in a fixed order.  Rows too long
// for the registers of a block go through the *_long kernels, which pass over
// the row in memory (it stays in L2).
#include "lg_feat.cuh"

#include "../../include/lanczos_b200.h"

namespace lg {
namespace feat {
namespace {

struct NormArgs {
  long long rows, ld_x, ld_g;
  int dim, nv, lg;       // row length, vectors per row, log2 of the team
  double eps;
  const void* w;         // weight and bias: the element type, or float
  const void* b;
  int w_float;
  int want_dw, want_db;
};

// One value of the weight or the bias.
template <typename T> __device__ __forceinline__ Acc<T> param(const void* p, int is_float, long long i) {
  return is_float ? (Acc<T>)static_cast<const float*>(p)[i] : to_acc(static_cast<const T*>(p)[i]);
}

__device__ __forceinline__ float rsqrt_acc(float v) { return 1.0f / sqrtf(v); }
__device__ __forceinline__ double rsqrt_acc(double v) { return 1.0 / sqrt(v); }

// Sum over a team of 1 << lg threads (lg <= 5: lanes of a warp; else the whole
// block, through shared memory); the result reaches every thread of the team.
template <typename A> __device__ __forceinline__ A team_sum(A v, int lg, A* scratch) {
  const int width = lg < 5 ? 1 << lg : 32;
  for (int o = width >> 1; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (lg <= 5) return v;
  const int warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[warp] = v;
  __syncthreads();
  A t = 0;
  for (int w = 0; w < nw; ++w) t += scratch[w];
  return t;
}

template <typename T, int V, int K>
__global__ void __launch_bounds__(1024) norm_forward_kernel(NormArgs a, const T* __restrict__ x, T* __restrict__ y,
                                                            Acc<T>* __restrict__ mean, Acc<T>* __restrict__ rstd) {
  typedef Acc<T> A;
  __shared__ A scratch[32];
  const int team = 1 << a.lg, me = threadIdx.x & (team - 1);
  const int per = blockDim.x >> a.lg;
  const A inv = (A)1 / (A)a.dim;
  for (long long r0 = (long long)blockIdx.x * per; r0 < a.rows; r0 += (long long)gridDim.x * per) {
    const long long row = r0 + (threadIdx.x >> a.lg);
    const bool on = row < a.rows;
    A v[K][V];
    A s = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = me + (k << a.lg);
      if (on && c < a.nv) {
        const Vec<T, V> t = load_vec<T, V>(x + row * a.ld_x + (long long)c * V);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          v[k][i] = to_acc(t.v[i]);
          s += v[k][i];
        }
      }
    }
    const A mu = team_sum(s, a.lg, scratch) * inv;
    s = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (on && me + (k << a.lg) < a.nv) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const A d = v[k][i] - mu;
          s += d * d;
        }
      }
    }
    const A r = rsqrt_acc(team_sum(s, a.lg, scratch) * inv + (A)a.eps);
    if (!on) continue;
    if (me == 0 && mean) {
      mean[row] = mu;
      rstd[row] = r;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = me + (k << a.lg);
      if (c < a.nv) {
        Vec<T, V> o;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          A h = (v[k][i] - mu) * r;
          if (a.w) h *= param<T>(a.w, a.w_float, (long long)c * V + i);
          if (a.b) h += param<T>(a.b, a.w_float, (long long)c * V + i);
          o.v[i] = from_acc<T>(h);
        }
        store_vec<T, V>(y + row * a.dim + (long long)c * V, o);
      }
    }
  }
}

template <typename T, int V, int K>
__global__ void __launch_bounds__(1024) norm_backward_kernel(NormArgs a, const T* __restrict__ x,
                                                             const T* __restrict__ g,
                                                             const Acc<T>* __restrict__ mean,
                                                             const Acc<T>* __restrict__ rstd, T* __restrict__ dx,
                                                             Acc<T>* __restrict__ dw_part,
                                                             Acc<T>* __restrict__ db_part) {
  typedef Acc<T> A;
  __shared__ A scratch[32];
  __shared__ A red[1024];
  const int team = 1 << a.lg, me = threadIdx.x & (team - 1);
  const int per = blockDim.x >> a.lg;
  const A inv = (A)1 / (A)a.dim;
  A dw[K][V], db[K][V];
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int i = 0; i < V; ++i) dw[k][i] = db[k][i] = 0;
  for (long long r0 = (long long)blockIdx.x * per; r0 < a.rows; r0 += (long long)gridDim.x * per) {
    const long long row = r0 + (threadIdx.x >> a.lg);
    const bool on = row < a.rows;
    const A mu = on ? mean[row] : (A)0, r = on ? rstd[row] : (A)0;
    A h[K][V], wg[K][V];
    A s0 = 0, s1 = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = me + (k << a.lg);
      if (on && c < a.nv) {
        const Vec<T, V> tx = load_vec<T, V>(x + row * a.ld_x + (long long)c * V);
        const Vec<T, V> tg = load_vec<T, V>(g + row * a.ld_g + (long long)c * V);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          h[k][i] = (to_acc(tx.v[i]) - mu) * r;
          const A gv = to_acc(tg.v[i]);
          dw[k][i] += gv * h[k][i];
          db[k][i] += gv;
          wg[k][i] = a.w ? gv * param<T>(a.w, a.w_float, (long long)c * V + i) : gv;
          s0 += wg[k][i];
          s1 += wg[k][i] * h[k][i];
        }
      }
    }
    if (!dx) continue;
    const A m0 = team_sum(s0, a.lg, scratch) * inv;
    const A m1 = team_sum(s1, a.lg, scratch) * inv;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = me + (k << a.lg);
      if (on && c < a.nv) {
        Vec<T, V> o;
#pragma unroll
        for (int i = 0; i < V; ++i) o.v[i] = from_acc<T>(r * (wg[k][i] - m0 - h[k][i] * m1));
        store_vec<T, V>(dx + row * a.dim + (long long)c * V, o);
      }
    }
  }
  // the block's partial rows: the teams' sums, added in order
  if (!a.want_dw && !a.want_db) return;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = me + (k << a.lg);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      for (int which = 0; which < 2; ++which) {
        A* part = which ? db_part : dw_part;
        if (!(which ? a.want_db : a.want_dw)) continue;
        __syncthreads();
        red[threadIdx.x] = which ? db[k][i] : dw[k][i];
        __syncthreads();
        if ((int)threadIdx.x < team && c < a.nv) {
          A s = 0;
          for (int q = 0; q < per; ++q) s += red[(q << a.lg) + me];
          part[(long long)blockIdx.x * a.dim + (long long)c * V + i] = s;
        }
      }
    }
  }
}

// Rows of any length: one block per row, the row read again for every pass.
template <typename T>
__global__ void __launch_bounds__(1024) norm_forward_long_kernel(NormArgs a, const T* __restrict__ x,
                                                                 T* __restrict__ y, Acc<T>* __restrict__ mean,
                                                                 Acc<T>* __restrict__ rstd) {
  typedef Acc<T> A;
  __shared__ A scratch[32];
  const A inv = (A)1 / (A)a.dim;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* p = x + row * a.ld_x;
    A s = 0;
    for (int c = threadIdx.x; c < a.dim; c += blockDim.x) s += to_acc(p[c]);
    const A mu = team_sum(s, 10, scratch) * inv;
    s = 0;
    for (int c = threadIdx.x; c < a.dim; c += blockDim.x) {
      const A d = to_acc(p[c]) - mu;
      s += d * d;
    }
    const A r = rsqrt_acc(team_sum(s, 10, scratch) * inv + (A)a.eps);
    if (threadIdx.x == 0 && mean) {
      mean[row] = mu;
      rstd[row] = r;
    }
    for (int c = threadIdx.x; c < a.dim; c += blockDim.x) {
      A h = (to_acc(p[c]) - mu) * r;
      if (a.w) h *= param<T>(a.w, a.w_float, c);
      if (a.b) h += param<T>(a.b, a.w_float, c);
      y[row * a.dim + c] = from_acc<T>(h);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(1024) norm_backward_long_kernel(NormArgs a, const T* __restrict__ x,
                                                                  const T* __restrict__ g,
                                                                  const Acc<T>* __restrict__ mean,
                                                                  const Acc<T>* __restrict__ rstd,
                                                                  T* __restrict__ dx, Acc<T>* __restrict__ dw_part,
                                                                  Acc<T>* __restrict__ db_part) {
  typedef Acc<T> A;
  __shared__ A scratch[32];
  const A inv = (A)1 / (A)a.dim;
  bool first = true;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x, first = false) {
    const T* px = x + row * a.ld_x;
    const T* pg = g + row * a.ld_g;
    const A mu = mean[row], r = rstd[row];
    A s0 = 0, s1 = 0;
    for (int c = threadIdx.x; c < a.dim; c += blockDim.x) {
      const A h = (to_acc(px[c]) - mu) * r, gv = to_acc(pg[c]);
      const A wg = a.w ? gv * param<T>(a.w, a.w_float, c) : gv;
      s0 += wg;
      s1 += wg * h;
      const long long o = (long long)blockIdx.x * a.dim + c;   // this thread's own columns
      if (a.want_dw) dw_part[o] = (first ? (A)0 : dw_part[o]) + gv * h;
      if (a.want_db) db_part[o] = (first ? (A)0 : db_part[o]) + gv;
    }
    if (!dx) continue;
    const A m0 = team_sum(s0, 10, scratch) * inv;
    const A m1 = team_sum(s1, 10, scratch) * inv;
    for (int c = threadIdx.x; c < a.dim; c += blockDim.x) {
      const A h = (to_acc(px[c]) - mu) * r, gv = to_acc(pg[c]);
      const A wg = a.w ? gv * param<T>(a.w, a.w_float, c) : gv;
      dx[row * a.dim + c] = from_acc<T>(r * (wg - m0 - h * m1));
    }
  }
}

// Team and vectors per thread for rows of nv vectors: up to 32 lanes with one
// vector, then up to a block of 1024 threads with four.
struct NormPlan {
  int lg, k, threads, per;   // k = 0: the long kernels
};

NormPlan norm_plan(int nv) {
  NormPlan p;
  p.lg = 0;
  while (p.lg < 5 && (1 << p.lg) < nv) ++p.lg;
  p.threads = 256;
  if (nv > 32 * 4) {
    p.lg = 8;
    while (p.lg < 10 && (4 << p.lg) < nv) ++p.lg;
    p.threads = 1 << p.lg;
  }
  const int k = (nv + (1 << p.lg) - 1) >> p.lg;
  p.k = k <= 1 ? 1 : k <= 2 ? 2 : k <= 4 ? 4 : 0;
  if (p.k == 0) p.threads = 1024, p.lg = 10;
  p.per = p.k == 0 ? 1 : p.threads >> p.lg;
  return p;
}

// Blocks of the backward pass, each of which leaves a partial row of dw and db.
int norm_backward_blocks(long long rows, int sms) {
  const long long most = 4LL * sms;
  return (int)(rows < most ? rows : most);
}

template <typename T, int V>
cudaError_t norm_forward(NormArgs a, const T* x, T* y, void* mean, void* rstd, cudaStream_t st) {
  a.nv = a.dim / V;
  const NormPlan p = norm_plan(a.nv);
  a.lg = p.lg;
  const long long need = (a.rows + p.per - 1) / p.per;
  const unsigned grid = (unsigned)(need < (1 << 30) ? need : (1 << 30));
  Acc<T>* m = static_cast<Acc<T>*>(mean);
  Acc<T>* r = static_cast<Acc<T>*>(rstd);
  switch (p.k) {
    case 1: norm_forward_kernel<T, V, 1><<<grid, p.threads, 0, st>>>(a, x, y, m, r); break;
    case 2: norm_forward_kernel<T, V, 2><<<grid, p.threads, 0, st>>>(a, x, y, m, r); break;
    case 4: norm_forward_kernel<T, V, 4><<<grid, p.threads, 0, st>>>(a, x, y, m, r); break;
    default: norm_forward_long_kernel<T><<<grid, 1024, 0, st>>>(a, x, y, m, r);
  }
  return cudaGetLastError();
}

template <typename T, int V>
cudaError_t norm_backward(NormArgs a, const T* x, const T* g, const void* mean, const void* rstd, T* dx, void* dw,
                          void* db, char* ws, int sms, cudaStream_t st) {
  typedef Acc<T> A;
  a.nv = a.dim / V;
  const NormPlan p = norm_plan(a.nv);
  a.lg = p.lg;
  const long long need = (a.rows + p.per - 1) / p.per;
  const int most = norm_backward_blocks(a.rows, sms);
  const int grid = (int)(need < most ? need : most);
  const A* m = static_cast<const A*>(mean);
  const A* r = static_cast<const A*>(rstd);
  A* dwp = reinterpret_cast<A*>(ws);
  A* dbp = reinterpret_cast<A*>(ws + (a.want_dw ? align_up((size_t)most * a.dim * sizeof(A)) : 0));
  switch (p.k) {
    case 1: norm_backward_kernel<T, V, 1><<<grid, p.threads, 0, st>>>(a, x, g, m, r, dx, dwp, dbp); break;
    case 2: norm_backward_kernel<T, V, 2><<<grid, p.threads, 0, st>>>(a, x, g, m, r, dx, dwp, dbp); break;
    case 4: norm_backward_kernel<T, V, 4><<<grid, p.threads, 0, st>>>(a, x, g, m, r, dx, dwp, dbp); break;
    default: norm_backward_long_kernel<T><<<grid, 1024, 0, st>>>(a, x, g, m, r, dx, dwp, dbp);
  }
  cudaError_t e = cudaGetLastError();
  for (int which = 0; which < 2 && e == cudaSuccess; ++which) {
    if (!(which ? a.want_db : a.want_dw)) continue;
    const A* part = which ? dbp : dwp;
    void* out = which ? db : dw;
    if (a.w_float) e = column_sum(part, grid, a.dim, a.dim, static_cast<float*>(out), st);
    else e = column_sum(part, grid, a.dim, a.dim, static_cast<T*>(out), st);
  }
  return e;
}

bool norm_args_ok(long long rows, int dim, int dtype, int pdtype) {
  return rows >= 1 && rows < 2147483647LL && dim >= 1 && dim <= (1 << 24) && elem_size(dtype) &&
         (pdtype == dtype || (pdtype == LG_F32 && dtype != LG_F64));
}

}  // namespace
}  // namespace feat
}  // namespace lg

using namespace lg;
using namespace lg::feat;

#define LG_NORM_DISPATCH(F)                                                             \
  switch (dtype) {                                                                      \
    case LG_F64: return vec >= 2 ? F(double, 2) : F(double, 1);                         \
    case LG_F32: return vec >= 4 ? F(float, 4) : F(float, 1);                           \
    case LG_F16: return vec >= 8 ? F(__half, 8) : vec >= 2 ? F(__half, 2) : F(__half, 1); \
    default:                                                                            \
      return vec >= 8 ? F(__nv_bfloat16, 8) : vec >= 2 ? F(__nv_bfloat16, 2) : F(__nv_bfloat16, 1); \
  }

extern "C" int lg_layer_norm_forward(long long rows, int dim, int dtype, const void* x, long long ld_x, int param_dtype,
                                     const void* weight, const void* bias, double eps, void* y, void* mean, void* rstd,
                                     void* stream) {
  if (!norm_args_ok(rows, dim, dtype, param_dtype) || !x || !y || ld_x < dim || !(eps >= 0.0) ||
      (mean == nullptr) != (rstd == nullptr))
    return bad_args("lg_layer_norm_forward: invalid arguments");
  NormArgs a = {};
  a.rows = rows;
  a.dim = dim;
  a.ld_x = ld_x;
  a.eps = eps;
  a.w = weight;
  a.b = bias;
  a.w_float = param_dtype == LG_F32;
  Align al(elem_size(dtype));
  al.address(x);
  al.address(y);
  al.elements(ld_x);
  al.elements(dim);
  const int vec = al.vec();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto run = [&]() -> cudaError_t {
#define LG_F(T, V) norm_forward<T, V>(a, static_cast<const T*>(x), static_cast<T*>(y), mean, rstd, st)
    LG_NORM_DISPATCH(LG_F)
#undef LG_F
  };
  return cuda_status(run(), "lg_layer_norm_forward");
}

extern "C" size_t lg_layer_norm_workspace_bytes(long long rows, int dim, int dtype, int want_weight, int want_bias) {
  if (!norm_args_ok(rows, dim, dtype, dtype)) return 0;
  const int sms = sm_count();
  if (sms < 1) return 0;
  const size_t one = align_up((size_t)norm_backward_blocks(rows, sms) * dim * acc_size(dtype));
  return one * ((want_weight ? 1 : 0) + (want_bias ? 1 : 0)) + 256;
}

extern "C" int lg_layer_norm_backward(long long rows, int dim, int dtype, const void* x, long long ld_x, const void* g,
                                      long long ld_g, int param_dtype, const void* weight, const void* mean,
                                      const void* rstd, void* dx, void* d_weight, void* d_bias, void* ws,
                                      size_t ws_bytes, void* stream) {
  if (!norm_args_ok(rows, dim, dtype, param_dtype) || !x || !g || ld_x < dim || ld_g < dim || !mean || !rstd ||
      (!dx && !d_weight && !d_bias) || ((d_weight || d_bias) && !ws))
    return bad_args("lg_layer_norm_backward: invalid arguments");
  const int sms = sm_count();
  if (sms < 1) return bad_args("lg_layer_norm_backward: no CUDA device");
  const size_t one = align_up((size_t)norm_backward_blocks(rows, sms) * dim * acc_size(dtype));
  if (ws_bytes < one * ((d_weight ? 1 : 0) + (d_bias ? 1 : 0)))
    return bad_args("lg_layer_norm_backward: workspace too small");
  NormArgs a = {};
  a.rows = rows;
  a.dim = dim;
  a.ld_x = ld_x;
  a.ld_g = ld_g;
  a.w = weight;
  a.w_float = param_dtype == LG_F32;
  a.want_dw = d_weight != nullptr;
  a.want_db = d_bias != nullptr;
  Align al(elem_size(dtype));
  al.address(x);
  al.address(g);
  if (dx) al.address(dx);
  al.elements(ld_x);
  al.elements(ld_g);
  al.elements(dim);
  const int vec = al.vec();
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto run = [&]() -> cudaError_t {
#define LG_F(T, V)                                                                                            \
  norm_backward<T, V>(a, static_cast<const T*>(x), static_cast<const T*>(g), mean, rstd, static_cast<T*>(dx), d_weight, \
                      d_bias, static_cast<char*>(ws), sms, st)
    LG_NORM_DISPATCH(LG_F)
#undef LG_F
  };
  return cuda_status(run(), "lg_layer_norm_backward");
}
