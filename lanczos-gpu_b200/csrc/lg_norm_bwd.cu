// lg_norm_bwd.cu — layer norm, backward (lg_norm.cuh has the formulas and the plan).
#include "lg_norm.cuh"

#include <type_traits>

namespace lg {
namespace feat {
namespace {

// V sums, in accesses of at most 16 bytes where the place is a multiple of that.
template <typename A, int V> __device__ __forceinline__ void store_values(A* p, const Vec<A, V>& x) {
  constexpr int W = sizeof(A) * V > 16 ? 16 / (int)sizeof(A) : V;
#pragma unroll
  for (int i = 0; i < V; i += W) {
    Vec<A, W> o;
#pragma unroll
    for (int j = 0; j < W; ++j) o.v[j] = x.v[i + j];
    store_vec<A, W>(p + i, o);
  }
}

// part: one row of 2 * dim sums per block, dw then db.
template <typename T, typename P, int V, int K, bool BLOCK, bool AFFINE>
__global__ void __launch_bounds__(BLOCK ? kBlock : 256) norm_backward_kernel(
    NormArgs a, const T* __restrict__ x, const T* __restrict__ g, const Acc<T>* __restrict__ mean,
    const Acc<T>* __restrict__ rstd, T* __restrict__ dx, Acc<T>* __restrict__ part) {
  typedef Acc<T> A;
  typedef Lane<T, V> L;
  constexpr int N = lanes<V>;
  __shared__ __align__(16) A scratch[BLOCK ? 128 : 1];
  if (BLOCK) clear_scratch(scratch, 128);
  __shared__ A red[BLOCK || !AFFINE ? 1 : 8][BLOCK || !AFFINE ? 1 : 32 * K * V];
  int half = 0;
  const Team<BLOCK> t(a.lg);
  Params<P, V> w[K];
  L dw[K][N], db[K][N];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int c = t.me + k * t.stride;
    if (AFFINE) w[k].load_or(c < a.nv ? a.w : nullptr, (long long)c * V, c < a.nv ? 1.0f : 0.0f);
#pragma unroll
    for (int n = 0; n < N; ++n) dw[k][n] = db[k][n] = spread<L>((A)0);
  }
  extern __shared__ __align__(16) char ring[];
  const T* const from[2] = {x, g};
  const long long ld[2] = {a.ld_x, a.ld_g};
  Rows<T, V, K, 2, BLOCK> rows(ring, t, a.rows, a.nv, from, ld, mean, rstd);
  T* dst = dx + t.row * a.dim + (long long)t.me * V;
  for (long long row = t.row, r0 = BLOCK ? row : (long long)blockIdx.x * (blockDim.x >> a.lg); r0 < a.rows;
       row += t.step, r0 += t.step, dst += t.step * a.dim) {
    const bool on = BLOCK || row < a.rows;
    A mu, r;
    Vec<T, V> got[2][K];
    rows.next(t, on, got, &mu, &r);
    Vec<T, V>(&vx)[K] = got[0];
    Vec<T, V>(&vg)[K] = got[1];
    const L minus = spread<L>(-mu), rr = spread<L>(r);
    L s0 = spread<L>((A)0), s1 = s0;
    L h[K][N], wg[K][N];
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int n = 0; n < N; ++n) {
        h[k][n] = mul(add(widen<T, V>(vx[k].v, n), minus), rr);
        const L gv = widen<T, V>(vg[k].v, n);
        if (AFFINE) {
          dw[k][n] = fma(gv, h[k][n], dw[k][n]);
          db[k][n] = add(db[k][n], gv);
        }
        wg[k][n] = AFFINE ? mul(gv, w[k].lane(n)) : gv;
        s0 = add(s0, wg[k][n]);
        s1 = fma(wg[k][n], h[k][n], s1);
      }
    }
    if (!dx) continue;
    A s[2] = {sum(s0), sum(s1)};
    team_sum<A, 2, BLOCK>(s, a.lg, scratch, half);
    const L m0 = spread<L>(-mean_of(s[0], a)), m1 = spread<L>(-about_mean(s[1], a));
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (on && rows.in[k]) {
        Vec<T, V> o;
#pragma unroll
        for (int n = 0; n < N; ++n) narrow<T, V>(mul(rr, fma(h[k][n], m1, add(wg[k][n], m0))), o.v, n);
        store_vec<T, V>(dst + k * t.stride * V, o);
      }
    }
  }
  if (!AFFINE || (!a.want_dw && !a.want_db)) return;
  A* out = part + (long long)blockIdx.x * 2 * a.dim;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if (!(which ? a.want_db : a.want_dw)) continue;
    if (BLOCK) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        const long long c = t.me + k * t.stride;
        if (c < a.nv) {
          Vec<A, V> o;
#pragma unroll
          for (int n = 0; n < N; ++n) narrow<A, V>(which ? db[k][n] : dw[k][n], o.v, n);
          store_values<A, V>(out + (long long)which * a.dim + c * V, o);
        }
      }
    } else {
      // the teams of a warp, then the warps, in order
      const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
      __syncthreads();
#pragma unroll
      for (int k = 0; k < K; ++k) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
          A v[2];
          narrow<A, V>(which ? db[k][n] : dw[k][n], v, 0);
#pragma unroll
          for (int i = 0; i < (V == 1 ? 1 : 2); ++i) {
            for (int o = t.stride; o < 32; o <<= 1) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
            if (lane < t.stride) red[warp][(lane + k * t.stride) * V + 2 * n + i] = v[i];
          }
        }
      }
      __syncthreads();
      for (int c = threadIdx.x; c < a.dim; c += blockDim.x) {
        A v = 0;
#pragma unroll
        for (int q = 0; q < 8; ++q) v += red[q][c];
        out[(long long)which * a.dim + c] = v;
      }
    }
  }
}

// Rows too long for a block's registers, in two passes over x and g (the second
// finds them in L2 where they fit): the two means of every row, a block of 1024
// threads a row; then dx, dw and db by blocks that own 256 vectors of columns and
// every gridDim.y-th row.
template <typename T, typename P, int V>
__global__ void __launch_bounds__(1024) norm_means_kernel(NormArgs a, const T* __restrict__ x, const T* __restrict__ g,
                                                          const Acc<T>* __restrict__ mean,
                                                          const Acc<T>* __restrict__ rstd, Acc<T>* __restrict__ means) {
  typedef Acc<T> A;
  typedef Lane<T, V> L;
  __shared__ __align__(16) A scratch[128];
  clear_scratch(scratch, 128);
  int half = 0;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* px = x + row * a.ld_x;
    const T* pg = g + row * a.ld_g;
    const L minus = spread<L>(-mean[row]), rr = spread<L>(rstd[row]);
    L s0 = spread<L>((A)0), s1 = s0;
    for (int c = threadIdx.x; c < a.nv; c += 1024) {
      const Vec<T, V> vx = load_vec<T, V>(px + (long long)c * V), vg = load_vec<T, V>(pg + (long long)c * V);
      Params<P, V> w;
      w.load_or(a.w, (long long)c * V, 1.0f);
#pragma unroll
      for (int n = 0; n < lanes<V>; ++n) {
        const L wg = mul(widen<T, V>(vg.v, n), w.lane(n));
        s0 = add(s0, wg);
        s1 = fma(wg, mul(add(widen<T, V>(vx.v, n), minus), rr), s1);
      }
    }
    A s[2] = {sum(s0), sum(s1)};
    team_sum<A, 2, true>(s, 0, scratch, half);
    if (threadIdx.x == 0) {
      means[2 * row] = mean_of(s[0], a);
      means[2 * row + 1] = about_mean(s[1], a);
    }
  }
}

template <typename T, typename P, int V>
__global__ void __launch_bounds__(256) norm_columns_kernel(NormArgs a, const T* __restrict__ x, const T* __restrict__ g,
                                                           const Acc<T>* __restrict__ mean,
                                                           const Acc<T>* __restrict__ rstd, const Acc<T>* __restrict__ means,
                                                           T* __restrict__ dx, Acc<T>* __restrict__ part) {
  typedef Acc<T> A;
  typedef Lane<T, V> L;
  constexpr int N = lanes<V>;
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.nv) return;
  const long long col = (long long)c * V;
  Params<P, V> w;
  w.load_or(a.w, col, 1.0f);
  L dw[N], db[N];
#pragma unroll
  for (int n = 0; n < N; ++n) dw[n] = db[n] = spread<L>((A)0);
#pragma unroll 4
  for (long long row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const Vec<T, V> vx = load_vec<T, V>(x + row * a.ld_x + col), vg = load_vec<T, V>(g + row * a.ld_g + col);
    const L minus = spread<L>(-mean[row]), rr = spread<L>(rstd[row]);
    L m0 = spread<L>((A)0), m1 = m0;
    if (dx) {
      m0 = spread<L>(-means[2 * row]);
      m1 = spread<L>(-means[2 * row + 1]);
    }
    Vec<T, V> o;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const L h = mul(add(widen<T, V>(vx.v, n), minus), rr), gv = widen<T, V>(vg.v, n);
      dw[n] = fma(gv, h, dw[n]);
      db[n] = add(db[n], gv);
      narrow<T, V>(mul(rr, fma(h, m1, add(mul(gv, w.lane(n)), m0))), o.v, n);
    }
    if (dx) store_vec<T, V>(dx + row * a.dim + col, o);
  }
  A* out = part + (long long)blockIdx.y * 2 * a.dim;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if (!(which ? a.want_db : a.want_dw)) continue;
    Vec<A, V> o;
#pragma unroll
    for (int n = 0; n < N; ++n) narrow<A, V>(which ? db[n] : dw[n], o.v, n);
    store_values<A, V>(out + (long long)which * a.dim + col, o);
  }
}

template <typename T, typename P, int V, int K, bool BLOCK, bool AFFINE>
cudaError_t launch_backward(const NormArgs& a, const NormPlan& p, const T* x, const T* g, const Acc<T>* mean,
                            const Acc<T>* rstd, T* dx, Acc<T>* part, int* parts, int sms, cudaStream_t st) {
  static Resident res;
  void (*f)(NormArgs, const T*, const T*, const Acc<T>*, const Acc<T>*, T*, Acc<T>*) =
      norm_backward_kernel<T, P, V, K, BLOCK, AFFINE>;
  const size_t smem = Rows<T, V, K, 2, BLOCK>::bytes(p.threads);
  int per_sm = res.get(reinterpret_cast<const void*>(f), p.threads, smem);
  if (per_sm < 1) return cudaErrorInvalidConfiguration;
  if (per_sm > 1024 / p.threads) per_sm = 1024 / p.threads;
  if (Rows<T, V, K, 2, BLOCK>::async) per_sm = in_flight(per_sm, p.threads, 2 * K);
  *parts = norm_grid(a.rows, p, sms, per_sm);
  f<<<*parts, p.threads, smem, st>>>(a, x, g, mean, rstd, dx, part);
  return cudaGetLastError();
}

template <typename T, typename P, int V>
cudaError_t norm_backward_rows(NormArgs a, const T* x, const T* g, const Acc<T>* m, const Acc<T>* r, T* dx,
                               Acc<T>* part, Acc<T>* means, int* parts, int sms, cudaStream_t st) {
  a.nv = a.dim / V;
  const NormPlan p = norm_plan(a.nv, KMax<T, V>::backward);
  a.lg = p.lg;
  if (p.k == 0) {
    if (dx) norm_means_kernel<T, P, V><<<norm_grid(a.rows, p, sms, 2), 1024, 0, st>>>(a, x, g, m, r, means);
    const int cols = (a.nv + 255) / 256, want = 4 * sms / cols > 1 ? 4 * sms / cols : 1;   // four blocks a SM
    *parts = (int)(a.rows < want ? a.rows : want);
    norm_columns_kernel<T, P, V><<<dim3(cols, *parts), 256, 0, st>>>(a, x, g, m, r, means, dx, part);
    return cudaGetLastError();
  }
  if constexpr (std::is_same<P, T>::value) {
    if (!a.w && !a.want_dw && !a.want_db) {
      LG_NORM_K(launch_backward, (KMax<T, V>::backward), false, a, p, x, g, m, r, dx, part, parts, sms, st)
    }
  }
  LG_NORM_K(launch_backward, (KMax<T, V>::backward), true, a, p, x, g, m, r, dx, part, parts, sms, st)
}

template <typename T, typename P, int V>
cudaError_t norm_backward(const NormArgs& a, const T* x, const T* g, const void* mean, const void* rstd, T* dx, void* dw,
                          void* db, void* ws, int sms, cudaStream_t st) {
  typedef Acc<T> A;
  A* means = static_cast<A*>(ws);   // two values a row, of long rows only
  A* part = reinterpret_cast<A*>(static_cast<char*>(ws) + align_up((size_t)a.rows * 2 * sizeof(A)));
  int parts = 0;
  const cudaError_t e = norm_backward_rows<T, P, V>(a, x, g, static_cast<const A*>(mean), static_cast<const A*>(rstd),
                                                    dx, part, means, &parts, sms, st);
  if (e != cudaSuccess || (!dw && !db)) return e;
  // dw and db lie side by side in a partial row: one sum over both, or over one of them
  const int dim = a.dim;
  if (dw && db) return column_sum2(part, parts, 2LL * dim, dim, static_cast<P*>(dw), static_cast<P*>(db), st);
  return column_sum(part + (dw ? 0 : dim), parts, 2LL * dim, dim, static_cast<P*>(dw ? dw : db), st);
}

}  // namespace
}  // namespace feat
}  // namespace lg

using namespace lg;
using namespace lg::feat;

extern "C" size_t lg_layer_norm_workspace_bytes(long long rows, int dim, int dtype) {
  if (!norm_args_ok(rows, dim, dtype, dtype)) return 0;
  const int sms = sm_count();
  if (sms < 1) return 0;
  return norm_workspace(rows, dim, dtype, sms);
}

extern "C" int lg_layer_norm_backward(long long rows, int dim, int dtype, const void* x, long long ld_x, const void* g,
                                      long long ld_g, int param_dtype, const void* weight, const void* mean,
                                      const void* rstd, void* dx, void* d_weight, void* d_bias, void* ws,
                                      size_t ws_bytes, void* stream) {
  if (!norm_args_ok(rows, dim, dtype, param_dtype) || !x || !g || ld_x < dim || ld_g < dim || !mean || !rstd ||
      (!dx && !d_weight && !d_bias) || !ws || !aligned(elem_size(dtype), x, g, dx) ||
      !aligned(elem_size(param_dtype), weight, d_weight, d_bias) || !aligned(acc_size(dtype), mean, rstd) ||
      !aligned(kWsAlign, ws))
    return bad_args("lg_layer_norm_backward: invalid arguments");
  const int sms = sm_count();
  if (sms < 1) return bad_args("lg_layer_norm_backward: no CUDA device");
  if (ws_bytes < norm_workspace(rows, dim, dtype, sms))
    return bad_args("lg_layer_norm_backward: workspace too small");
  NormArgs a = {};
  a.rows = rows;
  set_dim(a, dim);
  a.ld_x = ld_x;
  a.ld_g = ld_g;
  a.w = weight;
  a.want_dw = d_weight != nullptr;
  a.want_db = d_bias != nullptr;
  Align al(elem_size(dtype));
  al.address(x);
  al.address(g);
  if (dx) al.address(dx);
  al.elements(ld_x);
  al.elements(ld_g);
  al.elements(dim);
  const int vec = norm_vec(al, param_dtype, weight, nullptr);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto run = [&]() -> cudaError_t {
#define LG_F(T, P, V)                                                                                              \
  norm_backward<T, P, V>(a, static_cast<const T*>(x), static_cast<const T*>(g), mean, rstd, static_cast<T*>(dx), d_weight, \
                         d_bias, ws, sms, st)
    LG_NORM_DISPATCH(LG_F)
#undef LG_F
  };
  return cuda_status(run(), "lg_layer_norm_backward");
}
