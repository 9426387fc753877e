// lg_norm_fwd.cu — layer norm, forward (lg_norm.cuh has the formulas and the plan).
#include "lg_norm.cuh"

#include <type_traits>

namespace lg {
namespace feat {
namespace {

template <typename T, typename P, int V, int K, bool BLOCK, bool AFFINE>
__global__ void __launch_bounds__(BLOCK ? kBlock : 256) norm_forward_kernel(NormArgs a, const T* __restrict__ x,
                                                                          T* __restrict__ y, Acc<T>* __restrict__ mean,
                                                                          Acc<T>* __restrict__ rstd) {
  typedef Acc<T> A;
  typedef Lane<T, V> L;
  constexpr int N = lanes<V>;
  __shared__ __align__(16) A scratch[BLOCK ? 64 : 1];
  if (BLOCK) clear_scratch(scratch, 64);
  int half = 0;
  const Team<BLOCK> t(a.lg);
  const A count = (A)a.dim, inv = (A)1 / count;
  constexpr bool kept = K <= 4;   // weight and bias stay in registers; else they are read again (from L1) for every row
  Params<P, V> w[kept ? K : 1], b[kept ? K : 1];
  if (kept && AFFINE) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int c = t.me + k * t.stride;
      if (c < a.nv) {
        w[kept ? k : 0].load_or(a.w, (long long)c * V, 1.0f);
        b[kept ? k : 0].load_or(a.b, (long long)c * V, 0.0f);
      }
    }
  }
  extern __shared__ __align__(16) char ring[];
  const T* const from[1] = {x};
  const long long ld[1] = {a.ld_x};
  Rows<T, V, K, 1, BLOCK> rows(ring, t, a.rows, a.nv, from, ld);
  T* out = y + t.row * a.dim + (long long)t.me * V;
  // every thread of a warp takes the same number of turns
  for (long long row = t.row, r0 = BLOCK ? row : (long long)blockIdx.x * (blockDim.x >> a.lg); r0 < a.rows;
       row += t.step, r0 += t.step, out += t.step * a.dim) {
    const bool on = BLOCK || row < a.rows;
    Vec<T, V> got[1][K];
    rows.next(t, on, got);
    Vec<T, V>(&v)[K] = got[0];
    A s[1];
    L acc = spread<L>((A)0);
#pragma unroll
    for (int k = 0; k < K; ++k) {
#pragma unroll
      for (int n = 0; n < N; ++n) acc = add(acc, widen<T, V>(v[k].v, n));
    }
    s[0] = sum(acc);
    team_sum<A, 1, BLOCK>(s, a.lg, scratch, half);
    const A mu = mean_of(s[0], count, inv);
    const L minus = spread<L>(-mu);
    acc = spread<L>((A)0);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const L there = spread<L>((A)(rows.in[k] ? 1 : 0));
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const L d = add(widen<T, V>(v[k].v, n), minus);
        acc = fma(mul(d, there), d, acc);
      }
    }
    s[0] = sum(acc);
    team_sum<A, 1, BLOCK>(s, a.lg, scratch, half);
    const A r = rsqrt_acc(s[0] * inv + (A)a.eps);
    if (!on) continue;
    if (t.me == 0 && mean) {
      mean[row] = mu;
      rstd[row] = r;
    }
    const L rr = spread<L>(r);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (rows.in[k]) {
        const long long c = t.me + k * t.stride;
        if (!kept && AFFINE) {
          w[0].load_or(a.w, c * V, 1.0f);
          b[0].load_or(a.b, c * V, 0.0f);
        }
        Vec<T, V> o;
#pragma unroll
        for (int n = 0; n < N; ++n) {
          L h = mul(add(widen<T, V>(v[k].v, n), minus), rr);
          if (AFFINE) h = fma(h, w[kept ? k : 0].lane(n), b[kept ? k : 0].lane(n));
          narrow<T, V>(h, o.v, n);
        }
        store_vec<T, V>(out + k * t.stride * V, o);
      }
    }
  }
}

// Rows of any length: a block of 1024 threads per row.
template <typename T, typename P, int V>
__global__ void __launch_bounds__(1024) norm_forward_long_kernel(NormArgs a, const T* __restrict__ x,
                                                                 T* __restrict__ y, Acc<T>* __restrict__ mean,
                                                                 Acc<T>* __restrict__ rstd) {
  typedef Acc<T> A;
  __shared__ __align__(16) A scratch[64];
  clear_scratch(scratch, 64);
  int half = 0;
  const A count = (A)a.dim, inv = (A)1 / count;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* p = x + row * a.ld_x;
    A s[1] = {0};
    for (int c = threadIdx.x; c < a.nv; c += 1024) {
      const Vec<T, V> v = load_vec<T, V>(p + (long long)c * V);
#pragma unroll
      for (int i = 0; i < V; ++i) s[0] += to_acc(v.v[i]);
    }
    team_sum<A, 1, true>(s, 0, scratch, half);
    const A mu = mean_of(s[0], count, inv);
    s[0] = 0;
    for (int c = threadIdx.x; c < a.nv; c += 1024) {
      const Vec<T, V> v = load_vec<T, V>(p + (long long)c * V);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const A d = to_acc(v.v[i]) - mu;
        s[0] += d * d;
      }
    }
    team_sum<A, 1, true>(s, 0, scratch, half);
    const A r = rsqrt_acc(s[0] * inv + (A)a.eps);
    if (threadIdx.x == 0 && mean) {
      mean[row] = mu;
      rstd[row] = r;
    }
    for (int c = threadIdx.x; c < a.nv; c += 1024) {
      const Vec<T, V> v = load_vec<T, V>(p + (long long)c * V);
      Params<P, V> w, b;
      if (a.w) w.load(static_cast<const P*>(a.w) + (long long)c * V);
      if (a.b) b.load(static_cast<const P*>(a.b) + (long long)c * V);
      Vec<T, V> o;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        A h = (to_acc(v.v[i]) - mu) * r;
        if (a.w) h *= to_acc(w.value(i));
        if (a.b) h += to_acc(b.value(i));
        o.v[i] = from_acc<T>(h);
      }
      store_vec<T, V>(y + row * a.dim + (long long)c * V, o);
    }
  }
}

template <typename T, typename P, int V, int K, bool BLOCK, bool AFFINE>
cudaError_t launch_forward(const NormArgs& a, const NormPlan& p, const T* x, T* y, Acc<T>* mean, Acc<T>* rstd, int sms,
                           cudaStream_t st) {
  static Resident res;
  void (*f)(NormArgs, const T*, T*, Acc<T>*, Acc<T>*) = norm_forward_kernel<T, P, V, K, BLOCK, AFFINE>;
  const size_t smem = Rows<T, V, K, 1, BLOCK>::bytes(p.threads);
  int per_sm = res.get(reinterpret_cast<const void*>(f), p.threads, smem);
  if (per_sm < 1) return cudaErrorInvalidConfiguration;
  if (Rows<T, V, K, 1, BLOCK>::async) per_sm = in_flight(per_sm, p.threads, K);
  const int grid = norm_grid(a.rows, p, sms, per_sm);
  f<<<grid, p.threads, smem, st>>>(a, x, y, mean, rstd);
  return cudaGetLastError();
}

template <typename T, typename P, int V>
cudaError_t norm_forward(NormArgs a, const T* x, T* y, void* mean, void* rstd, int sms, cudaStream_t st) {
  a.nv = a.dim / V;
  const NormPlan p = norm_plan(a.nv, KMax<T, V>::forward);
  a.lg = p.lg;
  Acc<T>* m = static_cast<Acc<T>*>(mean);
  Acc<T>* r = static_cast<Acc<T>*>(rstd);
  if (p.k == 0) {
    norm_forward_long_kernel<T, P, V><<<norm_grid(a.rows, p, sms, 2), 1024, 0, st>>>(a, x, y, m, r);
    return cudaGetLastError();
  }
  if constexpr (std::is_same<P, T>::value) {
    if (!a.w && !a.b) { LG_NORM_K(launch_forward, (KMax<T, V>::forward), false, a, p, x, y, m, r, sms, st) }
  }
  LG_NORM_K(launch_forward, (KMax<T, V>::forward), true, a, p, x, y, m, r, sms, st)
}

}  // namespace
}  // namespace feat
}  // namespace lg

using namespace lg;
using namespace lg::feat;

extern "C" int lg_layer_norm_forward(long long rows, int dim, int dtype, const void* x, long long ld_x, int param_dtype,
                                     const void* weight, const void* bias, double eps, void* y, void* mean, void* rstd,
                                     void* stream) {
  if (!norm_args_ok(rows, dim, dtype, param_dtype) || !x || !y || ld_x < dim || !(eps >= 0.0) ||
      (mean == nullptr) != (rstd == nullptr) || !aligned(elem_size(dtype), x, y) ||
      !aligned(elem_size(param_dtype), weight, bias) || !aligned(acc_size(dtype), mean, rstd))
    return bad_args("lg_layer_norm_forward: invalid arguments");
  const int sms = sm_count();
  if (sms < 1) return bad_args("lg_layer_norm_forward: no CUDA device");
  NormArgs a = {};
  a.rows = rows;
  set_dim(a, dim);
  a.ld_x = ld_x;
  a.eps = eps;
  a.w = weight;
  a.b = bias;
  Align al(elem_size(dtype));
  al.address(x);
  al.address(y);
  al.elements(ld_x);
  al.elements(dim);
  const int vec = norm_vec(al, param_dtype, weight, bias);
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  auto run = [&]() -> cudaError_t {
#define LG_F(T, P, V) norm_forward<T, P, V>(a, static_cast<const T*>(x), static_cast<T*>(y), mean, rstd, sms, st)
    LG_NORM_DISPATCH(LG_F)
#undef LG_F
  };
  return cuda_status(run(), "lg_layer_norm_forward");
}
