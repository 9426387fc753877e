// lg_feat.cuh — what the node-feature kernels (lg_rows.cu, lg_norm_fwd.cu,
// lg_norm_bwd.cu, lg_edges.cu) share: element types, vector accesses, the stable sort of row
// ids, the column sum of partial rows.
//
// Element types are float, double, half and bfloat16.  Arithmetic and every
// sum are in Acc<T>: double for double, else float; a value is rounded to T
// once, when it is stored.
#pragma once

#include "lg_common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <cstring>
#include <string>

namespace lg {
extern thread_local std::string g_last_error;

namespace feat {

template <typename T> struct AccOf { typedef float type; };
template <> struct AccOf<double> { typedef double type; };
template <typename T> using Acc = typename AccOf<T>::type;

__device__ __forceinline__ float to_acc(float v) { return v; }
__device__ __forceinline__ double to_acc(double v) { return v; }
__device__ __forceinline__ float to_acc(__half v) { return __half2float(v); }
// A bfloat16 is the upper half of its float: a shift, where the conversion
// instruction goes through the slow unit (16 a cycle and SM; with it, layer
// norm's backward pass of 16384 x 4096 took 109 us).
__device__ __forceinline__ float to_acc(__nv_bfloat16 v) {
  return __uint_as_float((unsigned)__bfloat16_as_ushort(v) << 16);
}

template <typename T> __device__ __forceinline__ T from_acc(Acc<T> v);
template <> __device__ __forceinline__ float from_acc<float>(float v) { return v; }
template <> __device__ __forceinline__ double from_acc<double>(double v) { return v; }
template <> __device__ __forceinline__ __half from_acc<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_acc<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// V elements moved by one access (sizeof(T) * V is 2, 4, 8 or 16 bytes).
template <typename T, int V> struct alignas(sizeof(T) * V) Vec { T v[V]; };

template <int BYTES> struct Word;
template <> struct Word<2> { typedef unsigned short type; };
template <> struct Word<4> { typedef unsigned type; };
template <> struct Word<8> { typedef uint2 type; };
template <> struct Word<16> { typedef uint4 type; };

template <typename T, int V> __device__ __forceinline__ Vec<T, V> load_vec(const T* p) {
  typedef typename Word<sizeof(T) * V>::type W;
  const W w = *reinterpret_cast<const W*>(p);
  Vec<T, V> x;
  memcpy(&x, &w, sizeof(W));
  return x;
}
template <typename T, int V> __device__ __forceinline__ void store_vec(T* p, const Vec<T, V>& x) {
  typedef typename Word<sizeof(T) * V>::type W;
  W w;
  memcpy(&w, &x, sizeof(W));
  *reinterpret_cast<W*>(p) = w;
}

// ---------------------------------------------------------------------------
// Values of a vector in the accumulation type, two to a lane: sm_100 adds,
// multiplies and fuses two floats in one instruction (add / mul / fma
// .rn.f32x2), each half rounded as on its own.  A vector of one element is one
// single lane.
// ---------------------------------------------------------------------------
struct Single32 { float a; };
struct Pair32 { unsigned long long v; };
struct Single64 { double a; };
struct Pair64 { double a, b; };

template <typename A, int V> struct LaneOf { typedef Pair32 type; };
template <> struct LaneOf<float, 1> { typedef Single32 type; };
template <int V> struct LaneOf<double, V> { typedef Pair64 type; };
template <> struct LaneOf<double, 1> { typedef Single64 type; };
template <typename T, int V> using Lane = typename LaneOf<Acc<T>, V>::type;
template <int V> constexpr int lanes = V == 1 ? 1 : V / 2;

__device__ __forceinline__ Pair32 pair32(float a, float b) {
  Pair32 r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r.v) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 halves(Pair32 p) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(p.v));
  return r;
}
__device__ __forceinline__ Pair32 add(Pair32 x, Pair32 y) {
  Pair32 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(x.v), "l"(y.v));
  return r;
}
__device__ __forceinline__ Pair32 mul(Pair32 x, Pair32 y) {
  Pair32 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(x.v), "l"(y.v));
  return r;
}
__device__ __forceinline__ Pair32 fma(Pair32 x, Pair32 y, Pair32 z) {   // x y + z
  Pair32 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(x.v), "l"(y.v), "l"(z.v));
  return r;
}
__device__ __forceinline__ float sum(Pair32 p) {
  const float2 h = halves(p);
  return h.x + h.y;
}
__device__ __forceinline__ void spread(float v, Pair32& p) { p = pair32(v, v); }

__device__ __forceinline__ Single32 add(Single32 x, Single32 y) { return {x.a + y.a}; }
__device__ __forceinline__ Single32 mul(Single32 x, Single32 y) { return {x.a * y.a}; }
__device__ __forceinline__ Single32 fma(Single32 x, Single32 y, Single32 z) { return {fmaf(x.a, y.a, z.a)}; }
__device__ __forceinline__ float sum(Single32 p) { return p.a; }
__device__ __forceinline__ void spread(float v, Single32& p) { p.a = v; }

__device__ __forceinline__ Single64 add(Single64 x, Single64 y) { return {x.a + y.a}; }
__device__ __forceinline__ Single64 mul(Single64 x, Single64 y) { return {x.a * y.a}; }
__device__ __forceinline__ Single64 fma(Single64 x, Single64 y, Single64 z) { return {::fma(x.a, y.a, z.a)}; }
__device__ __forceinline__ double sum(Single64 p) { return p.a; }
__device__ __forceinline__ void spread(double v, Single64& p) { p.a = v; }

__device__ __forceinline__ Pair64 add(Pair64 x, Pair64 y) { return {x.a + y.a, x.b + y.b}; }
__device__ __forceinline__ Pair64 mul(Pair64 x, Pair64 y) { return {x.a * y.a, x.b * y.b}; }
__device__ __forceinline__ Pair64 fma(Pair64 x, Pair64 y, Pair64 z) {
  return {::fma(x.a, y.a, z.a), ::fma(x.b, y.b, z.b)};
}
__device__ __forceinline__ double sum(Pair64 p) { return p.a + p.b; }
__device__ __forceinline__ void spread(double v, Pair64& p) { p.a = p.b = v; }

template <typename L, typename A> __device__ __forceinline__ L spread(A v) {
  L l;
  spread(v, l);
  return l;
}

// Element pairs <-> lanes.
__device__ __forceinline__ Pair32 widen2(const float* p) { return pair32(p[0], p[1]); }
__device__ __forceinline__ Pair32 widen2(const __half* p) {
  const float2 f = __half22float2(*reinterpret_cast<const __half2*>(p));
  return pair32(f.x, f.y);
}
__device__ __forceinline__ Pair32 widen2(const __nv_bfloat16* p) {
  unsigned u;
  memcpy(&u, p, 4);
  return pair32(__uint_as_float(u << 16), __uint_as_float(u & 0xffff0000u));
}
__device__ __forceinline__ Pair64 widen2(const double* p) { return {p[0], p[1]}; }
__device__ __forceinline__ void narrow2(Pair32 v, float* p) {
  const float2 h = halves(v);
  p[0] = h.x;
  p[1] = h.y;
}
__device__ __forceinline__ void narrow2(Pair32 v, __half* p) {
  const float2 h = halves(v);
  *reinterpret_cast<__half2*>(p) = __floats2half2_rn(h.x, h.y);
}
__device__ __forceinline__ void narrow2(Pair32 v, __nv_bfloat16* p) {
  const float2 h = halves(v);
  *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(h.x, h.y);
}
__device__ __forceinline__ void narrow2(Pair64 v, double* p) {
  p[0] = v.a;
  p[1] = v.b;
}

// Lane n of V elements at p, and back.
template <typename T, int V> __device__ __forceinline__ Lane<T, V> widen(const T* p, int n) {
  if constexpr (V == 1) return {to_acc(p[0])};
  else return widen2(p + 2 * n);
}
template <typename T, int V> __device__ __forceinline__ void narrow(Lane<T, V> v, T* p, int n) {
  if constexpr (V == 1) p[0] = from_acc<T>(v.a);
  else narrow2(v, p + 2 * n);
}

inline int elem_size(int dtype) {
  switch (dtype) {
    case 0: return 4;   // LG_F32
    case 1: return 8;   // LG_F64
    case 2: return 2;   // LG_F16
    case 3: return 2;   // LG_BF16
    default: return 0;
  }
}
inline int acc_size(int dtype) { return dtype == 1 ? 8 : 4; }

// The widest vector (in elements, a power of two, at most 16 bytes) that
// divides every length, stride and address of a call.
struct Align {
  unsigned long long bits = 0;
  int size;
  explicit Align(int elem_bytes) : size(elem_bytes) {}
  void address(const void* p) { bits |= reinterpret_cast<uintptr_t>(p); }
  void elements(long long n) { bits |= (unsigned long long)n * (unsigned)size; }
  int vec() const {
    int b = 16;
    while (b > size && (bits & (unsigned long long)(b - 1))) b >>= 1;
    return b / size;
  }
};

// Whether every address (null allowed) is a multiple of `bytes`: one that is not
// would be a misaligned access on the device.
template <typename... P> inline bool aligned(size_t bytes, const P*... p) {
  return (... && (reinterpret_cast<uintptr_t>(p) % bytes == 0));
}
constexpr size_t kWsAlign = 16;   // of a workspace

inline int sm_count() {
  static std::atomic<int> cache[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return 0;
  if (dev >= 0 && dev < 64) {
    const int c = cache[dev].load(std::memory_order_acquire);
    if (c > 0) return c;
  }
  int n = 0;
  if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  if (dev >= 0 && dev < 64) cache[dev].store(n, std::memory_order_release);
  return n;
}

inline size_t align_up(size_t b) { return (b + 255) & ~(size_t)255; }

inline int bad_args(const char* what) {
  g_last_error = what;
  return -1;   // LG_ERR_INVALID
}
inline int cuda_status(cudaError_t e, const char* where) {
  if (e == cudaSuccess) return 0;
  g_last_error = std::string(where) + ": " + cudaGetErrorString(e);
  return -2;   // LG_ERR_CUDA
}

// ---------------------------------------------------------------------------
// Stable sort of row ids (lg_rows.cu).  Pairs (key, position): key = the id,
// or `rows` for an id that is out of range or equal to the padding id, so that
// those come last.  Equal keys keep the order of their positions.
// ---------------------------------------------------------------------------
size_t sort_ids_workspace(long long rows, long long n);
// *sorted points into ws after the call.  `zero`: nzero words set to zero on the
// way; `fill`: bytes set to zero beside the sort.
struct SideFill {
  void* p;
  size_t bytes;
};
cudaError_t sort_ids(long long rows, long long n, const void* ids, int ids64, long long pad, int has_pad, void* ws,
                     unsigned* zero, int nzero, SideFill fill, uint2** sorted, cudaStream_t st);

// ---------------------------------------------------------------------------
// out[c] = sum over r < nrows of part[r * ld + c] for c < dim; columns from
// `dim` on, up to 2 * dim, go to out2 (when given).  Rows in a fixed order:
// strided by 32 over the block's row groups, then the groups in turn.
// ---------------------------------------------------------------------------
template <typename A, typename O>
__global__ void __launch_bounds__(1024) column_sum_kernel(const A* __restrict__ part, int nrows, long long ld, int dim,
                                                          O* __restrict__ out, O* __restrict__ out2) {
  __shared__ A red[32][33];
  griddep_wait();
  const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5;
  const long long c = (long long)blockIdx.x * 32 + lane, width = out2 ? 2LL * dim : dim;
  A s = 0;
  if (c < width) {
    int r = grp;
    for (; r + 96 < nrows; r += 128) {
      const A a0 = part[r * ld + c], a1 = part[(r + 32) * ld + c], a2 = part[(r + 64) * ld + c],
              a3 = part[(r + 96) * ld + c];
      s += a0;
      s += a1;
      s += a2;
      s += a3;
    }
    for (; r < nrows; r += 32) s += part[r * ld + c];
  }
  red[grp][lane] = s;
  __syncthreads();
  if (grp == 0 && c < width) {
    A t = 0;
#pragma unroll
    for (int k = 0; k < 32; ++k) t += red[k][lane];
    if (c < dim) out[c] = from_acc<O>(t);
    else out2[c - dim] = from_acc<O>(t);
  }
}

template <typename A, typename O>
inline cudaError_t column_sum2(const A* part, int nrows, long long ld, int dim, O* out, O* out2, cudaStream_t st) {
  const long long width = out2 ? 2LL * dim : dim;
  return launch_pdl(column_sum_kernel<A, O>, dim3((unsigned)((width + 31) / 32)), dim3(1024), 0, st, part, nrows, ld,
                    dim, out, out2);
}
template <typename A, typename O>
inline cudaError_t column_sum(const A* part, int nrows, long long ld, int dim, O* out, cudaStream_t st) {
  return column_sum2(part, nrows, ld, dim, out, static_cast<O*>(nullptr), st);
}

}  // namespace feat
}  // namespace lg
