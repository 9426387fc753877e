// lg_feat.cuh — what the node-feature kernels (lg_rows.cu, lg_norm.cu,
// lg_edges.cu) share: element types, vector accesses, the stable sort of row
// ids, the column sum of partial rows.
//
// Element types are float, double, half and bfloat16.  Arithmetic and every
// sum are in Acc<T>: double for double, else float; a value is rounded to T
// once, when it is stored.
#pragma once

#include "lg_common.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

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
__device__ __forceinline__ float to_acc(__nv_bfloat16 v) { return __bfloat162float(v); }

template <typename T> __device__ __forceinline__ T from_acc(Acc<T> v);
template <> __device__ __forceinline__ float from_acc<float>(float v) { return v; }
template <> __device__ __forceinline__ double from_acc<double>(double v) { return v; }
template <> __device__ __forceinline__ __half from_acc<__half>(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_acc<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// V elements moved by one access (sizeof(T) * V is 2, 4, 8 or 16 bytes).
template <typename T, int V> struct alignas(sizeof(T) * V) Vec { T v[V]; };

template <typename T, int V> __device__ __forceinline__ Vec<T, V> load_vec(const T* p) {
  return *reinterpret_cast<const Vec<T, V>*>(p);
}
template <typename T, int V> __device__ __forceinline__ void store_vec(T* p, const Vec<T, V>& x) {
  *reinterpret_cast<Vec<T, V>*>(p) = x;
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
// *sorted points into ws after the call.
cudaError_t sort_ids(long long rows, long long n, const void* ids, int ids64, long long pad, int has_pad, void* ws,
                     uint2** sorted, cudaStream_t st);

// ---------------------------------------------------------------------------
// out[c] = sum over r < nrows of part[r * ld + c], rows in a fixed order:
// strided by 32 over the block's row groups, then the groups in turn.
// ---------------------------------------------------------------------------
template <typename A, typename O>
__global__ void __launch_bounds__(1024) column_sum_kernel(const A* __restrict__ part, int nrows, long long ld, int dim,
                                                          O* __restrict__ out) {
  __shared__ A red[32][33];
  const int lane = threadIdx.x & 31, grp = threadIdx.x >> 5;
  const long long c = (long long)blockIdx.x * 32 + lane;
  A s = 0;
  if (c < dim) {
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
  if (grp == 0 && c < dim) {
    A t = 0;
#pragma unroll
    for (int k = 0; k < 32; ++k) t += red[k][lane];
    out[c] = from_acc<O>(t);
  }
}

template <typename A, typename O>
inline cudaError_t column_sum(const A* part, int nrows, long long ld, int dim, O* out, cudaStream_t st) {
  column_sum_kernel<A, O><<<(unsigned)((dim + 31) / 32), 1024, 0, st>>>(part, nrows, ld, dim, out);
  return cudaGetLastError();
}

}  // namespace feat
}  // namespace lg
