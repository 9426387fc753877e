// lg_norm.cuh — what the two passes of layer norm share (lg_norm_fwd.cu,
// lg_norm_bwd.cu; two files so that they compile side by side).
//
//   mu = mean(x),  r = 1 / sqrt(mean((x - mu)^2) + eps),  h = (x - mu) r
//   y  = h w + b
//   dx = r (wg - mean(wg) - h mean(wg h)),   wg = w g
//   dw = sum over rows of g h,   db = sum over rows of g
//
// Memory is the bound: forward reads x and writes y, backward reads x and g and
// writes dx.  So a row stays in registers, in its own type, between the passes
// over it: the variance is the second pass, about the row's own mean, and the
// backward pass forms its two means and then dx from the same registers.  A row
// belongs to a team of threads, which keeps the same columns for every row it
// takes: weight and bias are loaded once per team, and dw and db grow in
// registers and leave as one partial row per block, added in a fixed order by
// column_sum.
//
// Teams: part of a warp for short rows (the fewest lanes that hold the row with
// at most four vectors each: the more rows a warp holds, the fewer times it
// issues the divide and square root of a row), a block for long ones.  Rows too
// long for a block's registers are read again for every pass (from L2).
#pragma once

#include "lg_feat.cuh"

#include "../../include/lanczos_b200.h"

namespace lg {
namespace feat {
namespace {

constexpr int kBlock = 512;   // most threads of a block that holds one row (128 registers each)

struct NormArgs {
  long long rows, ld_x, ld_g;
  int dim, nv, lg;       // row length, vectors per row, log2 of a part-warp team
  float dim32, inv32;    // the row length and its reciprocal, rounded
  double dim64, inv64;
  double eps;
  const void* w;         // weight and bias, of type P
  const void* b;
  int want_dw, want_db;
};

__device__ __forceinline__ float rsqrt_acc(float v) { return 1.0f / sqrtf(v); }
__device__ __forceinline__ double rsqrt_acc(double v) { return 1.0 / sqrt(v); }

// s / dim by its rounded reciprocal: the product and one residual step (Markstein, IBM
// J. Res. Dev. 34, 1990), which gives the quotient itself where that is a number of
// the type.  So a row of equal values whose sum is exact has h = 0; the product alone
// can be an ulp away, which r = 1 / sqrt(eps) enlarges (7 fp32 of 1000.0: y = -0.019).
// A division costs more: 10^6 x 3 fp64 forward 14.4 us instead of 12.4, 5003 x 1537
// fp32 backward 26.5 instead of 24.6.
__device__ __forceinline__ float mean_of(float s, float n, float inv) {
  const float q = s * inv;
  return fmaf(fmaf(-q, n, s), inv, q);
}
__device__ __forceinline__ double mean_of(double s, double n, double inv) {
  const double q = s * inv;
  return ::fma(::fma(-q, n, s), inv, q);
}
// The same, and a mean to a few ulp, with n and 1 / n taken from the kernel's arguments
// where they are used: the backward pass has no registers to spare (5003 x 1537 fp32:
// 20.0 us, 22.5 with them in registers).  Forward has (10^6 x 3 fp64: 14.4 us, 16.3 so).
__device__ __forceinline__ float mean_of(float s, const NormArgs& a) { return mean_of(s, a.dim32, a.inv32); }
__device__ __forceinline__ double mean_of(double s, const NormArgs& a) { return mean_of(s, a.dim64, a.inv64); }
__device__ __forceinline__ float about_mean(float s, const NormArgs& a) { return s * a.inv32; }
__device__ __forceinline__ double about_mean(double s, const NormArgs& a) { return s * a.inv64; }

// V parameters, in accesses of at most 16 bytes.
template <typename P, int V> struct Params {
  static constexpr int W = sizeof(P) * V > 16 ? 16 / (int)sizeof(P) : V;
  Vec<P, W> part[V / W];
  __device__ __forceinline__ void load(const P* p) {
#pragma unroll
    for (int i = 0; i < V / W; ++i) part[i] = load_vec<P, W>(p + i * W);
  }
  __device__ __forceinline__ P value(int i) const { return part[i / W].v[i % W]; }
  __device__ __forceinline__ auto lane(int n) const {
    if constexpr (V == 1) return widen<P, 1>(part[0].v, 0);
    else return widen<P, 2>(part[2 * n / W].v + 2 * n % W, 0);
  }
  // A missing weight is 1, a missing bias 0.
  __device__ __forceinline__ void load_or(const void* p, long long at, float missing) {
    if (p) {
      load(static_cast<const P*>(p) + at);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) part[i / W].v[i % W] = from_acc<P>((Acc<P>)missing);
    }
  }
};

// Sums over the team, to every thread of it: by shuffles inside a warp; in a
// block the warps' sums go through `scratch` (2 * N * 32 values, zero at the
// start; its halves alternate, so one barrier a call is enough) and every thread
// adds them up.  Two values share one set of shuffles: after the first, the lower
// half warp carries one and the upper half the other.
template <typename A> __device__ __forceinline__ A warps_total(const A* s) {
  A t = 0;
  const int n = (blockDim.x + 127) / 128;
  if constexpr (sizeof(A) == 4) {
    for (int i = 0; i < n; ++i) {
      const float4 q = reinterpret_cast<const float4*>(s)[i];
      t += (q.x + q.y) + (q.z + q.w);
    }
  } else {
    for (int i = 0; i < n; ++i) {
      const double2 p = reinterpret_cast<const double2*>(s)[2 * i], q = reinterpret_cast<const double2*>(s)[2 * i + 1];
      t += (p.x + p.y) + (q.x + q.y);
    }
  }
  return t;
}

template <typename A, int N, bool BLOCK>
__device__ __forceinline__ void team_sum(A (&v)[N], int lg, A* scratch, int& half) {
  if (!BLOCK) {
    for (int o = 1 << lg >> 1; o > 0; o >>= 1) {
#pragma unroll
      for (int n = 0; n < N; ++n) v[n] += __shfl_xor_sync(0xffffffffu, v[n], o);
    }
    return;
  }
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  A* s = scratch + half * N * 32;
  half ^= 1;
  if constexpr (N == 1) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v[0] += __shfl_xor_sync(0xffffffffu, v[0], o);
    if (lane == 0) s[warp] = v[0];
  } else {
    const bool upper = lane >= 16;
    A keep = upper ? v[1] : v[0];
    keep += __shfl_xor_sync(0xffffffffu, upper ? v[0] : v[1], 16);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) keep += __shfl_xor_sync(0xffffffffu, keep, o);
    if ((lane & 15) == 0) s[(lane << 1) + warp] = keep;
  }
  __syncthreads();
#pragma unroll
  for (int n = 0; n < N; ++n) v[n] = warps_total(s + n * 32);
}

template <typename A> __device__ __forceinline__ void clear_scratch(A* scratch, int n) {
  for (int i = threadIdx.x; i < n; i += blockDim.x) scratch[i] = 0;
  __syncthreads();
}

// Where this thread's team stands: its first row and column, the rows between
// its turns, the columns between its vectors.
template <bool BLOCK> struct Team {
  int me, stride;
  long long row, step;
  __device__ __forceinline__ explicit Team(int lg) {
    if (BLOCK) {
      me = threadIdx.x;
      stride = blockDim.x;
      row = blockIdx.x;
      step = gridDim.x;
    } else {
      const int per = blockDim.x >> lg;
      me = threadIdx.x & ((1 << lg) - 1);
      stride = 1 << lg;
      row = (long long)blockIdx.x * per + (threadIdx.x >> lg);
      step = (long long)gridDim.x * per;
    }
  }
};

// The rows that a block takes next, on their way to shared memory while one is
// worked on: two rows of K vectors of each of NA arrays.  Every thread
// copies the vectors that it will read itself, so its own wait is all the
// ordering it needs.  What is in flight is then not limited by the registers
// (16384 x 4096 bf16 forward: 93 us with loads to registers, 42 us so).  Narrower
// accesses and part-warp teams load to registers when they need a row: a 4-byte
// asynchronous copy moves a quarter of a line's sectors at a time (5003 x 1537 fp32
// forward: 28 us with them, 17 us with loads), and short rows have enough warps.
template <typename T, int V, int K, int NA, bool BLOCK> struct Rows {
  static constexpr bool async = BLOCK && sizeof(T) * V == 16;
  static constexpr int stages = 2;
  typedef Acc<T> A;
  static constexpr int stats = NA - 1;   // with g (NA = 2) a row's mean and 1 / deviation come along
  const T* src[NA];        // this thread's first vector of the next row to fetch
  const A *mean = nullptr, *rstd = nullptr;
  long long step;
  long long jump[NA];      // elements from one row of the team to its next
  unsigned base, warp, column, stage, turn;
  int left;                // rows still to fetch
  bool in[K];

  // p, ld: the arrays and their row strides.
  __device__ __forceinline__ Rows(char* smem, const Team<BLOCK>& t, long long rows, int nv, const T* const (&p)[NA],
                                  const long long (&ld)[NA], const A* m = nullptr, const A* r = nullptr) {
    mean = m + (stats ? t.row : 0);
    rstd = r + (stats ? t.row : 0);
    step = t.step;
#pragma unroll
    for (int k = 0; k < K; ++k) in[k] = t.me + k * t.stride < nv;
#pragma unroll
    for (int n = 0; n < NA; ++n) {
      src[n] = p[n] + t.row * ld[n] + (long long)t.me * V;
      jump[n] = t.step * ld[n];
    }
    left = t.row < rows ? (int)((rows - t.row + t.step - 1) / t.step) : 0;
    turn = 0;
    if (async) {
      base = (unsigned)__cvta_generic_to_shared(smem) + threadIdx.x * 16;
      column = blockDim.x * 16;
      stage = NA * K * column + stats * (blockDim.x >> 5) * 16;
      warp = (unsigned)__cvta_generic_to_shared(smem) + NA * K * column + (threadIdx.x >> 5) * 16;
#pragma unroll
      for (int q = 0; q < stages - 1; ++q) fetch(q);
    }
  }
  // Starts the copy of the next row into the given stage.
  __device__ __forceinline__ void fetch(unsigned to) {
    if (left > 0) {
      const unsigned dst = base + to * stage;
#pragma unroll
      for (int n = 0; n < NA; ++n) {
#pragma unroll
        for (int k = 0; k < K; ++k)
          if (in[k])
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + (n * K + k) * column),
                         "l"(src[n] + (size_t)(k * blockDim.x) * V) : "memory");
        src[n] += jump[n];
      }
      if (stats) {   // for the whole warp, by its first two lanes
        if ((threadIdx.x & 31) < 2)
          asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(warp + to * stage + (threadIdx.x & 1) * (unsigned)sizeof(A)),
                       "l"(threadIdx.x & 1 ? rstd : mean), "n"((int)sizeof(A)) : "memory");
        mean += step;
        rstd += step;
      }
      --left;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  }
  // The row of this turn, K vectors of every array; `on`: there is one.  What is
  // not there is zero, so that the arithmetic needs no branches, which would keep
  // the work of different vectors apart.
  __device__ __forceinline__ void next(const Team<BLOCK>& t, bool on, Vec<T, V> (&v)[NA][K], A* mu = nullptr,
                                       A* r = nullptr) {
    if (async) {
      if (stats) __syncwarp();   // every lane has read the slot that is filled next
      fetch((turn + stages - 1) & (stages - 1));
      asm volatile("cp.async.wait_group %0;" ::"n"(stages - 1) : "memory");
      const unsigned slot = (turn & (stages - 1)) * stage, from = base + slot;
      ++turn;
      if (stats) {
        __syncwarp();            // the first two lanes' copies have come
        if constexpr (sizeof(A) == 4)
          asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(*mu), "=f"(*r) : "r"(warp + slot) : "memory");
        else
          asm volatile("ld.shared.v2.f64 {%0, %1}, [%2];" : "=d"(*mu), "=d"(*r) : "r"(warp + slot) : "memory");
      }
#pragma unroll
      for (int n = 0; n < NA; ++n)
#pragma unroll
        for (int k = 0; k < K; ++k)
          {
            uint4 w = make_uint4(0, 0, 0, 0);
            if (in[k])
              asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(w.x), "=r"(w.y), "=r"(w.z), "=r"(w.w)
                           : "r"(from + (n * K + k) * column) : "memory");
            memcpy(&v[n][k], &w, sizeof(v[n][k]));
          }
    } else {
      if (stats) {
        *mu = on ? *mean : (A)0;
        *r = on ? *rstd : (A)0;
        mean += step;
        rstd += step;
      }
#pragma unroll
      for (int n = 0; n < NA; ++n) {
#pragma unroll
        for (int k = 0; k < K; ++k) {
          typename Word<sizeof(T) * V>::type w = {};
          if (on && in[k]) w = *reinterpret_cast<const decltype(w)*>(src[n] + k * t.stride * V);
          memcpy(&v[n][k], &w, sizeof(w));
        }
        src[n] += jump[n];
      }
    }
  }
  static size_t bytes(int threads) {
    return async ? (size_t)stages * (threads * NA * K * 16 + stats * threads / 32 * 16) : 0;
  }
};

// Vectors per thread: what its registers hold.  Forward only the row, in its
// own type; backward x and g of two rows, the weight and two sums per element.
template <typename T, int V> struct KMax {
  static constexpr int forward = sizeof(Acc<T>) == 8 && V == 2 ? 4 : 8;
  static constexpr int backward = (sizeof(Acc<T>) == 8 ? 8 : 16) / V < 8 ? (sizeof(Acc<T>) == 8 ? 8 : 16) / V : 8;
};

struct NormPlan {
  int block, lg, k, threads, per;   // k = 0: the long kernels; per: rows of a block at a time
};

// Rows of at most a warp of vectors go to part-warp teams: the fewest lanes with at
// most four vectors each, so that a warp's loads stay whole lines.  Longer ones go to
// blocks, of as few threads as hold them with four vectors each (two where the
// backward pass keeps so many), since a row's two sums over the block cost a thread
// as much as eight elements do.
NormPlan norm_plan(int nv, int kmax) {
  NormPlan p;
  const int kw = kmax < 4 ? kmax : 4;
  p.block = nv > 32;
  p.lg = 0;
  p.threads = 256;
  int k;
  if (!p.block) {
    while ((kw << p.lg) < nv) ++p.lg;
    k = (nv + (1 << p.lg) - 1) >> p.lg;
  } else {
    k = 1;
    while (k < kw && nv > 32 * k) k *= 2;
    while (k < kmax && nv > 256 * k) k *= 2;
    p.threads = ((nv + k - 1) / k + 31) / 32 * 32;
    if (p.threads > kBlock) k = 0;
  }
  p.k = k == 0 ? 0 : k <= 1 ? 1 : k <= 2 ? 2 : k <= 4 ? 4 : 8;
  if (p.k == 0) p.threads = 1024;
  p.per = p.block ? 1 : p.threads >> p.lg;
  return p;
}

// Blocks of `kernel` that an SM holds, asked once per device and block size.
struct Resident {
  std::atomic<int> blocks[64][33] = {};
  int get(const void* kernel, int threads, size_t smem) {
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 1;
    std::atomic<int>& c = blocks[dev][threads / 32];
    int b = c.load(std::memory_order_acquire);
    if (b > 0) return b;
    // the most that any block size of this kernel takes
    if (smem && cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                     (int)(smem / threads * kBlock)) != cudaSuccess) {
      (void)cudaGetLastError();
      return 0;
    }
    if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&b, kernel, threads, smem) != cudaSuccess || b < 1) {
      (void)cudaGetLastError();
      return 1;
    }
    c.store(b, std::memory_order_release);
    return b;
  }
};

// Blocks a SM that keep 32 KB of rows on their way (vectors of 16 bytes a thread):
// more of them read no faster but worse.  16384 x 2048 fp32 forward: 43 us with 32
// KB, 48 us with 56 KB; 16384 x 4096 bf16: 42 us with 32 KB, 51 us with 96 KB (four
// rows a block instead of two).
int in_flight(int per_sm, int threads, int vectors) {
  const int most = 2048 / (threads * vectors);
  const int cap = most > 2 ? most : 2;   // two, so that one block's sums run beside the other's loads
  return per_sm < cap ? per_sm : cap;
}

// Every block of a persistent grid is resident: `per_sm` of them on an SM.
int norm_grid(long long rows, const NormPlan& p, int sms, int per_sm) {
  const long long need = (rows + p.per - 1) / p.per, most = (long long)per_sm * sms;
  return (int)(need < most ? need : most);
}

// The backward pass runs at most 1024 threads a SM, which is enough to keep
// memory busy, and so leaves at most this many partial rows: a block of 32 t
// threads holds rows of up to 512 t elements, and part-warp teams come in blocks
// of 256.
int norm_parts(long long rows, int dim, int sms) {
  int per_sm = 16384 / dim;
  per_sm = per_sm < 4 ? 4 : per_sm > 32 ? 32 : per_sm;
  const long long most = (long long)sms * per_sm;
  return (int)(rows < most ? rows : most);
}

// The means of long rows (two a row), then the partial rows.
size_t norm_workspace(long long rows, int dim, int dtype, int sms) {
  return align_up((size_t)rows * 2 * acc_size(dtype)) + (size_t)norm_parts(rows, dim, sms) * 2 * dim * acc_size(dtype);
}

void set_dim(NormArgs& a, int dim) {
  a.dim = dim;
  a.dim32 = (float)dim;
  a.inv32 = 1.0f / a.dim32;
  a.dim64 = dim;
  a.inv64 = 1.0 / a.dim64;
}

// F<T, P, V, K, BLOCK, AFFINE>(...) for the plan's K; K <= KM, part-warp teams at
// most 4.
#define LG_NORM_CASE(F, K, KM, AFFINE, ...)                              \
  case K:                                                                \
    if constexpr (K <= KM) {                                             \
      if (p.block) return F<T, P, V, K, true, AFFINE>(__VA_ARGS__);      \
    }                                                                    \
    if constexpr (K <= KM && K <= 4) {                                   \
      if (!p.block) return F<T, P, V, K, false, AFFINE>(__VA_ARGS__);    \
    }                                                                    \
    break;
#define LG_NORM_K(F, KM, AFFINE, ...)                                    \
  switch (p.k) {                                                         \
    LG_NORM_CASE(F, 1, KM, AFFINE, __VA_ARGS__)                          \
    LG_NORM_CASE(F, 2, KM, AFFINE, __VA_ARGS__)                          \
    LG_NORM_CASE(F, 4, KM, AFFINE, __VA_ARGS__)                          \
    LG_NORM_CASE(F, 8, KM, AFFINE, __VA_ARGS__)                          \
    default: break;                                                      \
  }                                                                      \
  return cudaErrorInvalidValue;

bool norm_args_ok(long long rows, int dim, int dtype, int pdtype) {
  return rows >= 1 && rows < 2147483647LL && dim >= 1 && dim <= (1 << 24) && elem_size(dtype) &&
         (pdtype == dtype || (pdtype == LG_F32 && dtype != LG_F64));
}

// The vector width of a call whose parameters p, q (of type pdtype) are read
// in accesses of at most 16 bytes: a parameter at an odd place makes it 1.
int norm_vec(const Align& al, int pdtype, const void* p, const void* q) {
  const int v = al.vec();
  const unsigned bytes = v * elem_size(pdtype) < 16 ? v * elem_size(pdtype) : 16;
  return ((reinterpret_cast<uintptr_t>(p) | reinterpret_cast<uintptr_t>(q)) & (bytes - 1)) ? 1 : v;
}

}  // namespace
}  // namespace feat
}  // namespace lg

#define LG_NORM_DISPATCH(F)                                                                             \
  const bool pf = param_dtype == LG_F32;                                                                \
  switch (dtype) {                                                                                      \
    case LG_F64: return vec >= 2 ? F(double, double, 2) : F(double, double, 1);                         \
    case LG_F32: return vec >= 4 ? F(float, float, 4) : vec == 2 ? F(float, float, 2) : F(float, float, 1); \
    case LG_F16:                                                                                        \
      if (pf) return vec >= 8 ? F(__half, float, 8) : vec == 4 ? F(__half, float, 4)                    \
                     : vec == 2 ? F(__half, float, 2) : F(__half, float, 1);                            \
      return vec >= 8 ? F(__half, __half, 8) : vec == 4 ? F(__half, __half, 4)                          \
             : vec == 2 ? F(__half, __half, 2) : F(__half, __half, 1);                                  \
    default:                                                                                            \
      if (pf) return vec >= 8 ? F(__nv_bfloat16, float, 8) : vec == 4 ? F(__nv_bfloat16, float, 4)      \
                     : vec == 2 ? F(__nv_bfloat16, float, 2) : F(__nv_bfloat16, float, 1);              \
      return vec >= 8 ? F(__nv_bfloat16, __nv_bfloat16, 8) : vec == 4 ? F(__nv_bfloat16, __nv_bfloat16, 4) \
             : vec == 2 ? F(__nv_bfloat16, __nv_bfloat16, 2) : F(__nv_bfloat16, __nv_bfloat16, 1);      \
  }
