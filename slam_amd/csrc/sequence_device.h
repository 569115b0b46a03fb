// Device helpers of the sequence-layer kernels (rms_norm.hip, causal_conv.hip, selective_scan.hip, gemm_fp8.hip).
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

// these kernels are compared with tolerances, not bit for bit: products and sums may contract to fma
#pragma clang fp contract(fast)

namespace slamhip {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));

template <int V>
struct Floats {
  typedef float type __attribute__((ext_vector_type(V)));
};
template <int V>
using floats = typename Floats<V>::type;

// V consecutive elements of a row, at the element's own alignment: gfx950 takes unaligned global accesses, so rows of odd length
// and views at odd offsets use the same vector accesses as aligned ones.
template <typename T, int V>
struct Packed {
  typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T))));
};

template <typename T, int V>
using packed = typename Packed<T, V>::type;

// valid >= V: one vector access; fewer (also none): element by element, the rest zero.  As they are in memory: a value that is
// converted behind a condition is waited for there, one that is kept like this when it is used.
template <int V, typename T>
__device__ __forceinline__ packed<T, V> load_raw(const T* p, int valid) {
  packed<T, V> raw;
#pragma unroll
  for (int i = 0; i < V; ++i) raw[i] = (T)0.0f;
  if (valid >= V) {
    raw = *reinterpret_cast<const packed<T, V>*>(p);
  } else if (valid > 0) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < valid) raw[i] = p[i];
  }
  return raw;
}

template <typename T, int V>
__device__ __forceinline__ floats<V> to_floats(packed<T, V> raw) {
  floats<V> v;
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = (float)raw[i];
  return v;
}

template <int V, typename T>
__device__ __forceinline__ floats<V> loadv(const T* p, int valid) {
  return to_floats<T, V>(load_raw<V>(p, valid));
}

template <int V, typename T>
__device__ __forceinline__ void storev(T* p, floats<V> v, int valid) {
  if (valid >= V) {
    typename Packed<T, V>::type raw;
#pragma unroll
    for (int i = 0; i < V; ++i) raw[i] = (T)v[i];
    *reinterpret_cast<typename Packed<T, V>::type*>(p) = raw;
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < valid) p[i] = (T)v[i];
  }
}

template <typename T>
__device__ __forceinline__ void store8(T* p, f32x8 v, int valid) { storev<8>(p, v, valid); }

__device__ __forceinline__ float exp2_(float v) { return __builtin_amdgcn_exp2f(v); }
__device__ __forceinline__ float log2_(float v) { return __builtin_amdgcn_logf(v); }
__device__ __forceinline__ float rcp_(float v) { return __builtin_amdgcn_rcpf(v); }

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

// 1 / (1 + e^-v): 0 and 1 at the far ends, NaN stays NaN
__device__ __forceinline__ float sigmoid_(float v) { return rcp_(1.0f + exp2_(-kLog2e * v)); }

// out(c, sum over parts of part[p][c]), in an order that depends on the sizes alone.  Eight loads of a thread are under way at once:
// 1024 parts of 4096 columns take 5 us, one by one 10.
template <typename Out>
__global__ void __launch_bounds__(1024) column_sum_kernel(const float* __restrict__ part, long long parts, int columns, Out out) {
  __shared__ float sh[32][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + tx;
  float s = 0.0f;
  if (c < columns)
#pragma unroll 8
    for (long long p = ty; p < parts; p += 32) s += part[p * columns + c];
  sh[ty][tx] = s;
  __syncthreads();
  if (ty == 0 && c < columns) {
    s = 0.0f;
    for (int i = 0; i < 32; ++i) s += sh[i][tx];
    out(c, s);
  }
}

template <typename Out>
hipError_t column_sums(const float* part, long long parts, int columns, Out out, hipStream_t s) {
  hipLaunchKernelGGL((column_sum_kernel<Out>), dim3((columns + 31) / 32), dim3(1024), 0, s, part, parts, columns, out);
  return hipGetLastError();
}

}  // namespace
}  // namespace slamhip
