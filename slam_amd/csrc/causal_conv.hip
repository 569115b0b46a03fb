// Short causal convolution over time, one filter a channel, with an optional SiLU, and its backward pass.
//
//   pre[b,t,c] = bias[c] + sum_k w[c,k] xp[b,t+k,c],  y = pre sigmoid(pre)      xp = K - 1 rows of state, then x
//   backward: d = dy silu'(pre),  dxp[p] = sum_k w[k] d[p-k],  dw[c,k] = sum d[t] xp[t+k],  dbias = sum d
//
// A thread walks a few channels down a run of time steps with the last K rows in registers, so a row is read from memory
// once but for the K - 1 rows in front of a run (and, backward, as many behind it).  Bytes bound this: 8 x 2048 x 4096 bfloat16 takes
// 55 us forward (268 MB, 4.9 TB/s) and 99-106 us back (403 MB, 3.8-4.1 TB/s), in float32 101 and 183 us (5.3 and 4.4 TB/s); 32 x 1 x 4096
// with its states 5 us: a launch and two ways to memory.
#include <hip/hip_runtime.h>

#include "common.h"
#include "sequence_device.h"

namespace slamhip {
namespace {

struct ConvArgs {
  const void *x, *dy, *state_in, *d_state_out;
  const float *w, *bias;
  void *y, *state_out, *dx, *d_state_in;
  float* part;
  const int* lengths;
  long long xb, xt, yb, yt, dyb, dyt, dxb, dxt;   // strides of a sequence and of a time step, in elements
  int T, C, run, runs, silu;
  int lx_log2;   // a workgroup is 2^lx_log2 threads along the channels by 256 / 2^lx_log2 runs
};

// A thread's channels c .. c + V - 1 and steps from t0.  Where the row ends inside them they are the V that end with it, so that every
// load is one of V, and the first `skip` belong to the thread in front: worked on and not stored (element by element a row of 1021 is
// waited for several times: 8 x 2048 x 1021 forward and back 105 us, so 56).  n: how many there are (C < V).
struct Place {
  int c, n, skip, run, t0;
  bool live;
};

template <int V>
__device__ __forceinline__ Place conv_place(const ConvArgs& a) {
  const int lx = 1 << a.lx_log2;
  Place p;
  p.c = (blockIdx.x * lx + (threadIdx.x & (lx - 1))) * V;
  p.live = p.c < a.C;
  p.skip = 0;
  if (a.C >= V && p.c > a.C - V) {
    p.skip = p.c - (a.C - V);
    p.c = a.C - V;
  }
  p.n = a.C - p.c;
  p.run = blockIdx.y * (256 >> a.lx_log2) + (threadIdx.x >> a.lx_log2);
  p.t0 = p.run * a.run;
  p.live = p.live && p.run < a.runs;
  return p;
}

template <int V, typename T>
__device__ __forceinline__ void put(T* to, floats<V> v, const Place& p) {
  if (p.skip == 0) {
    storev<V>(to, v, p.n);
  } else {
#pragma unroll
    for (int i = 1; i < V; ++i)
      if (i >= p.skip) to[i] = (T)v[i];
  }
}

__device__ __forceinline__ int conv_length(const ConvArgs& a, int b) {
  if (!a.lengths) return a.T;
  const int n = a.lengths[b];
  return n < 0 ? 0 : (n > a.T ? a.T : n);
}

// row `t` of a sequence as it is in memory: state rows in front of it, zeros where it has neither
template <typename T, int K, int V>
__device__ __forceinline__ packed<T, V> conv_row(const ConvArgs& a, const T* x, const T* state, int t, int len, int c, int n) {
  const T* from = t >= 0 ? x + t * a.xt : state + (long long)(t + K - 1) * a.C;
  return load_raw<V>(from + c, t >= 0 ? (t < len ? n : 0) : (state ? n : 0));
}

// a thread's filters lie one behind the other: V K floats
template <int K, int V>
__device__ __forceinline__ void conv_weights(const ConvArgs& a, int c, int n, floats<V> (&w)[K], floats<V>& bias) {
  floats<V> flat[K];
#pragma unroll
  for (int k = 0; k < K; ++k) flat[k] = loadv<V>(a.w + (long long)c * K + k * V, n * K - k * V);
#pragma unroll
  for (int j = 0; j < V; ++j)
#pragma unroll
    for (int k = 0; k < K; ++k) w[k][j] = flat[(j * K + k) / V][(j * K + k) % V];
  bias = floats<V>{};
  if (a.bias) bias = loadv<V>(a.bias + c, n);
}

template <typename T, int K, int V>
__global__ void __launch_bounds__(256) causal_conv_fwd_kernel(ConvArgs a) {
  const Place p = conv_place<V>(a);
  const int b = blockIdx.z, len = conv_length(a, b);
  if (!p.live) return;
  const T* x = (const T*)a.x + b * a.xb;
  T* y = (T*)a.y + b * a.yb;
  const T* state = a.state_in ? (const T*)a.state_in + (long long)b * (K - 1) * a.C : nullptr;
  // all loads that a run begins with are under way before the first is converted
  packed<T, V> front[K - 1], left[K - 1];
#pragma unroll
  for (int k = 0; k < K - 1; ++k) front[k] = conv_row<T, K, V>(a, x, state, p.t0 + k - (K - 1), len, p.c, p.n);
  const bool leaves = p.run == 0 && a.state_out;
#pragma unroll
  for (int i = 0; i < K - 1; ++i) {
    const int t = len + i - (K - 1);
    left[i] = load_raw<V>(x + (t > 0 ? t : 0) * a.xt + p.c, leaves && t >= 0 ? p.n : 0);
  }
  floats<V> w[K], bias, win[K];
  conv_weights<K, V>(a, p.c, p.n, w, bias);
  const int t1 = min(p.t0 + a.run, a.T), last = min(t1, len);
  packed<T, V> next[4];
  auto fetch = [&](int t) {
#pragma unroll
    for (int i = 0; i < 4; ++i) next[i] = load_raw<V>(x + (t + i) * a.xt + p.c, t + i < last ? p.n : 0);
  };
  fetch(p.t0);
#pragma unroll
  for (int k = 0; k < K - 1; ++k) win[k] = to_floats<T, V>(front[k]);
  if (leaves) {   // win holds the state: it may be written over from here on
    T* out = (T*)a.state_out + (long long)b * (K - 1) * a.C;
#pragma unroll
    for (int i = 0; i < K - 1; ++i) {
      floats<V> v = to_floats<T, V>(left[i]);
#pragma unroll
      for (int k = 0; k < K - 1; ++k)
        if (len + i == k) v = win[k];
      put<V>(out + (long long)i * a.C + p.c, v, p);
    }
  }
  for (int t = p.t0; t < t1; t += 4) {
    packed<T, V> now[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) now[i] = next[i];
    if (t + 4 < t1) fetch(t + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      win[K - 1] = to_floats<T, V>(now[i]);
      floats<V> v = bias;
#pragma unroll
      for (int k = 0; k < K; ++k)
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] = fmaf(w[k][j], win[k][j], v[j]);
      if (a.silu)
#pragma unroll
        for (int j = 0; j < V; ++j) v[j] *= sigmoid_(v[j]);
      if (t + i >= len) v = floats<V>{};
      if (t + i < t1) put<V>(y + (t + i) * a.yt + p.c, v, p);
#pragma unroll
      for (int k = 0; k < K - 1; ++k) win[k] = win[k + 1];
    }
  }
}

// part [sequence][group of runs][K + 1][C]: dw and dbias of a workgroup's runs
template <typename T, int K, int V>
__global__ void __launch_bounds__(256) causal_conv_bwd_kernel(ConvArgs a) {
  constexpr int U = 2;   // rows under way
  __shared__ float sh[256 * V];
  const Place p = conv_place<V>(a);
  const int b = blockIdx.z, len = conv_length(a, b);
  floats<V> dw[K], db{};
#pragma unroll
  for (int k = 0; k < K; ++k) dw[k] = floats<V>{};
  if (p.live) {
    const T* x = (const T*)a.x + b * a.xb;
    const T* dy = (const T*)a.dy + b * a.dyb;
    T* dx = (T*)a.dx + b * a.dxb;
    const long long sbase = (long long)b * (K - 1) * a.C;
    const T* state = a.state_in ? (const T*)a.state_in + sbase : nullptr;
    const T* d_out = a.d_state_out ? (const T*)a.d_state_out + sbase : nullptr;
    T* d_in = a.d_state_in ? (T*)a.d_state_in + sbase : nullptr;
    packed<T, V> front[K - 1];
#pragma unroll
    for (int k = 0; k < K - 1; ++k) front[k] = conv_row<T, K, V>(a, x, state, p.t0 + k - (K - 1), len, p.c, p.n);
    floats<V> w[K], bias, win[K], d[K];
    conv_weights<K, V>(a, p.c, p.n, w, bias);
    const int t1 = min(p.t0 + a.run, a.T);
    const int first = p.run == 0 ? -(K - 1) : p.t0;   // the first run's rows begin with the state's
    const int last = min(t1 + K - 1, len), mine = min(t1, len);
    packed<T, V> next_x[U], next_y[U];
    auto fetch = [&](int t) {
#pragma unroll
      for (int i = 0; i < U; ++i) {
        next_x[i] = load_raw<V>(x + (t + i) * a.xt + p.c, t + i < last ? p.n : 0);
        next_y[i] = load_raw<V>(dy + (t + i) * a.dyt + p.c, t + i < last ? p.n : 0);
      }
    };
    fetch(p.t0);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      d[k] = floats<V>{};   // d[k] is the gradient at pre of step t - (K - 1) + k
      if (k < K - 1) win[k] = to_floats<T, V>(front[k]);
    }
    for (int t = p.t0; t < t1 + K - 1; t += U) {
      packed<T, V> nx[U], ny[U];
#pragma unroll
      for (int i = 0; i < U; ++i) nx[i] = next_x[i], ny[i] = next_y[i];
      if (t + U < t1 + K - 1) fetch(t + U);
#pragma unroll
      for (int i = 0; i < U; ++i) {
        const int now = t + i;
        if (now < t1 + K - 1) {
          win[K - 1] = to_floats<T, V>(nx[i]);
          floats<V> g{};
          if (now < len) {
            g = to_floats<T, V>(ny[i]);
            if (a.silu) {
              floats<V> pre = bias;
#pragma unroll
              for (int k = 0; k < K; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) pre[j] = fmaf(w[k][j], win[k][j], pre[j]);
#pragma unroll
              for (int j = 0; j < V; ++j) {
                const float s = sigmoid_(pre[j]);
                g[j] *= s * fmaf(pre[j], 1.0f - s, 1.0f);
              }
            }
          }
          d[K - 1] = g;
          if (now < mine) {   // behind the sequence there is no product, whatever its last rows or its state hold
            db += g;
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
              for (int j = 0; j < V; ++j) dw[k][j] = fmaf(g[j], win[k][j], dw[k][j]);
          }
          const int row = now - (K - 1);
          if (row >= first) {
            floats<V> v{};
#pragma unroll
            for (int k = 0; k < K; ++k)
#pragma unroll
              for (int j = 0; j < V; ++j) v[j] = fmaf(w[k][j], d[K - 1 - k][j], v[j]);
            const int i_state = row - len + K - 1;   // row of the state that leaves
            if (d_out && i_state >= 0 && i_state < K - 1) v += loadv<V>(d_out + (long long)i_state * a.C + p.c, p.n);
            if (row >= 0) {
              if (row >= len) v = floats<V>{};
              put<V>(dx + row * a.dxt + p.c, v, p);
            } else if (d_in) {
              put<V>(d_in + (long long)(row + K - 1) * a.C + p.c, v, p);
            }
          }
#pragma unroll
          for (int k = 0; k < K - 1; ++k) {
            win[k] = win[k + 1];
            d[k] = d[k + 1];
          }
        }
      }
    }
  }
  // the workgroup's runs meet in shared memory, in order
  const int lx = 1 << a.lx_log2, ly = 256 >> a.lx_log2;
  float* part = a.part + ((long long)b * gridDim.y + blockIdx.y) * (K + 1) * a.C;
#pragma unroll
  for (int k = 0; k <= K; ++k) {
    const floats<V> v = k < K ? dw[k < K ? k : 0] : db;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j >= p.skip) sh[(j - p.skip) * 256 + threadIdx.x] = v[j];
    __syncthreads();
    for (int i = threadIdx.x; i < lx * V; i += 256) {   // i = channel within the workgroup's
      float s = 0.0f;
      for (int r = 0; r < ly; ++r) s += sh[i % V * 256 + r * lx + i / V];
      const int c = blockIdx.x * lx * V + i;
      if (c < a.C) part[(long long)k * a.C + c] = s;
    }
  }
}

struct ConvShape {
  int run, runs, lx_log2, gx, gy;
};

constexpr int kChannels = 4;   // a thread's; eight take 146 and 209 registers: 67 and 206 us where four take 55 and 103

// Runs are as long as leaves `waves` waves (fewer rows are read twice); short sequences take shorter ones.  8 x 2048 x 4096 forward
// (forward and back) with runs of at most 8 (32) 57 (160) us, 16 (64) 55 (151), 32 (128) 56 (154); 1 x 8192 x 4096 forward and back with half
// the waves 95 us, these 85, twice 89.  Shortest runs of 4 rows rather than 8: 2 x 160 x 261 forward and back 21 us, not 26.
ConvShape conv_shape(int B, int T, int C, int V, int longest, int align, int waves) {
  ConvShape s;
  const int across = (C + V - 1) / V;
  const long long rows_per_thread = (long long)B * T * across / (waves * 64LL);
  long long run = (rows_per_thread + align - 1) / align * align;
  if (run < align) run = align;
  if (run > longest) run = longest;
  s.run = (int)run;
  s.runs = T > 0 ? (T + s.run - 1) / s.run : 1;
  s.lx_log2 = 0;
  while (s.lx_log2 < 8 && (1 << s.lx_log2) < across && (s.lx_log2 < 6 || (256 >> s.lx_log2) > s.runs)) ++s.lx_log2;
  s.gx = (across + (1 << s.lx_log2) - 1) >> s.lx_log2;
  const int ly = 256 >> s.lx_log2;
  s.gy = (s.runs + ly - 1) / ly;
  return s;
}

// the limits of the entry points; a size beyond them needs no workspace, because its call is refused
bool conv_fits(int B, int T, int C) { return B <= 65535 && T <= (1 << 20) && C <= (1 << 20); }

ConvShape fwd_shape(int B, int T, int C) { return conv_shape(B, T, C, kChannels, 16, 4, 8192); }
ConvShape bwd_shape(int B, int T, int C) { return conv_shape(B, T, C, kChannels, 64, 4, 4096); }

template <typename T>
int conv_fwd(const ConvArgs& a, int K, dim3 grid, hipStream_t s) {
  if (K == 2) hipLaunchKernelGGL((causal_conv_fwd_kernel<T, 2, kChannels>), grid, dim3(256), 0, s, a);
  if (K == 3) hipLaunchKernelGGL((causal_conv_fwd_kernel<T, 3, kChannels>), grid, dim3(256), 0, s, a);
  if (K == 4) hipLaunchKernelGGL((causal_conv_fwd_kernel<T, 4, kChannels>), grid, dim3(256), 0, s, a);
  SLAMHIP_HIP(hipGetLastError());
  return SLAMHIP_OK;
}

template <typename T>
int conv_bwd(const ConvArgs& a, int K, dim3 grid, hipStream_t s) {
  if (K == 2) hipLaunchKernelGGL((causal_conv_bwd_kernel<T, 2, kChannels>), grid, dim3(256), 0, s, a);
  if (K == 3) hipLaunchKernelGGL((causal_conv_bwd_kernel<T, 3, kChannels>), grid, dim3(256), 0, s, a);
  if (K == 4) hipLaunchKernelGGL((causal_conv_bwd_kernel<T, 4, kChannels>), grid, dim3(256), 0, s, a);
  SLAMHIP_HIP(hipGetLastError());
  return SLAMHIP_OK;
}

// part's columns are [K + 1][C]; dweight is [C][K]
struct ConvGradients {
  float *dw, *db;
  int C, K;
  __device__ void operator()(int i, float v) const {
    const int k = i / C, c = i - k * C;
    if (k < K)
      dw[(long long)c * K + k] = v;
    else if (db)
      db[c] = v;
  }
};

}  // namespace
}  // namespace slamhip

using namespace slamhip;

extern "C" {

int slamhip_causal_conv_fwd(const void* x, const long long* strides, const float* weight, const float* bias, const void* state_in,
                            const int32_t* lengths, int B, int T, int C, int K, int silu, int dtype, void* y, void* state_out,
                            void* stream) {
  SLAMHIP_REQUIRE(B >= 0 && T >= 0 && C > 0 && K >= 2 && K <= 4 && (dtype == SLAMHIP_F32 || dtype == SLAMHIP_BF16), SLAMHIP_E_ARG,
                  "causal_conv_fwd: need C >= 1, 2 <= K <= 4 and a known type");
  SLAMHIP_REQUIRE(conv_fits(B, T, C), SLAMHIP_E_SIZE, "causal_conv_fwd: at most 65535 sequences, 2^20 steps and channels");
  if (B == 0 || (T == 0 && !state_out)) return SLAMHIP_OK;
  SLAMHIP_REQUIRE(weight && (T == 0 || (x && y && strides)), SLAMHIP_E_ARG, "causal_conv_fwd: null pointer");
  ConvArgs a{};
  a.x = x, a.w = weight, a.bias = bias, a.state_in = state_in, a.y = y, a.state_out = state_out, a.lengths = lengths;
  if (strides) a.xb = strides[0], a.xt = strides[1], a.yb = strides[2], a.yt = strides[3];
  const ConvShape g = fwd_shape(B, T, C);
  a.T = T, a.C = C, a.run = g.run, a.runs = g.runs, a.silu = silu, a.lx_log2 = g.lx_log2;
  const dim3 grid(g.gx, g.gy, B);
  SLAMHIP_REQUIRE(g.gy <= 65535, SLAMHIP_E_SIZE, "causal_conv_fwd: too many steps");
  return dtype == SLAMHIP_BF16 ? conv_fwd<__bf16>(a, K, grid, (hipStream_t)stream) : conv_fwd<float>(a, K, grid, (hipStream_t)stream);
}

size_t slamhip_causal_conv_bwd_workspace_bytes(int B, int T, int C, int K) {
  if (B <= 0 || C <= 0 || T < 0 || K < 2 || K > 4 || !conv_fits(B, T, C)) return 0;
  return (size_t)B * bwd_shape(B, T, C).gy * (K + 1) * C * sizeof(float);
}

int slamhip_causal_conv_bwd(const void* dy, const void* x, const long long* strides, const float* weight, const float* bias,
                            const void* state_in, const void* d_state_out, const int32_t* lengths, int B, int T, int C, int K, int silu,
                            int dtype, void* dx, float* dweight, float* dbias, void* d_state_in, void* workspace,
                            size_t workspace_bytes, void* stream) {
  SLAMHIP_REQUIRE(B >= 0 && T >= 0 && C > 0 && K >= 2 && K <= 4 && (dtype == SLAMHIP_F32 || dtype == SLAMHIP_BF16), SLAMHIP_E_ARG,
                  "causal_conv_bwd: need C >= 1, 2 <= K <= 4 and a known type");
  SLAMHIP_REQUIRE(conv_fits(B, T, C), SLAMHIP_E_SIZE, "causal_conv_bwd: at most 65535 sequences, 2^20 steps and channels");
  SLAMHIP_REQUIRE(weight && dweight && (B == 0 || workspace) && (B == 0 || T == 0 || (dy && x && dx && strides)), SLAMHIP_E_ARG,
                  "causal_conv_bwd: null pointer");
  SLAMHIP_REQUIRE(workspace_bytes >= slamhip_causal_conv_bwd_workspace_bytes(B, T, C, K), SLAMHIP_E_ARG, "causal_conv_bwd: workspace too small");
  hipStream_t s = (hipStream_t)stream;
  const ConvShape g = bwd_shape(B, T, C);
  if (B > 0) {
    ConvArgs a{};
    a.x = x, a.dy = dy, a.w = weight, a.bias = bias, a.state_in = state_in, a.d_state_out = d_state_out, a.lengths = lengths;
    a.dx = dx, a.d_state_in = d_state_in, a.part = (float*)workspace;
    if (strides) a.dyb = strides[0], a.dyt = strides[1], a.xb = strides[2], a.xt = strides[3], a.dxb = strides[4], a.dxt = strides[5];
    a.T = T, a.C = C, a.run = g.run, a.runs = g.runs, a.silu = silu, a.lx_log2 = g.lx_log2;
    SLAMHIP_REQUIRE(g.gy <= 65535, SLAMHIP_E_SIZE, "causal_conv_bwd: too many steps");
    const int rc = dtype == SLAMHIP_BF16 ? conv_bwd<__bf16>(a, K, dim3(g.gx, g.gy, B), s) : conv_bwd<float>(a, K, dim3(g.gx, g.gy, B), s);
    if (rc != SLAMHIP_OK) return rc;
  }
  SLAMHIP_HIP(column_sums((const float*)workspace, (long long)B * g.gy, (K + 1) * C, ConvGradients{dweight, dbias, C, K}, s));
  return SLAMHIP_OK;
}

}  // extern "C"
