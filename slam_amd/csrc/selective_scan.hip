// Selective scan: a diagonal linear recurrence for each channel whose step, input and output weights depend on the time step.
//
//   dt = softplus(delta + delta_bias);  h_t[n] = exp(dt_t A[n]) h_{t-1}[n] + dt_t u_t B_t[n]
//   y_t = (sum_n C_t[n] h_t[n] + D u_t) silu(z_t)
// Backward, with e_t = dy_t silu(z_t) and g_t[n] = e_t C_t[n] + exp(dt_{t+1} A[n]) g_{t+1}[n], q_t = exp(dt_t A) g_t h_{t-1}:
//   dB_t[n] = sum_c g_t dt_t u_t      dC_t[n] = sum_c e_t h_t       dA[n] = sum_{b,t} q_t dt_t
//   du_t = dt_t sum_n g_t B_t + D e_t      ddt_t = u_t sum_n g_t B_t + sum_n q_t A      dz_t = dy_t inner_t silu'(z_t)
//
// Layout.  Four lanes (a DPP quad) hold one channel, P = N / 4 states each: sums over the states are two quad permutes, a wave
// is 16 channels.  What is needed once a step and channel (softplus, gates, stores) is done by lane k of the quad for
// steps k, k + 4, ... and handed on with quad permutes.  B_t and C_t are staged in shared memory in float32 for the workgroup's
// 64 channels.  Vector instructions bound it: an exponential (two issue slots), two products and two multiply-adds for every (step, channel,
// state), and once a step and channel softplus, gate, sums over the quad.  At 8 x 2048 x 2048 x 16 bfloat16 the passes of 99 and 180 us
// forward issue 23 and 34 vector instructions a step of a wave (16 and 20 of them the recurrence) and keep the units busy 81 and 84 % of
// the time; those of 108 and 495 us back 24 and 101, 83 %.  The bytes alone would take 153 us; float32 takes as long.  With 17 to 32 states the
// pass back needs 379 registers, which leaves one wave a SIMD, and keeps 68 bytes of them in memory: 8 x 2048 x 1024 x 32 takes 86 + 146 us
// forward and 91 + 577 us back.
// A long sequence is cut into chunks where there are too few channels to fill the chip: a first pass leaves each chunk's own end
// state and its sum of dt (the decay over a chunk is exp(A sum dt)), and every chunk of the second pass joins those in front of
// it.  The backward pass runs over the chunks the same way from behind, and recomputes the states of TB steps from the one that
// the forward pass kept in front of them.
#include <hip/hip_runtime.h>

#include <type_traits>

#include "common.h"
#include "sequence_device.h"

namespace slamhip {
namespace {

// steps that the states are kept apart, and that the backward pass works on at once: it holds as many states and decays of each
// of a lane's P in registers
constexpr int kept_steps(int P) { return P <= 2 ? 16 : 8; }
constexpr int kFwdSteps = 16;   // steps that the forward pass stages at once

struct ScanArgs {
  const void *u, *delta, *z, *Bm, *Cm, *dy;
  const float *A, *D, *bias, *state_in, *d_state_out;
  void *y, *du, *ddelta, *dz;
  float *state_out, *kept, *d_state_in;
  float *ends, *sums, *part, *part_bc;   // workspace
  const int* lengths;
  long long ub, ut, deltab, deltat, zb, zt, Bb, Bt, Cb, Ct, yb, yt;
  long long dyb, dyt, dub, dut, ddeltab, ddeltat, dzb, dzt;
  int T, C, N, chunk, chunks, softplus;
};

template <int CTRL>
__device__ __forceinline__ float dpp_(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}

template <int K>
__device__ __forceinline__ float quad_lane(float v) {
  return dpp_<K * 0x55>(v);
}

__device__ __forceinline__ float quad_sum(float v) {
  v += dpp_<0xB1>(v);
  return v + dpp_<0x4E>(v);
}

// v[k] summed over the quad, for the lane whose place in the quad is k
__device__ __forceinline__ float quad_sum_own(const float (&v)[4], int q) {
  const bool odd = q & 1, high = q & 2;
  const float a0 = (odd ? v[1] : v[0]) + dpp_<0xB1>(odd ? v[0] : v[1]);
  const float a1 = (odd ? v[3] : v[2]) + dpp_<0xB1>(odd ? v[2] : v[3]);
  return (high ? a1 : a0) + dpp_<0x4E>(high ? a0 : a1);
}

// ln(1 + e^v); the part of e that the rounding of 1 + e drops is added back, so that small results keep their relative precision
__device__ __forceinline__ float softplus_(float v, float e) {
  const float w = 1.0f + e;
  const float lost = e - (w - 1.0f);
  return fmaxf(v, 0.0f) + fmaf(log2_(w), kLn2, lost);
}

struct Lane {
  int q, c, cc, len, own, b;   // own: the lane's own length, 0 without a channel
  bool live;
};

__device__ __forceinline__ Lane scan_lane(const ScanArgs& a) {
  Lane l;
  l.q = threadIdx.x & 3;
  l.c = blockIdx.x * 64 + (threadIdx.x >> 2);
  l.live = l.c < a.C;
  l.cc = l.live ? l.c : a.C - 1;   // lanes without a channel read the last one's values, have steps of no length and store nothing
  l.b = blockIdx.z;
  l.len = a.T;
  if (a.lengths) {
    const int n = a.lengths[l.b];
    l.len = n < 0 ? 0 : (n > a.T ? a.T : n);
  }
  l.own = l.live ? l.len : 0;
  return l;
}

// a lane's P states of a row of N; all lanes' are there when N == 4 P
template <int P>
struct StateVector {
  typedef float type __attribute__((ext_vector_type(P), aligned(4)));
};
template <>
struct StateVector<1> {
  typedef float type;
};

template <int P>
__device__ __forceinline__ void load_states(const float* p, int N, int q, float (&v)[P]) {
  if (P > 1 && N == 4 * P) {
    const typename StateVector<P>::type r = *reinterpret_cast<const typename StateVector<P>::type*>(p + q * P);
    __builtin_memcpy(v, &r, sizeof(v));
  } else {
#pragma unroll
    for (int i = 0; i < P; ++i) v[i] = q * P + i < N ? p[q * P + i] : 0.0f;
  }
}

template <int P>
__device__ __forceinline__ void store_states(float* p, int N, int q, const float (&v)[P]) {
  if (P > 1 && N == 4 * P) {
    typename StateVector<P>::type r;
    __builtin_memcpy(&r, v, sizeof(v));
    *reinterpret_cast<typename StateVector<P>::type*>(p + q * P) = r;
  } else {
#pragma unroll
    for (int i = 0; i < P; ++i)
      if (q * P + i < N) p[q * P + i] = v[i];
  }
}

// B and C of a block of steps, one value a thread and pass; zeros beyond the sequence's end and beyond N.  The values stay in the
// sequences' type until they are put away: a conversion behind a guarded load would be waited for before the next load.
template <typename T, int P, int TB>
struct Staged {
  static constexpr int kPer = TB * 8 * P / 256 > 0 ? TB * 8 * P / 256 : 1;
  const T* p;           // value 0 of the thread; the next ones are `rows` steps on
  long long st;
  bool there;
  int row;
  T v[kPer];
  __device__ __forceinline__ Staged(const ScanArgs& a, const Lane& l, int t0) {
    const int at = threadIdx.x % (TB * 8 * P), n = at % (4 * P), which = at / (4 * P) & 1;
    st = which ? a.Ct : a.Bt;
    row = at / (8 * P);
    p = (which ? (const T*)a.Cm + l.b * a.Cb : (const T*)a.Bm + l.b * a.Bb) + n + (long long)(t0 + row) * st;
    there = n < a.N;
  }
  static constexpr int kRows = 256 / (8 * P);
  __device__ __forceinline__ void load(int t0, int len) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      v[i] = (T)0.0f;
      if (there && t0 + row + i * kRows < len) v[i] = p[i * kRows * st];
    }
  }
  __device__ __forceinline__ void advance(int steps) { p += steps * st; }
  __device__ __forceinline__ void put(float* sh) const {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (TB * 8 * P >= 256 || threadIdx.x < TB * 8 * P) sh[i * 256 + threadIdx.x] = (float)v[i];
  }
};

template <int P>
__device__ __forceinline__ void read_states(const float* sh, float (&v)[P]) {
#pragma unroll
  for (int i = 0; i < P; ++i) v[i] = sh[i];
}

// a lane's own steps of a block: t0 + q, t0 + q + 4, ...; the pointer moves with the block (a product of 64 bits for every access
// costs as much as the recurrence)
template <typename T, int G>
struct Rows {
  typedef T __attribute__((address_space(1))) Global;
  Global* p;        // step t0 + q
  long long four;   // four steps
  __device__ __forceinline__ Rows(const void* base, long long sb, long long st, const Lane& l, int t0)
      : p((Global*)base + l.b * sb + (t0 + l.q) * st + l.cc), four(4 * st) {}
  __device__ __forceinline__ void load(T (&v)[G], bool full, int t0, const Lane& l) const {
    if (full) {
#pragma unroll
      for (int i = 0; i < G; ++i) v[i] = p[i * four];
    } else {
#pragma unroll
      for (int i = 0; i < G; ++i) {
        v[i] = (T)0.0f;
        if (t0 + 4 * i + l.q < l.own) v[i] = p[i * four];
      }
    }
  }
  __device__ __forceinline__ void store(int i, float v) const { p[i * four] = (T)v; }
  __device__ __forceinline__ void advance(int fours) {
    p += fours * four;
    asm("" : "+v"(p));   // one pointer a tensor: the compiler would otherwise carry one for each of a block's rows
  }
};

// STATES: the first pass of a cut sequence: each chunk's end state from zero (the first chunk's from state_in) and its sum of dt
template <typename T, int P, bool STATES, bool Z>
__global__ void __launch_bounds__(256, 4) selective_scan_fwd_kernel(ScanArgs a) {
  constexpr int TB = kFwdSteps, G = TB / 4, TK = kept_steps(P);
  __shared__ float bc[2][TB * 8 * P];
  const Lane l = scan_lane(a);
  const int chunk = blockIdx.y, t_begin = chunk * a.chunk, t_end = min(t_begin + a.chunk, a.T);
  const long long bC = (long long)l.b * a.C + l.cc;
  const long long slots = a.chunks + 1;   // a.ends [B][chunks + 1][C][N]: state_in, then each chunk's end
  float h[P], A2[P];
  load_states<P>(a.A + (long long)l.cc * a.N, a.N, l.q, A2);
#pragma unroll
  for (int i = 0; i < P; ++i) {
    A2[i] *= kLog2e;
    h[i] = 0.0f;
  }
  if (STATES || a.chunks == 1) {
    if (chunk == 0 && a.state_in) load_states<P>(a.state_in + bC * a.N, a.N, l.q, h);
    if (STATES && chunk == 0 && l.live) store_states<P>(a.ends + ((long long)l.b * slots * a.C + l.c) * a.N, a.N, l.q, h);
  } else if (chunk == 0) {
    load_states<P>(a.ends + ((long long)l.b * slots * a.C + l.cc) * a.N, a.N, l.q, h);
  } else {
#pragma unroll 8
    for (int j = 0; j < chunk; ++j) {
      const float s = a.sums[((long long)l.b * a.chunks + j) * a.C + l.cc];
      float e[P];
      load_states<P>(a.ends + (((long long)l.b * slots + j + 1) * a.C + l.cc) * a.N, a.N, l.q, e);
#pragma unroll
      for (int i = 0; i < P; ++i) h[i] = fmaf(exp2_(A2[i] * s), h[i], e[i]);
    }
  }
  const float bias = a.bias ? a.bias[l.cc] : 0.0f, D = a.D ? a.D[l.cc] : 0.0f;
  const long long nkept = (a.T + TK - 1) / TK;
  float dt_sum = 0.0f;

  Staged<T, P, TB> next_bc(a, l, t_begin);
  Rows<T, G> ru(a.u, a.ub, a.ut, l, t_begin), rd(a.delta, a.deltab, a.deltat, l, t_begin), rz(a.z, a.zb, a.zt, l, t_begin);
  Rows<T, G> ry(a.y, a.yb, a.yt, l, t_begin);
  float* kept = a.kept + (((long long)l.b * nkept + t_begin / TK) * a.C + l.c) * a.N;
  const long long kept_step = (long long)a.C * a.N;
  T nu[G], nd[G], nz[G];
  auto fetch = [&](int t0) {
    const bool full = t0 + TB <= l.len;
    next_bc.load(t0, l.len);
    ru.load(nu, full, t0, l);
    rd.load(nd, full, t0, l);
    if (!STATES && Z) rz.load(nz, full, t0, l);
    next_bc.advance(TB);
    ru.advance(G);
    rd.advance(G);
    if (!STATES && Z) rz.advance(G);
  };
  if (t_begin < t_end) fetch(t_begin);
  int buf = 0;
  for (int t0 = t_begin; t0 < t_end; t0 += TB, buf ^= 1) {
    next_bc.put(bc[buf]);
    float u[G], dt[G], x[G], z[G];
#pragma unroll
    for (int i = 0; i < G; ++i) dt[i] = (float)nd[i] + bias;
    if (a.softplus)
#pragma unroll
      for (int i = 0; i < G; ++i) dt[i] = softplus_(dt[i], exp2_(-kLog2e * fabsf(dt[i])));
#pragma unroll
    for (int i = 0; i < G; ++i) {
      if (t0 + 4 * i + l.q >= l.own) dt[i] = 0.0f;
      u[i] = (float)nu[i];
      x[i] = dt[i] * u[i];
      if (STATES) dt_sum += dt[i];
      if (!STATES && Z) z[i] = (float)nz[i];
    }
    __syncthreads();   // bc[buf] is whole; bc[buf ^ 1] has been read by all
    if (t0 + TB < t_end) fetch(t0 + TB);
    // whole blocks run straight through; a block that ends inside asks for every four steps
    auto block = [&](auto whole) {
      constexpr bool WHOLE = decltype(whole)::value;
#pragma unroll
      for (int i = 0; i < G; ++i) {
        if (!STATES && i % (TK / 4) == 0 && a.kept) {
          if (l.live && (WHOLE || t0 + 4 * i < a.T)) store_states<P>(kept, a.N, l.q, h);
          kept += kept_step;
        }
        float inner[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (WHOLE || t0 + 4 * i < l.len) {
          auto step = [&](auto k) {
            constexpr int K = decltype(k)::value;
            const float* sh = bc[buf] + (4 * i + K) * 8 * P + l.q * P;
            float Bv[P], Cv[P];
            read_states<P>(sh, Bv);
            if (!STATES) read_states<P>(sh + 4 * P, Cv);
            const float d = quad_lane<K>(dt[i]), xv = quad_lane<K>(x[i]);
#pragma unroll
            for (int p = 0; p < P; ++p) {
              h[p] = fmaf(exp2_(A2[p] * d), h[p], xv * Bv[p]);
              if (!STATES) inner[K] = fmaf(h[p], Cv[p], inner[K]);
            }
          };
          step(std::integral_constant<int, 0>{});
          step(std::integral_constant<int, 1>{});
          step(std::integral_constant<int, 2>{});
          step(std::integral_constant<int, 3>{});
        }
        if (!STATES) {
          const int t = t0 + 4 * i + l.q;
          float v = fmaf(D, u[i], quad_sum_own(inner, l.q));
          if (Z) v *= z[i] * sigmoid_(z[i]);
          if (!WHOLE && t >= l.len) v = 0.0f;
          if (l.live && (WHOLE || t < t_end)) ry.store(i, v);
        }
      }
    };
    if (t0 + TB <= l.len)
      block(std::true_type{});
    else
      block(std::false_type{});
    if (!STATES) ry.advance(G);
  }
  if (STATES) {
    if (l.live) {
      store_states<P>(a.ends + (((long long)l.b * slots + chunk + 1) * a.C + l.c) * a.N, a.N, l.q, h);
      const float s = quad_sum(dt_sum);
      if (l.q == 0) a.sums[((long long)l.b * a.chunks + chunk) * a.C + l.c] = s;
    }
  } else if (a.state_out && chunk == a.chunks - 1 && l.live) {
    store_states<P>(a.state_out + bC * a.N, a.N, l.q, h);
  }
}

// One step (T = 1): the state comes and goes, nothing is handed on.  No staging, no barrier, few registers: all waves of 32 x 4096
// channels are on the chip at once.
template <typename T, int P, bool Z>
__global__ void __launch_bounds__(256) selective_scan_step_kernel(ScanArgs a) {
  const Lane l = scan_lane(a);
  if (!l.live) return;   // whole quads
  const long long bC = (long long)l.b * a.C + l.c;
  float h[P], A2[P];
#pragma unroll
  for (int i = 0; i < P; ++i) h[i] = 0.0f;
  if (a.state_in) load_states<P>(a.state_in + bC * a.N, a.N, l.q, h);
  float y = 0.0f;
  if (l.len > 0) {
    load_states<P>(a.A + (long long)l.c * a.N, a.N, l.q, A2);
    const floats<P> Bv = loadv<P>((const T*)a.Bm + l.b * a.Bb + l.q * P, a.N - l.q * P);
    const floats<P> Cv = loadv<P>((const T*)a.Cm + l.b * a.Cb + l.q * P, a.N - l.q * P);
    const float u = (float)((const T*)a.u)[l.b * a.ub + l.c];
    const float z = Z ? (float)((const T*)a.z)[l.b * a.zb + l.c] : 0.0f;
    float dt = (float)((const T*)a.delta)[l.b * a.deltab + l.c] + (a.bias ? a.bias[l.c] : 0.0f);
    if (a.softplus) dt = softplus_(dt, exp2_(-kLog2e * fabsf(dt)));
    float inner = 0.0f;
#pragma unroll
    for (int i = 0; i < P; ++i) {
      h[i] = fmaf(exp2_(A2[i] * kLog2e * dt), h[i], dt * u * Bv[i]);
      inner = fmaf(h[i], Cv[i], inner);
    }
    y = quad_sum(inner);
    if (a.D) y = fmaf(a.D[l.c], u, y);
    if (Z) y *= z * sigmoid_(z);
  }
  if (l.q == 0) ((T*)a.y)[l.b * a.yb + l.c] = (T)y;
  if (a.state_out) store_states<P>(a.state_out + bC * a.N, a.N, l.q, h);
}

// v[p] (p < P) and w[p] summed over the wave's 16 channels (lanes of equal place in the quad).  Swapping halves (rows) of two
// registers and adding them sums both at once, half a wave (a row) each; what is left are four channels of a row.
template <int P>
__device__ __forceinline__ void channel_sums(float (&v)[2 * P]) {
  // after the swaps, register r of lane row `row` holds the sum of value 4 r' + order[row]
  static_assert(P == 1 || P == 2 || P == 4 || P == 8, "");
  if constexpr (2 * P >= 4) {
#pragma unroll
    for (int i = 0; i < P; ++i) {
      auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[2 * i]), __float_as_uint(v[2 * i + 1]), false, false);
      v[i] = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
#pragma unroll
    for (int i = 0; i < P / 2; ++i) {
      auto s = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[2 * i]), __float_as_uint(v[2 * i + 1]), false, false);
      v[i] = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    }
#pragma unroll
    for (int i = 0; i < P / 2; ++i) {
      v[i] += dpp_<0x124>(v[i]);   // row_ror:4
      v[i] += dpp_<0x128>(v[i]);   // row_ror:8
    }
  } else {   // two values: one for each half of the wave, rows added with a further swap
    auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[0]), __float_as_uint(v[1]), false, false);
    v[0] = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v[0]), __float_as_uint(v[0]), false, false);
    v[0] = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    v[0] += dpp_<0x124>(v[0]);
    v[0] += dpp_<0x128>(v[0]);
  }
}

// what value of v register i of channel_sums() holds in row `row` of the wave
template <int P>
__device__ __forceinline__ int channel_sum_index(int i, int row) {
  if (P == 1) return row >> 1;                       // halves
  return 4 * i + 2 * (row & 1) + (row >> 1);         // row 0: 4i, row 1: 4i + 2, row 2: 4i + 1, row 3: 4i + 3
}

// CARRY: the first pass of a cut sequence: the gradient that each chunk by itself hands to the state in front of it
template <typename T, int P, bool CARRY, bool Z>
__global__ void __launch_bounds__(256, P == 8 && !CARRY ? 1 : 2) selective_scan_bwd_kernel(ScanArgs a) {
  constexpr int TB = kept_steps(P), G = TB / 4, V = TB * 8 * P;
  __shared__ float bc[2][V];
  __shared__ float bc_grad[CARRY ? 1 : 2][CARRY ? 1 : 4][CARRY ? 1 : V];
  const Lane l = scan_lane(a);
  const int wave = threadIdx.x >> 6;
  const int chunk = blockIdx.y + (CARRY ? 1 : 0), t_begin = chunk * a.chunk, t_end = min(t_begin + a.chunk, a.T);
  const long long bC = (long long)l.b * a.C + l.cc;
  float A2[P], g[P], dA[P];
  load_states<P>(a.A + (long long)l.cc * a.N, a.N, l.q, A2);
#pragma unroll
  for (int i = 0; i < P; ++i) {
    A2[i] *= kLog2e;
    g[i] = 0.0f;
    dA[i] = 0.0f;
  }
  if (!CARRY || chunk == a.chunks - 1)
    if (a.d_state_out) load_states<P>(a.d_state_out + bC * a.N, a.N, l.q, g);
  if (!CARRY)
#pragma unroll 8
    for (int j = a.chunks - 1; j > chunk; --j) {   // the last chunk's own carry holds d_state_out already
      const float s = a.sums[((long long)l.b * a.chunks + j) * a.C + l.cc];
      float e[P];
      load_states<P>(a.ends + (((long long)l.b * a.chunks + j) * a.C + l.cc) * a.N, a.N, l.q, e);
#pragma unroll
      for (int i = 0; i < P; ++i) g[i] = j == a.chunks - 1 ? e[i] : fmaf(exp2_(A2[i] * s), g[i], e[i]);
    }
  const float bias = a.bias ? a.bias[l.cc] : 0.0f, D = a.D ? a.D[l.cc] : 0.0f;
  const long long nkept = (a.T + TB - 1) / TB;
  const int groups = gridDim.x;
  float dt_sum = 0.0f, dD = 0.0f, dbias = 0.0f;

  // where the lane leaves its sums of channel_sums() of a group of four steps
  const int row_channel = threadIdx.x >> 2 & 3;
  int grad_at[P >= 2 ? P / 2 : 1];
#pragma unroll
  for (int r = 0; r < (P >= 2 ? P / 2 : 1); ++r) {
    const int at = channel_sum_index<P>(r, threadIdx.x >> 4 & 3);   // below P: dB of state at, else dC of state at - P
    grad_at[r] = row_channel * 8 * P + (at >= P ? 4 * P + at - P : at) + l.q * P;
  }
  const int t_last = t_begin + (t_end - 1 - t_begin) / TB * TB;
  Staged<T, P, TB> next_bc(a, l, t_last);
  Rows<T, G> ru(a.u, a.ub, a.ut, l, t_last), rd(a.delta, a.deltab, a.deltat, l, t_last), rz(a.z, a.zb, a.zt, l, t_last);
  Rows<T, G> ry(a.dy, a.dyb, a.dyt, l, t_last), rdu(a.du, a.dub, a.dut, l, t_last), rdd(a.ddelta, a.ddeltab, a.ddeltat, l, t_last);
  Rows<T, G> rdz(a.dz, a.dzb, a.dzt, l, t_last);
  const float* kept = a.kept + (((long long)l.b * nkept + t_last / TB) * a.C + l.cc) * a.N;
  T nu[G], nd[G], nz[G], ny[G];
  float nh[P];
  auto fetch = [&](int t0) {
    const bool full = t0 + TB <= l.len;
    next_bc.load(t0, l.len);
    if (!CARRY) {
      load_states<P>(kept, a.N, l.q, nh);
      kept -= (long long)a.C * a.N;
      ru.load(nu, full, t0, l);
      ru.advance(-G);
    }
    rd.load(nd, full, t0, l);
    ry.load(ny, full, t0, l);
    if (Z) rz.load(nz, full, t0, l);
    next_bc.advance(-TB);
    rd.advance(-G);
    ry.advance(-G);
    if (Z) rz.advance(-G);
  };
  // part_bc [B][T][groups][2][4 P]: a block's dB and dC of the workgroup's channels, once all waves have left theirs
  float* part_bc = a.part_bc + (((long long)l.b * a.T + t_last + threadIdx.x / (8 * P)) * groups + blockIdx.x) * 8 * P + threadIdx.x % (8 * P);
  const long long part_row = (long long)groups * 8 * P;
  auto put_part = [&](int t0, int buf) {
    if constexpr (!CARRY) {
      constexpr int kRows = 256 / (8 * P);
#pragma unroll
      for (int i = 0; i < (V + 255) / 256; ++i) {
        const int at = i * 256 + threadIdx.x;
        if (at < V && t0 + at / (8 * P) < t_end)
          part_bc[i * kRows * part_row] = (bc_grad[buf][0][at] + bc_grad[buf][1][at]) + (bc_grad[buf][2][at] + bc_grad[buf][3][at]);
      }
      part_bc -= TB * part_row;
    }
  };
  int buf = 0;
  if (t_begin < t_end) fetch(t_last);
  for (int t0 = t_last; t0 >= t_begin && t_begin < t_end; t0 -= TB, buf ^= 1) {
    float u[G], z[G], dy[G], raw[G], dt[G], e[G], h[P];
    next_bc.put(bc[buf]);
#pragma unroll
    for (int i = 0; i < G; ++i) dt[i] = raw[i] = (float)nd[i] + bias;
    if (a.softplus)
#pragma unroll
      for (int i = 0; i < G; ++i) dt[i] = softplus_(raw[i], exp2_(-kLog2e * fabsf(raw[i])));
#pragma unroll
    for (int i = 0; i < G; ++i) {   // behind the sequence u, dy and z are zero
      if (t0 + 4 * i + l.q >= l.own) dt[i] = 0.0f;
      // the sums over the channels take no part of a lane without one
      if (!CARRY) u[i] = l.live ? (float)nu[i] : 0.0f;
      e[i] = dy[i] = CARRY || l.live ? (float)ny[i] : 0.0f;
      if (CARRY) dt_sum += dt[i];
    }
    if (Z)
#pragma unroll
      for (int i = 0; i < G; ++i) {
        z[i] = (float)nz[i];
        e[i] *= z[i] * sigmoid_(z[i]);
      }
    if (!CARRY)
#pragma unroll
      for (int i = 0; i < P; ++i) h[i] = nh[i];
    __syncthreads();   // bc[buf] is whole, and so is the previous block's bc_grad; what was read two blocks ago may be written
    if (t0 - TB >= t_begin) fetch(t0 - TB);
    if constexpr (CARRY) {
#pragma unroll
      for (int i = G - 1; i >= 0; --i) {
        auto step = [&](auto k) {
          constexpr int K = decltype(k)::value;
          const float* sh = bc[buf] + (4 * i + K) * 8 * P + l.q * P;
          float Cv[P];
          read_states<P>(sh + 4 * P, Cv);
          const float d = quad_lane<K>(dt[i]), ev = quad_lane<K>(e[i]);
#pragma unroll
          for (int p = 0; p < P; ++p) g[p] = fmaf(ev, Cv[p], g[p]) * exp2_(A2[p] * d);
        };
        step(std::integral_constant<int, 3>{});
        step(std::integral_constant<int, 2>{});
        step(std::integral_constant<int, 1>{});
        step(std::integral_constant<int, 0>{});
      }
    } else {
      if (t0 + TB < t_end) put_part(t0 + TB, buf ^ 1);
      float hs[TB][P], as[TB][P];   // the state in front of each step, and its decay
#pragma unroll
      for (int i = 0; i < G; ++i) {
        const float x = dt[i] * u[i];
        auto step = [&](auto k) {
          constexpr int K = decltype(k)::value;
          const float* sh = bc[buf] + (4 * i + K) * 8 * P + l.q * P;
          float Bv[P];
          read_states<P>(sh, Bv);
          const float d = quad_lane<K>(dt[i]), xv = quad_lane<K>(x);
#pragma unroll
          for (int p = 0; p < P; ++p) {
            hs[4 * i + K][p] = h[p];
            as[4 * i + K][p] = exp2_(A2[p] * d);
            h[p] = fmaf(as[4 * i + K][p], h[p], xv * Bv[p]);
          }
        };
        step(std::integral_constant<int, 0>{});
        step(std::integral_constant<int, 1>{});
        step(std::integral_constant<int, 2>{});
        step(std::integral_constant<int, 3>{});
        __builtin_amdgcn_sched_barrier(0);
      }
      // what the steps back need again is read and spread over the quad again: kept since the steps forward it would cost 48 registers
      asm volatile("" ::: "memory");
#pragma unroll
      for (int i = 0; i < G; ++i) asm volatile("" : "+v"(dt[i]), "+v"(u[i]));
      auto reverse = [&](auto whole) {
        constexpr bool WHOLE = decltype(whole)::value;
#pragma unroll
        for (int i = G - 1; i >= 0; --i) {
          constexpr int R = P >= 2 ? P / 2 : 1;
          const float x = dt[i] * u[i];
          float inner[4], gb[4], qa[4], own_sum[R];
          auto step = [&](auto k) {
            constexpr int K = decltype(k)::value;
            const float* sh = bc[buf] + (4 * i + K) * 8 * P + l.q * P;
            float Bv[P], Cv[P], v[2 * P];
            read_states<P>(sh, Bv);
            read_states<P>(sh + 4 * P, Cv);
            const float d = quad_lane<K>(dt[i]), xv = quad_lane<K>(x), ev = quad_lane<K>(e[i]);
            const bool inside = t0 + 4 * i + K < l.len;
            float s_in = 0.0f, s_gb = 0.0f, s_qa = 0.0f;
#pragma unroll
            for (int p = 0; p < P; ++p) {
              g[p] = fmaf(ev, Cv[p], g[p]);
              if (Z) s_in = fmaf(h[p], Cv[p], s_in);
              v[P + p] = ev * h[p];
              v[p] = g[p] * xv;
              s_gb = fmaf(g[p], Bv[p], s_gb);
              g[p] *= as[4 * i + K][p];
              h[p] = hs[4 * i + K][p];
              const float q = g[p] * h[p];
              // behind the sequence d is zero, but its state (of a slot that is not used, say) may be no number
              if (WHOLE || inside) dA[p] = fmaf(q, d, dA[p]);
              s_qa = fmaf(q, A2[p], s_qa);
            }
            // the sums are finished here: left to the end of the group they would keep B, C and the products of all four steps
            asm volatile("" : "+v"(s_in), "+v"(s_gb), "+v"(s_qa));
            inner[K] = s_in;
            gb[K] = s_gb;
            qa[K] = s_qa;
            channel_sums<P>(v);
            // the four channels of a row hold the same sums: channel K keeps those of step K
#pragma unroll
            for (int r = 0; r < R; ++r) own_sum[r] = K == 3 || row_channel == K ? v[r] : own_sum[r];
            __builtin_amdgcn_sched_barrier(0);   // steps are not mixed: there are no registers for it
          };
          step(std::integral_constant<int, 3>{});
          step(std::integral_constant<int, 2>{});
          step(std::integral_constant<int, 1>{});
          step(std::integral_constant<int, 0>{});
#pragma unroll
          for (int r = 0; r < R; ++r) bc_grad[buf][wave][4 * i * 8 * P + grad_at[r]] = own_sum[r];
          const int t = t0 + 4 * i + l.q;
          const float gb_sum = quad_sum_own(gb, l.q), qa_sum = quad_sum_own(qa, l.q);
          const bool in = WHOLE || t < l.own;
          const float slope = a.softplus ? sigmoid_(raw[i]) : 1.0f;
          float du = fmaf(gb_sum, dt[i], D * e[i]);
          float dd = fmaf(gb_sum, u[i], qa_sum * kLn2) * slope;
          if (!in) du = dd = 0.0f;
          dD = fmaf(e[i], u[i], dD);
          dbias += dd;
          const bool there = l.live && (WHOLE || t < t_end);
          if (there) {
            rdu.store(i, du);
            rdd.store(i, dd);
          }
          if (Z) {
            const float s = sigmoid_(z[i]);
            float dz = dy[i] * fmaf(D, u[i], quad_sum_own(inner, l.q)) * s * fmaf(z[i], 1.0f - s, 1.0f);
            if (!in) dz = 0.0f;
            if (there) rdz.store(i, dz);
          }
        }
      };
      if (t0 + TB <= l.len)
        reverse(std::true_type{});
      else
        reverse(std::false_type{});
      rdu.advance(-G);
      rdd.advance(-G);
      if (Z) rdz.advance(-G);
    }
  }
  if constexpr (CARRY) {
    if (l.live) {
      store_states<P>(a.ends + (((long long)l.b * a.chunks + chunk) * a.C + l.c) * a.N, a.N, l.q, g);
      const float s = quad_sum(dt_sum);
      if (l.q == 0) a.sums[((long long)l.b * a.chunks + chunk) * a.C + l.c] = s;
    }
  } else {
    __syncthreads();
    put_part(t_begin, buf ^ 1);
    dD = quad_sum(dD);
    dbias = quad_sum(dbias);
    if (l.live) {
      if (a.d_state_in && chunk == 0) store_states<P>(a.d_state_in + bC * a.N, a.N, l.q, g);
      // part [B * chunks][C * N of dA, C of dD, C of the bias]
      float* part = a.part + ((long long)l.b * a.chunks + chunk) * a.C * (a.N + 2);
      store_states<P>(part + (long long)l.c * a.N, a.N, l.q, dA);
      if (l.q == 0) {
        part[(long long)a.C * a.N + l.c] = dD;
        part[(long long)a.C * (a.N + 1) + l.c] = dbias;
      }
    }
  }
}

// The parts of dB and dC (of the channel groups; a thread a value) and those of dA, dD and the bias (of sequences and chunks; 32
// columns a workgroup), in one launch: the first bc_groups workgroups take dB and dC.  Fixed orders.
template <typename T>
__global__ void __launch_bounds__(256) selective_scan_parts_kernel(ScanArgs a, int bc_groups, int groups, int np, int B, void* dB, void* dC,
                                                                   long long dBb, long long dBt, long long dCb, long long dCt, float* dA,
                                                                   float* dD, float* dbias) {
  if ((int)blockIdx.x < bc_groups) {
    const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
    const long long step = at / (2 * np);
    if (step >= (long long)B * a.T) return;
    const int v = (int)(at - step * 2 * np), which = v / np, n = v - which * np;
    if (n >= a.N) return;
    const int b = (int)(step / a.T), t = (int)(step - (long long)b * a.T);
    float s = 0.0f;
#pragma unroll 8
    for (int g = 0; g < groups; ++g) s += a.part_bc[(step * groups + g) * 2 * np + v];
    if (a.lengths && t >= a.lengths[b]) s = 0.0f;
    if (which)
      ((T*)dC)[b * dCb + t * dCt + n] = (T)s;
    else
      ((T*)dB)[b * dBb + t * dBt + n] = (T)s;
    return;
  }
  __shared__ float sh[8][33];
  const int tx = threadIdx.x & 31, ty = threadIdx.x >> 5, columns = a.C * (a.N + 2);
  const int c = (blockIdx.x - bc_groups) * 32 + tx, parts = B * a.chunks;
  float s = 0.0f;
  if (c < columns)
#pragma unroll 8
    for (int p = ty; p < parts; p += 8) s += a.part[(long long)p * columns + c];
  sh[ty][tx] = s;
  __syncthreads();
  if (ty || c >= columns) return;
  s = 0.0f;
  for (int i = 0; i < 8; ++i) s += sh[i][tx];
  if (c < a.C * a.N)
    dA[c] = s;
  else if (c < a.C * (a.N + 1)) {
    if (dD) dD[c - a.C * a.N] = s;
  } else if (dbias)
    dbias[c - a.C * (a.N + 1)] = s;
}

struct ScanShape {
  int P, groups, chunk, chunks;
};

// Chunks, where the channels alone give fewer waves than two a SIMD (2048): then as many as make eight (a first pass costs two
// thirds of the second whatever their number).  Measured at 8 x 2048 steps x 2048 channels x 16 states (1024 waves): whole 271 us
// forward and 665 us back, cut in 8 98 + 180 us and 105 + 495 us; at 1024 waves and more a short sequence stays whole (32 x 130 x
// 700 x 4 forward 22 us, cut 25 us).  A chunk also joins all those in front of it, one after the other, so none is shorter than
// the square root of the sequence: 1 x 4096 x 64 x 16 forward takes 83, 48, 36, 41 us in chunks of 16, 32, 64, 128.  What is shorter than
// two of the shortest chunks stays whole: 1 x 31 x 512 x 16 forward 6.8 us, cut 8.5.
// Back, the shortest chunks are 16 steps longer where they make more than 2048 waves, whose sums and joins cost more than their steps: us
// back with the shortest and the longer ones, 5 x 200 x 1000 x 8 34 and 31, 4 x 333 x 1024 x 16 50 and 44; below, 1 x 200 x 512 x 16
// 18 and 22, 2 x 500 x 300 x 32 41 and 49.
ScanShape scan_shape(int B, int T, int C, int N, bool back) {
  ScanShape s;
  s.P = N <= 4 ? 1 : N <= 8 ? 2 : N <= 16 ? 4 : 8;
  s.groups = (C + 63) / 64;
  const long long waves = (long long)(B > 0 ? B : 1) * s.groups * 4;   // without sequences the parameters' gradients are still asked for
  int shortest = 16;
  while ((long long)shortest * shortest < T) shortest += 16;
  const long long chunks = waves >= 2048 || (waves >= 1024 && T < 512) || T < 2 * shortest ? 1 : (8192 + waves - 1) / waves;
  if (back && waves * ((T + shortest - 1) / shortest) > 2048) shortest += 16;
  const int even = (int)(((T + chunks - 1) / chunks + 15) / 16 * 16);
  s.chunk = even > shortest ? even : shortest;
  s.chunks = T > 0 ? (T + s.chunk - 1) / s.chunk : 1;
  return s;
}

template <typename T, int P>
int scan_fwd(const ScanArgs& a, int groups, int B, hipStream_t s) {
  const dim3 grid(groups, a.chunks, B);
  if (a.T == 1 && !a.kept) {
    if (a.z)
      hipLaunchKernelGGL((selective_scan_step_kernel<T, P, true>), grid, dim3(256), 0, s, a);
    else
      hipLaunchKernelGGL((selective_scan_step_kernel<T, P, false>), grid, dim3(256), 0, s, a);
    SLAMHIP_HIP(hipGetLastError());
    return SLAMHIP_OK;
  }
  // nothing follows the last chunk: its end is not asked for
  if (a.chunks > 1) hipLaunchKernelGGL((selective_scan_fwd_kernel<T, P, true, false>), dim3(groups, a.chunks - 1, B), dim3(256), 0, s, a);
  if (a.z)
    hipLaunchKernelGGL((selective_scan_fwd_kernel<T, P, false, true>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((selective_scan_fwd_kernel<T, P, false, false>), grid, dim3(256), 0, s, a);
  SLAMHIP_HIP(hipGetLastError());
  return SLAMHIP_OK;
}

template <typename T, int P>
int scan_bwd(const ScanArgs& a, int groups, int B, hipStream_t s) {
  const dim3 grid(groups, a.chunks, B), carry(groups, a.chunks - 1, B);   // nothing is in front of the first chunk
  if (a.z) {
    if (a.chunks > 1) hipLaunchKernelGGL((selective_scan_bwd_kernel<T, P, true, true>), carry, dim3(256), 0, s, a);
    hipLaunchKernelGGL((selective_scan_bwd_kernel<T, P, false, true>), grid, dim3(256), 0, s, a);
  } else {
    if (a.chunks > 1) hipLaunchKernelGGL((selective_scan_bwd_kernel<T, P, true, false>), carry, dim3(256), 0, s, a);
    hipLaunchKernelGGL((selective_scan_bwd_kernel<T, P, false, false>), grid, dim3(256), 0, s, a);
  }
  SLAMHIP_HIP(hipGetLastError());
  return SLAMHIP_OK;
}

}  // namespace
}  // namespace slamhip

using namespace slamhip;

#define SLAMHIP_SCAN_DISPATCH(FN, P, ...)                     \
  (dtype == SLAMHIP_BF16 ? ((P) == 1   ? FN<__bf16, 1>(__VA_ARGS__)  \
                            : (P) == 2 ? FN<__bf16, 2>(__VA_ARGS__)  \
                            : (P) == 4 ? FN<__bf16, 4>(__VA_ARGS__)  \
                                       : FN<__bf16, 8>(__VA_ARGS__)) \
                         : ((P) == 1   ? FN<float, 1>(__VA_ARGS__)   \
                            : (P) == 2 ? FN<float, 2>(__VA_ARGS__)   \
                            : (P) == 4 ? FN<float, 4>(__VA_ARGS__)   \
                                       : FN<float, 8>(__VA_ARGS__)))

namespace {
// the limits of the entry points; a size beyond them needs no workspace, because its call is refused
bool scan_fits(int B, int T, int C) { return B <= 65535 && T <= (1 << 20) && C <= (1 << 20); }
}  // namespace

#define SLAMHIP_SCAN_SIZES(name)                                                                                               \
  SLAMHIP_REQUIRE(B >= 0 && T >= 0 && C > 0 && N > 0 && N <= 32 && (dtype == SLAMHIP_F32 || dtype == SLAMHIP_BF16), SLAMHIP_E_ARG, \
                  name ": need C >= 1, 1 <= N <= 32 and a known type");                                                        \
  SLAMHIP_REQUIRE(scan_fits(B, T, C), SLAMHIP_E_SIZE, name ": at most 65535 sequences, 2^20 steps and channels")

extern "C" {

size_t slamhip_selective_scan_kept_floats(int B, int T, int C, int N) {
  if (B <= 0 || T <= 0 || C <= 0 || N <= 0 || N > 32 || !scan_fits(B, T, C)) return 0;
  const int tb = kept_steps(scan_shape(B, T, C, N, false).P);
  return (size_t)B * ((T + tb - 1) / tb) * C * N;
}

size_t slamhip_selective_scan_fwd_workspace_bytes(int B, int T, int C, int N) {
  if (B <= 0 || T <= 0 || C <= 0 || N <= 0 || N > 32 || !scan_fits(B, T, C)) return 0;
  const ScanShape g = scan_shape(B, T, C, N, false);
  if (g.chunks == 1) return 0;
  return ((size_t)B * (g.chunks + 1) * C * N + (size_t)B * g.chunks * C) * sizeof(float);
}

int slamhip_selective_scan_fwd(const void* u, const void* delta, const void* z, const void* Bm, const void* Cm, const long long* strides,
                               const float* A, const float* D, const float* delta_bias, const float* state_in, const int32_t* lengths,
                               int B, int T, int C, int N, int softplus, int dtype, void* y, float* state_out, float* kept_states,
                               void* workspace, size_t workspace_bytes, void* stream) {
  SLAMHIP_SCAN_SIZES("selective_scan_fwd");
  if (B == 0 || (T == 0 && !state_out)) return SLAMHIP_OK;
  SLAMHIP_REQUIRE(A && strides && (T == 0 || (u && delta && Bm && Cm && y)), SLAMHIP_E_ARG, "selective_scan_fwd: null pointer");
  SLAMHIP_REQUIRE(workspace_bytes >= slamhip_selective_scan_fwd_workspace_bytes(B, T, C, N) &&
                      (workspace || slamhip_selective_scan_fwd_workspace_bytes(B, T, C, N) == 0),
                  SLAMHIP_E_ARG, "selective_scan_fwd: workspace too small");
  const ScanShape g = scan_shape(B, T, C, N, false);
  ScanArgs a{};
  a.u = u, a.delta = delta, a.z = z, a.Bm = Bm, a.Cm = Cm, a.A = A, a.D = D, a.bias = delta_bias, a.state_in = state_in;
  a.y = y, a.state_out = state_out, a.kept = kept_states, a.lengths = lengths;
  a.ub = strides[0], a.ut = strides[1], a.deltab = strides[2], a.deltat = strides[3], a.zb = strides[4], a.zt = strides[5];
  a.Bb = strides[6], a.Bt = strides[7], a.Cb = strides[8], a.Ct = strides[9], a.yb = strides[10], a.yt = strides[11];
  a.T = T, a.C = C, a.N = N, a.chunk = g.chunk, a.chunks = g.chunks, a.softplus = softplus;
  if (g.chunks > 1) {
    a.ends = (float*)workspace;
    a.sums = a.ends + (size_t)B * (g.chunks + 1) * C * N;
  }
  return SLAMHIP_SCAN_DISPATCH(scan_fwd, g.P, a, g.groups, B, (hipStream_t)stream);
}

size_t slamhip_selective_scan_bwd_workspace_bytes(int B, int T, int C, int N) {
  if (B <= 0 || T < 0 || C <= 0 || N <= 0 || N > 32 || !scan_fits(B, T, C)) return 0;
  const ScanShape g = scan_shape(B, T, C, N, true);
  const size_t carry = g.chunks > 1 ? (size_t)B * g.chunks * C * (N + 1) : 0;
  return (carry + (size_t)B * g.chunks * C * (N + 2) + (size_t)B * T * g.groups * 8 * g.P) * sizeof(float);
}

int slamhip_selective_scan_bwd(const void* dy, const void* u, const void* delta, const void* z, const void* Bm, const void* Cm,
                               const long long* strides, const float* A, const float* D, const float* delta_bias,
                               const float* kept_states, const float* d_state_out, const int32_t* lengths, int B, int T, int C, int N,
                               int softplus, int dtype, void* du, void* ddelta, void* dz, void* dB, void* dC, float* dA, float* dD,
                               float* d_delta_bias, float* d_state_in, void* workspace, size_t workspace_bytes, void* stream) {
  SLAMHIP_SCAN_SIZES("selective_scan_bwd");
  const bool work = B > 0, data = work && T > 0;
  SLAMHIP_REQUIRE(dA && (!work || (A && strides && workspace)) &&
                      (!data || (dy && u && delta && Bm && Cm && kept_states && du && ddelta && dB && dC)),
                  SLAMHIP_E_ARG, "selective_scan_bwd: null pointer");
  SLAMHIP_REQUIRE(!data || !z == !dz, SLAMHIP_E_ARG, "selective_scan_bwd: z and dz come together");
  SLAMHIP_REQUIRE(workspace_bytes >= slamhip_selective_scan_bwd_workspace_bytes(B, T, C, N), SLAMHIP_E_ARG, "selective_scan_bwd: workspace too small");
  hipStream_t s = (hipStream_t)stream;
  const ScanShape g = scan_shape(B, T, C, N, true);
  const long long columns = (long long)C * (N + 2), bc_groups = work ? ((long long)B * T * 8 * g.P + 255) / 256 : 0;
  const long long all_groups = bc_groups + (columns + 31) / 32;
  SLAMHIP_REQUIRE(all_groups < (1 << 24) && (long long)B * g.chunks < (1 << 30), SLAMHIP_E_SIZE, "selective_scan_bwd: too many steps or parameters");
  ScanArgs a{};
  a.T = T, a.C = C, a.N = N, a.chunk = g.chunk, a.chunks = g.chunks, a.softplus = softplus, a.lengths = lengths;
  a.part = (float*)workspace;
  if (work) {
    a.u = u, a.delta = delta, a.z = z, a.Bm = Bm, a.Cm = Cm, a.dy = dy, a.A = A, a.D = D, a.bias = delta_bias;
    a.d_state_out = d_state_out, a.kept = const_cast<float*>(kept_states);
    a.du = du, a.ddelta = ddelta, a.dz = dz, a.d_state_in = d_state_in;
    a.dyb = strides[0], a.dyt = strides[1], a.ub = strides[2], a.ut = strides[3], a.deltab = strides[4], a.deltat = strides[5];
    a.zb = strides[6], a.zt = strides[7], a.Bb = strides[8], a.Bt = strides[9], a.Cb = strides[10], a.Ct = strides[11];
    a.dub = strides[12], a.dut = strides[13], a.ddeltab = strides[14], a.ddeltat = strides[15], a.dzb = strides[16], a.dzt = strides[17];
    a.part_bc = a.part + (size_t)B * g.chunks * columns;
    a.ends = a.part_bc + (size_t)B * T * g.groups * 8 * g.P;
    a.sums = a.ends + (size_t)B * g.chunks * C * N;
    const int rc = SLAMHIP_SCAN_DISPATCH(scan_bwd, g.P, a, g.groups, B, s);
    if (rc != SLAMHIP_OK) return rc;
  }
  const long long none[4] = {0, 0, 0, 0}, *bc = work ? strides + 18 : none;
  const int parts_of = work ? B : 0;   // nothing to add: the parameters' gradients are zero
  if (dtype == SLAMHIP_BF16)
    hipLaunchKernelGGL((selective_scan_parts_kernel<__bf16>), dim3((unsigned)all_groups), dim3(256), 0, s, a, (int)bc_groups, g.groups,
                       4 * g.P, parts_of, dB, dC, bc[0], bc[1], bc[2], bc[3], dA, dD, d_delta_bias);
  else
    hipLaunchKernelGGL((selective_scan_parts_kernel<float>), dim3((unsigned)all_groups), dim3(256), 0, s, a, (int)bc_groups, g.groups,
                       4 * g.P, parts_of, dB, dC, bc[0], bc[1], bc[2], bc[3], dA, dD, d_delta_bias);
  SLAMHIP_HIP(hipGetLastError());
  return SLAMHIP_OK;
}

}  // extern "C"
