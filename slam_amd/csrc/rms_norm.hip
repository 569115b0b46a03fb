// Root-mean-square norm of rows with the residual's addition, its backward pass, and the 8-bit rows that feed the 8-bit product.
//
//   s = round(x + residual),  rstd = (mean(s^2) + eps)^(-1/2),  y = s rstd w
//   8 bits: for each 128 consecutive values of a row, scale = max(max|y| / 448, 2^-100), y8 = e4m3(y / scale)
//   backward: hat = s rstd, dx = rstd (w dy - hat mean(w dy hat)) + d_sum, dw = sum over rows of dy hat
//
// A row is read once and stays in registers until its statistics are known.  Bytes bound all of it: 16384 x 4096 bfloat16 with the
// residual takes 87-94 us forward (5.7-6.2 TB/s, partly from the cache), with an 8-bit output 85 us, and 105-110 us back with the sum's gradient
// (4.9-5.1 TB/s); float32 188 and 205 us (5.7 and 5.2 TB/s); 4 rows 5 us, a launch and the way to memory and back.
//
// Statistics and the quantised values are float32; s is rounded to the rows' type before its statistics are taken, because the
// backward pass and the next layer read the rounded s.
#include <hip/hip_runtime.h>

#include "common.h"
#include "sequence_device.h"

namespace slamhip {
namespace {

constexpr float kFp8Max = 448.0f;
constexpr float kMinScale = 7.888609052210118e-31f;   // 2^-100: the scale of a block of zeros
constexpr int kMaxNormC = 16384;
constexpr long long kMaxGroups = (1LL << 24) - 1;   // a launch has fewer than 2^32 threads

// Values c .. c + 7 of a row of C, zeros behind its end.  The last octet is loaded as the eight values that end with the row, which
// octet() moves down once all loads are under way: element by element its lanes would wait eight times (16384 x 1500 forward 60 us,
// so 36 us).
template <typename T>
__device__ __forceinline__ packed<T, 8> octet_raw(const T* row, int c, int C) {
  if (C < 8) return load_raw<8>(row + c, C - c);
  return load_raw<8>(row + min(c, C - 8), c < C ? 8 : 0);
}

template <typename T>
__device__ __forceinline__ f32x8 octet(packed<T, 8> raw, int c, int C) {
  f32x8 v = to_floats<T, 8>(raw);
  if (c + 8 > C && C >= 8) {
    const int by = (8 - C % 8) & 7;   // the same for all rows
#pragma unroll
    for (int m = 4; m; m >>= 1)
      if (by & m)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = i + m < 8 ? v[i + m] : 0.0f;
  }
  return v;
}

template <typename T>
__device__ __forceinline__ f32x8 load_octet(const T* row, int c, int C) { return octet<T>(octet_raw(row, c, C), c, C); }

template <int LANES>
__device__ __forceinline__ float row_sum(float v, float* sh) {
#pragma unroll
  for (int m = (LANES < 64 ? LANES : 64) / 2; m; m >>= 1) v += __shfl_xor(v, m);
  if (LANES > 64) {
    __syncthreads();   // the previous sum has been read
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.0f;
#pragma unroll
    for (int i = 0; i < LANES / 64; ++i) v += sh[i];
  }
  return v;
}

// Eight values of a 128-value block whose 16 octets lie in 16 consecutive lanes: the block's scale and the octet in e4m3.
// The maximum is taken over the bit patterns of |v|, so that a NaN is the maximum.
__device__ __forceinline__ float block_scale(f32x8 v) {
  unsigned m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
#pragma unroll
  for (int k = 8; k; k >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, k));
  const float s = __uint_as_float(m) / kFp8Max;
  return s < kMinScale ? kMinScale : s;
}

__device__ __forceinline__ float clamp_fp8(float v) {   // NaN stays NaN
  return v > kFp8Max ? kFp8Max : (v < -kFp8Max ? -kFp8Max : v);
}

// The quotients are correctly rounded (an error in the last bit would move values halfway between two of the format): the reciprocal
// is, a first correction by the exact remainder brings v r to within one unit, and a second one rounds correctly (Markstein 1990).
// 16384 x 8192 bfloat16 takes 84-92 us, 4.4-4.8 TB/s; with IEEE divisions 103 us; float32 112 us, 6.0 TB/s.  An exact zero loses its sign.
// A remainder may lose bits below 2^-149 where a scale is near its least; that is 2^-17 of the quotient's last place at most.
struct Quotient {
  float scale, r;
  __device__ __forceinline__ explicit Quotient(float s) : scale(s), r(1.0f / s) {
    if (r == 0.0f) scale = 0.0f;   // of an infinite block: finite values become 0, infinite ones NaN
  }
  __device__ __forceinline__ float operator()(float v) const {
    float q = v * r;
    q = fmaf(fmaf(-q, scale, v), r, q);
    q = fmaf(fmaf(-q, scale, v), r, q);
    return clamp_fp8(q);
  }
};

__device__ __forceinline__ uint2 to_fp8(f32x8 v, float scale) {
  const Quotient of(scale);
  uint2 q;
  int w = 0;
  w = __builtin_amdgcn_cvt_pk_fp8_f32(of(v[0]), of(v[1]), w, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(of(v[2]), of(v[3]), w, true);
  q.x = (unsigned)w;
  w = __builtin_amdgcn_cvt_pk_fp8_f32(of(v[4]), of(v[5]), w, false);
  w = __builtin_amdgcn_cvt_pk_fp8_f32(of(v[6]), of(v[7]), w, true);
  q.y = (unsigned)w;
  return q;
}

typedef unsigned u32x2_b __attribute__((ext_vector_type(2), aligned(1)));

__device__ __forceinline__ void store_fp8(uint8_t* p, uint2 q, int valid) {
  if (valid >= 8) {
    u32x2_b raw = {q.x, q.y};
    *reinterpret_cast<u32x2_b*>(p) = raw;
  } else {
    for (int i = 0; i < valid; ++i) p[i] = (uint8_t)((i < 4 ? q.x >> (8 * i) : q.y >> (8 * (i - 4))) & 0xffu);
  }
}

// LANES threads hold one row: octet i of thread t is octet i * LANES + t of the row.  sum_out and y may be x or residual: a thread stores
// an octet when it has loaded it, and what another thread loads beside its own (the last octet of a row) it drops.
template <typename T, int LANES, int ITER>
__global__ void __launch_bounds__(256)
rms_norm_fwd_kernel(const T* x, const T* residual, const float* __restrict__ w, float eps, long long rows,
                    int C, T* sum_out, T* y, uint8_t* __restrict__ y8, float* __restrict__ scales,
                    float* __restrict__ rstd_out) {
  __shared__ float sh[4];
  const int lane = threadIdx.x % LANES;
  const long long row = (long long)blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  if (row >= rows) return;   // LANES == 256: no row is left over; below: the row's lanes leave together, no barrier
  const long long base = row * C;
  packed<T, 8> raw_x[ITER], raw_r[ITER];
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    const int c = (i * LANES + lane) * 8;
    raw_x[i] = octet_raw(x + base, c, C);
    if (residual) raw_r[i] = octet_raw(residual + base, c, C);
  }
  f32x8 v[ITER];
  float ss = 0.0f;
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    const int c = (i * LANES + lane) * 8, n = C - c;
    v[i] = octet<T>(raw_x[i], c, C);
    if (residual) {
      v[i] += octet<T>(raw_r[i], c, C);
#pragma unroll
      for (int j = 0; j < 8; ++j) v[i][j] = (float)(T)v[i][j];
      if (sum_out && n > 0) store8(sum_out + base + c, v[i], n);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) ss = fmaf(v[i][j], v[i][j], ss);
  }
  ss = row_sum<LANES>(ss, sh);
  const float rstd = 1.0f / sqrtf(ss / (float)C + eps);
  if (rstd_out && lane == 0) rstd_out[row] = rstd;
  const int nblocks = (C + 127) / 128;
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    const int c = (i * LANES + lane) * 8, n = C - c;
    f32x8 o{};
    if (n > 0) {
      const f32x8 wv = load_octet(w, c, C);
#pragma unroll
      for (int j = 0; j < 8; ++j) o[j] = v[i][j] * rstd * wv[j];
      if (y) store8(y + base + c, o, n);
    }
    if (y8) {   // all lanes of a wave take part in the block's maximum
      const float scale = block_scale(o);
      if (n > 0) {
        store_fp8(y8 + base + c, to_fp8(o, scale), n);
        if ((lane & 15) == 0) scales[row * nblocks + c / 128] = scale;
      }
    }
  }
}

// A slot is LANES threads; slot k takes rows k, k + slots, ...; a workgroup's slots add up their parts of dw, part[workgroup][C].
// dx may be dy or d_sum, whose octets are loaded before dx's is stored.
template <typename T, int LANES, int ITER>
__global__ void __launch_bounds__(256)
rms_norm_bwd_kernel(const T* dy, const T* __restrict__ s, const float* __restrict__ w, const float* __restrict__ rstd,
                    const T* d_sum, long long rows, int C, T* dx, float* __restrict__ part) {
  __shared__ float sh[4];
  const int lane = threadIdx.x % LANES, slots = gridDim.x * (256 / LANES);
  const int slot = blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  f32x8 dw[ITER], wv[ITER];
#pragma unroll
  for (int i = 0; i < ITER; ++i) {
    const int c = (i * LANES + lane) * 8;
    dw[i] = f32x8{};
    wv[i] = load_octet(w, c, C);
  }
  for (long long row = slot; row < rows; row += slots) {
    const long long base = row * C;
    const float r = rstd[row];
    packed<T, 8> raw_g[ITER], raw_h[ITER], raw_d[ITER];
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      const int c = (i * LANES + lane) * 8;
      raw_g[i] = octet_raw(dy + base, c, C);
      raw_h[i] = octet_raw(s + base, c, C);
      if (d_sum) raw_d[i] = octet_raw(d_sum + base, c, C);
    }
    f32x8 g[ITER], h[ITER];
    float dot = 0.0f;
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      const int c = (i * LANES + lane) * 8;
      g[i] = octet<T>(raw_g[i], c, C);
      h[i] = octet<T>(raw_h[i], c, C) * r;
    }
#pragma unroll
    for (int i = 0; i < ITER; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        dw[i][j] = fmaf(g[i][j], h[i][j], dw[i][j]);
        g[i][j] *= wv[i][j];
        dot = fmaf(g[i][j], h[i][j], dot);
      }
    dot = row_sum<LANES>(dot, sh) / (float)C;
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      const int c = (i * LANES + lane) * 8, n = C - c;
      if (n > 0) {
        f32x8 o;
#pragma unroll
        for (int j = 0; j < 8; ++j) o[j] = r * (g[i][j] - h[i][j] * dot);
        if (d_sum) o += octet<T>(raw_d[i], c, C);
        store8(dx + base + c, o, n);
      }
    }
  }
  if constexpr (LANES == 256) {
#pragma unroll
    for (int i = 0; i < ITER; ++i) {
      const int c = (i * LANES + lane) * 8;
      if (c < C) store8(part + (long long)blockIdx.x * C + c, dw[i], C - c);
    }
  } else {
    constexpr int kRow = LANES * 8 * ITER;
    __shared__ float sums[256 / LANES][kRow];
#pragma unroll
    for (int i = 0; i < ITER; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) sums[threadIdx.x / LANES][(i * LANES + lane) * 8 + j] = dw[i][j];
    __syncthreads();
    for (int c = threadIdx.x; c < C; c += 256) {
      float v = 0.0f;
#pragma unroll
      for (int k = 0; k < 256 / LANES; ++k) v += sums[k][c];
      part[(long long)blockIdx.x * C + c] = v;
    }
  }
}

struct WeightGradient {
  float* dw;
  __device__ void operator()(int c, float v) const { dw[c] = v; }
};

// one octet a thread; 16 consecutive threads share a 128-value block of a row
template <typename T>
__global__ void __launch_bounds__(256)
quantize_fp8_kernel(const T* __restrict__ x, long long rows, int C, uint8_t* __restrict__ q, float* __restrict__ scales) {
  const int nblocks = C / 128 + (C % 128 != 0);
  const long long blk = (long long)blockIdx.x * 16 + threadIdx.x / 16;
  const bool live = blk < rows * nblocks;
  const long long row = live ? blk / nblocks : 0;
  const int b = live ? (int)(blk - row * nblocks) : 0;
  const int c = b * 128 + (threadIdx.x & 15) * 8, n = C - c;
  f32x8 v{};
  if (live) v = load_octet(x + row * C, c, C);
  const float scale = block_scale(v);
  if (live && n > 0) {
    store_fp8(q + row * C + c, to_fp8(v, scale), n);
    if ((threadIdx.x & 15) == 0) scales[blk] = scale;
  }
}

// one 128 x 128 block a workgroup: thread t holds octet t % 16 of rows t / 16 + 16 i.  16384 x 8192 bfloat16 takes 78 us, float32 118 us: bytes,
// 5.2 and 5.7 TB/s.
template <typename T>
__global__ void __launch_bounds__(256)
quantize_fp8_blocks_kernel(const T* __restrict__ x, int R, int C, uint8_t* __restrict__ q, float* __restrict__ scales) {
  __shared__ unsigned sh[4];
  const int c = blockIdx.x * 128 + (threadIdx.x & 15) * 8, n = C - c;
  const int r0 = blockIdx.y * 128 + threadIdx.x / 16;
  packed<T, 8> raw[8];
  f32x8 v[8];
  unsigned m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + 16 * i;
    raw[i] = octet_raw(x + (long long)min(r, R - 1) * C, r < R ? c : C, C);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    v[i] = octet<T>(raw[i], c, C);
#pragma unroll
    for (int j = 0; j < 8; ++j) m = max(m, __float_as_uint(v[i][j]) & 0x7fffffffu);
  }
#pragma unroll
  for (int k = 32; k; k >>= 1) m = max(m, (unsigned)__shfl_xor((int)m, k));
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = m;
  __syncthreads();
  m = max(max(sh[0], sh[1]), max(sh[2], sh[3]));
  const float s = __uint_as_float(m) / kFp8Max;
  const float scale = s < kMinScale ? kMinScale : s;
  if (threadIdx.x == 0) scales[(long long)blockIdx.y * gridDim.x + blockIdx.x] = scale;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const int r = r0 + 16 * i;
    if (r < R && n > 0) store_fp8(q + (long long)r * C + c, to_fp8(v[i], scale), n);
  }
}

// Lanes that hold a row.  us forward and back: 65536 x 128 28 with 16 lanes, 99 with 64, 143 with 256; 16384 x 512 29 with 64, 47 with 256;
// 16384 x 1024 54 with 64 (two octets each), 67 with 256; 16384 x 2048 131 with 64, 96 with 256.
int norm_lanes(int C) { return C <= 128 ? 16 : C <= 256 ? 32 : C <= 1024 ? 64 : 256; }

// Workgroups of the backward pass, a part of dw each: as many as are on the chip at once, whose registers hold dw.  us forward and back
// with 256 / 512 / 768 / 1024 of them: 16384 x 4096 218/202/205/212, 2000 x 8192 61/56/60/65, 2000 x 16384 123/132/139/149; one octet a
// thread leaves room for more: 16384 x 1504 -/93/-/76.
int norm_most_parts(int C) { return C > 8192 ? 256 : C > 1024 && C <= 2048 ? 1024 : 512; }

// Up to two rows a workgroup takes them all and its part is dw: with a second launch 2 x 4096 takes about as long (8.4, 9.2 us), 4 x 4096
// less (9.1, not 13).
int norm_parts(long long rows, int C) {
  const int per = 256 / norm_lanes(C);
  const long long all = (rows + per - 1) / per;
  return rows <= 0 ? 0 : rows <= 2 ? 1 : (int)(all < norm_most_parts(C) ? all : norm_most_parts(C));
}

template <typename T, int LANES, int ITER>
int norm_fwd(const void* x, const void* residual, const float* w, float eps, long long rows, int C, void* sum_out, void* y, void* y8,
             float* scales, float* rstd, hipStream_t s) {
  const long long per = 256 / LANES, grid = (rows + per - 1) / per;
  hipLaunchKernelGGL((rms_norm_fwd_kernel<T, LANES, ITER>), dim3((unsigned)grid), dim3(256), 0, s, (const T*)x, (const T*)residual, w,
                     eps, rows, C, (T*)sum_out, (T*)y, (uint8_t*)y8, scales, rstd);
  SLAMHIP_HIP(hipGetLastError());
  return SLAMHIP_OK;
}

template <typename T, int LANES, int ITER>
int norm_bwd(const void* dy, const void* sum, const float* w, const float* rstd, const void* d_sum, long long rows, int C, void* dx,
             float* dw, float* part, hipStream_t s) {
  const int parts = norm_parts(rows, C);
  if (parts == 1) part = dw;
  if (parts > 0)
    hipLaunchKernelGGL((rms_norm_bwd_kernel<T, LANES, ITER>), dim3(parts), dim3(256), 0, s, (const T*)dy, (const T*)sum, w, rstd,
                       (const T*)d_sum, rows, C, (T*)dx, part);
  SLAMHIP_HIP(hipGetLastError());
  if (parts != 1) SLAMHIP_HIP(column_sums(part, parts, C, WeightGradient{dw}, s));
  return SLAMHIP_OK;
}

}  // namespace
}  // namespace slamhip

using namespace slamhip;

#define SLAMHIP_NORM_LANES(FN, T, ...)                               \
  do {                                                               \
    switch (norm_lanes(C)) {                                         \
      case 16: return FN<T, 16, 1>(__VA_ARGS__);                     \
      case 32: return FN<T, 32, 1>(__VA_ARGS__);                     \
    }                                                                \
    if (C <= 512) return FN<T, 64, 1>(__VA_ARGS__);                  \
    if (C <= 1024) return FN<T, 64, 2>(__VA_ARGS__);                 \
    if (C <= 2048) return FN<T, 256, 1>(__VA_ARGS__);                \
    if (C <= 4096) return FN<T, 256, 2>(__VA_ARGS__);                \
    if (C <= 8192) return FN<T, 256, 4>(__VA_ARGS__);                \
    return FN<T, 256, 8>(__VA_ARGS__);                               \
  } while (0)

#define SLAMHIP_NORM_DISPATCH(FN, ...)                               \
  do {                                                               \
    if (dtype == SLAMHIP_BF16) SLAMHIP_NORM_LANES(FN, __bf16, __VA_ARGS__); \
    SLAMHIP_NORM_LANES(FN, float, __VA_ARGS__);                      \
  } while (0)

extern "C" {

int slamhip_rms_norm_fwd(const void* x, const void* residual, const float* weight, float eps, long long rows, int C, int dtype,
                         void* sum_out, void* y, void* y8, float* scales, float* rstd, void* stream) {
  SLAMHIP_REQUIRE(rows >= 0 && C > 0 && (dtype == SLAMHIP_F32 || dtype == SLAMHIP_BF16), SLAMHIP_E_ARG,
                  "rms_norm_fwd: need rows >= 0, C >= 1 and a known type");
  SLAMHIP_REQUIRE(C <= kMaxNormC && rows <= kMaxGroups, SLAMHIP_E_SIZE, "rms_norm_fwd: at most %d columns and 2^24 - 1 rows", kMaxNormC);
  if (rows == 0) return SLAMHIP_OK;
  SLAMHIP_REQUIRE(x && weight && (y || y8 || sum_out), SLAMHIP_E_ARG, "rms_norm_fwd: null pointer");
  SLAMHIP_REQUIRE(!y8 == !scales, SLAMHIP_E_ARG, "rms_norm_fwd: the 8-bit output and its scales come together");
  SLAMHIP_REQUIRE(residual || !sum_out, SLAMHIP_E_ARG, "rms_norm_fwd: sum_out without a residual");
  hipStream_t s = (hipStream_t)stream;
  SLAMHIP_NORM_DISPATCH(norm_fwd, x, residual, weight, eps, rows, C, sum_out, y, y8, scales, rstd, s);
}

size_t slamhip_rms_norm_bwd_workspace_bytes(long long rows, int C) {
  if (rows <= 0 || C <= 0 || C > kMaxNormC || rows > kMaxGroups) return 0;   // beyond the limits the call is refused
  const int parts = norm_parts(rows, C);
  return parts == 1 ? 0 : (size_t)parts * (size_t)C * sizeof(float);
}

int slamhip_rms_norm_bwd(const void* dy, const void* sum, const float* weight, const float* rstd, const void* d_sum, long long rows,
                         int C, int dtype, void* dx, float* dweight, void* workspace, size_t workspace_bytes, void* stream) {
  SLAMHIP_REQUIRE(rows >= 0 && C > 0 && (dtype == SLAMHIP_F32 || dtype == SLAMHIP_BF16), SLAMHIP_E_ARG,
                  "rms_norm_bwd: need rows >= 0, C >= 1 and a known type");
  SLAMHIP_REQUIRE(C <= kMaxNormC && rows <= kMaxGroups, SLAMHIP_E_SIZE, "rms_norm_bwd: at most %d columns and 2^24 - 1 rows", kMaxNormC);
  SLAMHIP_REQUIRE(dweight && (rows == 0 || (dy && sum && weight && rstd && dx)), SLAMHIP_E_ARG, "rms_norm_bwd: null pointer");
  const size_t need = slamhip_rms_norm_bwd_workspace_bytes(rows, C);
  SLAMHIP_REQUIRE(workspace_bytes >= need && (workspace || need == 0), SLAMHIP_E_ARG, "rms_norm_bwd: workspace too small");
  hipStream_t s = (hipStream_t)stream;
  SLAMHIP_NORM_DISPATCH(norm_bwd, dy, sum, weight, rstd, d_sum, rows, C, dx, dweight, (float*)workspace, s);
}

int slamhip_quantize_fp8(const void* x, long long rows, int C, int dtype, void* q, float* scales, void* stream) {
  SLAMHIP_REQUIRE(rows >= 0 && C > 0 && (dtype == SLAMHIP_F32 || dtype == SLAMHIP_BF16), SLAMHIP_E_ARG,
                  "quantize_fp8: need rows >= 0, C >= 1 and a known type");
  if (rows == 0) return SLAMHIP_OK;
  SLAMHIP_REQUIRE(x && q && scales, SLAMHIP_E_ARG, "quantize_fp8: null pointer");
  const int nblocks = C / 128 + (C % 128 != 0);
  SLAMHIP_REQUIRE(rows <= kMaxGroups * 16 / nblocks, SLAMHIP_E_SIZE, "quantize_fp8: more than 2^28 - 16 blocks of 128 values");
  const long long groups = (rows * nblocks + 15) / 16;
  hipStream_t s = (hipStream_t)stream;
  if (dtype == SLAMHIP_BF16)
    hipLaunchKernelGGL((quantize_fp8_kernel<__bf16>), dim3((unsigned)groups), dim3(256), 0, s, (const __bf16*)x, rows, C, (uint8_t*)q, scales);
  else
    hipLaunchKernelGGL((quantize_fp8_kernel<float>), dim3((unsigned)groups), dim3(256), 0, s, (const float*)x, rows, C, (uint8_t*)q, scales);
  SLAMHIP_HIP(hipGetLastError());
  return SLAMHIP_OK;
}

int slamhip_quantize_fp8_blocks(const void* x, int R, int C, int dtype, void* q, float* scales, void* stream) {
  SLAMHIP_REQUIRE(R >= 0 && C > 0 && (dtype == SLAMHIP_F32 || dtype == SLAMHIP_BF16), SLAMHIP_E_ARG,
                  "quantize_fp8_blocks: need R >= 0, C >= 1 and a known type");
  if (R == 0) return SLAMHIP_OK;
  SLAMHIP_REQUIRE(x && q && scales, SLAMHIP_E_ARG, "quantize_fp8_blocks: null pointer");
  SLAMHIP_REQUIRE(R <= 65535 * 128 && C <= kMaxGroups, SLAMHIP_E_SIZE, "quantize_fp8_blocks: at most 65535 * 128 rows and 2^24 - 1 columns");
  const dim3 grid((C + 127) / 128, (R + 127) / 128);
  hipStream_t s = (hipStream_t)stream;
  if (dtype == SLAMHIP_BF16)
    hipLaunchKernelGGL((quantize_fp8_blocks_kernel<__bf16>), grid, dim3(256), 0, s, (const __bf16*)x, R, C, (uint8_t*)q, scales);
  else
    hipLaunchKernelGGL((quantize_fp8_blocks_kernel<float>), grid, dim3(256), 0, s, (const float*)x, R, C, (uint8_t*)q, scales);
  SLAMHIP_HIP(hipGetLastError());
  return SLAMHIP_OK;
}

}  // extern "C"
