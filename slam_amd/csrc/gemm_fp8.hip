// Matrix product of 8-bit operands (e4m3) with a float32 scale for each 128 values of an activation row and for each 128 x 128
// block of the weights:
//
//   out[m,n] = sum_kb sa[m,kb] sb[n/128,kb] sum_{k in block kb} a[m,k] b[n,k]
//
// One v_mfma_f32_16x16x128_f8f6f4 is the inner sum of a 16 x 16 tile: it starts from zero, and its result is added to the tile's
// float32 accumulator with one multiply-add an element, the product of the two scales.  The weights are the matrix instruction's
// first operand: a lane then holds one activation row (one scale) and four consecutive columns of the output (one store).
// The matrix unit sums eight consecutive products after cutting each to 2^-13 of the largest one's power of two, and such sums in
// float32 (seen with single products beside each other): below bfloat16's half step of 2^-9 unless terms cancel, which is why
// bfloat16 is the only output.
// The order of k inside a block is the same for both operands and otherwise free: a lane takes 16-byte chunks g and g + 4 of a
// block's eight.
#include <hip/hip_runtime.h>

#include "common.h"
#include "sequence_device.h"

namespace slamhip {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

struct GemmArgs {
  const uint8_t *a, *b;
  const float *sa, *sb;
  __bf16* out;
  int M, N, K, KB;
};

__device__ __forceinline__ f32x4 mfma_fp8(i32x8 x, i32x8 y) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, f32x4{}, 0, 0, 0, 0, 0, 0);
}

__device__ __forceinline__ i32x8 join(i32x4 lo, i32x4 hi) {
  return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef bf16x4 bf16x4_b __attribute__((aligned(2)));

// four columns n .. n + 3 of row m
__device__ __forceinline__ void store_out(const GemmArgs& p, int m, int n, f32x4 v) {
  if (m >= p.M || n >= p.N) return;
  __bf16* o = p.out + (long long)m * p.N + n;
  if (n + 4 <= p.N) {
    *reinterpret_cast<bf16x4_b*>(o) = __builtin_convertvector(v, bf16x4);
  } else {
    for (int i = 0; i < p.N - n; ++i) o[i] = (__bf16)v[i];
  }
}

typedef __attribute__((address_space(3))) void* lds_ptr;

constexpr unsigned kBeyond = 0xffff0000u;   // an offset past every operand: both are smaller

// BM x BN outputs a workgroup, WM x WN waves; both operands' 128-deep slices go from memory straight into shared memory (two
// buffers).  A slice's row is eight 16-byte chunks, chunk c of row r at place c ^ (r & 7): the rows that a fragment read touches
// at once lie in different banks.  Chunks beyond the matrix are given an address beyond the buffer: they arrive as zeros.
template <int BM, int BN, int WM, int WN>
__global__ void __launch_bounds__(64 * WM * WN) gemm_fp8_kernel(GemmArgs p) {
  constexpr int kWaves = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16;
  constexpr int kSlice = (BM + BN) * 128;
  __shared__ __align__(1024) uint8_t sh[2 * kSlice];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int tiles_n = (p.N + BN - 1) / BN;
  const int m0 = blockIdx.x / tiles_n * BM, n0 = blockIdx.x % tiles_n * BN;
  const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
  const auto ra = __builtin_amdgcn_make_buffer_rsrc((void*)p.a, 0, (unsigned)((size_t)p.M * p.K), 0x00020000);
  const auto rb = __builtin_amdgcn_make_buffer_rsrc((void*)p.b, 0, (unsigned)((size_t)p.N * p.K), 0x00020000);

  // a wave's load moves 8 rows of a slice: lane l brings chunk (l & 7) ^ (row & 7) of row l >> 3
  const int lrow = lane >> 3, lchunk = (lane & 7) ^ (lrow & 7);
  auto load = [&](int kb, int buf) {
    const int k = kb * 128 + lchunk * 16;
#pragma unroll
    for (int i = 0; i < BM / 8 / kWaves; ++i) {
      const int r = (i * kWaves + wave) * 8;
      const unsigned off = k < p.K && m0 + r + lrow < p.M ? (unsigned)(m0 + r + lrow) * (unsigned)p.K + k : kBeyond;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_ptr)(sh + buf * kSlice + r * 128), 16, off, 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < BN / 8 / kWaves; ++i) {
      const int r = (i * kWaves + wave) * 8;
      const unsigned off = k < p.K && n0 + r + lrow < p.N ? (unsigned)(n0 + r + lrow) * (unsigned)p.K + k : kBeyond;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lds_ptr)(sh + buf * kSlice + (BM + r) * 128), 16, off, 0, 0, 0);
    }
  };
  const int frow = lane & 15, g = lane >> 4;
  const int c0 = (g ^ (frow & 7)) * 16, c1 = ((g + 4) ^ (frow & 7)) * 16;
  auto fragment = [&](const uint8_t* rows) {
    const i32x4 lo = *reinterpret_cast<const i32x4*>(rows + frow * 128 + c0);
    const i32x4 hi = *reinterpret_cast<const i32x4*>(rows + frow * 128 + c1);
    return join(lo, hi);
  };
  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{};
  load(0, 0);
  for (int kb = 0; kb < p.KB; ++kb) {
    float sa[TM], sb[TN];
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int m = min(m0 + wm + i * 16 + frow, p.M - 1);
      sa[i] = p.sa[(long long)m * p.KB + kb];
    }
#pragma unroll
    for (int j = 0; j < TN; ++j) sb[j] = p.sb[(long long)(min(n0 + wn + j * 16, p.N - 1) / 128) * p.KB + kb];
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();   // slice kb has arrived for all waves; the other buffer has been read
    if (kb + 1 < p.KB) load(kb + 1, (kb + 1) & 1);
    const uint8_t* base = sh + (kb & 1) * kSlice;
    i32x8 fb[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) fb[j] = fragment(base + (BM + wn + j * 16) * 128);
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const i32x8 fa = fragment(base + (wm + i * 16) * 128);
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const f32x4 d = mfma_fp8(fb[j], fa);
        const float s = sa[i] * sb[j];
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][j][r] = fmaf(d[r], s, acc[i][j][r]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) store_out(p, m0 + wm + i * 16 + frow, n0 + wn + j * 16 + g * 4, acc[i][j]);
}

// Few rows: the weights are read once, straight into registers; a workgroup's waves take every kWaves-th block of k for the same
// 16 columns and meet in shared memory.
template <int TM>
__global__ void __launch_bounds__(256) gemm_fp8_rows_kernel(GemmArgs p) {
  constexpr int kWaves = 4;
  __shared__ f32x4 sh[kWaves][TM][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int n0 = blockIdx.x * 16, row = lane & 15, g = lane >> 4;
  const uint8_t* b = p.b + (long long)min(n0 + row, p.N - 1) * p.K;
  f32x4 acc[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) acc[i] = f32x4{};
  for (int kb = wave; kb < p.KB; kb += kWaves) {
    const int k0 = kb * 128 + g * 16, k1 = k0 + 64;
    i32x4 z{};
    const i32x8 fb = join(k0 < p.K ? *reinterpret_cast<const i32x4*>(b + k0) : z, k1 < p.K ? *reinterpret_cast<const i32x4*>(b + k1) : z);
    const float sb = p.sb[(long long)(n0 / 128) * p.KB + kb];
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const int m = min(i * 16 + row, p.M - 1);   // rows beyond the last repeat it and are not stored
      const uint8_t* a = p.a + (long long)m * p.K;
      const i32x8 fa = join(k0 < p.K ? *reinterpret_cast<const i32x4*>(a + k0) : z, k1 < p.K ? *reinterpret_cast<const i32x4*>(a + k1) : z);
      const float s = p.sa[(long long)m * p.KB + kb] * sb;
      const f32x4 d = mfma_fp8(fb, fa);
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[i][r] = fmaf(d[r], s, acc[i][r]);
    }
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) sh[wave][i][lane] = acc[i];
  __syncthreads();
  for (int i = wave; i < TM; i += kWaves) {
    f32x4 v = sh[0][i][lane];
    for (int w = 1; w < kWaves; ++w) v += sh[w][i][lane];
    store_out(p, i * 16 + row, n0 + g * 4, v);
  }
}

int gemm(const GemmArgs& p, hipStream_t s) {
  if (p.M <= 64) {
    const dim3 grid((p.N + 15) / 16);
    if (p.M <= 16)
      hipLaunchKernelGGL((gemm_fp8_rows_kernel<1>), grid, dim3(256), 0, s, p);
    else if (p.M <= 32)
      hipLaunchKernelGGL((gemm_fp8_rows_kernel<2>), grid, dim3(256), 0, s, p);
    else
      hipLaunchKernelGGL((gemm_fp8_rows_kernel<4>), grid, dim3(256), 0, s, p);
  } else {
    const long long tiles = (long long)((p.M + 127) / 128) * ((p.N + 127) / 128);
    SLAMHIP_REQUIRE(tiles < (1 << 23), SLAMHIP_E_SIZE, "gemm_nt_fp8: too many tiles");
    hipLaunchKernelGGL((gemm_fp8_kernel<128, 128, 2, 2>), dim3((unsigned)tiles), dim3(256), 0, s, p);
  }
  SLAMHIP_HIP(hipGetLastError());
  return SLAMHIP_OK;
}

}  // namespace
}  // namespace slamhip

using namespace slamhip;

extern "C" {

int slamhip_gemm_nt_fp8(const void* a, const float* a_scales, const void* b, const float* b_scales, int M, int N, int K, void* out,
                        void* stream) {
  SLAMHIP_REQUIRE(M >= 0 && N >= 0 && K > 0, SLAMHIP_E_ARG, "gemm_nt_fp8: need M, N >= 0 and K >= 1");
  SLAMHIP_REQUIRE(K % 16 == 0, SLAMHIP_E_SIZE, "gemm_nt_fp8: K must be a multiple of 16");
  SLAMHIP_REQUIRE((long long)M * K < 0xffff0000LL && (long long)N * K < 0xffff0000LL, SLAMHIP_E_SIZE, "gemm_nt_fp8: an operand is larger than 4 GB");
  if (M == 0 || N == 0) return SLAMHIP_OK;
  SLAMHIP_REQUIRE(a && a_scales && b && b_scales && out, SLAMHIP_E_ARG, "gemm_nt_fp8: null pointer");
  SLAMHIP_REQUIRE(((uintptr_t)a & 15) == 0 && ((uintptr_t)b & 15) == 0, SLAMHIP_E_ARG, "gemm_nt_fp8: operands must be 16-byte aligned");
  const GemmArgs p{(const uint8_t*)a, (const uint8_t*)b, a_scales, b_scales, (__bf16*)out, M, N, K, (K + 127) / 128};
  return gemm(p, (hipStream_t)stream);
}

}  // extern "C"
