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
// What bounds it: with up to 16 rows the weights' bytes.  With tiles no unit is at its limit, by the counters: at 8192 x 8192 x 4096 (270-280 us,
// 2.0 PFLOP/s; a product of the same operands without scales in the vendor's library reaches 2.47) the matrix units are busy 45 % of the
// cycles, at a clock of about 2 GHz, and a wave is at a wait or barrier for 33 % of its time and waits for its turn for 33 %.  At 777 x 2056 x 4096 (16 us)
// the matrix units of the CUs that have work are busy 25 %, the L2 hands each of them 27 bytes a cycle (hits 80 %), and a wave is at a wait or
// barrier for 35 % of its time and waits for its turn for 28 %: what is left is how long a slice takes, with two waves a SIMD and one
// workgroup a CU to cover it.  There neither twice as many slices under way (through registers, 18 us), nor fewer reads of shared memory
// (64 x 64 a wave, 22 us), nor the weights straight in registers (23 us) came out faster.
// The order of k inside a block is the same for both operands and otherwise free: a lane takes 16-byte chunks g and g + 4 of a
// block's eight.
#include <hip/hip_runtime.h>

#include "common.h"
#include "gemm_fp8_plan.h"
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
  int per;       // blocks of k a workgroup, a multiple of 4; workgroups (.., y) begin at block y * per
  float* part;   // with more than one such part: their sums, float32 [parts][M][N]
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
  if (p.part) {
    storev<4>(p.part + ((long long)blockIdx.y * p.M + m) * p.N + n, v, p.N - n);
    return;
  }
  __bf16* o = p.out + (long long)m * p.N + n;
  if (n + 4 <= p.N) {
    *reinterpret_cast<bf16x4_b*>(o) = __builtin_convertvector(v, bf16x4);
  } else {
    for (int i = 0; i < p.N - n; ++i) o[i] = (__bf16)v[i];
  }
}

typedef __attribute__((address_space(3))) void* lds_ptr;

typedef const float __attribute__((address_space(4))) ConstFloat;

// until at most N of the wave's loads are under way, and none of its reads of shared memory
template <int N>
__device__ __forceinline__ void wait_loads() {
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory");
}

// floats that a wave reads alike and no kernel writes meanwhile: scalar loads
__device__ __forceinline__ ConstFloat* uniform_floats(const float* p) { return (ConstFloat*)p; }

// BM x BN outputs a workgroup, KW groups of WM x WN waves that take every KW-th block of k and meet in shared memory at the end;
// both operands' 128-deep slices and the rows' scales go from memory straight into shared memory (NS buffers of KW slices).  A
// slice's row is eight 16-byte chunks, chunk c of row r at place c ^ (r & 7): the rows that a fragment read touches at once lie in
// different banks.  Chunks beyond the matrix are given an address beyond the buffer: they arrive as zeros (1.6 % of 8192 x 8192 x 4096 is what
// it costs that this holds for the vector offset by itself).  Per block of k a wave does TM x TN matrix instructions; the multiply-adds of one row of tiles are issued
// behind the matrix instructions of the next, so that neither waits for the other.
template <int BM, int BN, int WM, int WN, int NS, int KW>
__global__ void __launch_bounds__(64 * WM * WN * KW, 2) gemm_fp8_kernel(GemmArgs p) {
  constexpr int kWaves = WM * WN, TM = BM / WM / 16, TN = BN / WN / 16, kLoadA = BM / 8 / kWaves, kLoadB = BN / 8 / kWaves, kLoads = kLoadA + kLoadB;
  constexpr int kSlice = (BM + BN) * 128, kScales = BM * 16, kLoadS = (BM / 16 + kWaves * KW - 1) / (kWaves * KW);
  static_assert(NS >= 2 && NS <= 4 && (KW == 1 || KW == 2) && 128 % (BN / WN) == 0, "a wave's columns share a scale");
  __shared__ __align__(1024) uint8_t sh[NS * KW * kSlice + 4 * kScales];
  static_assert(KW == 1 || NS * KW * kSlice >= BM * BN * 4, "the groups' sums meet where the slices were");
  const int lane = threadIdx.x & 63, all_waves = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wave = all_waves % kWaves, kg = all_waves / kWaves;
  // Workgroups of one XCD (every eighth) take neighbouring tiles, eight rows of tiles at a time: they share operands in its L2.
  const int tiles_m = (p.M + BM - 1) / BM, tiles_n = (p.N + BN - 1) / BN, total = tiles_m * tiles_n;
  const int per_xcd = (total + 7) / 8, work = (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3);
  if (work >= total) return;
  const int band = work / (8 * tiles_n), high = min(8, tiles_m - band * 8), in_band = work - band * 8 * tiles_n;
  const int m0 = (band * 8 + in_band % high) * BM, n0 = in_band / high * BN;
  const int wm = wave / WN * (BM / WM), wn = wave % WN * (BN / WN);
  const int kb_begin = blockIdx.y * p.per, kb_end = min(kb_begin + p.per, p.KB);
  const auto ra = __builtin_amdgcn_make_buffer_rsrc((void*)p.a, 0, (unsigned)((size_t)p.M * p.K), 0x00020000);
  const auto rb = __builtin_amdgcn_make_buffer_rsrc((void*)p.b, 0, (unsigned)((size_t)p.N * p.K), 0x00020000);
  const auto rs = __builtin_amdgcn_make_buffer_rsrc((void*)p.sa, 0, (unsigned)((size_t)p.M * p.KB * 4), 0x00020000);

  // A wave's load moves 8 rows of a slice: lane l brings chunk (l & 7) ^ (row & 7) of row l >> 3.
  const int lrow = lane >> 3, lchunk = (lane & 7) ^ (lrow & 7);
  const unsigned off_a = operand_offset(m0 + wave * 8 + lrow, lchunk, p.K), off_b = operand_offset(n0 + wave * 8 + lrow, lchunk, p.K);
  auto load = [&](int it, int buf) {
    const int kb = kb_begin + it * KW + kg;
    const unsigned block = block_offset(kb, p.KB);
    uint8_t* to = sh + (buf * KW + kg) * kSlice;
#pragma unroll
    for (int i = 0; i < kLoadA; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lds_ptr)(to + (i * kWaves + wave) * 1024), 16, operand_load(off_a, kb, lchunk, i * kWaves * 8, p.K), block, 0, 0);
#pragma unroll
    for (int i = 0; i < kLoadB; ++i)
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lds_ptr)(to + BM * 128 + (i * kWaves + wave) * 1024), 16, operand_load(off_b, kb, lchunk, i * kWaves * 8, p.K), block, 0, 0);
  };
  // The rows' scales come for four blocks of k at a time, 16 bytes a row: a row's scales are one after the other, and bringing one
  // for each row and block touches four times as many lines of memory (331 instead of 299 us at 8192 x 8192 x 4096).
  uint8_t* const scales = sh + NS * KW * kSlice;
  // A load is one float a lane, so that each is inside the rows' scales or not: 16 rows a wave.
  auto load_scales = [&](int four) {
#pragma unroll
    for (int i = 0; i < kLoadS; ++i) {
      const int group = i * kWaves * KW + all_waves;
      if (group < BM / 16)
        __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (lds_ptr)(scales + (four & 3) * kScales + group * 256), 4,
                                                 scale_load(m0 + group * 16 + (lane >> 2), four * 4 + (lane & 3), p.M, p.KB), 0, 0, 0);
    }
  };
  const int frow = lane & 15, g = lane >> 4;
  const int c0 = frow * 128 + (g ^ (frow & 7)) * 16, c1 = frow * 128 + ((g + 4) ^ (frow & 7)) * 16;
  auto fragment = [&](const uint8_t* rows) {
    return join(*reinterpret_cast<const i32x4*>(rows + c0), *reinterpret_cast<const i32x4*>(rows + c1));
  };
  ConstFloat* sbp = uniform_floats(p.sb + (long long)min((n0 + wn) / 128, (p.N - 1) / 128) * p.KB);
  f32x4 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x4{};
  load_scales(kb_begin >> 2);
  load_scales((kb_begin >> 2) + 1);
#pragma unroll
  for (int i = 0; i < NS; ++i) load(i, i);
  wait_loads<(NS - 1) * kLoads>();
  __syncthreads();
  i32x8 fb[TN], fa[2];
#pragma unroll
  for (int j = 0; j < TN; ++j) fb[j] = fragment(sh + kg * kSlice + (BM + wn + j * 16) * 128);
  fa[0] = fragment(sh + kg * kSlice + wm * 128);
  // The buffers change hands one row of tiles before a block's end: by then its fragments are all in registers, and while the next
  // block's first fragments are read (a column's as soon as its registers are free) the matrix unit has that row to work on.
  // The loop has no branch: behind the last block zeros are brought and not used.
  int buf = 0;
  float sb_next = sbp[min(kb_begin + kg, p.KB - 1)];
  for (int it = 0; kb_begin + it * KW < kb_end; ++it) {
    const int kb = kb_begin + it * KW + kg, next_buf = buf + 1 == NS ? 0 : buf + 1;
    const uint8_t* base = sh + (buf * KW + kg) * kSlice;
    const uint8_t* other = sh + (next_buf * KW + kg) * kSlice;
    const float sb = sb_next;
    sb_next = sbp[min(kb + KW, p.KB - 1)];
    float s[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) s[i] = *reinterpret_cast<const float*>(scales + (kb >> 2 & 3) * kScales + (wm + i * 16 + frow) * 16 + (kb & 3) * 4) * sb;
    if (KW > 1 && kb >= kb_end)   // the last round of a group that has no block left
#pragma unroll
      for (int i = 0; i < TM; ++i) s[i] = 0.0f;
    f32x4 d[2][2];
    // tiles in pairs: the multiply-adds of a pair are issued behind the matrix instructions of the next
    auto add = [&](int pair) {
      const int i = pair / (TN / 2), j = pair % (TN / 2) * 2;
#pragma unroll
      for (int r = 0; r < 8; ++r) acc[i][j + r / 4][r % 4] = fmaf(d[pair & 1][r / 4][r % 4], s[i], acc[i][j + r / 4][r % 4]);
    };
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      if (i + 1 < TM) fa[(i + 1) & 1] = fragment(base + (wm + (i + 1) * 16) * 128);
      if (i == TM - 1) {
        wait_loads<(NS - 2) * kLoads>();
        __syncthreads();   // the next slice has arrived for all waves, this one has been read by all
        load(it + NS, buf);
      }
#pragma unroll
      for (int j = 0; j < TN; j += 2) {
        const int pair = i * (TN / 2) + j / 2;
        d[pair & 1][0] = mfma_fp8(fb[j], fa[i & 1]);
        d[pair & 1][1] = mfma_fp8(fb[j + 1], fa[i & 1]);
        if (i == TM - 1) {
          fb[j] = fragment(other + (BM + wn + j * 16) * 128);
          fb[j + 1] = fragment(other + (BM + wn + j * 16 + 16) * 128);
        }
        if (pair > 0) add(pair - 1);
      }
    }
    fa[0] = fragment(other + wm * 128);
    add(TM * TN / 2 - 1);
    // the sums are finished here: beyond the branch the compiler would keep all matrix results until then
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) asm volatile("" : "+v"(acc[i][j]));
    // two fours ahead: before the last wait in front of their first use two slices are asked for, as many as may be under way then
    if ((it * KW & 3) == 0) load_scales(((kb_begin + it * KW) >> 2) + 2);
    buf = next_buf;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // nothing is under way to shared memory when the workgroup ends
  if constexpr (KW > 1) {
    f32x4* const sums = reinterpret_cast<f32x4*>(sh) + (wave * TM * TN) * 64 + lane;
    __syncthreads();
    if (kg == 1)
#pragma unroll
      for (int i = 0; i < TM * TN; ++i) sums[i * 64] = acc[i / TN][i % TN];
    __syncthreads();
    if (kg == 1) return;
#pragma unroll
    for (int i = 0; i < TM * TN; ++i) acc[i / TN][i % TN] += sums[i * 64];
  }
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) store_out(p, m0 + wm + i * 16 + frow, n0 + wn + j * 16 + g * 4, acc[i][j]);
}

// Up to 16 rows: the weights are read once, straight into registers (one fragment serves all rows); a workgroup's waves take every
// 16th block of k for the same 16 columns and meet in shared memory.  U blocks of a wave are under way at once, all of K = 4096.  Bound by
// the weights' bytes: 4 x 16384 x 4096 takes 15.3 us, 4.4 TB/s (8 waves and four blocks 16.6), 4 x 8192 x 4096 9.5 us (9.9).  From 17 rows on
// the tiles are faster (12 against 18 us at 32 rows).
__global__ void __launch_bounds__(1024) gemm_fp8_rows_kernel(GemmArgs p) {
  constexpr int kWaves = 16, U = 2;
  __shared__ f32x4 sh[kWaves][64];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int n0 = blockIdx.x * 16, row = lane & 15, g = lane >> 4;
  const int m = min(row, p.M - 1);   // rows beyond the last repeat it and are not stored
  const uint8_t* a = p.a + (long long)m * p.K;
  const float* sap = p.sa + (long long)m * p.KB;
  const uint8_t* b = p.b + (long long)min(n0 + row, p.N - 1) * p.K;
  ConstFloat* sbp = uniform_floats(p.sb + (long long)(n0 / 128) * p.KB);
  f32x4 acc{};
  const int kb_begin = blockIdx.y * p.per, kb_end = min(kb_begin + p.per, p.KB);
  for (int kb0 = kb_begin + wave; kb0 < kb_end; kb0 += kWaves * U) {
    i32x8 fb[U], fa[U];
    float s[U];
    const i32x4 zero{};
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int kb = kb0 + u * kWaves, k0 = kb * 128 + g * 16, k1 = k0 + 64;
      const bool in0 = k0 < p.K && kb < kb_end, in1 = k1 < p.K && kb < kb_end;
      fb[u] = join(in0 ? *reinterpret_cast<const i32x4*>(b + k0) : zero, in1 ? *reinterpret_cast<const i32x4*>(b + k1) : zero);
      fa[u] = join(in0 ? *reinterpret_cast<const i32x4*>(a + k0) : zero, in1 ? *reinterpret_cast<const i32x4*>(a + k1) : zero);
      s[u] = kb < kb_end ? sap[kb] * sbp[kb] : 0.0f;
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const f32x4 d = mfma_fp8(fb[u], fa[u]);
#pragma unroll
      for (int r = 0; r < 4; ++r) acc[r] = fmaf(d[r], s[u], acc[r]);
    }
  }
  sh[wave][lane] = acc;
  __syncthreads();
  if (wave == 0) {
    for (int w = 1; w < kWaves; ++w) acc += sh[w][lane];
    store_out(p, row, n0 + g * 4, acc);
  }
}

__global__ void __launch_bounds__(256) gemm_fp8_parts_kernel(const float* __restrict__ part, int parts, long long n, __bf16* __restrict__ out) {
  const long long at = ((long long)blockIdx.x * 256 + threadIdx.x) * 4;
  if (at >= n) return;
  const int valid = (int)min(n - at, 4LL);
  f32x4 v = loadv<4>(part + at, valid);
#pragma unroll 4
  for (int i = 1; i < parts; ++i) v += loadv<4>(part + i * n + at, valid);
  storev<4>(out + at, v, valid);
}

template <int BM, int BN, int WM, int WN, int NS, int KW>
void gemm_tiles(const GemmArgs& p, const GemmPlan& g, hipStream_t s) {
  hipLaunchKernelGGL((gemm_fp8_kernel<BM, BN, WM, WN, NS, KW>), dim3((unsigned)((g.groups + 7) / 8 * 8), g.parts), dim3(64 * WM * WN * KW), 0, s, p);
}

int gemm(const GemmArgs& p, const GemmPlan& g, hipStream_t s) {
  const dim3 rows((unsigned)g.groups, g.parts);
  switch (g.kind) {
    case GemmPlan::kRows: hipLaunchKernelGGL(gemm_fp8_rows_kernel, rows, dim3(1024), 0, s, p); break;
    case GemmPlan::k256: gemm_tiles<256, 256, 2, 4, 2, 1>(p, g, s); break;
    case GemmPlan::k128: gemm_tiles<128, 128, 2, 2, 2, 1>(p, g, s); break;
    case GemmPlan::k128KW: gemm_tiles<128, 128, 2, 2, 2, 2>(p, g, s); break;
    case GemmPlan::k64x128KW: gemm_tiles<64, 128, 2, 2, 3, 2>(p, g, s); break;
    case GemmPlan::k64KW: gemm_tiles<64, 64, 2, 2, 4, 2>(p, g, s); break;
  }
  SLAMHIP_HIP(hipGetLastError());
  if (g.parts > 1) {
    const long long n = (long long)p.M * p.N;
    hipLaunchKernelGGL(gemm_fp8_parts_kernel, dim3((unsigned)((n + 1023) / 1024)), dim3(256), 0, s, p.part, g.parts, n, p.out);
    SLAMHIP_HIP(hipGetLastError());
  }
  return SLAMHIP_OK;
}

}  // namespace
}  // namespace slamhip

using namespace slamhip;

extern "C" {

size_t slamhip_gemm_nt_fp8_workspace_bytes(int M, int N, int K) {
  if (M <= 0 || N <= 0 || K <= 0 || !gemm_fits(M, N, K)) return 0;
  const GemmPlan g = gemm_plan(M, N, K);
  return g.parts > 1 ? (size_t)g.parts * M * N * sizeof(float) : 0;
}

int slamhip_gemm_nt_fp8(const void* a, const float* a_scales, const void* b, const float* b_scales, int M, int N, int K, void* out,
                        void* workspace, size_t workspace_bytes, void* stream) {
  SLAMHIP_REQUIRE(M >= 0 && N >= 0 && K > 0, SLAMHIP_E_ARG, "gemm_nt_fp8: need M, N >= 0 and K >= 1");
  SLAMHIP_REQUIRE(K % 16 == 0, SLAMHIP_E_SIZE, "gemm_nt_fp8: K must be a multiple of 16");
  SLAMHIP_REQUIRE(gemm_fits(M, N, K), SLAMHIP_E_SIZE, "gemm_nt_fp8: an operand with 256 rows more is larger than 2 GB");
  if (M == 0 || N == 0) return SLAMHIP_OK;
  SLAMHIP_REQUIRE(a && a_scales && b && b_scales && out, SLAMHIP_E_ARG, "gemm_nt_fp8: null pointer");
  SLAMHIP_REQUIRE(((uintptr_t)a & 15) == 0 && ((uintptr_t)b & 15) == 0, SLAMHIP_E_ARG, "gemm_nt_fp8: operands must be 16-byte aligned");
  const GemmPlan g = gemm_plan(M, N, K);
  SLAMHIP_REQUIRE(g.groups < (1 << 22), SLAMHIP_E_SIZE, "gemm_nt_fp8: too many tiles");
  SLAMHIP_REQUIRE(g.parts == 1 || (workspace && workspace_bytes >= (size_t)g.parts * M * N * sizeof(float)), SLAMHIP_E_ARG,
                  "gemm_nt_fp8: workspace too small");
  const GemmArgs p{(const uint8_t*)a, (const uint8_t*)b, a_scales, b_scales, (__bf16*)out, M, N, K, (K + 127) / 128, g.per,
                   g.parts > 1 ? (float*)workspace : nullptr};
  return gemm(p, g, (hipStream_t)stream);
}

}  // extern "C"
