// How the 8-bit product (gemm_fp8.hip) is cut, and where its tiles' loads begin: plain arithmetic that the host compiles too.
#pragma once

namespace slamhip {
namespace {

// A tile's loads go through buffers of an operand's size, and those that would begin behind it arrive as zeros.  Which rows and
// columns of k an access belongs to is all in its vector offset, because the scalar offset may be left out of the range check: it holds
// the block of k alone, never one behind the last, and a vector offset inside the operand's row stays inside with it.

constexpr unsigned kBeyond = 0x80000000u;   // a vector offset past every operand, which are smaller, also with what is added to it

// chunk (16 bytes of a block's 128) of a row; rows behind the last are behind the operand by themselves ((rows + 256) K < 2^31)
constexpr unsigned operand_offset(int row, int chunk, int K) { return (unsigned)row * (unsigned)K + (unsigned)chunk * 16u; }

// the same for block kb of k, `rows_on` rows further: chunks behind the last of a row are behind the operand
constexpr unsigned operand_load(unsigned offset, int kb, int chunk, int rows_on, int K) {
  return (kb * 128 + chunk * 16 < K ? offset : kBeyond) + (unsigned)rows_on * (unsigned)K;
}

constexpr unsigned block_offset(int kb, int KB) { return (unsigned)(kb < KB ? kb : KB - 1) * 128u; }

// the scale of a row for block kb, one float
constexpr unsigned scale_load(int row, int kb, int rows, int KB) {
  return row < rows && kb < KB ? ((unsigned)row * (unsigned)KB + (unsigned)kb) * 4u : kBeyond;
}

// both operands below 2 GB with the rows that tiles have behind the last; a larger product is refused and needs no workspace
constexpr bool gemm_fits(int M, int N, int K) { return (M + 256LL) * K < (1LL << 31) && (N + 256LL) * K < (1LL << 31); }

// The kernel by the number of rows and tiles, and parts of k where that leaves most CUs idle.
struct GemmPlan {
  enum Kind { kRows, k256, k128, k128KW, k64x128KW, k64KW } kind;
  long long groups;
  int per, parts;
};

inline GemmPlan gemm_plan(int M, int N, int K) {
  GemmPlan g;
  auto tiles = [&](int bm, int bn) { return (long long)((M + bm - 1) / bm) * ((N + bn - 1) / bn); };
  auto pick = [&](GemmPlan::Kind kind, long long groups) { g.kind = kind, g.groups = groups; };
  // The smallest tiles while there is one for each of the 256 CUs at most (they wait least for each other), then larger ones, which read
  // operands less often: 256^2 where k is long enough for its start and end, and two groups of waves (KW = 2) where a CU has one
  // workgroup and k is long.  us, 256^2 / 128^2 / 128^2 KW / 64 x 128 KW / 64^2 KW: 4096x4096x4096 68/83/93/115/153, 2048x4096x4096
  // 59/42/48/59/77, 1024x4096x4096 57/28/26/31/40, 777x2056x4096 54/25/22/16/21, 1024x1024x4096 56/25/22/16/12, 645x1434x3584
  // 37/19/19/14/11, 306x6016x1408 28/12/13/9/13, 2225x7997x640 46/34/48/57/80, 1028x2864x896 19/9.5/10.7/14/15.
  const int KB = (K + 127) / 128;
  if (M <= 16) pick(GemmPlan::kRows, (N + 15) / 16);
  else if (tiles(64, 64) <= 256) pick(GemmPlan::k64KW, tiles(64, 64));
  else if (tiles(64, 128) <= 256) pick(GemmPlan::k64x128KW, tiles(64, 128));
  else if (tiles(256, 256) >= 192 && KB >= 8) pick(GemmPlan::k256, tiles(256, 256));
  else if (tiles(128, 128) <= 256 && KB > 16) pick(GemmPlan::k128KW, tiles(128, 128));
  else pick(GemmPlan::k128, tiles(128, 128));
  // Blocks of k that are worth a part of their own, and a launch more.  us with at least 8 / 12 / 16 / 32 of them: 40x478x7328 8.4/9.7/10.2/16.2,
  // 276x490x10512 14.3/14.2/14.7/20.4, 100x500x16384 13.5/12.1/12.1/14.3, 871x562x3152 13.6/13.6/12.3/12.4; few rows, whose weights
  // are read by more waves, 4x2048x4096 6.7/6.8/6.8/5.5.
  const int least = g.kind == GemmPlan::kRows ? 32 : 12;
  // a workgroup for each CU at most, of each XCD's 32 too: with 33 112x2598x12000 takes 27 us, with fewer parts 22
  long long parts = g.kind == GemmPlan::kRows ? 256 / g.groups : 32 / ((g.groups + 7) / 8);
  if (parts > KB / least) parts = KB / least;
  if (parts < 1) parts = 1;
  g.per = (int)(((KB + parts - 1) / parts + 3) / 4 * 4);
  g.parts = (KB + g.per - 1) / g.per;
  return g;
}

}  // namespace
}  // namespace slamhip
