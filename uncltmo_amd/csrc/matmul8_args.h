// Arguments of the 8-bit matrix product's kernels (matmul8.h), and the way to run one from another file.
#pragma once
#include "common.h"

struct MmArgs {
  const unsigned char *a, *b;
  const float *sa, *sb, *bias;
  const void* res;
  void* out;
  long long lda, ldb, ldr, ldo, sa_row, sa_blk, sb_row, sb_blk;
  int M, N, K, KB, act, out_dtype;
  // K split over gridDim.y workgroups a tile (64 x 64 tiles): fp32 partial results [gridDim.y][M][N rounded up to 8], `per` blocks each
  float* part;
  int per;
};

static inline long long mm_tiles(int M, int N, int t) { return (long long)((M + t - 1) / t) * ((N + t - 1) / t); }

// Which tiles, and their time in tenths of a round of 256 x 128 x 128 outputs.  Time goes by rounds of workgroups over the 256 CUs.  256 x 256
// tiles (8-bit instruction, b scaled by tiles) work one to a CU, four units a round; 128 x 128 ones two to a CU, two units a round, a
// tenth slower a unit (8192 x 4096 x 4096: 124 against 146 us; 4099 x 4096 x 2048, 8 units against 6: 65 against 51 us; a short K leaves
// nothing to hide the epilogue behind but another workgroup: 28800 x 1024 x 256 with GELU 35.8 against 33.4 us).  64 x 64 tiles, four to a CU,
// where 128 x 128 ones are at most one a CU (512 x 4096 x 4096: 19 against 27 us; 2048 x 2048 x 2048 16.4 against 16.0, x 512 8.2 against 8.1).
// All three at 14 outputs from 1024 x 1024 to 28800 x 1024 and K = 128 to 4096, without bias: for bf16 results the rule's tiles are the fastest or
// within 10 % of them, but for 256 x 256 ones under K = 768 (4096 x 4096 x 512: 16.0 against the chosen 17.9, 8192 x 2048 x 512 15.7 against
// 17.9); for exact sums 64 x 64 ones would be up to 20 % faster at 257 to 320 large tiles (2304 x 2048 x 1024: 18.0 against the chosen 21.7) and
// up to a third at K = 128 (4608 x 2048: 12.1 against 16.1): left to a rule of its own.
struct MmPlan {
  int tile;
  long long units;
};
static inline MmPlan mm_plan(int M, int N, int kb, bool large) {
  const long long t128 = mm_tiles(M, N, 128), u128 = 22 * ((t128 + 511) / 512), u256 = 40 * ((mm_tiles(M, N, 256) + 255) / 256);
  if (t128 <= 256) return {64, 12 * ((mm_tiles(M, N, 64) + 1023) / 1024)};
  if (large && kb >= 6 && u256 <= u128) return {256, u256};
  return {128, u128};
}

// workgroups that share a tile's K: 1, or enough for two a CU where 64 x 64 tiles leave CUs idle, at least four blocks each
static inline int mm_splits(int M, int N, int K) {
  const long long t = mm_tiles(M, N, 64);
  const int kb = (K + 127) / 128;
  if (M <= 64 || t >= 256 || kb < 8) return 1;
  long long s = (512 + t - 1) / t;
  if (s > kb / 4) s = kb / 4;
  if (s > 16) s = 16;
  const int per = (int)((kb + s - 1) / s);
  return (kb + per - 1) / per;
}
static inline size_t mm_split_bytes(int M, int N, int K) {
  const int s = mm_splits(M, N, K);
  return s > 1 ? (size_t)s * M * ((N + 7) & ~7) * sizeof(float) : 0;
}
int mm_run(const MmArgs& p, int a_fmt, bool b_tile, void* workspace, hipStream_t s);
