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

// workgroups that share a tile's K: 1, or enough for two a CU where 64 x 64 tiles leave CUs idle, at least four blocks each
static inline int mm_splits(int M, int N, int K) {
  const long long t = (long long)((M + 63) / 64) * ((N + 63) / 64);
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
