// Quantisers of the 8-bit matrix product: blocks of 1 x 128 (activations, gradients) or 128 x 128 (weights), one fp32 scale a block, from
// fp32 / bf16 / fp16 matrices, as they lie or transposed (the operands of a linear layer's two gradients have the other axis inside).
//
//   scale = max(amax, 2^-100) fl(1 / top),   q = round_even(x fl(1 / scale))
//
// One pass: a block is read once, its maximum found in registers (and LDS), and written in 8 bits: bound by HBM, 2 (or 4) + 1 bytes an
// element.
#include "row_ops.h"

namespace {

struct QuantArgs {
  const void* x;
  unsigned char* q;
  float* scale;
  long long rows, ldx, ldq, ss_row, ss_blk;
  int cols;
};

// 1 x 128 blocks along the row: sixteen lanes hold one block, a wave four
template <typename T, int FMT>
__global__ __launch_bounds__(256) void quant_rows_kernel(const QuantArgs a) {
  const int blocks = (a.cols + 127) >> 7, lane = threadIdx.x & 15;
  const long long total = a.rows * blocks, step = (long long)gridDim.x * 16;
  for (long long i0 = (long long)blockIdx.x * 16; i0 < total; i0 += step) {
    const long long i = i0 + (threadIdx.x >> 4);
    const long long row = i / blocks;
    const int kb = (int)(i - row * blocks), col = kb * 128 + lane * 8, n = i < total ? a.cols - col : 0;
    float v[8], m = 0.f;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
    if (n > 0) ro_load8(reinterpret_cast<const T*>(a.x) + row * a.ldx + col, n, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) m = fmaxf(m, ro_finite_abs(v[j]));
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
    const float s = ro_scale_of<FMT>(m), inv = 1.f / s;
    if (n <= 0) continue;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = ro_fit<FMT>(v[j], inv);
    ro_store8q(a.q + row * a.ldq + col, n, ro_pack4<FMT>(v[0], v[1], v[2], v[3]), ro_pack4<FMT>(v[4], v[5], v[6], v[7]));
    if (lane == 0) a.scale[row * a.ss_row + kb * a.ss_blk] = s;
  }
}

// One workgroup, one 128 x 128 tile of x, an 8 x 8 patch a thread.  TILE: one scale for the tile, else one for each output row's 128.
// TRANS: q is (cols, rows); the bytes turn round in LDS, whose rows are 144 bytes (16-byte aligned, 36 banks apart).
template <typename T, int FMT, bool TILE, bool TRANS>
__global__ __launch_bounds__(256) void quant_tile_kernel(const QuantArgs a) {
  __shared__ float red[TILE ? 4 : 16 * 128];
  __shared__ __align__(16) unsigned char turn[TRANS ? 128 * 144 : 16];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const long long row0 = (long long)blockIdx.y * 128;
  const int col0 = blockIdx.x * 128, col = col0 + tx * 8;
  float v[8][8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const long long row = row0 + ty * 8 + i;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] = 0.f;
    if (row < a.rows && col < a.cols) ro_load8(reinterpret_cast<const T*>(a.x) + row * a.ldx + col, a.cols - col, v[i]);
  }
  float inv[8];
  if constexpr (TILE) {
    float m = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 8; ++j) m = fmaxf(m, ro_finite_abs(v[i][j]));
    m = wave_max(m);
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    const float s = ro_scale_of<FMT>(fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3])));
    const float t = 1.f / s;
#pragma unroll
    for (int j = 0; j < 8; ++j) inv[j] = t;
    if (threadIdx.x == 0) a.scale[TRANS ? blockIdx.x * a.ss_row + blockIdx.y * a.ss_blk : blockIdx.y * a.ss_row + blockIdx.x * a.ss_blk] = s;
  } else {
    static_assert(TILE || TRANS, "rows as they lie have a kernel of their own");
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float m = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) m = fmaxf(m, ro_finite_abs(v[i][j]));
      red[ty * 128 + tx * 8 + j] = m;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float m = 0.f;
#pragma unroll
      for (int k = 0; k < 16; ++k) m = fmaxf(m, red[k * 128 + tx * 8 + j]);
      const float s = ro_scale_of<FMT>(m);
      inv[j] = 1.f / s;
      if (ty == 0 && col + j < a.cols) a.scale[(long long)(col + j) * a.ss_row + blockIdx.y * a.ss_blk] = s;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] = ro_fit<FMT>(v[i][j], inv[j]);
  if constexpr (!TRANS) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const long long row = row0 + ty * 8 + i;
      if (row < a.rows && col < a.cols)
        ro_store8q(a.q + row * a.ldq + col, a.cols - col, ro_pack4<FMT>(v[i][0], v[i][1], v[i][2], v[i][3]),
                   ro_pack4<FMT>(v[i][4], v[i][5], v[i][6], v[i][7]));
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const u32x2 b = {ro_pack4<FMT>(v[0][j], v[1][j], v[2][j], v[3][j]), ro_pack4<FMT>(v[4][j], v[5][j], v[6][j], v[7][j])};
      *reinterpret_cast<u32x2*>(&turn[(tx * 8 + j) * 144 + ty * 8]) = b;
    }
    __syncthreads();
    const long long n = a.rows - (row0 + tx * 8);
    if (n > 0)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = ty + 16 * i;
        if (col0 + c >= a.cols) break;
        const u32x2 b = *reinterpret_cast<const u32x2*>(&turn[c * 144 + tx * 8]);
        ro_store8q(a.q + (long long)(col0 + c) * a.ldq + row0 + tx * 8, n < 8 ? (int)n : 8, b[0], b[1]);
      }
  }
}

template <typename T, int FMT>
int launch_quant(const QuantArgs& a, int tile, int trans, hipStream_t s) {
  if (!tile && !trans) {
    const long long total = (a.rows * ((a.cols + 127) >> 7) + 15) / 16;
    quant_rows_kernel<T, FMT><<<(int)(total < 4096 ? total : 4096), 256, 0, s>>>(a);
  } else {
    const dim3 grid((a.cols + 127) / 128, (unsigned)((a.rows + 127) / 128));
    if (tile && trans) quant_tile_kernel<T, FMT, true, true><<<grid, 256, 0, s>>>(a);
    else if (tile) quant_tile_kernel<T, FMT, true, false><<<grid, 256, 0, s>>>(a);
    else quant_tile_kernel<T, FMT, false, true><<<grid, 256, 0, s>>>(a);
  }
  UNCL_CHECK_LAUNCH();
  return UNCL_OK;
}

}  // namespace

extern "C" int uncl_quant8(const void* x, int dtype, long long rows, int cols, long long ldx, void* q, long long ldq, int fmt, float* scale,
                           long long scale_row, long long scale_block, int tile, int transposed, void* stream) {
  if (!(dtype == UNCL_F32 || uncl_is_h16(dtype)) || (fmt != UNCL_E4M3 && fmt != UNCL_E5M2) || rows < 0 || cols < 0) return UNCL_ERR_ARG;
  if (rows == 0 || cols == 0) return UNCL_OK;
  if (!x || !q || !scale || ldx < cols || ldq < (transposed ? rows : cols)) return UNCL_ERR_ARG;
  if ((tile || transposed) && (rows + 127) / 128 > 65535) return UNCL_ERR_ARG;      // one workgroup a tile, rows along the grid's y
  const QuantArgs a{x, reinterpret_cast<unsigned char*>(q), scale, rows, ldx, ldq, scale_row, scale_block, cols};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define BY_TYPE(F)                                                                                          \
  (dtype == UNCL_F32 ? launch_quant<float, F>(a, tile, transposed, s)                                       \
                     : dtype == UNCL_BF16 ? launch_quant<bf16_t, F>(a, tile, transposed, s) : launch_quant<f16_t, F>(a, tile, transposed, s))
  return fmt == UNCL_E4M3 ? BY_TYPE(UNCL_E4M3) : BY_TYPE(UNCL_E5M2);
#undef BY_TYPE
}
