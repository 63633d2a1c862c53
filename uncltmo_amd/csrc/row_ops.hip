// Operators on rows of channels (a row = one pixel or graph node of a channel-last tensor): dropout from a counter, and the residual
// addition with the RMS norm behind it, forward (16 / 32-bit or 8-bit output) and backward.
//
//   drop:    y = res + k x s            k from Philox words (row_ops.h), s = 2^16 / (2^16 - limit); the mask is never stored, the
//                                       gradient is the same call on g
//   norm:    h = round(res + drop(x)),  r = 1 / sqrt(mean_c h^2 + eps),  y = h r w
//   back:    n = h r,  g_h = g_h' + r (gy w - n mean_c(gy w n)),  g_res = g_h,  g_x = drop(g_h),  g_w = sum_rows gy n
//
// All of them are bound by HBM: each input is read once, each output written once, the row lives in registers between the two passes
// over it.  A row is held by LANES threads, eight channels each per chunk, CH chunks: narrow maps (32 channels: 4 lanes) put sixteen rows
// into a wave, so that every access of a wave is 1 KB of consecutive memory whatever the width.
//
// Measured, bf16 (a copy of 1 GiB runs at 5.05 TB/s on the same card): dropout of 16 x 252 x 252 x 32 25.6 us = 5.1 TB/s (a Philox
// evaluation of ten rounds for each eight elements hides behind the loads); addition and norm of 8 x 252 x 252 x 32 28.3 us = 4.6 TB/s,
// the backward pass 25.4 us = 5.1 TB/s and 4.0 us for the weight gradient's fold; into 8 bits 28800 x 256 11.9 us = 4.4 TB/s; a single row
// 3.4 us, of which the launch is most.
#include "row_ops.h"

namespace {

struct NormArgs {
  const void *x, *res;
  const float* w;
  void *h, *y;
  float *rstd, *scale;
  long long rows, ldx, ldr, ldh, ldy, ss_row, ss_blk;
  int cols, groups;
  float eps, inv_cols;
  RoDrop drop;
};

// sum over the LANES threads that hold a row; every one of them gets it.  LANES = 256: the workgroup, through LDS (two buffers in turn:
// one barrier a row)
template <int LANES>
__device__ __forceinline__ float row_sum(float v, float* red, int& turn) {
#pragma unroll
  for (int o = (LANES < 64 ? LANES : 64) / 2; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  if constexpr (LANES > 64) {
    float* s = red + turn * 4;
    turn ^= 1;
    if ((threadIdx.x & 63) == 0) s[threadIdx.x >> 6] = v;
    __syncthreads();
    v = (s[0] + s[1]) + (s[2] + s[3]);
  }
  return v;
}

// Squares of values over about 2^63 leave fp32's range: the sum is then infinite, and is made again from 2^-64 of the values.  again: that sum
// over the row (infinite still where a value is)
#define RO_FAR 0x1p-64f
template <typename F>
__device__ __forceinline__ float inverse_rms(float sum, float inv_cols, float eps, F again) {
  if (__builtin_expect(sum == __builtin_inff(), 0)) return rsqrtf(again() * inv_cols + eps * (RO_FAR * RO_FAR)) * RO_FAR;
  return rsqrtf(sum * inv_cols + eps);
}

// FMT: UNCL_Q8_NONE = y in T; UNCL_E4M3 / UNCL_E5M2 = y in 8 bits with a scale for each 128 channels (sixteen lanes hold one block)
template <typename T, int LANES, int CH, int FMT>
__global__ __launch_bounds__(256) void norm_kernel(const NormArgs a) {
  constexpr int PER = 256 / LANES;
  __shared__ float red[8];
  int turn = 0;
  const int lane = threadIdx.x % LANES, slot = threadIdx.x / LANES;
  float w[CH][8];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int col = (lane + c * LANES) * 8;
    if (a.w && col < a.cols) {
      ro_load8(a.w + col, a.cols - col, w[c]);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) w[c][i] = 1.f;
    }
  }
  unsigned long long seed = a.drop.seed, offset = a.drop.offset;
  if (a.drop.limit && a.drop.dev) { seed = a.drop.dev[0]; offset += a.drop.dev[1]; }
  const long long step = (long long)gridDim.x * PER;
  for (long long row0 = (long long)blockIdx.x * PER; row0 < a.rows; row0 += step) {
    const long long row = row0 + slot;
    const bool live = row < a.rows;
    const unsigned long long fg = a.drop.limit ? ro_flag_group(a.drop, row, a.groups) : 0;
    float v[CH][8], sum = 0.f;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (lane + c * LANES) * 8, n = live ? a.cols - col : 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) v[c][i] = 0.f;
      if (n <= 0) continue;
      float r[8];
      ro_load8_two(reinterpret_cast<const T*>(a.x) + row * a.ldx + col, a.res ? reinterpret_cast<const T*>(a.res) + row * a.ldr + col : nullptr, n, v[c], r);
      if (a.drop.limit) ro_drop8(fg + (col >> 3), offset, seed, a.drop.limit, a.drop.scale, v[c]);
      if (a.res)
#pragma unroll
        for (int i = 0; i < 8; ++i) v[c][i] += r[i];
      // the sum is normalised AS STORED, so that the backward pass sees the numbers the forward pass used
#pragma unroll
      for (int i = 0; i < 8; ++i) v[c][i] = (float)(T)v[c][i];
      if (a.h) ro_store8(reinterpret_cast<T*>(a.h) + row * a.ldh + col, n, v[c]);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = i < n ? fmaf(v[c][i], v[c][i], sum) : sum;
    }
    const float r = inverse_rms(row_sum<LANES>(sum, red, turn), a.inv_cols, a.eps, [&]() {
      float far = 0.f;
#pragma unroll
      for (int c = 0; c < CH; ++c)
#pragma unroll
        for (int i = 0; i < 8; ++i) far = fmaf(v[c][i] * RO_FAR, v[c][i] * RO_FAR, far);        // (0 behind the row's end)
      return row_sum<LANES>(far, red, turn);
    });
    if (a.rstd && live && lane == 0) a.rstd[row] = r;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (lane + c * LANES) * 8, n = live ? a.cols - col : 0;
      float y[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) y[i] = v[c][i] * r * w[c][i];
      if constexpr (FMT == UNCL_Q8_NONE) {
        if (n > 0) ro_store8(reinterpret_cast<T*>(a.y) + row * a.ldy + col, n, y);
      } else {
        bool odd;
        const unsigned m = ro_max_lanes<(LANES < 16 ? LANES : 16)>(ro_size8(y, odd));
        const float s = ro_scale_of<FMT>(m), inv = 1.f / s;
        if (n > 0) {
          ro_store8q(reinterpret_cast<unsigned char*>(a.y) + row * a.ldy + col, n, ro_pack8<FMT>(y, inv, odd));
          if ((col & 127) == 0) a.scale[row * a.ss_row + (col >> 7) * a.ss_blk] = s;
        }
      }
    }
  }
}

// Rows that do not fit in registers (over 16384 channels): the same arithmetic, the second pass reads x and res (or h) again
template <typename T, int FMT>
__global__ __launch_bounds__(256) void norm_long_kernel(const NormArgs a) {
  __shared__ float red[8];
  int turn = 0;
  unsigned long long seed = a.drop.seed, offset = a.drop.offset;
  if (a.drop.limit && a.drop.dev) { seed = a.drop.dev[0]; offset += a.drop.dev[1]; }
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const unsigned long long fg = a.drop.limit ? ro_flag_group(a.drop, row, a.groups) : 0;
    auto sum8 = [&](int col, float* v) {
      ro_load8(reinterpret_cast<const T*>(a.x) + row * a.ldx + col, a.cols - col, v);
      if (a.drop.limit) ro_drop8(fg + (col >> 3), offset, seed, a.drop.limit, a.drop.scale, v);
      if (a.res) {
        float r[8];
        ro_load8(reinterpret_cast<const T*>(a.res) + row * a.ldr + col, a.cols - col, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += r[i];
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = (float)(T)v[i];
    };
    float sum = 0.f;
    for (int col = threadIdx.x * 8; col < a.cols; col += 2048) {
      float v[8];
      sum8(col, v);
#pragma unroll
      for (int i = 0; i < 8; ++i) sum = i < a.cols - col ? fmaf(v[i], v[i], sum) : sum;
    }
    const float r = inverse_rms(row_sum<256>(sum, red, turn), a.inv_cols, a.eps, [&]() {
      float far = 0.f;
      for (int col = threadIdx.x * 8; col < a.cols; col += 2048) {
        float v[8];
        sum8(col, v);
#pragma unroll
        for (int i = 0; i < 8; ++i) far = i < a.cols - col ? fmaf(v[i] * RO_FAR, v[i] * RO_FAR, far) : far;
      }
      return row_sum<256>(far, red, turn);
    });
    if (a.rstd && threadIdx.x == 0) a.rstd[row] = r;
    // whole waves stay in the loop: sixteen lanes share a block's maximum.  h is written here, behind the last read of x and res by
    // this thread, so that it may be one of them
    for (int c0 = 0; c0 < a.cols; c0 += 2048) {
      const int col = c0 + threadIdx.x * 8, n = a.cols - col;
      float v[8], w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) { v[i] = 0.f; w[i] = 1.f; }
      if (n > 0) {
        sum8(col, v);
        if (a.w) ro_load8(a.w + col, n, w);
        if (a.h) ro_store8(reinterpret_cast<T*>(a.h) + row * a.ldh + col, n, v);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = v[i] * r * w[i];
      if constexpr (FMT == UNCL_Q8_NONE) {
        if (n > 0) ro_store8(reinterpret_cast<T*>(a.y) + row * a.ldy + col, n, v);
      } else {
        bool odd;
        const unsigned m = ro_max_lanes<16>(ro_size8(v, odd));
        const float s = ro_scale_of<FMT>(m), inv = 1.f / s;
        if (n > 0) {
          ro_store8q(reinterpret_cast<unsigned char*>(a.y) + row * a.ldy + col, n, ro_pack8<FMT>(v, inv, odd));
          if ((col & 127) == 0) a.scale[row * a.ss_row + (col >> 7) * a.ss_blk] = s;
        }
      }
    }
  }
}

struct NormBackArgs {
  const void *gy, *gh, *h;
  const float *w, *rstd;
  void *g_res, *g_x;
  float* part;        // [gridDim.x][cols] partial sums of g_w, or NULL
  long long rows, ldgy, ldgh, ldh, ldgr, ldgx;
  int cols, groups;
  float inv_cols;
  RoDrop drop;
};

template <typename T, int LANES, int CH>
__global__ __launch_bounds__(256) void norm_back_kernel(const NormBackArgs a) {
  constexpr int PER = 256 / LANES;
  __shared__ float red[8];
  __shared__ float fold[LANES < 64 ? 4 * LANES * 8 : (LANES < 256 ? 4 * LANES * 8 * CH : 1)];
  int turn = 0;
  const int lane = threadIdx.x % LANES, slot = threadIdx.x / LANES;
  float w[CH][8], gw[CH][8];
#pragma unroll
  for (int c = 0; c < CH; ++c) {
    const int col = (lane + c * LANES) * 8;
#pragma unroll
    for (int i = 0; i < 8; ++i) { w[c][i] = 1.f; gw[c][i] = 0.f; }
    if (a.w && col < a.cols) ro_load8(a.w + col, a.cols - col, w[c]);
  }
  unsigned long long seed = a.drop.seed, offset = a.drop.offset;
  if (a.drop.limit && a.drop.dev) { seed = a.drop.dev[0]; offset += a.drop.dev[1]; }
  const long long step = (long long)gridDim.x * PER;
  for (long long row0 = (long long)blockIdx.x * PER; row0 < a.rows; row0 += step) {
    const long long row = row0 + slot;
    const bool live = row < a.rows;
    const float r = live ? a.rstd[row] : 0.f;
    const unsigned long long fg = a.drop.limit && a.g_x ? ro_flag_group(a.drop, row, a.groups) : 0;
    float n_[CH][8], g[CH][8], dot = 0.f;
    RoRaw8<T> early;                                         // gh's, which waits for nobody
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (lane + c * LANES) * 8, n = live ? a.cols - col : 0;
#pragma unroll
      for (int i = 0; i < 8; ++i) { n_[c][i] = 0.f; g[c][i] = 0.f; }
      if (CH == 1 && a.gh && n >= 8) early.load(reinterpret_cast<const T*>(a.gh) + row * a.ldgh + col);
      if (n <= 0 || !a.gy) continue;
      ro_load8_two(reinterpret_cast<const T*>(a.h) + row * a.ldh + col, reinterpret_cast<const T*>(a.gy) + row * a.ldgy + col, n, n_[c], g[c]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        n_[c][i] *= r;
        gw[c][i] = fmaf(g[c][i], n_[c][i], gw[c][i]);
        g[c][i] *= w[c][i];
        dot = fmaf(g[c][i], n_[c][i], dot);
      }
    }
    const float mean = row_sum<LANES>(dot, red, turn) * a.inv_cols;
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (lane + c * LANES) * 8, n = live ? a.cols - col : 0;
      if (n <= 0) continue;
      if (a.gy)                                              // (without a gradient of y, 1 / rms counts for nothing, whatever it is)
#pragma unroll
        for (int i = 0; i < 8; ++i) g[c][i] = r * (g[c][i] - n_[c][i] * mean);
      if (a.gh) {
        float q[8];
        if (CH == 1 && n >= 8) early.get(q);
        else ro_load8(reinterpret_cast<const T*>(a.gh) + row * a.ldgh + col, n, q);
#pragma unroll
        for (int i = 0; i < 8; ++i) g[c][i] += q[i];
      }
      if (a.g_res) ro_store8(reinterpret_cast<T*>(a.g_res) + row * a.ldgr + col, n, g[c]);
      if (a.g_x) {
        if (a.drop.limit) ro_drop8(fg + (col >> 3), offset, seed, a.drop.limit, a.drop.scale, g[c]);
        ro_store8(reinterpret_cast<T*>(a.g_x) + row * a.ldgx + col, n, g[c]);
      }
    }
  }
  if (!a.part) return;
  // the slots of the workgroup hold the same columns: lanes of a wave by shuffles, the four waves through LDS, in a fixed order
  float* out = a.part + (long long)blockIdx.x * a.cols;
  if constexpr (LANES == 256) {
#pragma unroll
    for (int c = 0; c < CH; ++c) {
      const int col = (lane + c * LANES) * 8;
      if (col < a.cols) ro_store8(out + col, a.cols - col, gw[c]);
    }
  } else {
    const int wave = threadIdx.x >> 6;
#pragma unroll
    for (int c = 0; c < CH; ++c)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float v = gw[c][i];
#pragma unroll
        for (int o = LANES; o < 64; o <<= 1) v += __shfl_xor(v, o, 64);
        if ((threadIdx.x & 63) < LANES) fold[((wave * CH + c) * LANES + lane) * 8 + i] = v;
      }
    __syncthreads();
    for (int k = threadIdx.x; k < CH * LANES * 8; k += 256)
      if (k < a.cols) out[k] = (fold[k] + fold[CH * LANES * 8 + k]) + (fold[2 * CH * LANES * 8 + k] + fold[3 * CH * LANES * 8 + k]);
  }
}

// over 16384 channels: the second pass reads h and gy again; the partial sums of g_w are added up in the workgroup's own row of `part`
template <typename T>
__global__ __launch_bounds__(256) void norm_back_long_kernel(const NormBackArgs a) {
  __shared__ float red[8];
  int turn = 0;
  unsigned long long seed = a.drop.seed, offset = a.drop.offset;
  if (a.drop.limit && a.drop.dev) { seed = a.drop.dev[0]; offset += a.drop.dev[1]; }
  float* out = a.part ? a.part + (long long)blockIdx.x * a.cols : nullptr;
  bool first = true;
  for (long long row = blockIdx.x; row < a.rows; row += gridDim.x, first = false) {
    const float r = a.rstd[row];
    const unsigned long long fg = a.drop.limit ? ro_flag_group(a.drop, row, a.groups) : 0;
    float dot = 0.f;
    if (a.gy)
      for (int col = threadIdx.x * 8; col < a.cols; col += 2048) {
        float nv[8], g[8], w[8];
        const int n = a.cols - col;
        ro_load8(reinterpret_cast<const T*>(a.h) + row * a.ldh + col, n, nv);
        ro_load8(reinterpret_cast<const T*>(a.gy) + row * a.ldgy + col, n, g);
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = 1.f;
        if (a.w) ro_load8(a.w + col, n, w);
#pragma unroll
        for (int i = 0; i < 8; ++i) dot = fmaf(g[i] * w[i], nv[i] * r, dot);
      }
    const float mean = row_sum<256>(dot, red, turn) * a.inv_cols;
    for (int col = threadIdx.x * 8; col < a.cols; col += 2048) {
      float nv[8], g[8], w[8], p[8];
      const int n = a.cols - col;
#pragma unroll
      for (int i = 0; i < 8; ++i) { nv[i] = g[i] = p[i] = 0.f; w[i] = 1.f; }
      if (a.gy) {
        ro_load8(reinterpret_cast<const T*>(a.h) + row * a.ldh + col, n, nv);
        ro_load8(reinterpret_cast<const T*>(a.gy) + row * a.ldgy + col, n, g);
      }
      if (a.w) ro_load8(a.w + col, n, w);
      if (out && !first) ro_load8(out + col, n, p);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (!a.gy) continue;
        nv[i] *= r;
        p[i] = fmaf(g[i], nv[i], p[i]);
        g[i] = r * (g[i] * w[i] - nv[i] * mean);
      }
      if (out) ro_store8(out + col, n, p);
      if (a.gh) {
        float q[8];
        ro_load8(reinterpret_cast<const T*>(a.gh) + row * a.ldgh + col, n, q);
#pragma unroll
        for (int i = 0; i < 8; ++i) g[i] += q[i];
      }
      if (a.g_res) ro_store8(reinterpret_cast<T*>(a.g_res) + row * a.ldgr + col, n, g);
      if (a.g_x) {
        if (a.drop.limit) ro_drop8(fg + (col >> 3), offset, seed, a.drop.limit, a.drop.scale, g);
        ro_store8(reinterpret_cast<T*>(a.g_x) + row * a.ldgx + col, n, g);
      }
    }
  }
}

// out[c] = sum of `blocks` partial rows, in a fixed order: 32 columns x 32 row lanes a workgroup
__global__ __launch_bounds__(1024) void fold_rows_kernel(const float* __restrict__ part, int blocks, int cols, float* __restrict__ out) {
  __shared__ float s[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  float v = 0.f;
  if (c < cols)
#pragma unroll 4
    for (int b = threadIdx.y; b < blocks; b += 32) v += part[(long long)b * cols + c];
  s[threadIdx.y][threadIdx.x] = v;
  __syncthreads();
  float t = s[threadIdx.x][threadIdx.y];        // transposed: a wave's half adds up one column
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) t += __shfl_xor(t, o, 32);
  const int cc = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && cc < cols) out[cc] = t;
}

struct DropArgs {
  const void *x, *res;
  void* y;
  long long rows, ldx, ldr, ldy;
  int cols, groups, lanes;     // lanes: threads along a row, a power of two up to 256
  RoDrop drop;
};

template <typename T>
__global__ __launch_bounds__(256) void dropout_kernel(const DropArgs a) {
  const int lane = threadIdx.x & (a.lanes - 1), per = 256 / a.lanes;
  unsigned long long seed = a.drop.seed, offset = a.drop.offset;
  if (a.drop.dev) { seed = a.drop.dev[0]; offset += a.drop.dev[1]; }
  const long long step = (long long)gridDim.x * per;
  for (long long row = (long long)blockIdx.x * per + threadIdx.x / a.lanes; row < a.rows; row += step) {
    const unsigned long long fg = ro_flag_group(a.drop, row, a.groups);
    for (int g = lane; g < a.groups; g += a.lanes) {
      const int col = g * 8, n = a.cols - col;
      float v[8];
      ro_load8(reinterpret_cast<const T*>(a.x) + row * a.ldx + col, n, v);
      if (a.drop.limit) ro_drop8(fg + g, offset, seed, a.drop.limit, a.drop.scale, v);
      if (a.res) {
        float r[8];
        ro_load8(reinterpret_cast<const T*>(a.res) + row * a.ldr + col, n, r);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] += r[i];
      }
      ro_store8(reinterpret_cast<T*>(a.y) + row * a.ldy + col, n, v);
    }
  }
}

int pow2_at_least(int v, int most) {
  int p = 1;
  while (p < v && p < most) p <<= 1;
  return p;
}

// threads that hold a row and chunks of eight channels each: the fewest lanes that leave CH small
bool row_shape(int cols, int& lanes, int& ch) {
  const int groups = (cols + 7) / 8;
  if (groups <= 64) { lanes = pow2_at_least(groups, 64); ch = 1; return true; }
  if (groups <= 256) { lanes = 64; ch = groups <= 128 ? 2 : 4; return true; }
  if (groups <= 2048) { lanes = 256; ch = groups <= 512 ? 2 : (groups <= 1024 ? 4 : 8); return true; }
  return false;
}

int grid_of(long long rows, int per, int most) {
  const long long b = (rows + per - 1) / per;
  return (int)(b < most ? b : most);
}

// workgroups of the backward pass, a function of the shape alone (the workspace holds a row of partial sums for each): as many as there is
// work for up to 1024 (20000 x 4096 bf16: 107 us; 512 156, 2048 116), but over 256 at least eight rows each, so that the partial sums stay
// under a sixteenth of what is read and written
int back_blocks(long long rows, int cols) {
  int lanes = 256, ch = 0;
  const bool fits = row_shape(cols, lanes, ch);
  const int per = fits ? 256 / lanes : 1;
  long long b = (rows + per - 1) / per;
  if (b > 256) {
    const long long most = rows / 8 > 256 ? rows / 8 : 256;
    b = b < most ? b : most;
  }
  return (int)(b > 1024 ? 1024 : b);
}

template <typename T, int FMT>
int launch_norm(const NormArgs& a, hipStream_t s) {
  int lanes, ch;
  if (!row_shape(a.cols, lanes, ch)) {
    norm_long_kernel<T, FMT><<<grid_of(a.rows, 1, 2048), 256, 0, s>>>(a);
    UNCL_CHECK_LAUNCH();
    return UNCL_OK;
  }
  const int grid = grid_of(a.rows, 256 / lanes, 2048);
#define GO(L, C) norm_kernel<T, L, C, FMT><<<grid, 256, 0, s>>>(a)
  switch (lanes) {
    case 1: GO(1, 1); break;
    case 2: GO(2, 1); break;
    case 4: GO(4, 1); break;
    case 8: GO(8, 1); break;
    case 16: GO(16, 1); break;
    case 32: GO(32, 1); break;
    case 64: if (ch == 1) GO(64, 1); else if (ch == 2) GO(64, 2); else GO(64, 4); break;
    default: if (ch == 2) GO(256, 2); else if (ch == 4) GO(256, 4); else GO(256, 8); break;
  }
#undef GO
  UNCL_CHECK_LAUNCH();
  return UNCL_OK;
}

template <typename T>
int launch_norm_back(const NormBackArgs& a, int grid, hipStream_t s) {
  int lanes, ch;
  if (!row_shape(a.cols, lanes, ch)) {
    norm_back_long_kernel<T><<<grid, 256, 0, s>>>(a);
    UNCL_CHECK_LAUNCH();
    return UNCL_OK;
  }
#define GO(L, C) norm_back_kernel<T, L, C><<<grid, 256, 0, s>>>(a)
  switch (lanes) {
    case 1: GO(1, 1); break;
    case 2: GO(2, 1); break;
    case 4: GO(4, 1); break;
    case 8: GO(8, 1); break;
    case 16: GO(16, 1); break;
    case 32: GO(32, 1); break;
    case 64: if (ch == 1) GO(64, 1); else if (ch == 2) GO(64, 2); else GO(64, 4); break;
    default: if (ch == 2) GO(256, 2); else if (ch == 4) GO(256, 4); else GO(256, 8); break;
  }
#undef GO
  UNCL_CHECK_LAUNCH();
  return UNCL_OK;
}

bool dtype_ok(int d) { return d == UNCL_F32 || uncl_is_h16(d); }

// columns step in int by up to 2048 behind the last one, flag groups (rows * cols / 8) in 64 bits
bool extent_ok(long long rows, int cols) { return rows >= 0 && rows <= (1ll << 32) && cols >= 0 && cols <= (1 << 30); }
bool drop_ok(float p, long long span) { return p >= 0.f && p <= 1.f && span >= 1; }

}  // namespace

int ro_fold_rows(const float* part, int blocks, int cols, float* out, hipStream_t s) {
  fold_rows_kernel<<<dim3((cols + 31) / 32), dim3(32, 32), 0, s>>>(part, blocks, cols, out);
  UNCL_CHECK_LAUNCH();
  return UNCL_OK;
}

extern "C" int uncl_dropout(const void* x, long long ldx, const void* res, long long ldr, void* y, long long ldy, int dtype, long long rows,
                            int cols, float p, long long span, const unsigned long long* seed_dev, unsigned long long seed,
                            unsigned long long offset, void* stream) {
  if (!dtype_ok(dtype) || !extent_ok(rows, cols)) return UNCL_ERR_ARG;
  if (rows == 0 || cols == 0) return UNCL_OK;
  if (!x || !y || !drop_ok(p, span) || ldx < cols || ldy < cols || (res && ldr < cols)) return UNCL_ERR_ARG;
  DropArgs a{x, res, y, rows, ldx, ldr, ldy, cols, (cols + 7) / 8, 0, {seed_dev, seed, offset, span, 0, 1.f}};
  ro_drop_setup(a.drop, p);
  a.lanes = pow2_at_least(a.groups, 256);
  const int grid = grid_of(rows, 256 / a.lanes, 8192);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (dtype == UNCL_F32) dropout_kernel<float><<<grid, 256, 0, s>>>(a);
  else if (dtype == UNCL_BF16) dropout_kernel<bf16_t><<<grid, 256, 0, s>>>(a);
  else dropout_kernel<f16_t><<<grid, 256, 0, s>>>(a);
  UNCL_CHECK_LAUNCH();
  return UNCL_OK;
}

extern "C" int uncl_rmsnorm(const uncl_rmsnorm_desc* d, void* stream) {
  if (!d || !dtype_ok(d->dtype) || !extent_ok(d->rows, d->cols)) return UNCL_ERR_ARG;
  if (d->rows == 0 || d->cols == 0) return UNCL_OK;
  const int fmt = d->y_fmt;
  if (fmt != UNCL_Q8_NONE && fmt != UNCL_E4M3 && fmt != UNCL_E5M2) return UNCL_ERR_ARG;
  if (!d->x || !d->y || !(d->eps > 0.f) || d->ldx < d->cols || d->ldy < d->cols || (d->res && d->ldr < d->cols) || (d->h && d->ldh < d->cols))
    return UNCL_ERR_ARG;
  if (!drop_ok(d->p, d->span) || (fmt != UNCL_Q8_NONE && !d->y_scale)) return UNCL_ERR_ARG;
  NormArgs a{};
  a.x = d->x; a.res = d->res; a.w = d->weight; a.h = d->h; a.y = d->y; a.rstd = d->rstd; a.scale = d->y_scale;
  a.rows = d->rows; a.ldx = d->ldx; a.ldr = d->ldr; a.ldh = d->ldh; a.ldy = d->ldy; a.ss_row = d->scale_row; a.ss_blk = d->scale_block;
  a.cols = d->cols; a.groups = (d->cols + 7) / 8; a.eps = d->eps; a.inv_cols = 1.f / (float)d->cols;
  a.drop = {d->seed_dev, d->seed, d->offset, d->span, 0, 1.f};
  ro_drop_setup(a.drop, d->p);
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define BY_TYPE(F) (d->dtype == UNCL_F32 ? launch_norm<float, F>(a, s) : d->dtype == UNCL_BF16 ? launch_norm<bf16_t, F>(a, s) : launch_norm<f16_t, F>(a, s))
  if (fmt == UNCL_Q8_NONE) return BY_TYPE(UNCL_Q8_NONE);
  if (fmt == UNCL_E4M3) return BY_TYPE(UNCL_E4M3);
  return BY_TYPE(UNCL_E5M2);
#undef BY_TYPE
}

extern "C" size_t uncl_rmsnorm_backward_workspace_bytes(long long rows, int cols) {
  if (rows <= 0 || cols <= 0) return 0;
  return (size_t)back_blocks(rows, cols) * cols * sizeof(float);
}

extern "C" int uncl_rmsnorm_backward(const uncl_rmsnorm_bwd_desc* d, void* workspace, void* stream) {
  if (!d || !dtype_ok(d->dtype) || !extent_ok(d->rows, d->cols)) return UNCL_ERR_ARG;
  if (d->cols == 0) return UNCL_OK;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (d->rows == 0) {
    return d->g_w ? ro_fold_rows(nullptr, 0, d->cols, d->g_w, s) : UNCL_OK;
  }
  if (!d->h || !d->rstd || d->ldh < d->cols || (d->gy && d->ldgy < d->cols) || (d->gh && d->ldgh < d->cols) ||
      (d->g_res && d->ldgr < d->cols) || (d->g_x && d->ldgx < d->cols) || (d->g_w && !workspace) || !drop_ok(d->p, d->span))
    return UNCL_ERR_ARG;
  NormBackArgs a{};
  a.gy = d->gy; a.gh = d->gh; a.h = d->h; a.w = d->weight; a.rstd = d->rstd; a.g_res = d->g_res; a.g_x = d->g_x;
  a.part = d->g_w ? reinterpret_cast<float*>(workspace) : nullptr;
  a.rows = d->rows; a.ldgy = d->ldgy; a.ldgh = d->ldgh; a.ldh = d->ldh; a.ldgr = d->ldgr; a.ldgx = d->ldgx;
  a.cols = d->cols; a.groups = (d->cols + 7) / 8; a.inv_cols = 1.f / (float)d->cols;
  a.drop = {d->seed_dev, d->seed, d->offset, d->span, 0, 1.f};
  ro_drop_setup(a.drop, d->p);
  const int grid = back_blocks(d->rows, d->cols);
  const int rc = d->dtype == UNCL_F32 ? launch_norm_back<float>(a, grid, s)
                                      : d->dtype == UNCL_BF16 ? launch_norm_back<bf16_t>(a, grid, s) : launch_norm_back<f16_t>(a, grid, s);
  if (rc != UNCL_OK) return rc;
  return d->g_w ? ro_fold_rows(a.part, grid, d->cols, d->g_w, s) : UNCL_OK;
}
