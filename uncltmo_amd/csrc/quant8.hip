// Quantisers of the 8-bit matrix product: blocks of 1 x 128 (activations, gradients) or 128 x 128 (weights), one fp32 scale a block, from
// fp32 / bf16 / fp16 matrices, as they lie or transposed (the operands of a linear layer's two gradients have the other axis inside).
//
//   scale = max(amax, 2^-100) fl(1 / top),   q = round_even(x fl(1 / scale))
//
// One pass: a block is read once, its maximum found in registers (and LDS), and written in 8 bits: bound by HBM, 2 (or 4) + 1 bytes an
// element.  By rows, bf16: 28800 x 256 7.4 us = 3.0 TB/s, 8192 x 4096 20.3 us = 5.0 TB/s.  Tiles: 4099 x 2048 8.6 us = 2.9 TB/s; transposed rows
// 10.6 us, transposed tiles of 4099 x 4096 14.0 us = 3.6 TB/s.  Both ways from one read (1 + 1 bytes written): 4099 x 2048 15.5 us = 2.2 TB/s, with
// the columns' sums 4099 x 4096 24.8 us = 2.7 TB/s -- 528 and 1056 workgroups of one tile each, whose read, maxima, conversion and writes
// follow one another at the same time on every CU: the short grids leave little of another tile's traffic to fill the gaps.
#include "matmul8_args.h"
#include "row_ops.h"

namespace {

struct QuantArgs {
  const void* x;
  unsigned char* q;
  float* scale;
  long long rows, ldx, ldq, ss_row, ss_blk;
  int cols;
  bool lost;                             // infinities become NaN, not the largest number
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
    float v[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = 0.f;
    if (n > 0) ro_load8(reinterpret_cast<const T*>(a.x) + row * a.ldx + col, n, v);
    bool odd;
    const unsigned m = ro_max_lanes<16>(ro_size8(v, odd));
    const float s = ro_scale_of<FMT>(m), inv = 1.f / s;
    if (n <= 0) continue;
    ro_store8q(a.q + row * a.ldq + col, n, ro_pack8<FMT>(v, inv, odd, a.lost));
    if (lane == 0) a.scale[row * a.ss_row + kb * a.ss_blk] = s;
  }
}

// One workgroup, one 128 x 128 tile of x, an 8 x 8 patch a thread, read once.  TILE: one scale for the tile, else one for each row's 128
// (q) and one for each column's 128 (its transpose).  WAYS: 1 = q as x lies, 2 = transposed, 3 = both; SUMS: the columns' sums too (the bias
// gradient of a linear layer whose output gradient this is), as partial sums [tiles of rows][cols].  The bytes of the transpose turn
// round in LDS: rows of 132 bytes put the eight lanes that write at once eight banks apart (384 cycles of conflicts are left in a workgroup).
// eight neighbours of a row as they lie in memory; their sizes (bits without the sign) compare as integers of the type's own width, two at a
// time for the 16-bit types
template <typename T>
struct Bits {
  typedef unsigned short U;
};
template <>
struct Bits<float> {
  typedef unsigned U;
};
template <typename T>
struct Eight {
  typedef typename Bits<T>::U U;
  typedef U U8 __attribute__((ext_vector_type(8)));
  static constexpr U sign = (U)1 << (8 * sizeof(U) - 1);
  static constexpr U inf = sizeof(U) == 4 ? (U)RO_INF_BITS : (U)(__is_same(T, bf16_t) ? 0x7f80 : 0x7c00);
  U8 raw;
  __device__ __forceinline__ void load(const T* p, int n) {
    if (n >= 8) {
      __builtin_memcpy(&raw, p, sizeof(raw));
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) raw[j] = j < n ? __builtin_bit_cast(U, p[j]) : (U)0;
    }
  }
  __device__ __forceinline__ float value(int j) const {
    const U u = raw[j];
    return (float)__builtin_bit_cast(T, u);
  }
  template <bool ODD>
  __device__ __forceinline__ U8 sizes() const {
    U8 s = raw & (U)(sign - 1);
    if constexpr (ODD)
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] = s[j] >= inf ? (U)0 : s[j];
    return s;
  }
  static __device__ __forceinline__ unsigned fp32_bits(U u) { return __builtin_bit_cast(unsigned, (float)__builtin_bit_cast(T, u)); }
};

// largest sizes of an 8 x 8 patch by row and by column
template <typename T, bool ODD>
__device__ __forceinline__ void patch_sizes(const Eight<T> (&v)[8], typename Eight<T>::U (&by_row)[8], typename Eight<T>::U8& by_col) {
  typedef typename Eight<T>::U U;
  typedef U U4 __attribute__((ext_vector_type(4)));
  typedef U U2 __attribute__((ext_vector_type(2)));
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const auto s = v[i].template sizes<ODD>();
    by_col = i == 0 ? s : __builtin_elementwise_max(by_col, s);
    const U4 t = __builtin_elementwise_max(s.lo, s.hi);
    const U2 u = __builtin_elementwise_max(t.lo, t.hi);
    by_row[i] = u[0] > u[1] ? u[0] : u[1];
  }
}

template <typename T, int FMT, bool TILE, int WAYS, bool SUMS>
__global__ __launch_bounds__(256, 2) void quant_tile_kernel(const QuantArgs a, const QuantArgs at, float* __restrict__ sums) {
  __shared__ unsigned red[SUMS || (!TILE && (WAYS & 2)) ? 16 * 128 : 4];      // sizes, and sums and inverses as their bits
  __shared__ __align__(16) unsigned char turn[(WAYS & 2) ? 128 * 132 : 16];
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const long long row0 = (long long)blockIdx.y * 128;
  const int col0 = blockIdx.x * 128, col = col0 + tx * 8;
  Eight<T> v[8];
  const T* from = reinterpret_cast<const T*>(a.x) + (row0 + ty * 8) * a.ldx + col;
  if (row0 + 128 <= a.rows && col0 + 128 <= a.cols) {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i].load(from + i * a.ldx, 8);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i].load(from + i * a.ldx, row0 + ty * 8 + i < a.rows ? a.cols - col : 0);
  }
  typename Eight<T>::U by_row[8], all = 0;
  typename Eight<T>::U8 by_col;
  patch_sizes<T, false>(v, by_row, by_col);
#pragma unroll
  for (int i = 0; i < 8; ++i) all = by_row[i] > all ? by_row[i] : all;
  const bool odd = all >= Eight<T>::inf;
  if (odd) {
    patch_sizes<T, true>(v, by_row, by_col);
    all = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) all = by_row[i] > all ? by_row[i] : all;
  }
  if constexpr (SUMS) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float t = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) t += v[i].value(j);
      red[ty * 128 + tx * 8 + j] = __builtin_bit_cast(unsigned, t);
    }
    __syncthreads();
    if (threadIdx.x < 128 && col0 + (int)threadIdx.x < a.cols) {
      float t = 0.f;
#pragma unroll
      for (int k = 0; k < 16; ++k) t += __builtin_bit_cast(float, red[k * 128 + threadIdx.x]);
      sums[(long long)blockIdx.y * a.cols + col0 + threadIdx.x] = t;
    }
    __syncthreads();
  }
  float inv[8], inv_col[8];
  if constexpr (TILE) {
    unsigned m = Eight<T>::fp32_bits(all);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) m = ro_max(m, (unsigned)__shfl_xor((int)m, o, 64));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = m;
    __syncthreads();
    const float s = ro_scale_of<FMT>(ro_max(ro_max(red[0], red[1]), ro_max(red[2], red[3])));
    const float t = 1.f / s;
    if (threadIdx.x == 0) {
      if (WAYS & 1) a.scale[blockIdx.y * a.ss_row + blockIdx.x * a.ss_blk] = s;
      if (WAYS & 2) at.scale[blockIdx.x * at.ss_row + blockIdx.y * at.ss_blk] = s;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) inv[j] = inv_col[j] = t;
  } else if constexpr ((WAYS & 2) != 0) {
#pragma unroll
    for (int j = 0; j < 8; ++j) red[ty * 128 + tx * 8 + j] = Eight<T>::fp32_bits(by_col[j]);
    __syncthreads();
    if (threadIdx.x < 128) {                    // one thread a column: its maximum, scale and inverse
      unsigned m = 0;
#pragma unroll
      for (int k = 0; k < 16; ++k) m = ro_max(m, red[k * 128 + threadIdx.x]);
      const float s = ro_scale_of<FMT>(m);
      if (col0 + (int)threadIdx.x < a.cols) at.scale[(long long)(col0 + threadIdx.x) * at.ss_row + blockIdx.y * at.ss_blk] = s;
      red[threadIdx.x] = __builtin_bit_cast(unsigned, 1.f / s);
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < 8; ++j) inv_col[j] = __builtin_bit_cast(float, red[tx * 8 + j]);
  }
  if constexpr (!TILE && (WAYS & 1) != 0)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float s = ro_scale_of<FMT>(ro_max_lanes<16>(Eight<T>::fp32_bits(by_row[i])));
      inv[i] = 1.f / s;
      if (tx == 0 && row0 + ty * 8 + i < a.rows) a.scale[(row0 + ty * 8 + i) * a.ss_row + blockIdx.x * a.ss_blk] = s;
    }
  if constexpr ((WAYS & 2) != 0) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float f[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = v[i].value(j);
      const u32x2 b = ro_pack8<FMT>(f, inv_col[j], odd, a.lost);
      unsigned* to = reinterpret_cast<unsigned*>(&turn[(tx * 8 + j) * 132 + ty * 8]);
      to[0] = b[0];
      to[1] = b[1];
    }
  }
  if constexpr ((WAYS & 1) != 0) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const long long row = row0 + ty * 8 + i;
      float f[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) f[j] = v[i].value(j);
      if (row < a.rows && col < a.cols) ro_store8q(a.q + row * a.ldq + col, a.cols - col, ro_pack8<FMT>(f, inv[i], odd, a.lost));
    }
  }
  if constexpr ((WAYS & 2) != 0) {
    __syncthreads();
    const long long n = a.rows - (row0 + tx * 8);
    if (n > 0)
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int c = ty + 16 * i;
        if (col0 + c >= a.cols) break;
        const unsigned* b = reinterpret_cast<const unsigned*>(&turn[c * 132 + tx * 8]);
        ro_store8q(at.q + (long long)(col0 + c) * at.ldq + row0 + tx * 8, n < 8 ? (int)n : 8, u32x2{b[0], b[1]});
      }
  }
}

template <typename T, int FMT, bool TILE, int WAYS, bool SUMS = false>
int launch_tiles(const QuantArgs& a, const QuantArgs& at, float* sums, hipStream_t s) {
  const dim3 grid((a.cols + 127) / 128, (unsigned)((a.rows + 127) / 128));
  quant_tile_kernel<T, FMT, TILE, WAYS, SUMS><<<grid, 256, 0, s>>>(a, at, sums);
  UNCL_CHECK_LAUNCH();
  return UNCL_OK;
}

template <typename T, int FMT>
int launch_quant(const QuantArgs& a, int tile, int trans, hipStream_t s) {
  if (tile) return trans ? launch_tiles<T, FMT, true, 2>(a, a, nullptr, s) : launch_tiles<T, FMT, true, 1>(a, a, nullptr, s);
  if (trans) return launch_tiles<T, FMT, false, 2>(a, a, nullptr, s);
  const long long total = (a.rows * ((a.cols + 127) >> 7) + 15) / 16;
  quant_rows_kernel<T, FMT><<<(int)(total < 4096 ? total : 4096), 256, 0, s>>>(a);
  UNCL_CHECK_LAUNCH();
  return UNCL_OK;
}

}  // namespace

extern "C" int uncl_quant8(const void* x, int dtype, long long rows, int cols, long long ldx, void* q, long long ldq, int fmt, float* scale,
                           long long scale_row, long long scale_block, int tile, int transposed, void* stream) {
  if (!(dtype == UNCL_F32 || uncl_is_h16(dtype)) || (fmt != UNCL_E4M3 && fmt != UNCL_E5M2) || rows < 0 || rows > (1ll << 32) || cols < 0 || cols > (1 << 30)) return UNCL_ERR_ARG;
  if (rows == 0 || cols == 0) return UNCL_OK;
  if (!x || !q || !scale || ldx < cols || ldq < (transposed ? rows : cols)) return UNCL_ERR_ARG;
  if ((tile || transposed) && (rows + 127) / 128 > 65535) return UNCL_ERR_ARG;      // one workgroup a tile, rows along the grid's y
  const QuantArgs a{x, reinterpret_cast<unsigned char*>(q), scale, rows, ldx, ldq, scale_row, scale_block, cols, false};
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define BY_TYPE(F)                                                                                          \
  (dtype == UNCL_F32 ? launch_quant<float, F>(a, tile, transposed, s)                                       \
                     : dtype == UNCL_BF16 ? launch_quant<bf16_t, F>(a, tile, transposed, s) : launch_quant<f16_t, F>(a, tile, transposed, s))
  return fmt == UNCL_E4M3 ? BY_TYPE(UNCL_E4M3) : BY_TYPE(UNCL_E5M2);
#undef BY_TYPE
}

// ---- the linear layer of a training step -----------------------------------------------------------------------------------------------
// y = x w^T + b, gx = gy w, gw = gy^T x with 8-bit operands.  x and w are read once in the forward pass, for its own product (x by rows, w
// by tiles) and, where gradients are wanted, for theirs (both transposed: a quarter to a half of the bytes that keeping x and w would
// take); gy is read once in the backward pass for both products and the bias.  An infinity is quantised to NaN: as the largest number of its
// block it would make finite results of a step that has overflowed, and a loss scale that looks for such steps would miss it.
namespace {

struct LinearPlan {                      // the operands' places in one buffer, 256-byte aligned
  size_t xq, xs, wq, ws, xt, xts, wt, wts, gq, gs, gt, gts, sums, split_y, split_gx, split_gw;
};
size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }
// rows of operands begin on lines of memory: a block of 128 across two of them is two requests for the product and half-written lines here
// (4099 rows of 2048 transposed: pitch 4112 or 4224)
long long pitch128(long long v) { return (v + 127) & ~127ll; }
long long blocks128(long long v) { return (v + 127) >> 7; }

// what the backward pass needs from the forward one: x and w transposed
size_t plan_saved(long long M, int N, int K, bool x, bool w, LinearPlan& p) {
  size_t at = 0;
  auto put = [&](size_t& f, size_t bytes, bool want) { f = at; at += want ? up256(bytes) : 0; };
  put(p.xt, (size_t)K * pitch128(M), x);
  put(p.xts, (size_t)blocks128(M) * K * 4, x);
  put(p.wt, (size_t)K * pitch128(N), w);
  put(p.wts, (size_t)blocks128(K) * blocks128(N) * 4, w);
  return at;
}
size_t plan_forward(long long M, int N, int K, LinearPlan& p) {
  size_t at = 0;
  auto put = [&](size_t& f, size_t bytes) { f = at; at += up256(bytes); };
  put(p.xq, (size_t)M * pitch128(K));
  put(p.xs, (size_t)blocks128(K) * M * 4);
  put(p.wq, (size_t)N * pitch128(K));
  put(p.ws, (size_t)blocks128(N) * blocks128(K) * 4);
  put(p.split_y, mm_split_bytes((int)M, N, K));
  return at;
}
size_t plan_backward(long long M, int N, int K, LinearPlan& p) {
  size_t at = 0;
  auto put = [&](size_t& f, size_t bytes) { f = at; at += up256(bytes); };
  put(p.gq, (size_t)M * pitch128(N));
  put(p.gs, (size_t)blocks128(N) * M * 4);
  put(p.gt, (size_t)N * pitch128(M));
  put(p.gts, (size_t)blocks128(M) * N * 4);
  put(p.sums, (size_t)blocks128(M) * N * 4);
  put(p.split_gx, mm_split_bytes((int)M, K, N));
  put(p.split_gw, mm_split_bytes(N, K, (int)M));
  return at;
}

bool linear_ok(const uncl_linear8_desc* d) {
  if (!d || d->M < 0 || d->N <= 0 || d->K <= 0 || d->M > (1 << 22) || d->N > (1 << 22) || d->K > (1 << 22)) return false;      // each is a product's K
  const bool x = d->dtype == UNCL_F32 || uncl_is_h16(d->dtype), w = d->w_dtype == UNCL_F32 || uncl_is_h16(d->w_dtype);
  return x && w && (d->grad_fmt == UNCL_E4M3 || d->grad_fmt == UNCL_E5M2);
}
QuantArgs quant_args(const void* x, long long rows, int cols, long long ldx, char* q, long long ldq, char* scale, long long row, long long blk) {
  return {x, reinterpret_cast<unsigned char*>(q), reinterpret_cast<float*>(scale), rows, ldx, ldq, row, blk, cols, true};
}

// x by rows and (t) by its columns' 128s; w by tiles, as it lies and (t) transposed; gy both ways and its columns' sums
template <typename T>
int quant_x(const QuantArgs& a, const QuantArgs& t, bool both, hipStream_t s) {
  return both ? launch_tiles<T, UNCL_E4M3, false, 3>(a, t, nullptr, s) : launch_quant<T, UNCL_E4M3>(a, 0, 0, s);
}
template <typename T>
int quant_w(const QuantArgs& a, const QuantArgs& t, bool both, hipStream_t s) {
  return both ? launch_tiles<T, UNCL_E4M3, true, 3>(a, t, nullptr, s) : launch_tiles<T, UNCL_E4M3, true, 1>(a, t, nullptr, s);
}
template <typename T>
int quant_g(const QuantArgs& a, const QuantArgs& t, int fmt, bool both, float* sums, hipStream_t s) {
  if (!both) return fmt == UNCL_E4M3 ? launch_tiles<T, UNCL_E4M3, false, 1, true>(a, t, sums, s) : launch_tiles<T, UNCL_E5M2, false, 1, true>(a, t, sums, s);
  return fmt == UNCL_E4M3 ? launch_tiles<T, UNCL_E4M3, false, 3, true>(a, t, sums, s) : launch_tiles<T, UNCL_E5M2, false, 3, true>(a, t, sums, s);
}
#define LIN_BY_TYPE(DT, F, ...) ((DT) == UNCL_F32 ? F<float>(__VA_ARGS__) : (DT) == UNCL_BF16 ? F<bf16_t>(__VA_ARGS__) : F<f16_t>(__VA_ARGS__))

MmArgs product(const char* a, long long lda, const char* sa, const char* b, long long ldb, const char* sb, long long sb_row, long long sb_blk, int M, int N, int K,
               void* out, long long ldo, int dtype) {
  MmArgs p{};
  p.a = reinterpret_cast<const unsigned char*>(a);
  p.b = reinterpret_cast<const unsigned char*>(b);
  p.sa = reinterpret_cast<const float*>(sa);
  p.sb = reinterpret_cast<const float*>(sb);
  p.lda = lda; p.ldb = ldb; p.sa_row = 1; p.sa_blk = M; p.sb_row = sb_row; p.sb_blk = sb_blk;
  p.M = M; p.N = N; p.K = K; p.out = out; p.ldo = ldo; p.out_dtype = dtype;
  return p;
}

}  // namespace

extern "C" size_t uncl_linear8_saved_bytes(long long M, int N, int K, int for_x, int for_w) {
  LinearPlan p;
  return M > 0 && N > 0 && K > 0 ? plan_saved(M, N, K, for_w != 0, for_x != 0, p) : 0;
}
extern "C" size_t uncl_linear8_workspace_bytes(long long M, int N, int K, int backward) {
  LinearPlan p;
  return M > 0 && N > 0 && K > 0 && M <= (1 << 22) ? (backward ? plan_backward(M, N, K, p) : plan_forward(M, N, K, p)) : 0;
}

extern "C" int uncl_linear8_forward(const uncl_linear8_desc* d, void* saved, void* workspace, void* stream) {
  if (!linear_ok(d)) return UNCL_ERR_ARG;
  if (d->M == 0) return UNCL_OK;
  if (!d->x || !d->w || !d->y || !workspace || d->ldx < d->K || d->ldw < d->K || d->ldy < d->N || ((d->for_x || d->for_w) && !saved)) return UNCL_ERR_ARG;
  const int M = d->M, N = d->N, K = d->K;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  LinearPlan p{};
  plan_saved(M, N, K, d->for_w, d->for_x, p);
  plan_forward(M, N, K, p);
  char *ws = reinterpret_cast<char*>(workspace), *sv = reinterpret_cast<char*>(saved);
  const QuantArgs x = quant_args(d->x, M, K, d->ldx, ws + p.xq, pitch128(K), ws + p.xs, 1, M);
  const QuantArgs xt = quant_args(d->x, M, K, d->ldx, sv + p.xt, pitch128(M), sv + p.xts, 1, K);
  const QuantArgs w = quant_args(d->w, N, K, d->ldw, ws + p.wq, pitch128(K), ws + p.ws, blocks128(K), 1);
  const QuantArgs wt = quant_args(d->w, N, K, d->ldw, sv + p.wt, pitch128(N), sv + p.wts, blocks128(N), 1);
  int rc = LIN_BY_TYPE(d->dtype, quant_x, x, xt, d->for_w != 0, s);
  if (rc == UNCL_OK) rc = LIN_BY_TYPE(d->w_dtype, quant_w, w, wt, d->for_x != 0, s);
  if (rc != UNCL_OK) return rc;
  MmArgs m = product(ws + p.xq, pitch128(K), ws + p.xs, ws + p.wq, pitch128(K), ws + p.ws, blocks128(K), 1, M, N, K, d->y, d->ldy, d->dtype);
  m.bias = d->bias;
  return mm_run(m, UNCL_E4M3, true, ws + p.split_y, s);
}

extern "C" int uncl_linear8_backward(const uncl_linear8_desc* d, const void* saved, void* workspace, void* stream) {
  if (!linear_ok(d)) return UNCL_ERR_ARG;
  if (d->M == 0) return UNCL_OK;
  if (!d->gy || !workspace || d->ldgy < d->N || ((d->gx || d->gw) && !saved) || (d->gx && (d->ldgx < d->K || !d->for_x)) || (d->gw && (d->ldgw < d->K || !d->for_w)))
    return UNCL_ERR_ARG;
  const int M = d->M, N = d->N, K = d->K;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  LinearPlan p{};
  plan_saved(M, N, K, d->for_w, d->for_x, p);
  plan_backward(M, N, K, p);
  char* ws = reinterpret_cast<char*>(workspace);
  const char* sv = reinterpret_cast<const char*>(saved);
  const QuantArgs g = quant_args(d->gy, M, N, d->ldgy, ws + p.gq, pitch128(N), ws + p.gs, 1, M);
  const QuantArgs gt = quant_args(d->gy, M, N, d->ldgy, ws + p.gt, pitch128(M), ws + p.gts, 1, N);
  float* sums = reinterpret_cast<float*>(ws + p.sums);
  int rc = LIN_BY_TYPE(d->dtype, quant_g, g, gt, d->grad_fmt, d->gw != nullptr, sums, s);
  if (rc == UNCL_OK && d->gx)
    rc = mm_run(product(ws + p.gq, pitch128(N), ws + p.gs, sv + p.wt, pitch128(N), sv + p.wts, blocks128(N), 1, M, K, N, d->gx, d->ldgx, d->dtype), d->grad_fmt,
                true, ws + p.split_gx, s);
  if (rc == UNCL_OK && d->gw)
    rc = mm_run(product(ws + p.gt, pitch128(M), ws + p.gts, sv + p.xt, pitch128(M), sv + p.xts, 1, K, N, K, M, d->gw, d->ldgw, d->w_dtype), d->grad_fmt, false,
                ws + p.split_gw, s);
  if (rc == UNCL_OK && d->gb) rc = ro_fold_rows(sums, (int)blocks128(M), N, d->gb, s);
  return rc;
}
