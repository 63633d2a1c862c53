// Matrix product of 8-bit operands: few rows, and the choice of a kernel (the tiles: matmul8.h).
#include "matmul8.h"

namespace {

// scale of the four columns n .. n + 3 (b scaled by rows) in block kb
__device__ __forceinline__ f32x4 mm_sb4(const MmArgs& p, int n, int kb) {
  f32x4 s;
#pragma unroll
  for (int i = 0; i < 4; ++i) s[i] = p.sb[(n + i < p.N ? n + i : p.N - 1) + kb * p.sb_blk];
  return s;
}

// columns n .. n + 3 of row m in the output's type
template <typename T>
__device__ __forceinline__ void mm_store4(const MmArgs& p, long long m, int n, f32x4 x) {
  const int left = p.N - n;
  if (left <= 0) return;
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = x[i] + (p.bias && i < left ? p.bias[n + i] : 0.f);
  mm_act<4>(v, p.act);
  T* out = reinterpret_cast<T*>(p.out) + m * p.ldo + n;
  const T* res = reinterpret_cast<const T*>(p.res) + m * p.ldr + n;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < left) out[i] = (T)(v[i] + (p.res ? (float)res[i] : 0.f));
}

// ---- few rows ------------------------------------------------------------------------------------------------------------------------
// Up to 64 rows: b is read once and is nearly all there is to read (so the sums are the exact ones for every type).  A workgroup owns 16
// columns, its WAVES waves take the blocks of K in turn, operands come straight from global memory into registers, and the waves' sums
// join in LDS in a fixed order.  1 x 4096 x 4096: 8.0 us, where 17 MB at the copy rate are 3.3: 256 workgroups, one a CU, eight waves with one
// block each in flight -- four blocks a wave, so a chain of four round trips to memory, the join and the launch.
template <int FA, bool BT, int TM, int WAVES>
__global__ __launch_bounds__(WAVES * 64) void mm_rows_kernel(const MmArgs p) {
  __shared__ f32x4 red[WAVES][TM][64];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, q = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16, nr = n0 + q < p.N ? n0 + q : p.N - 1;
  const unsigned char* gb = p.b + (long long)nr * p.ldb;
  const unsigned char* ga[TM];
  const float* sa[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = i * 16 + q < p.M ? i * 16 + q : p.M - 1;
    ga[i] = p.a + (long long)m * p.lda;
    sa[i] = p.sa + (long long)m * p.sa_row;
  }
  const int last = (p.K - 1) & ~15;
  f32x4 acc[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  for (int kb = wave; kb < p.KB; kb += WAVES) {
    const int c0 = kb * 128 + g * 16, c1 = c0 + 64;
    const int r0 = c0 < last ? c0 : last, r1 = c1 < last ? c1 : last;
    auto frag = [&](const unsigned char* row) {
      i32x4 lo = *reinterpret_cast<const i32x4*>(row + r0), hi = *reinterpret_cast<const i32x4*>(row + r1);
      if (kb * 128 + 128 > p.K) {                            // clear what lies behind K, byte by byte
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const int k0 = p.K - (c0 + w * 4), k1 = p.K - (c1 + w * 4);
          lo[w] = k0 >= 4 ? lo[w] : (k0 <= 0 ? 0 : lo[w] & ((1 << (8 * k0)) - 1));
          hi[w] = k1 >= 4 ? hi[w] : (k1 <= 0 ? 0 : hi[w] & ((1 << (8 * k1)) - 1));
        }
      }
      return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };
    const Wide fb[1] = {mm_widen<UNCL_E4M3>(frag(gb))};
    float t = 1.f;
    f32x4 sn = {1.f, 1.f, 1.f, 1.f};
    if constexpr (BT) t = p.sb[(long long)(n0 >> 7) * p.sb_row + kb * p.sb_blk];
    else sn = mm_sb4(p, n0 + g * 4, kb);
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const float s = sa[i][(long long)kb * p.sa_blk] * t;
      f32x4 d[1];
      mm_block<FA, 1>(fb, mm_widen<FA>(frag(ga[i])), d);
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][e] = fmaf(d[0][e], BT ? s : s * sn[e], acc[i][e]);
    }
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) red[wave][i][lane] = acc[i];
  __syncthreads();
  for (int i = wave; i < TM; i += WAVES) {
    f32x4 v = red[0][i][lane];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) v += red[w][i][lane];
    if (i * 16 + q >= p.M) continue;
    if (p.out_dtype == UNCL_BF16) mm_store4<bf16_t>(p, i * 16 + q, n0 + g * 4, v);
    else if (p.out_dtype == UNCL_F16) mm_store4<f16_t>(p, i * 16 + q, n0 + g * 4, v);
    else mm_store4<float>(p, i * 16 + q, n0 + g * 4, v);
  }
}

// a grid's axis holds under 2^32 threads (2^27 columns, sixteen to a workgroup of 512; more wrap round without an error): in parts
constexpr int ROWS_PART = 1 << 26;
template <int FA, bool BT>
int launch_rows(const MmArgs& args, hipStream_t s) {
  const int e = args.out_dtype == UNCL_F32 ? 4 : 2;
  for (int n = 0; n < args.N; n += ROWS_PART) {
    MmArgs p = args;
    p.N = args.N - n < ROWS_PART ? args.N - n : ROWS_PART;
    p.b += n * p.ldb;
    p.sb += BT ? (n >> 7) * p.sb_row : n;
    if (p.bias) p.bias += n;
    if (p.res) p.res = reinterpret_cast<const char*>(p.res) + (long long)n * e;
    p.out = reinterpret_cast<char*>(p.out) + (long long)n * e;
    const int grid = (p.N + 15) / 16;
    if (p.M <= 16) mm_rows_kernel<FA, BT, 1, 8><<<grid, 512, 0, s>>>(p);
    else if (p.M <= 32) mm_rows_kernel<FA, BT, 2, 8><<<grid, 512, 0, s>>>(p);
    else mm_rows_kernel<FA, BT, 4, 8><<<grid, 512, 0, s>>>(p);
    UNCL_CHECK_LAUNCH();
  }
  return UNCL_OK;
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

namespace {

int run_rows(const MmArgs& p, int a_fmt, bool tile, hipStream_t s) {
  if (a_fmt == UNCL_E4M3) return tile ? launch_rows<UNCL_E4M3, true>(p, s) : launch_rows<UNCL_E4M3, false>(p, s);
  return tile ? launch_rows<UNCL_E5M2, true>(p, s) : launch_rows<UNCL_E5M2, false>(p, s);
}

// Up to 64 rows behind the last whole 128 that would cost the tiles a round, or the larger tiles: they go to small tiles of their own, in a
// launch before the others.  (Not to the few rows' kernel, whose sums are the exact ones for every type: a row's result must not depend on its
// place.)  That launch took 2.6 us and 3.3 (bf16 results) to 4.5 ns a k for 256 to 16384 columns; a unit took 0.25 to 0.39 ns a k in its ten
// tenths (0.18 where the rest would change to smaller tiles: not then).  At once / apart, bf16 with b by tiles: 4099 x 4096 x 512 22.5 / 24.2,
// x 1024 32.1 / 29.3, x 2048 52.7 / 46.0; 8195 x 4096 x 4096 158 / 133; 4099 x 16384 x 1024 101 / 91; 8195 x 1024 x 2048 30.6 / 32.7; fp32:
// 4099 x 2048 x 1024 32.7 / 32.1, x 4096 94.8 / 86.8, 8195 x 4096 x 2048 149 / 148.
int ragged_rows(const MmArgs& p, bool large) {
  const int tail = p.M & 127;
  if (p.M <= 128 || tail == 0 || tail > 64 || p.part) return 0;
  const MmPlan all = mm_plan(p.M, p.N, p.KB, large), rest = mm_plan(p.M - tail, p.N, p.KB, large);
  const double rounds = (p.N + 65535ll) / 65536;              // of the small tiles, four to a CU
  return rest.tile >= all.tile && (double)(all.units - rest.units) * p.K * 0.26 > rounds * (2600. + 4. * p.K) ? tail : 0;
}

int run_tiles(const MmArgs& p, int a_fmt, bool tile, hipStream_t s) {
  if (p.out_dtype == UNCL_BF16) return mm_tiles_bf16(p, a_fmt, tile, s);
  return p.out_dtype == UNCL_F16 ? mm_tiles_f16(p, a_fmt, tile, s) : mm_tiles_f32(p, a_fmt, tile, s);
}

}  // namespace

int mm_run(const MmArgs& args, int a_fmt, bool tile, void* workspace, hipStream_t s) {
  MmArgs p = args;
  p.KB = (p.K + 127) / 128;
  if (p.M <= 64) return run_rows(p, a_fmt, tile, s);
  const int splits = workspace ? mm_splits(p.M, p.N, p.K) : 1;
  p.part = splits > 1 ? reinterpret_cast<float*>(workspace) : nullptr;
  p.per = (p.KB + splits - 1) / splits;
  if (const int tail = ragged_rows(p, tile && p.out_dtype == UNCL_BF16)) {
    MmArgs q = p;
    const long long at = p.M -= tail, e = p.out_dtype == UNCL_F32 ? 4 : 2;
    q.M = tail;
    q.a += at * p.lda;
    q.sa += at * p.sa_row;
    q.out = reinterpret_cast<char*>(p.out) + at * p.ldo * e;
    if (p.res) q.res = reinterpret_cast<const char*>(p.res) + at * p.ldr * e;
    const int rc = run_tiles(q, a_fmt, tile, s);
    if (rc != UNCL_OK) return rc;
  }
  return run_tiles(p, a_fmt, tile, s);
}

extern "C" size_t uncl_matmul8_workspace_bytes(int M, int N, int K) { return M > 0 && N > 0 && K > 0 ? mm_split_bytes(M, N, K) : 0; }

extern "C" int uncl_matmul8(const uncl_matmul8_desc* d, void* workspace, void* stream) {
  if (!d || d->M < 0 || d->N < 0 || d->K < 0 || (d->a_fmt != UNCL_E4M3 && d->a_fmt != UNCL_E5M2) || d->b_fmt != UNCL_E4M3) return UNCL_ERR_ARG;
  if (d->out_dtype != UNCL_F32 && !uncl_is_h16(d->out_dtype)) return UNCL_ERR_ARG;
  if (d->act < UNCL_ACT_NONE || d->act > UNCL_ACT_MSIG) return UNCL_ERR_ARG;
  if (d->M == 0 || d->N == 0) return UNCL_OK;
  if (d->K == 0 || !d->a || !d->b || !d->a_scale || !d->b_scale || !d->out) return UNCL_ERR_ARG;
  if (d->M > (1 << 30) || d->N > (1 << 30) || d->lda < d->K || d->ldb < d->K || (d->lda & 15) || (d->ldb & 15) || !aligned16(d->a) || !aligned16(d->b)) return UNCL_ERR_ARG;
  // a tile's rows and scales are addressed with 32 bits from its first one
  if (d->lda > (1 << 22) || d->ldb > (1 << 22) || d->a_scale_row < 0 || d->b_scale_row < 0 || d->a_scale_row > (1 << 20) || d->b_scale_row > (1 << 20))
    return UNCL_ERR_ARG;
  if (!d->b_tile && d->b_scale_row != 1 && d->N > 1) return UNCL_ERR_ARG;
  if (d->ldo < d->N || (d->res && d->ldr < d->N)) return UNCL_ERR_ARG;
  if (mm_tiles(d->M, d->N, 128) >= 1 << 24) return UNCL_ERR_ARG;      // one workgroup of 256 threads each, under 2^32 in all
  MmArgs p{};
  p.a = reinterpret_cast<const unsigned char*>(d->a); p.b = reinterpret_cast<const unsigned char*>(d->b);
  p.sa = d->a_scale; p.sb = d->b_scale; p.bias = d->bias; p.res = d->res; p.out = d->out;
  p.lda = d->lda; p.ldb = d->ldb; p.ldr = d->ldr; p.ldo = d->ldo;
  p.sa_row = d->a_scale_row; p.sa_blk = d->a_scale_block; p.sb_row = d->b_scale_row; p.sb_blk = d->b_scale_block;
  p.M = d->M; p.N = d->N; p.K = d->K; p.KB = (d->K + 127) / 128; p.act = d->act; p.out_dtype = d->out_dtype;
  return mm_run(p, d->a_fmt, d->b_tile != 0, workspace, reinterpret_cast<hipStream_t>(stream));
}
