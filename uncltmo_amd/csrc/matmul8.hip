// Matrix product of 8-bit floating-point operands with one fp32 scale for each block of 128 along the common axis:
//
//   out[m][n] = act( sum_kb sa[m][kb] sb[..][kb] sum_{k in kb} a[m][k] b[n][k] + bias[n] ) + res[m][n]
//
// a (M, K) rows, b (N, K) rows; sa one scale a row and block, sb one a 128 x 128 tile (weights) or a row and block (gradients).  The
// matrix instructions add up one block of 128 from zero, and the block joins the fp32 sum with one multiply-add an element: the scales
// never touch the operands.  b is the instruction's first operand, so that a lane's four results are four neighbouring columns of one
// row m: one scale a lane, one store of 8 or 16 bytes.  Which k a lane's 32 bytes are does not matter as long as both operands agree: a
// lane takes the 16-byte chunks g and g + 4 of its row's 128 (g = lane / 16).
//
// Two ways to add up a block.  The 8-bit instruction (16x16x128) adds products eight at a time on a common exponent and cuts each of them
// off 13 bits under the largest power of two in its group (measured, the same for all of the card's 8-bit forms; between groups it adds
// in fp32): about 1e-4 of a result of random signs.  That is a tenth of a rounding to bf16, so results in bf16 take it.  Results in fp16
// and fp32 would show it: there the operands are widened to bf16 in registers (exact: three or four significant bits, any exponent) and
// go through the bf16 instruction, whose sums measured 2^-23 of the products' sizes, at half the rate.
#include "row_ops.h"

namespace {

struct MmArgs {
  const unsigned char *a, *b;
  const float *sa, *sb, *bias;
  const void* res;
  void* out;
  long long lda, ldb, ldr, ldo, sa_row, sa_blk, sb_row, sb_blk;
  int M, N, K, KB, act, out_dtype;
};

// a lane's 32 bytes of one row, as they are or widened to bf16
struct Wide {
  bf16x8 v[4];
};
template <int F>
__device__ __forceinline__ Wide mm_widen(const i32x8& x) {
  typedef bf16_t bf16x2 __attribute__((ext_vector_type(2)));
  Wide w;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    bf16x2 lo, hi;
    if constexpr (F == UNCL_E4M3) {
      lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[i], 1.f, false);
      hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x[i], 1.f, true);
    } else {
      lo = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(x[i], 1.f, false);
      hi = __builtin_amdgcn_cvt_scalef32_pk_bf16_bf8(x[i], 1.f, true);
    }
    w.v[i >> 1][(i & 1) * 4 + 0] = lo[0];
    w.v[i >> 1][(i & 1) * 4 + 1] = lo[1];
    w.v[i >> 1][(i & 1) * 4 + 2] = hi[0];
    w.v[i >> 1][(i & 1) * 4 + 3] = hi[1];
  }
  return w;
}
template <int F, bool EXACT>
__device__ __forceinline__ auto mm_frag(const i32x8& x) {
  if constexpr (EXACT) return mm_widen<F>(x);
  else return x;
}
// one block of 128: b's 16 rows by a's 16 rows
template <int FA, int FB>
__device__ __forceinline__ f32x4 mm_block(const i32x8& b, const i32x8& a) {
  const f32x4 z = {0.f, 0.f, 0.f, 0.f};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b, a, z, FB - 1, FA - 1, 0, 0, 0, 0);
}
template <int FA, int FB>
__device__ __forceinline__ f32x4 mm_block(const Wide& b, const Wide& a) {
  f32x4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i) d = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b.v[i], a.v[i], d, 0, 0, 0);
  return d;
}

// four neighbouring columns n .. n + 3 of row m (`left` of them exist), residual added, in the output's type
template <typename T>
__device__ __forceinline__ void mm_put(T* out, const T* res, int left, f32x4 v) {
  T r[4];
  if (left >= 4) {
    if (res) {
      __builtin_memcpy(r, res, sizeof(r));
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] += (float)r[i];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) r[i] = (T)v[i];
    __builtin_memcpy(out, r, sizeof(r));
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < left) out[i] = (T)(v[i] + (res ? (float)res[i] : 0.f));
  }
}
__device__ __forceinline__ void mm_store(const MmArgs& p, long long m, int n, f32x4 v) {
  const int left = p.N - n;
  if (left <= 0) return;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < left) {
      if (p.bias) v[i] += p.bias[n + i];
      v[i] = uncl_act(v[i], p.act);
    }
  const long long o = m * p.ldo + n, r = m * p.ldr + n;
#define MM_PUT(T) mm_put(reinterpret_cast<T*>(p.out) + o, p.res ? reinterpret_cast<const T*>(p.res) + r : nullptr, left, v)
  if (p.out_dtype == UNCL_F32) MM_PUT(float);
  else if (p.out_dtype == UNCL_BF16) MM_PUT(bf16_t);
  else MM_PUT(f16_t);
#undef MM_PUT
}

// scale of the four columns n .. n + 3 (b scaled by rows) in block kb
__device__ __forceinline__ f32x4 mm_sb4(const MmArgs& p, int n, int kb) {
  f32x4 s;
#pragma unroll
  for (int i = 0; i < 4; ++i) s[i] = p.sb[(long long)(n + i < p.N ? n + i : p.N - 1) * p.sb_row + kb * p.sb_blk];
  return s;
}

__device__ __forceinline__ void mm_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// ---- tiles ---------------------------------------------------------------------------------------------------------------------------
// A workgroup of four waves (2 x 2) owns BM x BN outputs; a stage of LDS holds 128 bytes of each of its BM + BN rows, two stages.  Rows
// come in by asynchronous 16-byte loads straight to LDS; chunk c of row r lies at position c ^ (r & 7), so that the eight rows that a
// quarter of a wave reads at once fall on different banks.  The loads write LDS in lane order, hence the swizzle is in the lane's
// global address.
template <int FA, int FB, bool BT, bool EXACT, int BM, int BN>
__global__ __launch_bounds__(256) void mm_tile_kernel(const MmArgs p) {
  constexpr int TM = BM / 32, TN = BN / 32, STAGE = (BM + BN) * 128;
  constexpr int LA = BM / 32, LB = BN / 32;                 // 16-byte loads a thread and stage
  __shared__ __align__(16) unsigned char lds[2 * STAGE];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave & 1, wn = wave >> 1;
  const int tiles_n = (p.N + BN - 1) / BN;
  const int m0 = (blockIdx.x / tiles_n) * BM, n0 = (blockIdx.x % tiles_n) * BN;

  const int lr = lane >> 3, lc = (lane & 7) ^ lr;
  const unsigned char *ga[LA], *gb[LB];
#pragma unroll
  for (int i = 0; i < LA; ++i) {
    const int r = m0 + (i * 4 + wave) * 8 + lr;
    ga[i] = p.a + (long long)(r < p.M ? r : p.M - 1) * p.lda;
  }
#pragma unroll
  for (int i = 0; i < LB; ++i) {
    const int r = n0 + (i * 4 + wave) * 8 + lr;
    gb[i] = p.b + (long long)(r < p.N ? r : p.N - 1) * p.ldb;
  }
  const int last = (p.K - 1) & ~15;
  typedef __attribute__((address_space(3))) void* lptr;
  typedef const __attribute__((address_space(1))) void* gptr;
  auto fetch = [&](int kb, int st) {
    int col = kb * 128 + lc * 16;
    col = col < last ? col : last;                          // behind K: a chunk that exists; its bytes are cleared before use
    unsigned char* base = lds + st * STAGE + wave * 1024;
#pragma unroll
    for (int i = 0; i < LA; ++i) __builtin_amdgcn_global_load_lds((gptr)(ga[i] + col), (lptr)(base + i * 4096), 16, 0, 0);
#pragma unroll
    for (int i = 0; i < LB; ++i) __builtin_amdgcn_global_load_lds((gptr)(gb[i] + col), (lptr)(base + BM * 128 + i * 4096), 16, 0, 0);
  };

  f32x4 acc[TN][TM];
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int i = 0; i < TM; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int q = lane & 15, g = lane >> 4;
  const float* sa[TM];
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = m0 + (wm * TM + i) * 16 + q;
    sa[i] = p.sa + (long long)(m < p.M ? m : p.M - 1) * p.sa_row;
  }
  const int nb = n0 + wn * TN * 16;                           // the wave's columns lie inside one 128-column tile of b's scales

  fetch(0, 0);
  for (int kb = 0; kb < p.KB; ++kb) {
    float sm[TM];
#pragma unroll
    for (int i = 0; i < TM; ++i) sm[i] = sa[i][(long long)kb * p.sa_blk];
    f32x4 sn[TN];
    if constexpr (BT) {
      const float t = p.sb[(long long)((nb < p.N ? nb : p.N - 1) >> 7) * p.sb_row + kb * p.sb_blk];
#pragma unroll
      for (int i = 0; i < TM; ++i) sm[i] *= t;
    } else {
#pragma unroll
      for (int j = 0; j < TN; ++j) sn[j] = mm_sb4(p, nb + j * 16 + g * 4, kb);
    }
    if (kb + 1 < p.KB) {
      fetch(kb + 1, (kb + 1) & 1);
      if constexpr (LA + LB == 8) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
      else asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
    } else {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    mm_barrier();
    unsigned char* st = lds + (kb & 1) * STAGE;
    const int have = p.K - kb * 128;
    if (have < 128) {                                        // the last block is short: clear what lies behind K
      for (int t = threadIdx.x; t < (BM + BN) * 8; t += 256) {
        const int r = t >> 3, c = t & 7;
        unsigned char* at = st + r * 128 + ((c ^ (r & 7)) << 4);
        const int keep = have - c * 16;
        if (keep <= 0) *reinterpret_cast<i32x4*>(at) = i32x4{0, 0, 0, 0};
        else
          for (int k = keep; k < 16; ++k) at[k] = 0;
      }
      mm_barrier();
    }
    auto frag = [&](int row) {
      const unsigned char* r = st + row * 128;
      const i32x4 lo = *reinterpret_cast<const i32x4*>(r + ((g ^ (row & 7)) << 4));
      const i32x4 hi = *reinterpret_cast<const i32x4*>(r + (((g + 4) ^ (row & 7)) << 4));
      return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    };
    decltype(mm_frag<FB, EXACT>(i32x8{})) fb[TN];
#pragma unroll
    for (int j = 0; j < TN; ++j) fb[j] = mm_frag<FB, EXACT>(frag(BM + (wn * TN + j) * 16 + q));
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const auto fa = mm_frag<FA, EXACT>(frag((wm * TM + i) * 16 + q));
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const f32x4 t = mm_block<FA, FB>(fb[j], fa);
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[j][i][e] = fmaf(t[e], BT ? sm[i] : sm[i] * sn[j][e], acc[j][i][e]);
      }
    }
    mm_barrier();                                            // the stage may be written again
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = m0 + (wm * TM + i) * 16 + q;
    if (m < p.M)
#pragma unroll
      for (int j = 0; j < TN; ++j) mm_store(p, m, nb + j * 16 + g * 4, acc[j][i]);
  }
}

// ---- few rows ------------------------------------------------------------------------------------------------------------------------
// Up to 64 rows: b is read once and is nearly all there is to read (so the sums are the exact ones for every type).  A workgroup owns 16 columns, its WAVES waves take the blocks of K in
// turn, operands come straight from global memory into registers, and the waves' sums join in LDS in a fixed order.
template <int FA, int FB, bool BT, int TM, int WAVES>
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
#pragma unroll 2
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
    const Wide fb = mm_widen<FB>(frag(gb));
    float t = 1.f;
    f32x4 sn = {1.f, 1.f, 1.f, 1.f};
    if constexpr (BT) t = p.sb[(long long)(n0 >> 7) * p.sb_row + kb * p.sb_blk];
    else sn = mm_sb4(p, n0 + g * 4, kb);
#pragma unroll
    for (int i = 0; i < TM; ++i) {
      const float s = sa[i][(long long)kb * p.sa_blk] * t;
      const f32x4 d = mm_block<FA, FB>(fb, mm_widen<FA>(frag(ga[i])));
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[i][e] = fmaf(d[e], BT ? s : s * sn[e], acc[i][e]);
    }
  }
#pragma unroll
  for (int i = 0; i < TM; ++i) red[wave][i][lane] = acc[i];
  __syncthreads();
  for (int i = wave; i < TM; i += WAVES) {
    f32x4 v = red[0][i][lane];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) v += red[w][i][lane];
    if (i * 16 + q < p.M) mm_store(p, i * 16 + q, n0 + g * 4, v);
  }
}

template <int FA, int FB, bool BT>
int launch_mm(const MmArgs& p, hipStream_t s) {
  if (p.M <= 64) {
    const int grid = (p.N + 15) / 16;
    if (p.M <= 16) mm_rows_kernel<FA, FB, BT, 1, 8><<<grid, 512, 0, s>>>(p);
    else if (p.M <= 32) mm_rows_kernel<FA, FB, BT, 2, 8><<<grid, 512, 0, s>>>(p);
    else mm_rows_kernel<FA, FB, BT, 4, 8><<<grid, 512, 0, s>>>(p);
  } else {
    const long long big = (long long)((p.M + 127) / 128) * ((p.N + 127) / 128);
    // 128 x 128 tiles read half as much of LDS a product; 64 x 64 ones where the large ones would leave half of the 256 CUs idle
    const long long small = (long long)((p.M + 63) / 64) * ((p.N + 63) / 64);
    const bool exact = p.out_dtype != UNCL_BF16;
    if (big >= 256) {
      if (exact) mm_tile_kernel<FA, FB, BT, true, 128, 128><<<(unsigned)big, 256, 0, s>>>(p);
      else mm_tile_kernel<FA, FB, BT, false, 128, 128><<<(unsigned)big, 256, 0, s>>>(p);
    } else {
      if (exact) mm_tile_kernel<FA, FB, BT, true, 64, 64><<<(unsigned)small, 256, 0, s>>>(p);
      else mm_tile_kernel<FA, FB, BT, false, 64, 64><<<(unsigned)small, 256, 0, s>>>(p);
    }
  }
  UNCL_CHECK_LAUNCH();
  return UNCL_OK;
}

bool fmt_ok(int f) { return f == UNCL_E4M3 || f == UNCL_E5M2; }
bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

extern "C" int uncl_matmul8(const uncl_matmul8_desc* d, void* stream) {
  if (!d || d->M < 0 || d->N < 0 || d->K < 0 || !fmt_ok(d->a_fmt) || !fmt_ok(d->b_fmt)) return UNCL_ERR_ARG;
  if (d->out_dtype != UNCL_F32 && !uncl_is_h16(d->out_dtype)) return UNCL_ERR_ARG;
  if (d->act < UNCL_ACT_NONE || d->act > UNCL_ACT_MSIG) return UNCL_ERR_ARG;
  if (d->M == 0 || d->N == 0) return UNCL_OK;
  if (d->K == 0 || !d->a || !d->b || !d->a_scale || !d->b_scale || !d->out) return UNCL_ERR_ARG;
  if (d->M > (1 << 30) || d->N > (1 << 30) || d->K > (1 << 30) || d->lda < d->K || d->ldb < d->K || (d->lda & 15) || (d->ldb & 15) || !aligned16(d->a) || !aligned16(d->b)) return UNCL_ERR_ARG;
  if (d->ldo < d->N || (d->res && d->ldr < d->N)) return UNCL_ERR_ARG;
  if ((long long)((d->M + 63) / 64) * ((d->N + 63) / 64) > 0x7fffffffll) return UNCL_ERR_ARG;
  MmArgs p{};
  p.a = reinterpret_cast<const unsigned char*>(d->a); p.b = reinterpret_cast<const unsigned char*>(d->b);
  p.sa = d->a_scale; p.sb = d->b_scale; p.bias = d->bias; p.res = d->res; p.out = d->out;
  p.lda = d->lda; p.ldb = d->ldb; p.ldr = d->ldr; p.ldo = d->ldo;
  p.sa_row = d->a_scale_row; p.sa_blk = d->a_scale_block; p.sb_row = d->b_scale_row; p.sb_blk = d->b_scale_block;
  p.M = d->M; p.N = d->N; p.K = d->K; p.KB = (d->K + 127) / 128; p.act = d->act; p.out_dtype = d->out_dtype;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define BY_TILE(FA, FB) (d->b_tile ? launch_mm<FA, FB, true>(p, s) : launch_mm<FA, FB, false>(p, s))
  if (d->a_fmt == UNCL_E4M3) return d->b_fmt == UNCL_E4M3 ? BY_TILE(UNCL_E4M3, UNCL_E4M3) : BY_TILE(UNCL_E4M3, UNCL_E5M2);
  return d->b_fmt == UNCL_E4M3 ? BY_TILE(UNCL_E5M2, UNCL_E4M3) : BY_TILE(UNCL_E5M2, UNCL_E5M2);
#undef BY_TILE
}
