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
// in fp32): at most 7 x 2^-13 of the groups' largest products, added up.  Normal operands, K = 256 to 8192: 1.4e-5 of the results' rms, at
// most 1.3e-4; positive ones 3.6e-6 of the result.  That is a hundredth of a rounding to bf16 (1.7e-3), so results in bf16 take it: one to
// three in a hundred of them round the other way, and their distance from the 64-bit value is that of the fp32 sum's rounding to four digits.
// It goes with the PRODUCTS' sizes: of a result that cancels it may be any part.  Results in fp16 and fp32 would show it: there the operands
// are widened to bf16 in registers (exact: three or four significant bits, any exponent) and go through the bf16 instruction, whose sums
// measured 2^-23 of the products' sizes, at half the rate.
#pragma once
#include "matmul8_args.h"
#include "row_ops.h"

#include <type_traits>

// the tiled kernels, one file for each type of result: bf16 through the 8-bit instruction, fp16 and fp32 through the bf16 one
int mm_tiles_bf16(const MmArgs& p, int a_fmt, bool b_tile, hipStream_t s);
int mm_tiles_f16(const MmArgs& p, int a_fmt, bool b_tile, hipStream_t s);
int mm_tiles_f32(const MmArgs& p, int a_fmt, bool b_tile, hipStream_t s);

namespace {

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
// one block of 128, b's TN x 16 rows by a's 16 rows: TN results
template <int FA, int TN>
__device__ __forceinline__ void mm_block(const i32x8 (&b)[TN], const i32x8& a, f32x4 (&d)[TN]) {
  const f32x4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int j = 0; j < TN; ++j) d[j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(b[j], a, z, UNCL_E4M3 - 1, FA - 1, 0, 0, 0, 0);
}
template <int FA, int TN>
__device__ __forceinline__ void mm_block(const Wide (&b)[TN], const Wide& a, f32x4 (&d)[TN]) {
#pragma unroll
  for (int j = 0; j < TN; ++j) d[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) d[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[j].v[i], a.v[i], d[j], 0, 0, 0);
}

// x Phi(x) = max(x, 0) - |x| (1 - Phi(|x|)), the tail by Abramowitz and Stegun 7.1.26 (erf off by at most 1.5e-7): the library's erff took
// half of a short product's time.  |x| stops at 64, where the tail is 0 long since, so that infinity times it is not NaN: infinity stays,
// minus infinity becomes 0.
__device__ __forceinline__ float mm_gelu(float x) {
  const float a = fminf(__builtin_fabsf(x), 64.f);
  const float t = __builtin_amdgcn_rcpf(fmaf(0.3275911f * 0.70710678118654752f, a, 1.f));
  float q = fmaf(t, 0.5f * 1.061405429f, 0.5f * -1.453152027f);
  q = fmaf(t, q, 0.5f * 1.421413741f);
  q = fmaf(t, q, 0.5f * -0.284496736f);
  q = fmaf(t, q, 0.5f * 0.254829592f);
  const float e = __builtin_amdgcn_exp2f(x * x * (-0.5f * 1.44269504088896341f));
  return fmaxf(x, 0.f) - a * (q * t * e);
}
// the rarer activations, one copy of their code
__device__ __attribute__((noinline)) float mm_act_rare(float v, int act) { return uncl_act(v, act); }

// the activation of E sums
template <int E>
__device__ __forceinline__ void mm_act(float* v, int act) {
  if (act == UNCL_ACT_GELU) {
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = mm_gelu(v[i]);
  } else if (act == UNCL_ACT_RELU) {
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = v[i] < 0.f ? 0.f : v[i];             // (NaN stays)
  } else if (act != UNCL_ACT_NONE) {
#pragma unroll
    for (int i = 0; i < E; ++i) v[i] = mm_act_rare(v[i], act);
  }
}

__device__ __forceinline__ int mm_turn(int row) { return (row >> 1) & 7; }

// everything this wave has in flight has arrived, and every wave of the workgroup says so
__device__ __forceinline__ void mm_arrive() { asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

// The lanes of a wave hand numbers to each other through its own part of LDS: the hardware keeps a wave's LDS operations in order, this keeps the
// compiler's (which sees one thread) in that order too.  No instruction.
__device__ __forceinline__ void mm_wave_order() {
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  __builtin_amdgcn_wave_barrier();
}

// bytes from a row of a matrix on, bounds-checked by the hardware: `rows` rows `pitch` bytes apart, `len` bytes of each
__device__ __forceinline__ __amdgpu_buffer_rsrc_t mm_buffer(const void* p, long long rows, long long pitch, long long len) {
  const long long n = (rows - 1) * pitch + len;
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(p), (short)0, (int)(n < 0x7fffffffll ? n : 0x7fffffffll), 0x00020000);
}

// ---- tiles ---------------------------------------------------------------------------------------------------------------------------
// A workgroup of WM x WN waves owns BM x BN outputs; a stage of LDS holds 128 bytes of each of its BM + BN rows, two stages.  Rows
// come in by asynchronous 16-byte loads straight to LDS, a block ahead of the products, and the block's scales with them: one barrier
// a block says both that this block has arrived and that nobody reads the stage that the next one overwrites.  Chunk c of row r lies at
// position c ^ mm_turn(r), so that the rows that a part of a wave reads at once fall on different banks (conflicts counted: 256 cycles a
// workgroup of 128 x 128 at K = 256 and at 4096 alike, all of them where the results turn round at the end).  The loads write LDS in lane order,
// hence the swizzle is in the lane's global address.  Rows behind M or N are out of the buffers' bounds (their results are not stored);
// bytes behind K, of the next row or out of bounds, are cleared in LDS.
//
// Workgroups go to the card's eight XCDs in turn, each with an L2 of its own: the b-th workgroup takes the (b / 8)-th tile of its XCD's
// share, and a share runs through groups of eight rows of tiles, so that the 32 tiles at work on an XCD have few rows and columns.
// (The second launch bound, waves a SIMD: two workgroups of 128 x 128 a CU, four or more of 64 x 64 -- and under 257 registers a wave the
// compiler leaves the matrix instructions' results where the multiply-adds can read them.)
template <typename T, int FA, bool BT, bool EXACT, int BM, int BN, int WM, int WN>
__global__ __launch_bounds__(WM * WN * 64, BM > 64 ? 2 : 4) void mm_tile_kernel(const MmArgs p) {
  constexpr int NT = WM * WN * 64, TM = BM / WM / 16, TN = BN / WN / 16, STAGE = (BM + BN) * 128;
  constexpr int LA = BM * 8 / NT, LB = BN * 8 / NT;         // 16-byte loads a thread and stage
  constexpr int SB = BT ? (BN > 128 ? BN / 128 : 1) : BN / 64;   // waves that fetch b's scales
  constexpr int SCALES = (BM + SB * 64) * 4;                 // a block's scales, behind the two stages
  __shared__ __align__(16) unsigned char lds[2 * (STAGE + SCALES)];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wm = wave % WM, wn = wave / WM;
  const int tm = (p.M + BM - 1) / BM, tn = (p.N + BN - 1) / BN, total = tm * tn;
  int id = blockIdx.x;
  {
    const int x = id & 7, share = total >> 3, more = total & 7;
    id = x * share + (x < more ? x : more) + (id >> 3);
  }
  const int gr = id / (8 * tn), gm = gr * 8, rows = tm - gm < 8 ? tm - gm : 8, in = id - gr * 8 * tn;
  const int m0 = (gm + in % rows) * BM, n0 = (in / rows) * BN;

  const int lr = lane >> 3, lc0 = lane & 7, k16 = (p.K + 15) & ~15;
  const __amdgpu_buffer_rsrc_t ra = mm_buffer(p.a + (long long)m0 * p.lda, p.M - m0, p.lda, k16);
  const __amdgpu_buffer_rsrc_t rb = mm_buffer(p.b + (long long)n0 * p.ldb, p.N - n0, p.ldb, k16);
  const int lc = lc0 ^ mm_turn(wave * 8 + lr);                // NT / 8 rows further on the swizzle is the same
  const int va = (wave * 8 + lr) * (int)p.lda + lc * 16, vb = (wave * 8 + lr) * (int)p.ldb + lc * 16;
  const int sta = (NT / 8) * (int)p.lda, stb = (NT / 8) * (int)p.ldb;
  typedef __attribute__((address_space(3))) void* lptr;
  auto fetch_one = [&](int kb, int x) {                      // the x-th of a wave's LA + LB loads of a block
    unsigned char* base = lds + (kb & 1) * STAGE + wave * 1024;
    if (x < LA) __builtin_amdgcn_raw_ptr_buffer_load_lds(ra, (lptr)(base + x * NT * 16), 16, va + x * sta, kb * 128, 0, 0);
    else __builtin_amdgcn_raw_ptr_buffer_load_lds(rb, (lptr)(base + BM * 128 + (x - LA) * NT * 16), 16, vb + (x - LA) * stb, kb * 128, 0, 0);
  };
  auto fetch = [&](int kb) {
#pragma unroll
    for (int x = 0; x < LA + LB; ++x) fetch_one(kb, x);
  };

  f32x4 acc[TN][TM];
#pragma unroll
  for (int j = 0; j < TN; ++j)
#pragma unroll
    for (int i = 0; i < TM; ++i) acc[j][i] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int q = lane & 15, g = lane >> 4;
  const int mb = m0 + wm * TM * 16, nb = n0 + wn * TN * 16;
  const float* sap = p.sa + (long long)m0 * p.sa_row;
  // one wave for each 64 of a's rows, and for each 64 of b's columns or each tile of b's scales (64 copies of it)
  auto fetch_scales = [&](int kb) {
    unsigned char* to = lds + 2 * STAGE + (kb & 1) * SCALES + wave * 256;
    const int x = wave - BM / 64;
    if (x < 0) {
      const __amdgpu_buffer_rsrc_t r = mm_buffer(sap + kb * p.sa_blk, p.M - m0, p.sa_row * 4, 4);
      __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lptr)to, 4, (wave * 64 + lane) * (int)p.sa_row * 4, 0, 0, 0);
    } else if (x < SB) {
      if constexpr (BT) {
        const int last_tile = (p.N - 1) >> 7, tile = (n0 >> 7) + x;
        const __amdgpu_buffer_rsrc_t r = mm_buffer(p.sb + (tile < last_tile ? tile : last_tile) * p.sb_row + kb * p.sb_blk, 1, 4, 4);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lptr)to, 4, 0, 0, 0, 0);
      } else {
        const __amdgpu_buffer_rsrc_t r = mm_buffer(p.sb + n0 + kb * p.sb_blk, p.N - n0, 4, 4);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (lptr)to, 4, (x * 64 + lane) * 4, 0, 0, 0);
      }
    }
  };
  float sb = 1.f;                                            // b's scale (BT), of the block at work
  f32x4 sn[BT ? 1 : TN];                                     // or those of the lane's columns
  auto scales = [&](int kb) { return reinterpret_cast<const float*>(lds + 2 * STAGE + (kb & 1) * SCALES); };
  auto take_scales = [&](int kb) {
    if constexpr (BT) sb = scales(kb)[BM + ((wn * TN * 16) >> 7) * 64 + lane];
    else
#pragma unroll
      for (int j = 0; j < TN; ++j) sn[j] = *reinterpret_cast<const f32x4*>(scales(kb) + BM + wn * TN * 16 + g * 4 + j * 16);
  };
  auto scale_a = [&](int kb, int i) { return scales(kb)[(wm * TM + i) * 16 + q]; };

  int k0 = 0, k1 = p.KB;
  if constexpr (BM == 64)
    if (p.part) { k0 = blockIdx.y * p.per; k1 = k0 + p.per < p.KB ? k0 + p.per : p.KB; }
  fetch(k0);
  fetch_scales(k0);
  auto stage = [&](int kb) { return lds + (kb & 1) * STAGE; };
  // block kb has arrived (and nobody reads the other stage any more); a short last block: what lies behind K is cleared
  auto arrive = [&](int kb) {
    mm_arrive();
    const int have = p.K - kb * 128;
    if (have >= 128) return;
    for (int t = threadIdx.x; t < (BM + BN) * 8; t += NT) {
      const int r = t >> 3, c = t & 7;
      unsigned char* at = stage(kb) + r * 128 + ((c ^ mm_turn(r)) << 4);
      const int keep = have - c * 16;
      if (keep <= 0) *reinterpret_cast<i32x4*>(at) = i32x4{0, 0, 0, 0};
      else
        for (int k = keep; k < 16; ++k) at[k] = 0;
    }
    mm_arrive();
  };
  auto frag = [&](const unsigned char* st, int row) {
    const unsigned char* r = st + row * 128;
    const i32x4 lo = *reinterpret_cast<const i32x4*>(r + ((g ^ mm_turn(row)) << 4));
    const i32x4 hi = *reinterpret_cast<const i32x4*>(r + (((g + 4) ^ mm_turn(row)) << 4));
    return i32x8{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  };
  const int rowa = wm * TM * 16 + q, rowb = BM + wn * TN * 16 + q;
  // the products of a's rows i run while those of rows i - 1 join their sums: a matrix instruction's result is never waited for
  f32x4 t[2][TN];
  auto join_one = [&](int i, int j, float scale) {
#pragma unroll
    for (int e = 0; e < 4; ++e) acc[j][i][e] = fmaf(t[i & 1][j][e], BT ? scale : scale * sn[BT ? 0 : j][e], acc[j][i][e]);
  };
  auto join = [&](int i, float scale) {
#pragma unroll
    for (int j = 0; j < TN; ++j) join_one(i, j, scale);
  };
  if constexpr (BM == 256) {
    // One workgroup a CU: nobody else works while this one waits.  The next block's arrival is waited for before this block's last
    // products, whose time its first LDS reads then have; its loads are spread over the first half of this block's products (64 at once
    // kept the waves from issuing anything else); the last sums join in the next block.  8192 x 8192 x 8192: 468 -> 441 us; the smaller
    // tiles, two to four workgroups a CU, lost 5 - 10 % by it.
    i32x8 fb[TN], fa[2];
    float sm[2] = {0.f, 0.f};
#pragma unroll
    for (int j = 0; j < TN; ++j) t[(TM - 1) & 1][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto multiply = [&](int i, int j) {
      const f32x4 z = {0.f, 0.f, 0.f, 0.f};
      t[i & 1][j] = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(fb[j], fa[i & 1], z, UNCL_E4M3 - 1, FA - 1, 0, 0, 0, 0);
    };
    constexpr int HALF = TM / 2, EACH = (LA + LB + HALF - 1) / HALF;     // loads of the next block: spread over the first half
    auto all_but_last = [&](int kb, auto more) {
      const unsigned char* st = stage(kb);
#pragma unroll
      for (int i = 0; i + 1 < TM; ++i) {
        fa[(i + 1) & 1] = frag(st, rowa + (i + 1) * 16);
#pragma unroll
        for (int j = 0; j < TN; ++j) multiply(i, j);
        join((i + TM - 1) % TM, i == 0 ? sm[1] : sm[(i + 1) & 1] * sb);           // (rows TM - 1: of the last block, scaled already)
        sm[(i + 1) & 1] = scale_a(kb, i + 1);
        if constexpr (more)
#pragma unroll
          for (int x = i * EACH; x < (i + 1) * EACH && x < LA + LB; ++x) fetch_one(kb + 1, x);
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);                        // LDS reads of the next rows
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                      // a matrix instruction,
          __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x002, 4, 0);                      // the last rows' multiply-adds under it
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    };
    // what has been joined stays joined: left to itself the compiler moves all multiply-adds behind the next branch, their operands with them
    auto pin = [&]() {
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j)
          if (i != TM - 2) asm volatile("" : "+v"(acc[j][i]));
    };
    arrive(k0);
    fa[0] = frag(stage(k0), rowa);
#pragma unroll
    for (int j = 0; j < TN; ++j) fb[j] = frag(stage(k0), rowb + j * 16);
    take_scales(k0);
    sm[0] = scale_a(k0, 0);
    for (int kb = k0; kb + 1 < k1; ++kb) {
      fetch_scales(kb + 1);
      all_but_last(kb, std::true_type{});
      pin();
      arrive(kb + 1);
      const unsigned char* next = stage(kb + 1);
      sm[0] *= sb;
      sm[1] *= sb;
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int j = 0; j < TN; ++j) {                                              // (in this order: the next operand takes the last one's registers)
        multiply(TM - 1, j);
        __builtin_amdgcn_sched_barrier(0);
        fb[j] = frag(next, rowb + j * 16);
        join_one(TM - 2, j, sm[0]);
        __builtin_amdgcn_sched_barrier(0);
      }
      fa[0] = frag(next, rowa);
      take_scales(kb + 1);
      sm[0] = scale_a(kb + 1, 0);
    }
    all_but_last(k1 - 1, std::false_type{});
    pin();
#pragma unroll
    for (int j = 0; j < TN; ++j) multiply(TM - 1, j);
    join(TM - 2, sm[0] * sb);
    join(TM - 1, sm[1] * sb);
  } else {
    for (int kb = k0; kb < k1; ++kb) {
      arrive(kb);
      take_scales(kb);
      if (kb + 1 < k1) {
        fetch(kb + 1);
        fetch_scales(kb + 1);
      }
      const unsigned char* st = stage(kb);
      decltype(mm_frag<UNCL_E4M3, EXACT>(i32x8{})) fb[TN], fa[2];
      fa[0] = mm_frag<FA, EXACT>(frag(st, rowa));
#pragma unroll
      for (int j = 0; j < TN; ++j) fb[j] = mm_frag<UNCL_E4M3, EXACT>(frag(st, rowb + j * 16));
      float sm[2];
#pragma unroll
      for (int i = 0; i <= TM; ++i) {
        i32x8 raw;
        if (i + 1 < TM) raw = frag(st, rowa + (i + 1) * 16);
        if (i < TM) sm[i & 1] = scale_a(kb, i);
        if (i < TM) mm_block<FA, TN>(fb, fa[i & 1], t[i & 1]);
        if (i > 0) join(i - 1, BT ? sm[(i - 1) & 1] * sb : sm[(i - 1) & 1]);
        if (i + 1 < TM) fa[(i + 1) & 1] = mm_frag<FA, EXACT>(raw);
        if (i < TM) {
          if (i + 1 < TM) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
          for (int j = 0; j < (EXACT ? 4 : 1) * TN; ++j) {
            __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
            __builtin_amdgcn_sched_group_barrier(0x002, EXACT ? (BT ? 2 : 3) : 8, 0);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  }
  // A lane's results are four columns of sixteen different rows: they turn round in LDS, 32 rows of the wave at a time, so that eight (or
  // four) lanes hold one row's columns and memory sees whole lines.  Each wave has its own part of LDS, whose operations stay in order.
  constexpr int COLS = TN * 16, PITCH = COLS + 4, LPR = COLS / 8, RPP = 64 / LPR, PASSES = 32 / RPP;
  static_assert(BM < 256 || (BT && !EXACT), "the largest tiles are built for the 8-bit instruction and b scaled by tiles");
  static_assert(WM * WN * 32 * PITCH * 4 <= 2 * STAGE && TM % 2 == 0 && BM / 64 + SB <= WM * WN, "the turned rows fit where the stages were");
  mm_arrive();
  float* w = reinterpret_cast<float*>(lds) + wave * 32 * PITCH;
  const int r0 = lane / LPR, c0 = (lane % LPR) * 8, n = nb + c0, left = p.N - n;
  T* out = reinterpret_cast<T*>(p.out);
  const T* res = reinterpret_cast<const T*>(p.res);
  if constexpr (BM == 64)
    if (p.part) {
      const int n8 = (p.N + 7) & ~7;
      float* part = p.part + (long long)blockIdx.y * p.M * n8 + n;
#pragma unroll
      for (int ch = 0; ch < TM / 2; ++ch) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < TN; ++j) *reinterpret_cast<f32x4*>(w + (i * 16 + q) * PITCH + j * 16 + g * 4) = acc[j][ch * 2 + i];
        mm_wave_order();
#pragma unroll
        for (int t = 0; t < PASSES; ++t) {
          const int m = mb + ch * 32 + t * RPP + r0;
          const float* at = w + (t * RPP + r0) * PITCH + c0;
          const f32x4 lo = *reinterpret_cast<const f32x4*>(at), hi = *reinterpret_cast<const f32x4*>(at + 4);
          if (m < p.M && left > 0) {
            *reinterpret_cast<f32x4*>(part + (long long)m * n8) = lo;
            *reinterpret_cast<f32x4*>(part + (long long)m * n8 + 4) = hi;
          }
        }
        mm_wave_order();
      }
      return;
    }
  float bias[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) bias[e] = 0.f;
  if (p.bias && left > 0) ro_load8(p.bias + n, left, bias);
  // Where all columns exist the residual's loads need no branches and go out together (bf16, inputs of four sets in turn: 8192 x 4096 x 4096
  // 153 -> 146 us, 28800 x 1024 x 256 47 -> 36).  Rows behind M read the last one again, for nothing.
  const bool whole = res && nb + COLS <= p.N;
#pragma unroll
  for (int ch = 0; ch < TM / 2; ++ch) {
    float r[PASSES][8];
    if (whole) {
      RoRaw8<T> raw[PASSES];
#pragma unroll
      for (int t = 0; t < PASSES; ++t) {
        const int m = mb + ch * 32 + t * RPP + r0;
        raw[t].load(res + (long long)(m < p.M ? m : p.M - 1) * p.ldr + n);
      }
#pragma unroll
      for (int t = 0; t < PASSES; ++t) raw[t].get(r[t]);
    } else if (res)
#pragma unroll
      for (int t = 0; t < PASSES; ++t) {
        const int m = mb + ch * 32 + t * RPP + r0;
        if (m < p.M && left > 0) ro_load8(res + (long long)m * p.ldr + n, left, r[t]);
      }
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j) *reinterpret_cast<f32x4*>(w + (i * 16 + q) * PITCH + j * 16 + g * 4) = acc[j][ch * 2 + i];
    mm_wave_order();
#pragma unroll
    for (int t = 0; t < PASSES; ++t) {
      const int m = mb + ch * 32 + t * RPP + r0;
      float v[8];
      const float* at = w + (t * RPP + r0) * PITCH + c0;
      const f32x4 lo = *reinterpret_cast<const f32x4*>(at), hi = *reinterpret_cast<const f32x4*>(at + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) { v[e] = lo[e] + bias[e]; v[4 + e] = hi[e] + bias[4 + e]; }
      mm_act<8>(v, p.act);
      if (res)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] += r[t][e];
      if (m < p.M && left > 0) ro_store8(out + (long long)m * p.ldo + n, left, v);
    }
    mm_wave_order();
  }
}

template <typename T, int FA, bool BT, bool EXACT>
int launch_tiles(const MmArgs& p, hipStream_t s) {
  const MmPlan plan = mm_plan(p.M, p.N, p.KB, BT && !EXACT);
  if constexpr (BT && !EXACT)
    if (plan.tile == 256) mm_tile_kernel<T, FA, BT, EXACT, 256, 256, 2, 4><<<(unsigned)mm_tiles(p.M, p.N, 256), 512, 0, s>>>(p);
  if (plan.tile == 128) mm_tile_kernel<T, FA, BT, EXACT, 128, 128, 2, 2><<<(unsigned)mm_tiles(p.M, p.N, 128), 256, 0, s>>>(p);
  if (plan.tile == 64)
    mm_tile_kernel<T, FA, BT, EXACT, 64, 64, 2, 2><<<dim3((unsigned)mm_tiles(p.M, p.N, 64), p.part ? (p.KB + p.per - 1) / p.per : 1), 256, 0, s>>>(p);
  UNCL_CHECK_LAUNCH();
  return UNCL_OK;
}

// the split tiles' partial sums, in order, with the epilogue of a whole tile
template <typename T>
__global__ __launch_bounds__(256) void mm_join_kernel(const MmArgs p, int splits) {
  const int n8 = (p.N + 7) & ~7, per_row = n8 >> 3;
  const long long total = (long long)p.M * per_row;
  for (long long t = (long long)blockIdx.x * 256 + threadIdx.x; t < total; t += (long long)gridDim.x * 256) {
    const long long m = t / per_row;
    const int n = (int)(t - m * per_row) * 8, left = p.N - n;
    const float* at = p.part + m * n8 + n;
    float v[8], x[8];
    ro_load8(at, 8, v);
#pragma unroll 4
    for (int s = 1; s < splits; ++s) {
      ro_load8(at + (long long)s * p.M * n8, 8, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += x[e];
    }
    if (p.bias) {
      ro_load8(p.bias + n, left, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += x[e];
    }
    mm_act<8>(v, p.act);
    if (p.res) {
      ro_load8(reinterpret_cast<const T*>(p.res) + m * p.ldr + n, left, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += x[e];
    }
    ro_store8(reinterpret_cast<T*>(p.out) + m * p.ldo + n, left, v);
  }
}

template <typename T, bool EXACT>
int launch_by_format(const MmArgs& p, int a_fmt, bool b_tile, hipStream_t s) {
  int rc;
  if (a_fmt == UNCL_E4M3) rc = b_tile ? launch_tiles<T, UNCL_E4M3, true, EXACT>(p, s) : launch_tiles<T, UNCL_E4M3, false, EXACT>(p, s);
  else rc = b_tile ? launch_tiles<T, UNCL_E5M2, true, EXACT>(p, s) : launch_tiles<T, UNCL_E5M2, false, EXACT>(p, s);
  if (rc != UNCL_OK || !p.part) return rc;
  const long long blocks = ((long long)p.M * ((p.N + 7) >> 3) + 255) / 256;
  mm_join_kernel<T><<<(unsigned)(blocks < 2048 ? blocks : 2048), 256, 0, s>>>(p, (p.KB + p.per - 1) / p.per);
  UNCL_CHECK_LAUNCH();
  return UNCL_OK;
}

}  // namespace
