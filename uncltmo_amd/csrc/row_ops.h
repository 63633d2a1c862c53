// Shared pieces of the operators on rows of channels (row_ops.hip, quant8.hip, matmul8.hip).
#pragma once
#include "common.h"

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef int i32x4 __attribute__((ext_vector_type(4)));
typedef int i32x8 __attribute__((ext_vector_type(8)));

// Eight consecutive elements of a row <-> fp32.  n = elements of the row from p on: a whole group moves in 16-byte accesses (unaligned
// ones are legal on gfx950, so an odd pitch costs no other path), the row's last group element by element.
template <typename T>
__device__ __forceinline__ void ro_load8(const T* p, int n, float* f) {
  if (n >= 8) {
    if constexpr (sizeof(T) == 2) {
      typename Elem<T>::vec v;
      __builtin_memcpy(&v, p, 16);
      Elem<T>::unpack(v, f);
    } else {
      f32x4 a, b;
      __builtin_memcpy(&a, p, 16);
      __builtin_memcpy(&b, p + 4, 16);
#pragma unroll
      for (int i = 0; i < 4; ++i) { f[i] = a[i]; f[4 + i] = b[i]; }
    }
  } else {
    T e[8];                                                 // (n > 0; without branches, so that none waits for another)
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = p[i < n ? i : 0];
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = i < n ? (float)e[i] : 0.f;
  }
}
template <typename T>
__device__ __forceinline__ void ro_store8(T* p, int n, const float* f) {
  if (n >= 8) {
    if constexpr (sizeof(T) == 2) {
      const typename Elem<T>::vec v = Elem<T>::pack(f);
      __builtin_memcpy(p, &v, 16);
    } else {
      const f32x4 a = {f[0], f[1], f[2], f[3]}, b = {f[4], f[5], f[6], f[7]};
      __builtin_memcpy(p, &a, 16);
      __builtin_memcpy(p + 4, &b, 16);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = (T)f[i];
  }
}

// eight whole elements as they lie, for loads that are not waited for at once
template <typename T>
struct RoRaw8 {
  f32x4 v[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p) { __builtin_memcpy(v, p, 8 * sizeof(T)); }
  __device__ __forceinline__ void get(float* f) const {
    if constexpr (sizeof(T) == 2) {
      typename Elem<T>::vec x;
      __builtin_memcpy(&x, v, 16);
      Elem<T>::unpack(x, f);
    } else {
#pragma unroll
      for (int i = 0; i < 4; ++i) { f[i] = v[0][i]; f[4 + i] = v[1][i]; }
    }
  }
};

// up to eight elements of each of two rows (q NULL: of one, and b is 0); both loads go out before either is waited for where all eight exist
// (bf16, inputs of four sets in turn: the norm of 508032 x 32 28.4 -> 26.2 us, its backward pass, with gh's load as early, 28.8 -> 27.5 and of
// 20000 x 4096 133 -> 120; dropout, whose flags the first wait hides, lost 8 %)
template <typename T>
__device__ __forceinline__ void ro_load8_two(const T* p, const T* q, int n, float* a, float* b) {
  if (n >= 8) {
    RoRaw8<T> x, y;
    x.load(p);
    if (q) y.load(q);
    x.get(a);
    if (q) {
      y.get(b);
      return;
    }
  } else {
    ro_load8(p, n, a);
    if (q) {
      ro_load8(q, n, b);
      return;
    }
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) b[i] = 0.f;
}

// Philox4x32-10 (Salmon, Moraes, Dror, Shaw: "Parallel random numbers: as easy as 1, 2, 3", SC 2011): counter (group, stream), key = seed.
__device__ __forceinline__ void ro_philox(unsigned long long group, unsigned long long stream, unsigned long long seed, unsigned* w) {
  unsigned c0 = (unsigned)group, c1 = (unsigned)(group >> 32), c2 = (unsigned)stream, c3 = (unsigned)(stream >> 32);
  unsigned k0 = (unsigned)seed, k1 = (unsigned)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 10; ++r) {
    const unsigned long long x = (unsigned long long)c0 * 0xD2511F53u, y = (unsigned long long)c2 * 0xCD9E8D57u;
    c0 = (unsigned)(y >> 32) ^ c1 ^ k0;
    c1 = (unsigned)y;
    c2 = (unsigned)(x >> 32) ^ c3 ^ k1;
    c3 = (unsigned)x;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  w[0] = c0; w[1] = c1; w[2] = c2; w[3] = c3;
}

// What dropping needs: flags are 16-bit words against `limit` = round(p 2^16); kept elements are multiplied by 2^16 / (2^16 - limit), so
// the expectation is exact for the rounded p.  `span` consecutive rows share their flags (a sample's pixels: whole channels are dropped).
struct RoDrop {
  const unsigned long long* dev;   // {seed, offset} in device memory (read by every launch: a captured graph replays new flags), or NULL
  unsigned long long seed, offset; // host values; offset is added to the device's
  long long span;
  int limit;                       // 0: nothing is dropped
  float scale;
};

// p in [0, 1] -> limit and scale
static inline void ro_drop_setup(RoDrop& d, float p) {
  d.limit = (int)((double)p * 65536.0 + 0.5);
  d.scale = d.limit < 65536 ? (float)(65536.0 / (65536 - d.limit)) : 0.f;
}

// first flag group of a row
__device__ __forceinline__ unsigned long long ro_flag_group(const RoDrop& d, long long row, int groups) {
  return (unsigned long long)(d.span == 1 ? row : row / d.span) * (unsigned)groups;
}

// the eight flags of (flag row, group) applied to f: dropped elements become 0 whatever they held, kept ones are scaled
__device__ __forceinline__ void ro_drop8(unsigned long long group, unsigned long long stream, unsigned long long seed, int limit,
                                         float scale, float* f) {
#pragma clang fp contract(off)
  unsigned w[4];
  ro_philox(group, stream, seed, w);
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const unsigned u = (i & 1) ? (w[i >> 1] >> 16) : (w[i >> 1] & 0xffffu);
    f[i] = u >= (unsigned)limit ? f[i] * scale : 0.f;
  }
}

// ---- 8-bit floating point (OCP e4m3fn / e5m2), blocks of 128 -------------------------------------------------------------------------
// scale = max(amax, 2^-100) * fl(1 / top), inverse = fl(1 / scale), q = round_even(x * inverse) kept inside +-top.  amax is over the
// FINITE values of the block: an infinity then becomes +-top (or NaN, where the caller asks for it), a NaN stays NaN, and neither reaches
// its neighbours.
#define RO_AMAX_MIN 7.8886090522101181e-31f   /* 2^-100: the scale of a block of zeros, its inverse finite */
template <int FMT>
struct RoF8 {
  static constexpr float top = FMT == UNCL_E4M3 ? 448.f : 57344.f;
};
// Sizes are compared as integers (|x| without its sign orders like its bits; no canonicalising of inputs, three to an instruction): an
// infinity or a NaN is then the largest, and only a thread that meets one (ODD) pays for leaving it out and for the clamp below.
#define RO_INF_BITS 0x7f800000u
template <bool ODD>
__device__ __forceinline__ unsigned ro_size(float v) {
  const unsigned u = __builtin_bit_cast(unsigned, v) & 0x7fffffffu;
  return ODD && u >= RO_INF_BITS ? 0u : u;
}
__device__ __forceinline__ unsigned ro_max(unsigned a, unsigned b) { return a > b ? a : b; }
// maximum over LANES (1 .. 16) neighbouring lanes; every one of them gets it.  Quads, mirrored halves and rows of sixteen by data-parallel
// moves: no trip through LDS
template <int CTRL>
__device__ __forceinline__ unsigned ro_moved(unsigned v) {
  return (unsigned)__builtin_amdgcn_update_dpp((int)v, (int)v, CTRL, 0xf, 0xf, false);
}
template <int LANES>
__device__ __forceinline__ unsigned ro_max_lanes(unsigned m) {
  if constexpr (LANES >= 2) m = ro_max(m, ro_moved<0xB1>(m));      // lanes 1 0 3 2 of each four
  if constexpr (LANES >= 4) m = ro_max(m, ro_moved<0x4E>(m));      // lanes 2 3 0 1
  if constexpr (LANES >= 8) m = ro_max(m, ro_moved<0x141>(m));     // eight lanes mirrored: the other four
  if constexpr (LANES >= 16) m = ro_max(m, ro_moved<0x140>(m));    // sixteen lanes mirrored: the other eight
  return m;
}
// largest finite size of eight; odd: whether one of them is not finite
__device__ __forceinline__ unsigned ro_size8(const float* v, bool& odd) {
  unsigned m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = ro_max(m, ro_size<false>(v[i]));
  odd = m >= RO_INF_BITS;
  if (odd) {
    m = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) m = ro_max(m, ro_size<true>(v[i]));
  }
  return m;
}
template <int FMT>
__device__ __forceinline__ float ro_scale_of(unsigned amax_bits) {
#pragma clang fp contract(off)
  return fmaxf(__builtin_bit_cast(float, amax_bits), RO_AMAX_MIN) * (1.0f / RoF8<FMT>::top);
}
// x / scale kept inside +-top, ready to be rounded (the quotient of a block's largest may be one fp32 step over top, which the conversion
// would make a NaN).  lost: an infinity becomes a NaN instead (of the two formats one has no infinity), for a caller whose results must
// not hide it.
template <int FMT, bool ODD>
__device__ __forceinline__ float ro_fit(float v, float inv, bool lost) {
#pragma clang fp contract(off)
  const float q = v * inv;
  if (!ODD) return __builtin_amdgcn_fmed3f(q, -RoF8<FMT>::top, RoF8<FMT>::top);
  const float c = fminf(fmaxf(q, -RoF8<FMT>::top), RoF8<FMT>::top);
  return q != q || (lost && ro_size<false>(v) >= RO_INF_BITS) ? __builtin_nanf("") : c;
}
template <int FMT>
__device__ __forceinline__ unsigned ro_pack4(float a, float b, float c, float d) {
  int v;
  if constexpr (FMT == UNCL_E4M3) {
    v = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    v = __builtin_amdgcn_cvt_pk_fp8_f32(c, d, v, true);
  } else {
    v = __builtin_amdgcn_cvt_pk_bf8_f32(a, b, 0, false);
    v = __builtin_amdgcn_cvt_pk_bf8_f32(c, d, v, true);
  }
  return (unsigned)v;
}
template <int FMT>
__device__ __forceinline__ u32x2 ro_pack8(const float* v, float inv, bool odd, bool lost = false) {
  float f[8];
  if (odd) {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = ro_fit<FMT, true>(v[i], inv, lost);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = ro_fit<FMT, false>(v[i], inv, false);
  }
  return u32x2{ro_pack4<FMT>(f[0], f[1], f[2], f[3]), ro_pack4<FMT>(f[4], f[5], f[6], f[7])};
}
// eight 8-bit values to a row whose next n bytes exist
__device__ __forceinline__ void ro_store8q(unsigned char* p, int n, u32x2 v) {
  if (n >= 8) {
    __builtin_memcpy(p, &v, 8);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) p[i] = (unsigned char)(v[i >> 2] >> (8 * (i & 3)));
  }
}

// out[c] = sum of `blocks` partial rows of `cols` columns, in a fixed order (row_ops.hip)
int ro_fold_rows(const float* part, int blocks, int cols, float* out, hipStream_t s);
