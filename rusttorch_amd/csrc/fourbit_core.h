// Codes of the 4-bit cache (fourbit.h) as bf16, f32 rows as bf16 parts, and the
// bf16 matrix instructions that take them.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "bf16_split.h"
#include "fourbit.h"
#include "qrows.h"

namespace rtg {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

// Scale bytes as the f32 that the conversions take; byte 255 is infinity, for
// which they give NaN.
__device__ __forceinline__ float scale_of(unsigned byte) { return __uint_as_float(byte << 23); }

// Codes 2 SEL and 2 SEL + 1 of w under a scale as two bf16.
template <int SEL>
__device__ __forceinline__ unsigned two_bf16(unsigned w, float scale) {
  return __builtin_bit_cast(unsigned, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL));
}
// The 8 codes of w.
__device__ __forceinline__ u4v eight_bf16(unsigned w, float scale) {
  return u4v{two_bf16<0>(w, scale), two_bf16<1>(w, scale), two_bf16<2>(w, scale), two_bf16<3>(w, scale)};
}
__device__ __forceinline__ unsigned low_halves(unsigned a, unsigned b) {  // a's in the low half
  return __builtin_amdgcn_perm(b, a, 0x05040100u);
}
__device__ __forceinline__ unsigned high_halves(unsigned a, unsigned b) {
  return __builtin_amdgcn_perm(b, a, 0x07060302u);
}

// Columns c8 .. c8 + 7 of a row of n as f32, those from n on 0; vec (the same for
// all threads): n % 8 == 0 and the eight are aligned to 16 bytes (f32: both halves).
template <class T>
__device__ __forceinline__ void load8(const T* row, int c8, int n, bool vec, float (&x)[8]) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      const float4 a = load4(row, c8, n, true), b = load4(row, c8 + 4, n, true);
      x[0] = a.x, x[1] = a.y, x[2] = a.z, x[3] = a.w, x[4] = b.x, x[5] = b.y, x[6] = b.z, x[7] = b.w;
    } else {
      typedef T T8 __attribute__((ext_vector_type(8)));
      T8 v = {};
      if (c8 < n) v = *reinterpret_cast<const T8*>(row + c8);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] = (float)v[e];
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = c8 + e < n ? (float)row[c8 + e] : 0.f;
}
template <class T>
__device__ __forceinline__ void store8(T* row, int c8, int n, const float (&x)[8], bool vec) {
  store4(row, c8, n, make_float4(x[0], x[1], x[2], x[3]), vec);
  store4(row, c8 + 4, n, make_float4(x[4], x[5], x[6], x[7]), vec);
}
// Whether rows of n channels can be taken 8 at a time by load8.
inline bool by_eights(const QRows& r, int n, QType type) {
  const long e = type == Q_F32 ? 4 : 8;  // elements of 16 bytes
  return n % 8 == 0 && reinterpret_cast<uintptr_t>(r.p) % 16 == 0 && r.seq % e == 0 && r.tok % e == 0 && r.head % e == 0;
}

// x as bf16 parts, each what the ones before it leave over, cut: 8 bits of x a
// part. One part: to nearest instead.
template <int N>
__device__ __forceinline__ void bf16_parts(const float (&x)[8], u4v (&p)[N]) {
  if constexpr (N == 3) {
    split3(x, p[0], p[1], p[2]);
  } else if constexpr (N == 2) {
    u4v lo;
    unsigned h[8];
    float r[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      h[e] = __float_as_uint(x[e]) & 0xffff0000u;
      r[e] = x[e] - __uint_as_float(h[e]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      p[0][i] = high_halves(h[2 * i], h[2 * i + 1]);
      const bf16x2 l = {(__bf16)r[2 * i], (__bf16)r[2 * i + 1]};
      lo[i] = __builtin_bit_cast(unsigned, l);
    }
    p[1] = lo;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const bf16x2 v = {(__bf16)x[2 * i], (__bf16)x[2 * i + 1]};
      p[0][i] = __builtin_bit_cast(unsigned, v);
    }
  }
}

__device__ __forceinline__ f32x4 mfma16(const u4v& a, const u4v& b, const f32x4& c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(a), as_bf16x8(b), c, 0, 0, 0);
}

// The scale of the scores: its sign goes into the queries, and where it is far from
// 1 a power of two, so that sums stay within f32 where the scores do (exactly: parts
// of bf16 have f32's range); the rest is a factor of the sums, log2 e included. A
// scale of 0 makes the queries 0.
struct ScoreScale {
  float query, sum;
};
inline ScoreScale score_scale(float scale) {
  int e = 0;
  const double x = (double)scale * 1.4426950408889634074;
  const double m = frexp(fabs(x), &e);  // [0.5, 1)
  if (m == 0.0) return {0.f, 1.f};
  // (a power of two that f32 does not hold goes into the factor)
  const int in = abs(e) <= 20 ? 0 : e - 1 < -126 ? -126 : e - 1 > 127 ? 127 : e - 1;
  return {copysignf(ldexpf(1.f, in), scale), (float)ldexp(m, e - in)};
}

// Two neighbouring floats of a partial, past the L2 caches (workgroups of other
// XCDs read them).
__device__ __forceinline__ void store2(float* p, float x, float y) {
  const unsigned long long v = (unsigned long long)__float_as_uint(y) << 32 | __float_as_uint(x);
  __hip_atomic_store(reinterpret_cast<unsigned long long*>(p), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 load2(const float* p) {
  const unsigned long long v = __hip_atomic_load(reinterpret_cast<const unsigned long long*>(p), __ATOMIC_RELAXED,
                                                 __HIP_MEMORY_SCOPE_AGENT);
  return make_float2(__uint_as_float((unsigned)v), __uint_as_float((unsigned)(v >> 32)));
}

// The sum over a wave, in every lane.
__device__ __forceinline__ int wave_sum(int v) {
  v += __builtin_amdgcn_update_dpp(0, v, 0xB1, 0xF, 0xF, false);   // quad_perm [1,0,3,2]
  v += __builtin_amdgcn_update_dpp(0, v, 0x4E, 0xF, 0xF, false);   // quad_perm [2,3,0,1]
  v += __builtin_amdgcn_update_dpp(0, v, 0x124, 0xF, 0xF, false);  // row_ror:4
  v += __builtin_amdgcn_update_dpp(0, v, 0x128, 0xF, 0xF, false);  // row_ror:8
  const auto x = __builtin_amdgcn_permlane16_swap((unsigned)v, (unsigned)v, false, false);
  v = (int)(x[0] + x[1]);
  const auto y = __builtin_amdgcn_permlane32_swap((unsigned)v, (unsigned)v, false, false);
  return __builtin_amdgcn_readfirstlane((int)(y[0] + y[1]));
}

// The sum over this lane and those before it; the largest of numbers >= 0.
#define RTG_SCAN(combine)                                                       \
  RTG_STEP(combine, 0x111, 0xF); /* row_shr:1 */                                \
  RTG_STEP(combine, 0x112, 0xF); /* row_shr:2 */                                \
  RTG_STEP(combine, 0x114, 0xF); /* row_shr:4 */                                \
  RTG_STEP(combine, 0x118, 0xF); /* row_shr:8 */                                \
  RTG_STEP(combine, 0x142, 0xA); /* row_bcast:15 */                             \
  RTG_STEP(combine, 0x143, 0xC)  /* row_bcast:31 */
#define RTG_STEP(combine, ctrl, rows) v = combine(v, __builtin_amdgcn_update_dpp(0, v, ctrl, rows, 0xF, false))
__device__ __forceinline__ int wave_scan(int v) {
  auto sum = [](int a, int b) { return a + b; };
  RTG_SCAN(sum);
  return v;
}
__device__ __forceinline__ int wave_max_scan(int v) {
  auto most = [](int a, int b) { return max(a, b); };
  RTG_SCAN(most);
  return v;
}
#undef RTG_STEP
#undef RTG_SCAN

// Query i of a sequence of len tokens, the last `count` of which ask: keys it sees.
__device__ __forceinline__ int keys_seen(int len, int count, int i) { return i < count ? max(len - count + i + 1, 0) : 0; }

}  // namespace rtg
