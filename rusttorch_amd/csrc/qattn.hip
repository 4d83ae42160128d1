// Attention over the 8-bit key/value cache (qcache.h) on i8 matrix instructions.
//
// The codes go into v_mfma_i32_16x16x64_i8 as they lie in memory; what they
// multiply is held as fixed-point numbers of three signed 8-bit digits, an MFMA
// for each digit, so every product and sum is exact:
//   scores  S[key][query] = K Q^T: q = sq * (d2 2^16 + d1 2^8 + d0) with sq from
//           the largest |q| of the row: 24 bits, as f32 has;
//   output  O[column][query] = V^T P^T: p of a tile of 64 keys, times its
//           block's scale, over the tile's largest such product: 24 bits again.
// This goes for 16-bit types too: a query's channel much larger than the rest would
// take the others' bits (with two digits f16 results were off by 8e-4 at a channel
// 100 times the rest), and 128 probabilities of 16 bits move a result by 1e-4 of
// itself, of bf16's steps by one in 40. (2047 tokens of 32 heads of 128 behind 12001
// in bf16: 693 us; two digits for the probabilities 593, for both 510.)
// A wave holds 16 columns, a column being a (query, head) pair that reads one
// key/value head. Scores are computed transposed, so the lanes of a column hold
// 16 of a tile's keys each: the softmax statistics are lane-local up to two
// exchanges, and as the values' bytes are stored in the order in which a lane
// holds its keys (qcache.h), a lane's probabilities are its MFMA operand.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "attn_core.h"
#include "f16_pair.h"
#include "lds_direct.h"
#include "qcache.h"
#include "qrows.h"
#include "qwrite.h"

namespace rtg {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

// Largest fixed-point value of three balanced digits (127 * 65536 + 127 * 256 +
// 127), less a margin for the rounding of its scale.
constexpr float kFixedMax = 8355000.f;

__device__ __forceinline__ unsigned perm(unsigned a, unsigned b, unsigned sel) {
  return __builtin_amdgcn_perm(a, b, sel);  // bytes 0-3 of sel: of b, 4-7: of a
}

// Digit planes of four fixed-point values whose digits are the bytes of u0 .. u3,
// but for the top one plus 128: d[i] holds digit i of the four.
__device__ __forceinline__ void planes(unsigned u0, unsigned u1, unsigned u2, unsigned u3, unsigned (&d)[3]) {
  const unsigned a = perm(u1, u0, 0x05010400), b = perm(u3, u2, 0x05010400);  // [x0 y0 x1 y1]
  d[0] = perm(b, a, 0x05040100) ^ 0x80808080u;
  d[1] = perm(b, a, 0x07060302) ^ 0x80808080u;
  d[2] = perm(perm(u3, u2, 0x0c0c0602), perm(u1, u0, 0x0c0c0602), 0x05040100);
}

// Sums over the digits -> their value, in units of 256 (the lowest digit's sum
// enters as its rounded 256th).
template <int KS>
__device__ __forceinline__ i32x4 fixed_mfma(const i32x4 (&a)[KS], const i32x4 (&b)[KS][3]) {
  i32x4 lo = {128, 128, 128, 128}, hi = {0, 0, 0, 0};
#pragma unroll
  for (int k = 0; k < KS; ++k) lo = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[k], b[k][0], lo, 0, 0, 0);
  i32x4 mid = lo >> 8;
#pragma unroll
  for (int k = 0; k < KS; ++k) mid = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[k], b[k][1], mid, 0, 0, 0);
#pragma unroll
  for (int k = 0; k < KS; ++k) hi = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[k], b[k][2], hi, 0, 0, 0);
  return (hi << 8) + mid;
}

// A query as three digit planes: this lane's 16 elements (of each 64) group * 16 + e,
// q[k][digit] bytes e. Returns the score in units of log2 e of 256
// units of the fixed-point sums, but for the key's scale; NaN for a row with a
// value that is not finite. The four lanes 16 apart hold a row.
template <int KS, class T>
__device__ __forceinline__ float fixed_query(const T* qrow, int hd, bool vec, int group, float scale,
                                             i32x4 (&q)[KS][3]) {
  float4 x[KS][4];
  unsigned top = 0;  // (bits order like the values, NaN above infinity)
#pragma unroll
  for (int k = 0; k < KS; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[k][e] = load4(qrow, k * 64 + group * 16 + e * 4, hd, vec);
      top = max(max(top, __float_as_uint(x[k][e].x) & 0x7FFFFFFFu), __float_as_uint(x[k][e].y) & 0x7FFFFFFFu);
      top = max(max(top, __float_as_uint(x[k][e].z) & 0x7FFFFFFFu), __float_as_uint(x[k][e].w) & 0x7FFFFFFFu);
    }
  const auto r = __builtin_amdgcn_permlane16_swap(top, top, false, false);
  top = max(r[0], r[1]);
  const auto r2 = __builtin_amdgcn_permlane32_swap(top, top, false, false);
  top = max(r2[0], r2[1]);
  float amax = __uint_as_float(top);
  const bool fine = top < 0x7F800000u;
  float down = 1.f;
  if (__builtin_amdgcn_ballot_w64(amax < 7.9e-31f)) {
    asm volatile("");
    // rows below 2^-100 are taken 2^100 times as large, so that 1 / amax is a number
    const bool tiny = amax < 7.9e-31f;
    const float up = tiny ? 1.2676506e30f : 1.f;
    amax *= up;
    down = tiny ? 7.888609e-31f : 1.f;
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        x[k][e] = make_float4(x[k][e].x * up, x[k][e].y * up, x[k][e].z * up, x[k][e].w * up);
  }
  // (a negative scale goes into the digits: the factor of the sums is not negative;
  // it comes from inv as it was rounded, or all scores would be off by its rounding)
  const float inv = fine && amax > 0.f ? copysignf(kFixedMax, scale) / amax : 0.f;
  constexpr float bias = 8421504.f;  // 0x808080: every digit plus 128
#pragma unroll
  for (int k = 0; k < KS; ++k)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float xe[4] = {x[k][e].x, x[k][e].y, x[k][e].z, x[k][e].w};
      unsigned u[4], d[3];
#pragma unroll
      for (int i = 0; i < 4; ++i) u[i] = (unsigned)rintf(fmaf(xe[i], inv, bias));  // (NaN and infinity: sq says so)
      planes(u[0], u[1], u[2], u[3], d);
      d[2] ^= 0x80808080u;
#pragma unroll
      for (int i = 0; i < 3; ++i) q[k][i][e] = (int)d[i];
    }
  // (in this order neither a large scale of small queries nor a small one of large ones leaves f32's range)
  return !fine ? NAN : amax > 0.f ? 1.4426950408889634f * 256.f / fabsf(inv) * fabsf(scale) * down : 0.f;
}

// A wave's 16 columns: lane = group * 16 + column; the group's 16 (of 64) query
// elements, and 16 of a tile's keys: t * 16 + group * 4 + i.
template <int HDP>
struct Cols {
  static constexpr int KS = HDP / 64, DT = HDP / 16;
  i32x4 q[KS][3];
  float sq;  // score units of log2 e per unit of the fixed-point sums, without the key scale
  float m, l;
  float o[DT][4];
  int lim;  // keys that this lane's column sees

  // qrow: the column's query
  template <class T>
  __device__ __forceinline__ void init(const T* qrow, int hd, bool vec, int group, float scale, int lim_) {
    lim = lim_;
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[d][i] = 0.f;
    sq = fixed_query<KS>(qrow, hd, vec, group, scale, q);
  }
};

// The scales (keys', values') of block lane % nb of those that begin at a tile.
__device__ __forceinline__ float2 block_scale(const float* sp, int tile, int nb, int shift, int lane) {
  return reinterpret_cast<const float2*>(sp)[(tile << (6 - shift)) + (lane & (nb - 1))];
}

// A tile of keys and values in registers.
template <int HDP>
struct Tile {
  static constexpr int KS = HDP / 64, DT = HDP / 16;
  i32x4 k[4][KS], v[DT];
  float2 s;  // lane i: the scales (keys', values') of the tile's block i, over and over
  // sp: the (sequence, head)'s scales
  __device__ __forceinline__ void load_s(const float* sp, int tile, int shift, int lane) {
    s = block_scale(sp, tile, kQTile >> shift, shift, lane);
  }
  // the same for lane i: the scales of the tile's key i
  __device__ __forceinline__ void load_s64(const float* sp, int tile, int shift, int lane) {
    s = reinterpret_cast<const float2*>(sp)[(tile * kQTile + lane) >> shift];
  }
  // kp, vp: the (sequence, head)'s codes
  __device__ __forceinline__ void load_k(const int8_t* kp, int tile, int lane) {
    const int8_t* p = kp + (size_t)tile * kQTile * HDP + (lane & 15) * HDP + (lane >> 4) * 16;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int s = 0; s < KS; ++s) k[t][s] = *reinterpret_cast<const i32x4*>(p + t * 16 * HDP + s * 64);
  }
  __device__ __forceinline__ void load_v(const int8_t* vp, int tile, int lane) {
    const int8_t* p = vp + (size_t)tile * kQTile * HDP + ((lane >> 4) * HDP + (lane & 15)) * 16;
#pragma unroll
    for (int d = 0; d < DT; ++d) v[d] = *reinterpret_cast<const i32x4*>(p + d * 16 * 16);
  }
};

__device__ __forceinline__ float lane_of(float v, int lane) {
  return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), lane));
}
__device__ __forceinline__ float row_max(float v) {
  v = fmaxf(v, dpp_row<0xB1>(v));
  v = fmaxf(v, dpp_row<0x4E>(v));
  v = fmaxf(v, dpp_row<0x124>(v));
  v = fmaxf(v, dpp_row<0x128>(v));
  return v;
}
__device__ __forceinline__ float xmax(float v) { return xor32_max_k(xor16_max_k(v)); }
__device__ __forceinline__ float xsum(float v) { return xor32_sum_k(xor16_sum_k(v)); }

// Scores (in units of log2 e) up to which rounding cannot take the tile's largest
// probability further above 1 than fixed_max leaves room for; beyond, the
// exponents are clamped. (A tile's fixed-point probabilities with a bit less
// doubled the error of f32 results: 8.7e-7 against 4.7e-7 of 64 bits.)
constexpr float kLargeScore = 256.f;

// The scales of NG * 16 keys (one tile, or two) in blocks of 2^SH for a wave: of
// each block f (scores) and r = v scale / vmax as lr = log2 r and 1 / r. vmax counts
// blocks that a column may not see yet, or whose scores keep them out. So where an r
// is below kLeastRatio (or 0) the blocks are taken one by one, each as the only one:
// `only` (-1: all of them) says which: it is set to 0 here where that begins, and
// the tile is taken again with the next one.
// (The test and the loops' own advance cost many columns of 128 2 to 3 %.)
constexpr float kLeastRatio = 0.000244140625f;  // 2^-12: lr's last place is 2^-20 or less, of a product's 1
template <int NG, int SH>
struct TileScales {
  static constexpr int NB = NG * 16 >> SH;
  float f[NB], lr[NB], rinv[NB], vmax;
  unsigned bad;  // bit b: the values of block b read back as NaN
  static constexpr int block(int i) { return i * 16 >> SH; }  // of the i-th 16 keys
};
// sl: a lane's (keys', values') scales, those of the keys' blocks on lanes 0 ..
// and over and over; live: keys of these that are in the cache (or more).
template <int NG, int SH>
__device__ __forceinline__ TileScales<NG, SH> tile_scales(float2 sl, int live, int lane, int& only) {
  TileScales<NG, SH> t;
  constexpr int NB = TileScales<NG, SH>::NB;
  const int block = lane & (NB - 1);
  bool in = (block << SH) < live && (only < 0 || block == only);  // blocks behind the last key are not read as numbers
  float v = in ? sl.y : 0.f;
  float m = v;  // (fmaxf skips NaN)
  if (NB > 1) m = fmaxf(m, dpp_row<0xB1>(m));
  if (NB > 2) m = fmaxf(m, dpp_row<0x4E>(m));
  if (NB > 4) m = fmaxf(m, dpp_row<0x124>(m));
  m = fmaxf(m, 0.f);
  if (NB > 1 && only < 0 && __builtin_amdgcn_ballot_w64(in && v < m * kLeastRatio)) {
    only = 0;
    in = block == 0;
    v = in ? v : 0.f;
    m = fmaxf(lane_of(v, 0), 0.f);
  }
  const float k = in ? sl.x : 0.f;
  t.bad = (unsigned)__builtin_amdgcn_ballot_w64(v != v) & ((1u << NB) - 1);
  t.vmax = m;
  // (r to the last place: it is the same for a block's every key. Keys of the other
  // blocks score 0 * sum - infinity)
  const float r = m > 0.f && v > 0.f ? v * __builtin_amdgcn_rcpf(m) : 1.f;
  const float lr = in ? __builtin_amdgcn_logf(r) : -INFINITY, ri = in ? __builtin_amdgcn_rcpf(r) : 0.f;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    t.f[b] = lane_of(k, b);
    t.lr[b] = lane_of(lr, b);
    t.rinv[b] = lane_of(ri, b);
  }
  return t;
}
// Whether the blocks of NG * 16 keys have all been taken (only is then -1 again);
// else only is the next one.
template <int NG, int SH>
__device__ __forceinline__ bool all_taken(int live, int& only) {
  only = only < 0 || (only + 1) << SH >= min(live, NG * 16) ? -1 : only + 1;
  return only < 0;
}

// A tile's keys (NG = 4), or two tiles' (8), for a wave's columns. EDGE: some
// column does not see all of them. The running maximum is of score + lr, that is
// of the probability times the value's scale, so that the largest such product
// here is 1 and needs no second reduction; each probability itself is 1 / r of it.

// k: 16 keys; s[4]: a lane's fixed-point sums of them.
template <int HDP>
__device__ __forceinline__ void tile_sums(const Cols<HDP>& c, const i32x4 (&k)[HDP / 64], float (&s)[4]) {
  const i32x4 d = fixed_mfma<HDP / 64>(k, c.q);
#pragma unroll
  for (int e = 0; e < 4; ++e) s[e] = (float)d[e];
}

// s: the keys' fixed-point sums. pd: the probabilities' digits, w: what
// their products with the values' codes are to be multiplied with.
template <bool EDGE, int HDP, int NG, int SH>
__device__ __forceinline__ void tile_probs(Cols<HDP>& c, float (&s)[NG][4], const TileScales<NG, SH>& ts, int j0,
                                           int group, i32x4 (&pd)[NG / 4][3], float& w) {
  constexpr int DT = HDP / 16, NB = TileScales<NG, SH>::NB, PER = NG / NB;  // 16s per block
  float f[NB], cc[NB];
  float top = -INFINITY;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    f[b] = c.sq * ts.f[b];
    float most = -INFINITY;
#pragma unroll
    for (int i = b * PER; i < (b + 1) * PER; ++i) {
      if (EDGE) {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          s[i][e] = j0 + i * 16 + group * 4 + e < c.lim ? fmaf(s[i][e], f[b], ts.lr[b]) : -INFINITY;
      }
      most = fmaxf(most, fmaxf(fmaxf(s[i][0], s[i][1]), fmaxf(s[i][2], s[i][3])));
    }
    top = fmaxf(top, EDGE ? most : fmaf(most, f[b], ts.lr[b]));  // (f >= 0)
  }
  top = xmax(top);
  const float base = top == -INFINITY ? 0.f : top;  // (no key here: every p is 2^-inf = 0)
#pragma unroll
  for (int b = 0; b < NB; ++b) cc[b] = ts.lr[b] - base;
#pragma unroll
  for (int i = 0; i < NG; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[i][e] = EDGE ? s[i][e] - base : fmaf(s[i][e], f[i / PER], cc[i / PER]);
  if (!EDGE && __builtin_amdgcn_ballot_w64(fabsf(top) > kLargeScore)) {
#pragma unroll
    for (int i = 0; i < NG; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        asm volatile("" : "+v"(s[i][e]));  // (stays behind the branch, which is hardly ever taken)
        s[i][e] = s[i][e] > 0.f ? 0.f : s[i][e];
      }
  }
  float sum = 0.f;
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    float part = 0.f;
#pragma unroll
    for (int i = b * PER; i < (b + 1) * PER; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) s[i][e] = __builtin_amdgcn_exp2f(s[i][e]);
      part += (s[i][0] + s[i][1]) + (s[i][2] + s[i][3]);
    }
    sum = fmaf(part, ts.rinv[b], sum);
  }
  if (ts.bad) {
    asm volatile("");
    // every column that sees a key of such a block is NaN
#pragma unroll
    for (int i = 0; i < NG; ++i)
      if ((ts.bad >> i / PER & 1) && j0 + i * 16 + group * 4 < c.lim) sum = NAN;
  }
  const float mn = fmaxf(c.m, top), mb = mn == -INFINITY ? 0.f : mn;
  const float corr = __builtin_amdgcn_exp2f(c.m - mb), g = __builtin_amdgcn_exp2f(top - mb);
  c.l = fmaf(c.l, corr, sum * g);
  // (without a branch for maxima that stay: it cost more copies of registers than it saved)
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int i = 0; i < 4; ++i) c.o[d][i] *= corr;
  c.m = mn;
  w = g * ts.vmax * (256.f / kFixedMax);
  // rounded to an integer, the digits below the top one plus 128, in the low bits of the sum with 2^23
  constexpr float magic = 8421504.f;  // 2^23 + 0x8080
#pragma unroll
  for (int i = 0; i < NG; ++i) {
    unsigned u[4], d[3];
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = __float_as_uint(fmaf(s[i][e], kFixedMax, magic));
    planes(u[0], u[1], u[2], u[3], d);
#pragma unroll
    for (int n = 0; n < 3; ++n) pd[i / 4][n][i & 3] = (int)d[n];
  }
}

// v: 16 columns of the tiles' values; o[4]: the results of them.
template <int NT>
__device__ __forceinline__ void tile_product(const i32x4 (&v)[NT], const i32x4 (&pd)[NT][3], float w, float (&o)[4]) {
  const i32x4 r = fixed_mfma<NT>(v, pd);
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] = fmaf((float)r[i], w, o[i]);
}

struct AttnArgs {
  QStore c;
  const int* len;
  int len_stride, extra;
  QRows q;
  int n_q, n_q_head, group;  // group: query heads per key/value head
  unsigned group_inv;        // ceil(2^32 / group)
  const int* counts;
  float scale;
  QOut out;
  bool qvec, ovec;
  int cblocks;               // blocks of columns per (sequence, head)
  float* part;               // partial results of split keys
  unsigned* joined;          // per block of columns: how many of its splits are done (0 between calls)
  int splits;
  QRows new_k, new_v;        // of a decode step: its token's
};

// Column x of a key/value head's (x < 2^22, group <= 1024): query x / group, and
// the query head x % group of the head's.
__device__ __forceinline__ int by_group(const AttnArgs& a, int x) {
  return a.group == 1 ? x : (int)__umulhi((unsigned)x, a.group_inv);
}
struct Column {
  int i, h;
};
__device__ __forceinline__ Column column(const AttnArgs& a, int x) {
  const int i = by_group(a, x);
  return Column{i, x - i * a.group};
}

// The sequence's queries and keys.
struct Seq {
  int len, count;
};
__device__ __forceinline__ Seq seq_of(const AttnArgs& a, int seq) {
  Seq r;
  r.len = min(max(a.len[(size_t)seq * a.len_stride] + a.extra, 0), a.c.capacity);
  r.count = a.counts ? min(max(a.counts[seq], 0), a.n_q) : a.n_q;
  return r;
}
// Keys that query i sees.
__device__ __forceinline__ int visible(const Seq& r, int i) { return max(r.len - r.count + i + 1, 0); }

// The query of a column of key/value head `head`; of one that is none, some row.
template <class T>
__device__ __forceinline__ const T* query_row(const AttnArgs& a, int seq, int head, const Column& c) {
  return static_cast<const T*>(a.q.p) + (long)seq * a.q.seq + (long)min(c.i, a.n_q - 1) * a.q.tok +
         (long)(head * a.group + c.h) * a.q.head;
}

// Where the results of (sequence, query i, head) go.
template <class T, int KIND>
struct RowOut {
  T* p;
  uint16_t* pair;
  const float* scale;
  int col0, seq;
  __device__ __forceinline__ RowOut(const AttnArgs& a, int seq_, int i, int head) {
    seq = seq_;
    col0 = head * a.c.hd;
    if constexpr (KIND == QO_ROWS) {
      p = static_cast<T*>(a.out.rows.p) + (long)seq * a.out.rows.seq + (long)i * a.out.rows.tok + (long)head * a.out.rows.head;
    } else if constexpr (KIND == QO_PAIR) {
      pair = a.out.pair + pair_index((size_t)seq * a.n_q + i, 0, a.n_q_head * a.c.hd);
      scale = a.out.scale + col0;
    }
  }
  // columns c4 .. c4 + 3
  __device__ __forceinline__ void put(const AttnArgs& a, int c4, const float4& x) const {
    if constexpr (KIND == QO_ROWS) {
      store4(p, c4, a.c.hd, x, a.ovec);
    } else {
      const float xe[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (c4 + e >= a.c.hd) continue;
        if constexpr (KIND == QO_PAIR) {
          // (the scale brings the bound of the unrounded values to 2^15 at most;
          // rounded to 8 bits they are below twice that, which f16 just misses)
          float y = xe[e] * scale[c4 + e];
          if (fabsf(y) > 65504.f && fabsf(y) <= 65536.f) y = copysignf(65504.f, y);
          unsigned h, l;
          f16_split(y, &h, &l);
          uint16_t* q = pair + pair_index(0, col0 + c4 + e, 0);
          q[0] = (uint16_t)h;
          q[32] = (uint16_t)l;
        } else {
          a.out.xt[xt_index(seq, col0 + c4 + e, a.c.n_seq, a.out.tk)] = xe[e];
        }
      }
    }
  }
};

// ---- many columns: every wave has 16 of its own and takes all of their keys ----
//
// Two tiles at a time: 128 keys share the maximum, the scales and the conversion
// of their products with the values (a third of the vector work, which bounds
// this kernel: about 237 instructions per 64 keys and 16 columns of 64 and 277 of
// 128, 86 and 69 % of the cycles; matrix instructions take 24 and 38 %. 16 x 1023
// tokens of 20 heads in f32: 120 us; 2047 tokens of 32 heads of 128 behind 12001 in
// bf16: 693 us, 630 TFLOP/s, its 194 registers leave two waves a SIMD). A workgroup's
// four waves read them from LDS, where LDS-direct loads put the next pair's keys
// once every wave has this pair's sums, and its values once every wave has its
// products. (Codes widened to f16, whose products need no joining of digits, take
// 340 instead of 513 vector instructions a pair, but twice the LDS reads, which
// then bound it: 211 against 169 us for 16 x 1023 tokens of 20 heads.)
constexpr int kPair = 2 * kQTile;

template <int HDP>
struct SharedPair {
  static constexpr int CH = HDP / 16, U = kPair * CH / 256;  // 16-byte chunks per row; units per thread
  // Rows of keys lie in chunks xor'ed with the row, so that the 16 rows of a
  // matrix operand fall on all 64 banks; values lie as in memory.
  static __device__ __forceinline__ int swizzle(int row) { return HDP == 64 ? (row >> 2) & 3 : (row >> 1) & 7; }
  static __device__ __forceinline__ int k_at(int row, int chunk) { return row * CH + (chunk ^ swizzle(row)); }
  i32x4 k[kPair * CH], v[kPair * CH];
};

template <int HDP, int SH, int KIND, class T>
__global__ __launch_bounds__(256, HDP == 64 ? 4 : 2) void q_attend_cols_kernel(AttnArgs a) {
  using Pair = SharedPair<HDP>;
  constexpr int U = Pair::U, CH = Pair::CH, KS = HDP / 64;
  __shared__ Pair t;
  const int tid = threadIdx.x, lane = tid & 63, col = lane & 15, group = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int sh = blockIdx.x, seq = sh / a.c.n_head, head = sh - seq * a.c.n_head;
  const int cb0 = a.cblocks - 1 - (int)blockIdx.y * 4, cb = cb0 - wave;  // the longest first
  const Seq r = seq_of(a, seq);
  // keys that the columns of block b see: at least, at most
  // (the later blocks of columns may be padding: the last that is not sees most;
  // columns that are none may see anything, their results go nowhere)
  const int top_cb = r.count > 0 ? min(cb0, (r.count * a.group - 1) / 16) : -1, low_cb = max(cb0 - 3, 0);
  const int live = top_cb >= low_cb ? visible(r, min(by_group(a, top_cb * 16 + 15), r.count - 1)) : 0;
  if (live == 0) {  // (all four blocks are padding, or before the first token)
    const Column cl = column(a, max(cb, 0) * 16 + col);
    if (cb < 0 || cl.i >= a.n_q) return;
    const RowOut<T, KIND> out(a, seq, cl.i, head * a.group + cl.h);
#pragma unroll
    for (int d = 0; d < HDP / 16; ++d) out.put(a, d * 16 + group * 4, make_float4(0.f, 0.f, 0.f, 0.f));
    return;
  }
  const int pairs = (live + kPair - 1) / kPair;
  // pairs that every column sees whole
  const int full = min(visible(r, by_group(a, low_cb * 16)) / kPair, pairs);
  const int8_t *kp = a.c.k + a.c.codes(sh), *vp = a.c.v + a.c.codes(sh);
  const float* sp = a.c.s + a.c.scales(sh);
  // unit u * 256 + tid of a pair in LDS: a wave's 64 are 1 KB of one tile
  const unsigned kv = (unsigned)(tid / CH * CH + ((tid % CH) ^ Pair::swizzle(tid / CH))) * 16, vv = (unsigned)tid * 16;
  const unsigned lk = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)t.k + wave * 1024;
  const unsigned lv = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)t.v + wave * 1024;
  auto fetch = [&](const int8_t* p, int j, unsigned voff, unsigned lds) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // (a second tile behind the capacity is the first once more: no key of it is seen)
      const bool second = u >= U / 2;
      const int tile = second && 2 * j + 1 < a.c.tiles ? 2 * j + 1 : 2 * j;
      load_lds16(voff, p + (size_t)tile * kQTile * HDP + (u - (second ? U / 2 : 0)) * 4096, lds + u * 4096);
    }
  };
  // a pair whose second tile no column sees is taken by its first alone
  auto half = [&](int j) { return live - j * kPair <= kQTile; };
  // (blocks of a second tile behind the capacity are those of the last one)
  auto load_s = [&](int j) {
    const int nb = (half(j) ? kQTile : kPair) >> SH, last = (a.c.tiles * kQTile >> SH) - 1;
    return reinterpret_cast<const float2*>(sp)[min((j * kPair >> SH) + (lane & (nb - 1)), last)];
  };
  fetch(kp, 0, kv, lk);
  fetch(vp, 0, vv, lv);
  float2 sl = load_s(0);
  Cols<HDP> c;
  const Column cl = column(a, max(cb, 0) * 16 + col);
  c.init(query_row<T>(a, seq, head, cl), a.c.hd, a.qvec, group, a.scale, cb >= 0 && cl.i < r.count ? visible(r, cl.i) : 0);
  wait_and_sync();
  int only = -1;
  auto step = [&](int j, auto edge, auto groups) {  // groups: of 16 keys
    constexpr int NG = decltype(groups)::value;
    float s[NG][4], w;
#pragma unroll
    for (int n = 0; n < NG; ++n) {
      i32x4 k[KS];
#pragma unroll
      for (int e = 0; e < KS; ++e) k[e] = t.k[Pair::k_at(n * 16 + col, e * 4 + group)];
      tile_sums<HDP>(c, k, s[n]);
      if (n & 1) __builtin_amdgcn_sched_barrier(0);  // (two at a time in flight: fewer registers)
    }
    wait_and_sync();  // the keys are read; the values of this pair are there
    const TileScales<NG, SH> ts = tile_scales<NG, SH>(sl, live - j * kPair, lane, only);
    const bool done = all_taken<NG, SH>(live - j * kPair, only), more = done && NG == 8 && j + 1 < pairs;
    if (more) {
      fetch(kp, j + 1, kv, lk);
      sl = load_s(j + 1);
    }
    i32x4 pd[NG / 4][3];
    tile_probs<decltype(edge)::value>(c, s, ts, j * kPair, group, pd, w);
#pragma unroll
    for (int d = 0; d < HDP / 16; ++d) {
      i32x4 v[NG / 4];
#pragma unroll
      for (int i = 0; i < NG / 4; ++i) v[i] = t.v[(i * 4 + group) * HDP + d * 16 + col];
      tile_product<NG / 4>(v, pd, w, c.o[d]);
      if (d & 1) __builtin_amdgcn_sched_barrier(0);
    }
    if (more) {
      wait_and_sync();  // the values are read; the next pair's keys are there
      fetch(vp, j + 1, vv, lv);
    }
    return (int)done;
  };
  using Pairs = std::integral_constant<int, 8>;
  int j = 0;
  while (j < full) j += step(j, std::false_type(), Pairs());
  while (j < pairs && !half(j)) j += step(j, std::true_type(), Pairs());
  while (j < pairs) j += step(j, std::true_type(), std::integral_constant<int, 4>());
  const float l = xsum(c.l);
  if (cb < 0 || cl.i >= a.n_q) return;
  const float inv = c.lim > 0 ? 1.f / l : 0.f;
  const RowOut<T, KIND> out(a, seq, cl.i, head * a.group + cl.h);
#pragma unroll
  for (int d = 0; d < HDP / 16; ++d) {
    const float* o = c.o[d];
    out.put(a, d * 16 + group * 4,
            c.lim > 0 ? make_float4(o[0] * inv, o[1] * inv, o[2] * inv, o[3] * inv) : make_float4(0.f, 0.f, 0.f, 0.f));
  }
}

// ---- few columns: the keys are split over workgroups and over their waves ----
//
// (five tokens of 16 heads of six sequences behind 700: 7 us, all of it latency:
// the launch, the queries, a tile or two, the waves' results through LDS)

// Tiles per split for `tiles` tiles over at most `splits` workgroups. All of them
// up to as many as a workgroup takes in the time of a split (2.5 to 3.5 us: the
// partials' way through memory and back): 8 heads of 128, 1000 tokens: 9.1 us
// whole, 10.1 split, 1250: 11.2 and 10.5; 16 of 64, 2000: 6.9 and 8.1, 3000: 8.1
// both; 7 columns a head of 64, 1500: 8.1 and 8.9; 8 a head of 128, 750: 8.4 and
// 9.6, 1000: 9.7 both. Then at least two or one per wave; for 16 columns, whose
// join is longer, also so many that the splits to join cost no more than their
// tiles (16 columns a head of 128, 32000: 15 tiles each 20.3 us, 8 each 26.6).
template <int HDP, int W>
__device__ __forceinline__ int split_tiles(int tiles, int splits) {
  constexpr int whole = W == 16 ? HDP == 64 ? 28 : 12 : HDP == 64 ? 40 : 16, least = HDP == 64 ? 16 : 8;
  if (tiles <= whole) return max(tiles, 1);
  const int per = W == 16 ? (int)__builtin_amdgcn_sqrtf((HDP == 64 ? 0.5f : 0.75f) * tiles) / 4 * 4 : 0;
  return max(max((tiles + splits - 1) / splits, least), per);
}

// A column's partial: m, l, o[hdp]. Blocks of W columns.
template <int HDP, int W>
__device__ __forceinline__ float* part_of(const AttnArgs& a, int sh, int cb, int z, int col) {
  return a.part + ((((size_t)sh * a.cblocks + cb) * a.splits + z) * W + col) * (HDP + 2);
}

// The waves' results of a workgroup: statistics per column and rows of o.
template <int HDP, int W, int NW>
struct Merge {
  float m[NW][W], l[NW][W];
  __attribute__((aligned(16))) float o[NW][W][HDP + 4];
  int last;
};

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

// Joins the waves' results in s (written, not yet synchronised) for the W
// columns of block cb: to the results where the keys were not split, else to the
// partials; the last of a block's workgroups to come here joins those.
template <int HDP, int W, int NW, int KIND, class T>
__device__ __forceinline__ void finish(const AttnArgs& a, Merge<HDP, W, NW>& s, const Seq& r, int seq, int sh, int head,
                                       int cb, int z, int tiles, int per) {
  constexpr int C4 = HDP / 4, NT = 64 * NW, CPP = NT / C4;
  const int tid = threadIdx.x, c4 = (tid % C4) * 4;
  const bool whole = per >= tiles;
  auto put = [&](int col, float l, const float4& x) {
    const Column cl = column(a, cb * W + col);
    const bool any = cl.i < r.count && visible(r, cl.i) > 0;
    const float inv = 1.f / l;
    RowOut<T, KIND>(a, seq, cl.i, head * a.group + cl.h).put(
        a, c4, any ? make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv) : make_float4(0.f, 0.f, 0.f, 0.f));
  };
  const int cols = min(W, a.n_q * a.group - cb * W);
  __syncthreads();
  for (int col = tid / C4; col < cols; col += CPP) {
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) m = fmaxf(m, s.m[w][col]);
    const float base = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = __builtin_amdgcn_exp2f(s.m[w][col] - base);
      const float4 y = *reinterpret_cast<const float4*>(&s.o[w][col][c4]);
      l = fmaf(f, s.l[w][col], l);
      x = make_float4(fmaf(f, y.x, x.x), fmaf(f, y.y, x.y), fmaf(f, y.z, x.z), fmaf(f, y.w, x.w));
    }
    if (whole) {
      put(col, l, x);
    } else {
      float* p = part_of<HDP, W>(a, sh, cb, z, col);
      if (c4 == 0) store2(p, m, l);
      store2(p + 2 + c4, x.x, x.y);
      store2(p + 4 + c4, x.z, x.w);
    }
  }
  if (whole) return;
  const int n = (tiles + per - 1) / per;
  __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0): the stores have completed
  __syncthreads();
  if (tid == 0) {
    unsigned* count = a.joined + ((size_t)sh * a.cblocks + cb) * kQTicketStride;
    s.last = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)n - 1;
    if (s.last) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!s.last) return;
  // A split's row over C4 threads; as many such groups to a column as there are
  // (a power of two), each taking every gpc-th split.
  constexpr int GPW = 64 / C4;  // groups per wave
  int gpc = 1;
  while (gpc * 2 * cols <= CPP) gpc *= 2;
  const int g = tid / C4, wave = tid >> 6, zg = g & (gpc - 1);
  for (int col0 = 0; col0 < cols; col0 += CPP / gpc) {
    const int col = min(col0 + g / gpc, cols - 1);
    float m = -INFINITY, l = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    // (their way through memory takes over a microsecond: U at a time)
    constexpr int U = W == 16 ? 8 : 4;
    for (int z0 = zg; z0 < n; z0 += gpc * U) {
      float2 ml[U], y[U][2];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float* p = part_of<HDP, W>(a, sh, cb, min(z0 + u * gpc, n - 1), col);
        ml[u] = load2(p);
        y[u][0] = load2(p + 2 + c4);
        y[u][1] = load2(p + 4 + c4);
      }
      float most = m;
#pragma unroll
      for (int u = 0; u < U; ++u) most = fmaxf(most, ml[u].x);
      const float base = most == -INFINITY ? 0.f : most, corr = __builtin_amdgcn_exp2f(m - base);
      m = most;
      l *= corr;
      x = make_float4(x.x * corr, x.y * corr, x.z * corr, x.w * corr);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (z0 + u * gpc >= n) break;
        const float f = __builtin_amdgcn_exp2f(ml[u].x - base);
        l = fmaf(f, ml[u].y, l);
        x = make_float4(fmaf(f, y[u][0].x, x.x), fmaf(f, y[u][0].y, x.y), fmaf(f, y[u][1].x, x.z), fmaf(f, y[u][1].y, x.w));
      }
    }
    // takes another group's results m2, l2, x2 in
    auto add = [&](float m2, float l2, const float4& x2) {
      const float most = fmaxf(m, m2), base = most == -INFINITY ? 0.f : most;
      const float f = __builtin_amdgcn_exp2f(m - base), f2 = __builtin_amdgcn_exp2f(m2 - base);
      m = most;
      l = fmaf(f, l, f2 * l2);
      x = make_float4(fmaf(f, x.x, f2 * x2.x), fmaf(f, x.y, f2 * x2.y), fmaf(f, x.z, f2 * x2.z), fmaf(f, x.w, f2 * x2.w));
    };
    for (int w = 1; w < gpc && w < GPW; w *= 2)
      add(__shfl_xor(m, w * C4), __shfl_xor(l, w * C4),
          make_float4(__shfl_xor(x.x, w * C4), __shfl_xor(x.y, w * C4), __shfl_xor(x.z, w * C4), __shfl_xor(x.w, w * C4)));
    const bool first = zg == 0;
    if (gpc > GPW) {  // (uniform) a column's waves meet in LDS
      if ((tid & 63) < C4) *reinterpret_cast<float4*>(&s.o[wave][0][c4]) = x;
      if ((tid & 63) == 0) {
        s.m[wave][0] = m;
        s.l[wave][0] = l;
      }
      __syncthreads();
      if (first)
        for (int w = 1; w < gpc / GPW; ++w)
          add(s.m[wave + w][0], s.l[wave + w][0], *reinterpret_cast<const float4*>(&s.o[wave + w][0][c4]));
      __syncthreads();
    }
    if (first && col0 + g / gpc < cols) put(col, l, x);
  }
}

template <int HDP, int SH, int KIND, class T>
__global__ __launch_bounds__(256) void q_attend_split_kernel(AttnArgs a) {
  constexpr int NW = 4;
  __shared__ Merge<HDP, 16, NW> s;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, group = lane >> 4;
  const int sh = blockIdx.x, seq = sh / a.c.n_head, head = sh - seq * a.c.n_head, cb = blockIdx.y, z = blockIdx.z;
  const Seq r = seq_of(a, seq);
  const Column cl = column(a, cb * 16 + col);
  const int firstq = by_group(a, cb * 16);
  const int last = min(by_group(a, cb * 16 + 15), r.count - 1);
  const int live = firstq < r.count ? visible(r, last) : 0;
  const int least = firstq < r.count ? visible(r, firstq) : 0;
  const int tiles = (live + kQTile - 1) / kQTile, per = split_tiles<HDP, 16>(tiles, a.splits);
  const int t0 = z * per, t1 = min(t0 + per, tiles);
  if (z > 0 && t0 >= tiles) return;  // (the whole workgroup; split 0 also writes rows without keys)
  Cols<HDP> c;
  c.init(query_row<T>(a, seq, head, cl), a.c.hd, a.qvec, group, a.scale, cl.i < r.count ? visible(r, cl.i) : 0);
  const int8_t *kp = a.c.k + a.c.codes(sh), *vp = a.c.v + a.c.codes(sh);
  const float* sp = a.c.s + a.c.scales(sh);
  Tile<HDP> t;
  int j = t0 + wave;
  auto load = [&](Tile<HDP>& x, int tile) {
    x.load_s(sp, tile, SH, lane);
    x.load_k(kp, tile, lane);
    x.load_v(vp, tile, lane);
  };
  if (j < t1) load(t, j);
  auto take = [&](const TileScales<4, SH>& ts, bool edge) {
    float sums[4][4];
    i32x4 pd[1][3];
    float w;
#pragma unroll
    for (int i = 0; i < 4; ++i) tile_sums<HDP>(c, t.k[i], sums[i]);
    if (edge) tile_probs<true>(c, sums, ts, j * kQTile, group, pd, w);
    else tile_probs<false>(c, sums, ts, j * kQTile, group, pd, w);
#pragma unroll
    for (int d = 0; d < HDP / 16; ++d) {
      const i32x4 v[1] = {t.v[d]};
      tile_product<1>(v, pd, w, c.o[d]);
    }
  };
  bool left = false;  // tiles whose scales lie far apart
  auto step = [&] {
    int only = -1;
    const TileScales<4, SH> ts = tile_scales<4, SH>(t.s, live - j * kQTile, lane, only);
    if (only < 0) take(ts, j * kQTile + kQTile > least);
    else left = true;
  };
  for (; j + NW < t1; j += NW) {
    Tile<HDP> n;
    load(n, j + NW);
    step();
    t = n;
  }
  if (j < t1) step();
  if (left) {
    // (a loop of its own: above, it would keep more in registers)
    for (j = t0 + wave; j < t1; j += NW)
      for (int only = -1;;) {
        load(t, j);
        const bool first = only < 0;
        const TileScales<4, SH> ts = tile_scales<4, SH>(t.s, live - j * kQTile, lane, only);
        if (first && only < 0) break;
        take(ts, true);
        if (all_taken<4, SH>(live - j * kQTile, only)) break;
      }
  }
  const float l = xsum(c.l);
  if (group == 0) {
    s.m[wave][col] = c.m;
    s.l[wave][col] = l;
  }
#pragma unroll
  for (int d = 0; d < HDP / 16; ++d)
    *reinterpret_cast<float4*>(&s.o[wave][col][d * 16 + group * 4]) = make_float4(c.o[d][0], c.o[d][1], c.o[d][2], c.o[d][3]);
  finish<HDP, 16, NW, KIND, T>(a, s, r, seq, sh, head, cb, z, tiles, per);
}

// ---- up to four columns: one new token of a head, or of four that share their keys ----
//
// The matrix instructions' other way round: the digits of the queries are the
// rows, the keys of a tile the columns, so the digits' sums of a score lie in one
// lane's registers 4 g .. 4 g + 2. One column (NC = 1): the 16 keys t of a tile
// meet a copy of the query that sits in rows 4 t .. 4 t + 2, all into one
// accumulator, so each of the 64 lanes has the score of one of the 64 keys. Four
// columns (NC = 4): each has four rows, a lane has four keys of one of them. The
// probabilities' digits pass through LDS into the same rows for P V, which leaves
// a lane with one result of 64 (or with every 16th of its column's). A tile then
// takes about 140 vector instructions at 64 columns (NC = 4: 300 at 128) where a
// wave of 16 columns takes 400 (700), and memory bounds long caches: 50001 tokens of 16 heads 21 us (4.8 TB/s, where a
// large copy has 5.4), 8 x 32000 of 8 heads of 128 with four columns each 81 us
// (4.9 TB/s); 16 x 960 tokens of 25 heads take 10 us, 3 of them latency.
template <int HDP, int NC>
struct FewCols {
  static constexpr int KS = HDP / 64, DT = HDP / 16, NO = NC == 1 ? HDP / 64 : DT;
  i32x4 q[NC == 1 ? 4 : 1][KS];
  float sq, m, l;
  float o[NO];
  int lim;

  // qrow: this lane's row's column's query (lane & 15: rows); lane >> 4 selects 16 of its elements
  template <class T>
  __device__ __forceinline__ void init(const T* qrow, int hd, bool vec, int lane, float scale) {
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int i = 0; i < NO; ++i) o[i] = 0.f;
    i32x4 d[KS][3];
    const float sr = fixed_query<KS>(qrow, hd, vec, lane >> 4, scale, d);
    const int row = lane & 15;
    i32x4 mine[KS];
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int x = (row & 3) == 0 ? d[k][0][e] : (row & 3) == 1 ? d[k][1][e] : d[k][2][e];
        mine[k][e] = (row & 3) == 3 ? 0 : x;
      }
    if constexpr (NC == 1) {
      sq = sr;
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int k = 0; k < KS; ++k)
#pragma unroll
          for (int e = 0; e < 4; ++e) q[t][k][e] = row >> 2 == t ? mine[k][e] : 0;
    } else {
      // this lane's column is lane >> 4: rows 4 * column + digit
      sq = __shfl(sr, (lane >> 4) * 4);
#pragma unroll
      for (int k = 0; k < KS; ++k) q[0][k] = mine[k];
    }
  }
};

__device__ __forceinline__ int fixed_sum(const i32x4& d) { return (d[2] << 8) + d[1] + ((d[0] + 128) >> 8); }
// the same with the row of ones, in units w of 256, plus what there is
__device__ __forceinline__ float add_sum(const i32x4& d, float w, float o) {
  return fmaf((float)((d[3] << 15) + (d[2] << 8) + d[1]), w, fmaf((float)d[0], w * 0.00390625f, o));
}

// A tile's largest probability as a fixed-point number from 0 to 2^24: its digits
// are those of 2^23 less, and the row behind them holds ones, whose sum times 2^23
// is what is missing: a bit more than the three digits have for numbers that are
// not negative. (Of the integers below 2^24 - 0x8080 less a margin for roundings
// the one whose inverse is nearest to a float.)
constexpr float kFewMax = 16741781.f;

// image: this wave's digit planes, [NC][4][4][16] bytes, those of digit 3 one
template <int HDP, int NC>
__device__ __forceinline__ void few_step(FewCols<HDP, NC>& c, const Tile<HDP>& t, int j0, bool edge, int live, int lane,
                                         unsigned char* image) {
  constexpr int KS = HDP / 64, DT = HDP / 16, NT = NC == 1 ? 1 : 4;  // keys per lane
  const int row = lane & 15, group = lane >> 4;
  const i32x4 zero = {0, 0, 0, 0};
  float s[NT], sv[NT];
  // key i of the lane: NC = 1: the lane's own; NC = 4: i * 16 + row
  auto key = [&](int i) { return NC == 1 ? lane : i * 16 + row; };
  float top = -INFINITY;
  if constexpr (NC == 1) {
    i32x4 d = zero;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int k = 0; k < KS; ++k) d = __builtin_amdgcn_mfma_i32_16x16x64_i8(c.q[i][k], t.k[i][k], d, 0, 0, 0);
    s[0] = (float)fixed_sum(d) * (c.sq * t.s.x);
    sv[0] = t.s.y;
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      i32x4 d = zero;
#pragma unroll
      for (int k = 0; k < KS; ++k) d = __builtin_amdgcn_mfma_i32_16x16x64_i8(c.q[0][k], t.k[i][k], d, 0, 0, 0);
      s[i] = (float)fixed_sum(d) * (c.sq * lane_of(t.s.x, i * 16));
      sv[i] = lane_of(t.s.y, i * 16);
    }
  }
  bool poison = false;  // a key that the column sees reads back as NaN
  if (edge) {
#pragma unroll
    for (int i = 0; i < NT; ++i) {
      const bool see = j0 + key(i) < c.lim;
      if (!see) {
        s[i] = -INFINITY;
        sv[i] = 0.f;
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    poison |= sv[i] != sv[i];
    top = fmaxf(top, s[i]);
  }
  top = row_max(top);
  if constexpr (NC == 1) top = xmax(top);
  const float mn = fmaxf(c.m, top), base = mn == -INFINITY ? 0.f : mn;
  const float corr = __builtin_amdgcn_exp2f(c.m - base);
  float sum = 0.f, ptop = 0.f;
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    const float p = __builtin_amdgcn_exp2f(s[i] - base);
    sum += p;
    s[i] = p * sv[i];
    ptop = fmaxf(ptop, s[i]);
  }
  if (poison) sum = NAN;
  c.l = fmaf(c.l, corr, sum);
  c.m = mn;
  ptop = row_max(ptop);
  if constexpr (NC == 1) ptop = xmax(ptop);
  const float pinv = ptop >= 1.2e-38f ? __builtin_amdgcn_rcpf(ptop) : 0.f;
  // 1 / pinv, not ptop: the instruction's error would be in all results
  const float w = fmaf(ptop, fmaf(-ptop, pinv, 1.f), ptop) * (256.f / kFewMax);
  const int column = NC == 1 ? 0 : group;
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    // the bytes of the number less 2^23 plus 0x8080 are the digits, plus 128 but for the top one
    const unsigned u = ((unsigned)rintf(s[i] * pinv * kFewMax) - 0x7F7F80u) ^ 0x8080u;
    unsigned char* p = image + column * 256 + ((key(i) >> 2) & 3) * 16 + (key(i) >> 4) * 4 + (key(i) & 3);
    p[0] = (unsigned char)u;
    p[64] = (unsigned char)(u >> 8);
    p[128] = (unsigned char)(u >> 16);
  }
  // (one wave's LDS accesses are in order; the fences are for the compiler)
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  const i32x4 pd = *reinterpret_cast<const i32x4*>(image + (NC == 1 ? 0 : (row >> 2) * 256) + (row & 3) * 64 + group * 16);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  i32x4 r[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) r[d] = __builtin_amdgcn_mfma_i32_16x16x64_i8(pd, t.v[d], zero, 0, 0, 0);
  if constexpr (NC == 1) {
    // every group of rows holds the same sums: the lanes of group g take columns 16 g .. 16 g + 15 (of each 64)
#pragma unroll
    for (int h = 0; h < HDP / 64; ++h) {
      i32x4 x;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int lo = (group & 1) ? r[h * 4 + 1][e] : r[h * 4][e], hi = (group & 1) ? r[h * 4 + 3][e] : r[h * 4 + 2][e];
        x[e] = (group & 2) ? hi : lo;
      }
      c.o[h] = add_sum(x, w, c.o[h] * corr);
    }
  } else {
#pragma unroll
    for (int d = 0; d < DT; ++d) c.o[d] = add_sum(r[d], w, c.o[d] * corr);
  }
}

constexpr int kFewWaves = 8;

// STEP: a model's decode step. The key and value of the sequence's new token,
// whose query this is, are first written into the cache by the workgroup that has
// the last tile: no other reads a key of the block that this can change.
template <int HDP, int NC, int KIND, class T, bool STEP>
__global__ __launch_bounds__(64 * kFewWaves) void q_attend_few_kernel(AttnArgs a) {
  constexpr int NW = kFewWaves;
  __shared__ Merge<HDP, NC, NW> s;
  __shared__ __attribute__((aligned(16))) unsigned char image[NW][NC * 256];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, row = lane & 15, group = lane >> 4;
  const int sh = blockIdx.x, seq = sh / a.c.n_head, head = sh - seq * a.c.n_head, z = blockIdx.z;
  const Seq r = seq_of(a, seq);
  const int live = r.count > 0 ? visible(r, r.count - 1) : 0, least = r.count > 0 ? visible(r, 0) : 0;
  const int tiles = (live + kQTile - 1) / kQTile, per = split_tiles<HDP, NC>(tiles, a.splits);
  const int t0 = z * per, t1 = min(t0 + per, tiles);
  if (z > 0 && t0 >= tiles) return;  // (the whole workgroup)
  const int8_t *kp = a.c.k + a.c.codes(sh), *vp = a.c.v + a.c.codes(sh);
  const float* sp = a.c.s + a.c.scales(sh);
  const int shift = a.c.block_shift;
  Tile<HDP> t;
  int j = t0 + wave;
  auto load = [&](Tile<HDP>& x, int tile) {
    x.load_k(kp, tile, lane);
    x.load_v(vp, tile, lane);
    x.load_s64(sp, tile, shift, lane);
  };
  const bool fresh = STEP && j == tiles - 1;  // (this wave's first tile is the one that is written to)
  if (j < t1 && !fresh) load(t, j);
  for (int i = lane; i < NC * 64; i += 64) reinterpret_cast<unsigned*>(image[wave])[i] = (i & 63) < 48 ? 0 : 0x01010101u;
  FewCols<HDP, NC> c;
  if constexpr (STEP) {
    const bool writes = t1 == tiles;
    const OneToken<HDP, T, NW> token(a.c, seq, head, a.new_k, a.new_v, writes);
    c.init(query_row<T>(a, seq, head, column(a, 0)), a.c.hd, a.qvec, lane, a.scale);
    if (writes) {
      token.write(a.c, Place{r.len - 1, r.len - 1, r.len, r.len - 1, 0}, sh);
      __syncthreads();  // (a workgroup's stores are seen by its loads behind a barrier)
      if (fresh) load(t, j);
    }
  } else {
    c.init(query_row<T>(a, seq, head, column(a, NC == 1 ? 0 : row >> 2)), a.c.hd, a.qvec, lane, a.scale);
  }
  const int qi = by_group(a, NC == 1 ? 0 : group);
  c.lim = qi < r.count ? visible(r, qi) : 0;
  auto step = [&] { few_step<HDP, NC>(c, t, j * kQTile, j * kQTile + kQTile > least, live, lane, image[wave]); };
  for (; j + NW < t1; j += NW) {
    Tile<HDP> n;
    load(n, j + NW);
    step();
    t = n;
  }
  if (j < t1) step();  // (a load behind the last tile, though nobody needs it, would be waited for)
  float l = row16_sum_k(c.l);
  if constexpr (NC == 1) l = xsum(l);
  if (row == 0 && (NC > 1 || group == 0)) {
    s.m[wave][NC == 1 ? 0 : group] = c.m;
    s.l[wave][NC == 1 ? 0 : group] = l;
  }
#pragma unroll
  for (int i = 0; i < FewCols<HDP, NC>::NO; ++i) {
    if constexpr (NC == 1) s.o[wave][0][i * 64 + group * 16 + row] = c.o[i];
    else s.o[wave][group][i * 16 + row] = c.o[i];
  }
  finish<HDP, NC, NW, KIND, T>(a, s, r, seq, sh, head, 0, z, tiles, per);
}

// Workgroups of split keys: as many as the device holds at once, which the
// registers decide (few columns: 120 and 181 of them, 16 columns: 156 and 249).
template <int HDP>
constexpr int parts(bool few) {
  return few ? HDP == 64 ? 512 : 256 : HDP == 64 ? 768 : 512;
}
constexpr int kParts = 1024;

// Blocks of 16 columns from which every wave takes all keys of its own. hdp 64:
// 1.4 for each of the device's 1024 SIMDs; below, splitting the keys fills it
// better (1264 blocks: 184 against 231 us over 15000 keys, 19.2 against 21.0 for
// prompts of 1023), above it only reads them more often (1548: 13.3 against 10.4,
// 2000: 46.7 against 24.7). hdp 128: what it reads counts earlier (bf16, 640: 204
// against 244 us over 12000 keys, 14.5 against 11.7 for a prompt of 320; 800: 248
// against 244, 17.3 against 14.4 for one of 400).
template <int HDP>
constexpr long kManyBlocks = HDP == 64 ? 1400 : 800;

// How many workgroups split a (sequence, head)'s block of columns' keys, at most.
template <int HDP>
dim3 split_grid(AttnArgs& a, bool few) {
  const long heads = (long)a.c.n_seq * a.c.n_head;
  if (few) a.cblocks = 1;
  const int most = (a.c.tiles + 7) / 8;
  a.splits = (int)std::max<long>(1, std::min<long>(most, parts<HDP>(few) / (heads * a.cblocks)));
  return dim3((unsigned)heads, (unsigned)a.cblocks, (unsigned)a.splits);
}

template <int HDP, int KIND, class T>
void attend(hipStream_t s, AttnArgs& a) {
  const long heads = (long)a.c.n_seq * a.c.n_head;
  const int columns = a.n_q * a.group, sh = a.c.block_shift;
  const dim3 grid = split_grid<HDP>(a, columns <= 4);
  if (columns == 1) {
    if constexpr (KIND == QO_ROWS) q_attend_few_kernel<HDP, 1, KIND, T, false><<<grid, 64 * kFewWaves, 0, s>>>(a);
  } else if (columns <= 4) {
    q_attend_few_kernel<HDP, 4, KIND, T, false><<<grid, 64 * kFewWaves, 0, s>>>(a);
  } else if (heads * a.cblocks >= kManyBlocks<HDP>) {
    const dim3 wide((unsigned)heads, (unsigned)((a.cblocks + 3) / 4));
    if (sh == 4) q_attend_cols_kernel<HDP, 4, KIND, T><<<wide, 256, 0, s>>>(a);
    else if (sh == 5) q_attend_cols_kernel<HDP, 5, KIND, T><<<wide, 256, 0, s>>>(a);
    else q_attend_cols_kernel<HDP, 6, KIND, T><<<wide, 256, 0, s>>>(a);
  } else {
    if (sh == 4) q_attend_split_kernel<HDP, 4, KIND, T><<<grid, 256, 0, s>>>(a);
    else if (sh == 5) q_attend_split_kernel<HDP, 5, KIND, T><<<grid, 256, 0, s>>>(a);
    else q_attend_split_kernel<HDP, 6, KIND, T><<<grid, 256, 0, s>>>(a);
  }
}

bool vec4(const QRows& r, int hd, size_t size) {
  return hd % 4 == 0 && r.seq % 4 == 0 && r.tok % 4 == 0 && r.head % 4 == 0 &&
         reinterpret_cast<uintptr_t>(r.p) % (4 * size) == 0;
}

template <class T>
void attend_t(hipStream_t s, AttnArgs& a) {
  if constexpr (sizeof(T) == 4) {
    if (a.out.kind == QO_PAIR) return attend<64, QO_PAIR, T>(s, a);
  }
  if (a.c.hdp == 64) attend<64, QO_ROWS, T>(s, a);
  else attend<128, QO_ROWS, T>(s, a);
}

}  // namespace

// the partials, then the counters
static size_t part_bytes(int hdp) { return (size_t)kParts * 16 * (hdp + 2) * 4; }
size_t qattn_work_bytes(int hdp) { return part_bytes(hdp) + (size_t)kParts * kQTicketStride * 4; }
void qattn_work_clear(hipStream_t s, void* work, int hdp) {
  (void)hipMemsetAsync(static_cast<char*>(work) + part_bytes(hdp), 0, (size_t)kParts * kQTicketStride * 4, s);
}

namespace {
AttnArgs attn_args(const QStore& c, QLen len, int extra, QType type, const QRows& q, int n_q, int n_q_head,
                   const int* counts, float scale, const QOut& out, void* work) {
  AttnArgs a{};
  a.c = c;
  a.len = len.p;
  a.len_stride = len.stride;
  a.extra = extra;
  a.q = q;
  a.n_q = n_q;
  a.n_q_head = n_q_head;
  a.group = n_q_head / c.n_head;
  a.group_inv = (unsigned)((0x100000000ull + a.group - 1) / a.group);
  a.counts = counts;
  a.scale = scale;
  a.out = out;
  const size_t size = type == Q_F32 ? 4 : 2;
  a.qvec = vec4(q, c.hd, size);
  a.ovec = out.kind == QO_ROWS && vec4(out.rows, c.hd, size);
  a.cblocks = (int)(((long)n_q * a.group + 15) / 16);
  a.part = static_cast<float*>(work);
  a.joined = reinterpret_cast<unsigned*>(static_cast<char*>(work) + part_bytes(c.hdp));
  return a;
}
}  // namespace

void launch_q_attend(hipStream_t s, const QStore& c, QLen len, int extra, QType type, const QRows& q, int n_q,
                     int n_q_head, const int* counts, float scale, const QOut& out, void* work) {
  AttnArgs a = attn_args(c, len, extra, type, q, n_q, n_q_head, counts, scale, out, work);
  if (type == Q_F32) attend_t<float>(s, a);
  else if (type == Q_BF16) attend_t<__bf16>(s, a);
  else attend_t<_Float16>(s, a);
}

void launch_q_step(hipStream_t s, const QStore& c, QLen len, const QRows& k, const QRows& v, const QRows& q,
                   float scale, const QOut& out, void* work) {
  AttnArgs a = attn_args(c, len, 1, Q_F32, q, 1, c.n_head, nullptr, scale, out, work);
  a.new_k = k;
  a.new_v = v;
  const dim3 grid = split_grid<64>(a, true);
  if (out.kind == QO_XT) q_attend_few_kernel<64, 1, QO_XT, float, true><<<grid, 64 * kFewWaves, 0, s>>>(a);
  else if (out.kind == QO_PAIR) q_attend_few_kernel<64, 1, QO_PAIR, float, true><<<grid, 64 * kFewWaves, 0, s>>>(a);
  else q_attend_few_kernel<64, 1, QO_ROWS, float, true><<<grid, 64 * kFewWaves, 0, s>>>(a);
}

}  // namespace rtg
