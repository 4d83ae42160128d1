// Attention over the 8-bit key/value cache (qcache.h) on i8 matrix instructions.
//
// The codes go into v_mfma_i32_16x16x64_i8 as they lie in memory; what they
// multiply is held as fixed-point numbers of ND signed 8-bit digits, an MFMA
// for each digit, so every product and sum is exact:
//   scores  S[key][query] = K Q^T: q = sq * (d2 2^16 + d1 2^8 + d0) with sq from
//           the largest |q| of the row: 24 bits, as f32 has;
//   output  O[column][query] = V^T P^T: p of a tile of 64 keys, times its
//           block's scale, over the tile's largest such product: 24 bits again.
// Results of 16-bit types take two digits (16 bits: 1.5e-5 of the row's or the
// tile's largest value, against 2e-3 and 2.4e-4 half steps of bf16 and f16).
// A wave holds 16 columns, a column being a (query, head) pair that reads one
// key/value head. Scores are computed transposed, so the lanes of a column hold
// 16 of a tile's keys each: the softmax statistics are lane-local up to two
// exchanges, and as the values' bytes are stored in the order in which a lane
// holds its keys (qcache.h), a lane's probabilities are its MFMA operand.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "attn_core.h"
#include "f16_pair.h"
#include "qcache.h"
#include "qrows.h"

namespace rtg {
namespace {

typedef int i32x4 __attribute__((ext_vector_type(4)));

// Largest fixed-point values of 3 and 2 balanced digits (127 * 65536 + 127 * 256
// + 127 and 127 * 256 + 127), less a margin for the rounding of their scales.
template <int ND>
__device__ __forceinline__ constexpr float fixed_max() {
  return ND == 3 ? 8355000.f : 32600.f;
}

__device__ __forceinline__ unsigned perm(unsigned a, unsigned b, unsigned sel) {
  return __builtin_amdgcn_perm(a, b, sel);  // bytes 0-3 of sel: of b, 4-7: of a
}

// Digit planes of four fixed-point values whose digits are the bytes of u0 .. u3
// plus 128 (the top one of ND = 3 as it is): d[i] holds digit i of the four.
template <int ND>
__device__ __forceinline__ void planes(unsigned u0, unsigned u1, unsigned u2, unsigned u3, unsigned (&d)[ND]) {
  const unsigned a = perm(u1, u0, 0x05010400), b = perm(u3, u2, 0x05010400);  // [x0 y0 x1 y1]
  d[0] = perm(b, a, 0x05040100) ^ 0x80808080u;
  d[1] = perm(b, a, 0x07060302) ^ 0x80808080u;
  if constexpr (ND == 3) d[2] = perm(perm(u3, u2, 0x0c0c0602), perm(u1, u0, 0x0c0c0602), 0x05040100);
}

// acc[0 .. ND): sums over the digits -> their value; in units of 256 for ND = 3
// (the lowest digit's sum enters as its rounded 256th).
template <int ND, int KS>
__device__ __forceinline__ i32x4 fixed_mfma(const i32x4 (&a)[KS], const i32x4 (&b)[KS][ND]) {
  const i32x4 zero = {0, 0, 0, 0};
  i32x4 lo = ND == 3 ? i32x4{128, 128, 128, 128} : zero, mid, hi = zero;
#pragma unroll
  for (int k = 0; k < KS; ++k) lo = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[k], b[k][0], lo, 0, 0, 0);
  if constexpr (ND == 3) {
    mid = lo >> 8;
#pragma unroll
    for (int k = 0; k < KS; ++k) mid = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[k], b[k][1], mid, 0, 0, 0);
  } else {
    mid = lo;
  }
#pragma unroll
  for (int k = 0; k < KS; ++k) hi = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[k], b[k][ND - 1], hi, 0, 0, 0);
  return (hi << 8) + mid;
}

// A wave's 16 columns: lane = group * 16 + column; the group's 16 (of 64) query
// elements, and 16 of a tile's keys: t * 16 + group * 4 + i.
template <int HDP, int ND>
struct Cols {
  static constexpr int KS = HDP / 64, DT = HDP / 16;
  i32x4 q[KS][ND];
  float sq;  // score units of log2 e per unit of the fixed-point sums, without the key scale
  float m, l;
  float o[DT][4];
  int lim;  // keys that this lane's column sees

  // qrow: the column's query (null: an unused column)
  template <class T>
  __device__ __forceinline__ void init(const T* qrow, int hd, bool vec, int group, float scale, int lim_) {
    lim = lim_;
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) o[d][i] = 0.f;
    float4 x[KS][4];
    unsigned top = 0;
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        x[k][e] = qrow ? load4(qrow, k * 64 + group * 16 + e * 4, hd, vec) : make_float4(0.f, 0.f, 0.f, 0.f);
        top = max(max(top, __float_as_uint(x[k][e].x) & 0x7FFFFFFFu), __float_as_uint(x[k][e].y) & 0x7FFFFFFFu);
        top = max(max(top, __float_as_uint(x[k][e].z) & 0x7FFFFFFFu), __float_as_uint(x[k][e].w) & 0x7FFFFFFFu);
      }
    {
      const auto r = __builtin_amdgcn_permlane16_swap(top, top, false, false);
      top = max(r[0], r[1]);
      const auto r2 = __builtin_amdgcn_permlane32_swap(top, top, false, false);
      top = max(r2[0], r2[1]);
    }
    // (bits order like the values, NaN above infinity)
    const float amax = __uint_as_float(top);
    const bool fine = top < 0x7F800000u;
    // below 2^-100 a row is as good as 0: no score that exp could tell from 0
    const bool zero = amax < 7.9e-31f;
    const float inv = fine && !zero ? fixed_max<ND>() / amax : 0.f;
    sq = !fine ? NAN : zero ? 0.f : amax * (scale * 1.4426950408889634f * (ND == 3 ? 256.f : 1.f) / fixed_max<ND>());
    constexpr int bias = ND == 3 ? 0x808080 : 0x8080;
#pragma unroll
    for (int k = 0; k < KS; ++k)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float xe[4] = {x[k][e].x, x[k][e].y, x[k][e].z, x[k][e].w};
        unsigned u[4], d[ND];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          u[i] = (unsigned)((int)rintf(fine ? xe[i] * inv : 0.f) + bias);
          if constexpr (ND == 3) u[i] ^= 0x800000u;  // (the top digit of planes() carries no 128)
        }
        planes<ND>(u[0], u[1], u[2], u[3], d);
#pragma unroll
        for (int i = 0; i < ND; ++i) q[k][i][e] = (int)d[i];
      }
  }
};

// A tile of keys and values in registers.
template <int HDP>
struct Tile {
  static constexpr int KS = HDP / 64, DT = HDP / 16;
  i32x4 k[4][KS], v[DT];
  float2 s;  // lane i: the scales (keys', values') of the tile's block i, over and over
  // sp: the (sequence, head)'s scales
  __device__ __forceinline__ void load_s(const float* sp, int tile, int shift, int lane) {
    s = reinterpret_cast<const float2*>(sp)[(tile << (6 - shift)) + (lane & ((1 << (6 - shift)) - 1))];
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
__device__ __forceinline__ float xmax(float v) { return xor32_max_k(xor16_max_k(v)); }
__device__ __forceinline__ float xsum(float v) { return xor32_sum_k(xor16_sum_k(v)); }

// One tile (tokens j0 .. j0 + 63) for a wave's columns. edge: some column does
// not see all of its keys; live: keys below this are in the cache (uniform).
template <int HDP, int ND>
__device__ __forceinline__ void tile_step(Cols<HDP, ND>& c, const Tile<HDP>& t, int shift, int j0, bool edge, int live,
                                          int group) {
  constexpr int DT = HDP / 16;
  // the tile's scales: of each 16 tokens; those of blocks behind the last key are not read as numbers
  float fk[4], rv[4];
  float vmax = 0.f;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int b = (i * 16) >> shift;
    const bool in = j0 + i * 16 < live;
    fk[i] = in ? lane_of(t.s.x, b) : 0.f;
    rv[i] = in ? lane_of(t.s.y, b) : 0.f;
    vmax = fmaxf(vmax, rv[i]);  // (skips NaN)
    bad |= rv[i] != rv[i];
  }
  const float rinv = vmax > 0.f ? 1.f / vmax : 0.f;
  float s[4][4];
  float top = -INFINITY;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const i32x4 d = fixed_mfma<ND, Cols<HDP, ND>::KS>(t.k[i], c.q);
    const float f = c.sq * fk[i];
#pragma unroll
    for (int e = 0; e < 4; ++e) s[i][e] = (float)d[e] * f;
  }
  if (edge) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (j0 + i * 16 + group * 4 + e >= c.lim) s[i][e] = -INFINITY;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) top = fmaxf(top, s[i][e]);
  const float mn = fmaxf(c.m, xmax(top));
  const float base = mn == -INFINITY ? 0.f : mn;  // (no key yet: every p is 2^-inf = 0)
  const float corr = __builtin_amdgcn_exp2f(c.m - base);
  float sum = 0.f, ptop = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float r = rv[i] * rinv;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float p = __builtin_amdgcn_exp2f(s[i][e] - base);
      sum += p;
      s[i][e] = edge && j0 + i * 16 + group * 4 + e >= c.lim ? 0.f : p * r;
      ptop = fmaxf(ptop, s[i][e]);
    }
  }
  if (bad) {  // a block that reads back as NaN: every column that sees a key of it is NaN
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (rv[i] != rv[i] && j0 + i * 16 + group * 4 < c.lim) sum = NAN;
  }
  c.l = c.l * corr + sum;
  if (__builtin_amdgcn_ballot_w64(mn != c.m)) {
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int i = 0; i < 4; ++i) c.o[d][i] *= corr;
  }
  c.m = mn;
  ptop = xmax(ptop);
  // (a tile whose largest product is below 2^-100 of its largest scale adds nothing)
  const float pinv = ptop > 7.9e-31f ? fixed_max<ND>() * __builtin_amdgcn_rcpf(ptop) : 0.f;
  const float w = ptop * vmax * ((ND == 3 ? 256.f : 1.f) / fixed_max<ND>());
  // p * pinv rounded to an integer and biased, in the low bits of the sum with 2^23
  constexpr float magic = ND == 3 ? 8421504.f : 8388608.f + 32896.f;  // 2^23 + 0x8080
  i32x4 pd[1][ND];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    unsigned u[4], d[ND];
#pragma unroll
    for (int e = 0; e < 4; ++e) u[e] = __float_as_uint(fmaf(s[i][e], pinv, magic));
    planes<ND>(u[0], u[1], u[2], u[3], d);
#pragma unroll
    for (int n = 0; n < ND; ++n) pd[0][n][i] = (int)d[n];
  }
#pragma unroll
  for (int d = 0; d < DT; ++d) {
    const i32x4 va[1] = {t.v[d]};
    const i32x4 r = fixed_mfma<ND, 1>(va, pd);
#pragma unroll
    for (int i = 0; i < 4; ++i) c.o[d][i] = fmaf((float)r[i], w, c.o[d][i]);
  }
}

struct AttnArgs {
  QStore c;
  const int* len;
  int len_stride, extra;
  QRows q;
  int n_q, n_q_head, group;  // group: query heads per key/value head
  const int* counts;
  float scale;
  QOut out;
  bool qvec, ovec;
  int cblocks;               // blocks of columns per (sequence, head)
  float* part;               // partial results of split keys
  int splits;
};

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

// Four neighbouring results of (sequence, query i, head): columns c4 .. c4 + 3.
template <class T>
__device__ __forceinline__ void put4(const AttnArgs& a, int seq, int i, int head, int c4, const float4& x) {
  const int hd = a.c.hd;
  if (a.out.kind == QO_ROWS) {
    T* p = static_cast<T*>(a.out.rows.p) + (long)seq * a.out.rows.seq + (long)i * a.out.rows.tok + (long)head * a.out.rows.head;
    store4(p, c4, hd, x, a.ovec);
  } else if (c4 < hd) {
    const int col = head * hd + c4, d = a.n_q_head * hd;
    const float xe[4] = {x.x, x.y, x.z, x.w};
    if (a.out.kind == QO_PAIR) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (c4 + e >= hd) continue;
        // (the scale brings the bound of the unrounded values to 2^15 at most;
        // rounded to 8 bits they are below twice that, which f16 just misses)
        float y = xe[e] * a.out.scale[col + e];
        if (fabsf(y) > 65504.f && fabsf(y) <= 65536.f) y = copysignf(65504.f, y);
        unsigned h, l;
        f16_split(y, &h, &l);
        uint16_t* p = a.out.pair + pair_index((size_t)seq * a.n_q + i, col + e, d);
        p[0] = (uint16_t)h;
        p[32] = (uint16_t)l;
      }
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (c4 + e < hd) a.out.xt[xt_index(seq, col + e, a.c.n_seq, a.out.tk)] = xe[e];
    }
  }
}

// ---- many columns: every wave has 16 of its own and takes all of their keys ----
template <int HDP, int ND, class T>
__global__ __launch_bounds__(256) void q_attend_cols_kernel(AttnArgs a) {
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, group = lane >> 4;
  const int sh = blockIdx.x, seq = sh / a.c.n_head, head = sh - seq * a.c.n_head;
  const int cb = (a.cblocks - 1 - (int)blockIdx.y * 4) - wave;  // the longest first
  if (cb < 0) return;
  const Seq r = seq_of(a, seq);
  const int ci = cb * 16 + col, i = ci / a.group, qh = head * a.group + ci - i * a.group;
  const bool mine = i < a.n_q, used = i < r.count;
  const int last = min((cb * 16 + 15) / a.group, r.count - 1);  // the wave's last query
  const int firstq = cb * 16 / a.group;
  if (firstq >= a.n_q) return;
  Cols<HDP, ND> c;
  const T* qrow = static_cast<const T*>(a.q.p) + (long)seq * a.q.seq + (long)i * a.q.tok + (long)qh * a.q.head;
  c.init(used ? qrow : nullptr, a.c.hd, a.qvec, group, a.scale, used ? visible(r, i) : 0);
  const int live = firstq < r.count ? visible(r, last) : 0;
  const int least = firstq < r.count ? visible(r, firstq) : 0;
  const int tiles = (live + kQTile - 1) / kQTile;
  const int8_t *kp = a.c.k + a.c.codes(sh), *vp = a.c.v + a.c.codes(sh);
  const float* sp = a.c.s + a.c.scales(sh);
  const int shift = a.c.block_shift;
  Tile<HDP> t;
  if (tiles) {
    t.load_s(sp, 0, shift, lane);
    t.load_k(kp, 0, lane);
  }
  for (int j = 0; j < tiles; ++j) {
    t.load_v(vp, j, lane);
    Tile<HDP> n;
    n.load_s(sp, min(j + 1, tiles - 1), shift, lane);
    n.load_k(kp, min(j + 1, tiles - 1), lane);
    tile_step(c, t, shift, j * kQTile, j * kQTile + kQTile > least, live, group);
#pragma unroll
    for (int x = 0; x < 4; ++x)
#pragma unroll
      for (int y = 0; y < Cols<HDP, ND>::KS; ++y) t.k[x][y] = n.k[x][y];
    t.s = n.s;
  }
  const float l = xsum(c.l);
  if (!mine) return;
  const float inv = c.lim > 0 ? 1.f / l : 0.f;
#pragma unroll
  for (int d = 0; d < HDP / 16; ++d) {
    const float4 x = c.lim > 0 ? make_float4(c.o[d][0] * inv, c.o[d][1] * inv, c.o[d][2] * inv, c.o[d][3] * inv)
                               : make_float4(0.f, 0.f, 0.f, 0.f);
    put4<T>(a, seq, i, qh, d * 16 + group * 4, x);
  }
}

// ---- few columns: the keys are split over workgroups and over their waves ----

constexpr int kMinTiles = 4;  // a workgroup's share of the keys is at least this many tiles

// Tiles per split and splits used for `tiles` tiles.
__device__ __forceinline__ int split_tiles(int tiles, int splits) {
  return max((tiles + splits - 1) / splits, kMinTiles);
}

// A column's partial: m, l, o[hdp].
template <int HDP>
__device__ __forceinline__ float* part_of(const AttnArgs& a, int sh, int cb, int z, int col) {
  return a.part + ((((size_t)sh * a.cblocks + cb) * a.splits + z) * 16 + col) * (HDP + 2);
}

template <int HDP, int ND, class T>
__global__ __launch_bounds__(256) void q_attend_split_kernel(AttnArgs a) {
  constexpr int NW = 4, DT = HDP / 16;
  __shared__ float sm[NW][16], sl[NW][16];
  __shared__ __attribute__((aligned(16))) float so[NW][16][HDP + 4];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, group = lane >> 4;
  const int sh = blockIdx.x, seq = sh / a.c.n_head, head = sh - seq * a.c.n_head, cb = blockIdx.y, z = blockIdx.z;
  const Seq r = seq_of(a, seq);
  const int ci = cb * 16 + col, i = ci / a.group, qh = head * a.group + ci - i * a.group;
  const bool mine = i < a.n_q, used = i < r.count;
  const int firstq = cb * 16 / a.group;
  const int last = min((cb * 16 + 15) / a.group, r.count - 1);
  const int live = firstq < r.count ? visible(r, last) : 0;
  const int least = firstq < r.count ? visible(r, firstq) : 0;
  const int tiles = (live + kQTile - 1) / kQTile, per = split_tiles(tiles, a.splits);
  const int t0 = z * per, t1 = min(t0 + per, tiles);
  if (z > 0 && t0 >= tiles) return;  // (the whole workgroup; split 0 also writes rows without keys)
  const bool whole = per >= tiles;
  Cols<HDP, ND> c;
  const T* qrow = static_cast<const T*>(a.q.p) + (long)seq * a.q.seq + (long)i * a.q.tok + (long)qh * a.q.head;
  c.init(used ? qrow : nullptr, a.c.hd, a.qvec, group, a.scale, used ? visible(r, i) : 0);
  const int8_t *kp = a.c.k + a.c.codes(sh), *vp = a.c.v + a.c.codes(sh);
  const float* sp = a.c.s + a.c.scales(sh);
  const int shift = a.c.block_shift;
  Tile<HDP> t;
  int j = t0 + wave;
  if (j < t1) {
    t.load_s(sp, j, shift, lane);
    t.load_k(kp, j, lane);
    t.load_v(vp, j, lane);
  }
  for (; j < t1; j += NW) {
    Tile<HDP> n;
    const int nj = min(j + NW, tiles - 1);
    n.load_s(sp, nj, shift, lane);
    n.load_k(kp, nj, lane);
    n.load_v(vp, nj, lane);
    tile_step(c, t, shift, j * kQTile, j * kQTile + kQTile > least, live, group);
    t = n;
  }
  const float l = xsum(c.l);
  if (group == 0) {
    sm[wave][col] = c.m;
    sl[wave][col] = l;
  }
#pragma unroll
  for (int d = 0; d < DT; ++d)
    *reinterpret_cast<float4*>(&so[wave][col][d * 16 + group * 4]) = make_float4(c.o[d][0], c.o[d][1], c.o[d][2], c.o[d][3]);
  __syncthreads();
  // four threads' worth of columns at a time: thread = (column, 4 results)
  constexpr int C4 = HDP / 4, CPP = 256 / C4;
  const int c4 = (threadIdx.x % C4) * 4;
  for (int cc = threadIdx.x / C4; cc < 16; cc += CPP) {
    const int cj = cb * 16 + cc, qi = cj / a.group, h = head * a.group + cj - qi * a.group;
    if (qi >= a.n_q) break;
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) m = fmaxf(m, sm[w][cc]);
    const float base = m == -INFINITY ? 0.f : m;
    float ls = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float f = __builtin_amdgcn_exp2f(sm[w][cc] - base);
      const float4 y = *reinterpret_cast<const float4*>(&so[w][cc][c4]);
      ls = fmaf(f, sl[w][cc], ls);
      x.x = fmaf(f, y.x, x.x);
      x.y = fmaf(f, y.y, x.y);
      x.z = fmaf(f, y.z, x.z);
      x.w = fmaf(f, y.w, x.w);
    }
    if (whole) {
      const bool any = qi < r.count && visible(r, qi) > 0;
      const float inv = 1.f / ls;
      put4<T>(a, seq, qi, h, c4,
              any ? make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv) : make_float4(0.f, 0.f, 0.f, 0.f));
    } else {
      float* p = part_of<HDP>(a, sh, cb, z, cc);
      if (c4 == 0) {
        p[0] = m;
        p[1] = ls;
      }
      p[2 + c4] = x.x;
      p[3 + c4] = x.y;
      p[4 + c4] = x.z;
      p[5 + c4] = x.w;
    }
  }
}

// Joins the splits of the columns that have more than one: a workgroup per
// column, its threads 4 results of a split each.
template <int HDP, class T>
__global__ __launch_bounds__(256) void q_attend_join_kernel(AttnArgs a) {
  constexpr int C4 = HDP / 4, ZS = 256 / C4;
  __shared__ float sm[4];
  __shared__ __attribute__((aligned(16))) float4 so[4][C4];
  __shared__ float sl[4];
  const int sh = blockIdx.x, seq = sh / a.c.n_head, head = sh - seq * a.c.n_head;
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int ci = blockIdx.y, cb = ci >> 4, qi = ci / a.group, h = head * a.group + ci - qi * a.group;
  const Seq r = seq_of(a, seq);
  const int last = min((cb * 16 + 15) / a.group, r.count - 1);
  const int live = cb * 16 / a.group < r.count ? visible(r, last) : 0;
  const int tiles = (live + kQTile - 1) / kQTile, per = split_tiles(tiles, a.splits);
  if (per >= tiles) return;
  const int n = (tiles + per - 1) / per;
  float m = -INFINITY;
  for (int z = tid; z < n; z += 256) m = fmaxf(m, part_of<HDP>(a, sh, cb, z, ci & 15)[0]);
  for (int w = 1; w < 64; w <<= 1) m = fmaxf(m, __shfl_xor(m, w));
  if (lane == 0) sm[wave] = m;
  __syncthreads();
  m = fmaxf(fmaxf(sm[0], sm[1]), fmaxf(sm[2], sm[3]));
  const float base = m == -INFINITY ? 0.f : m;
  const int c4 = (tid % C4) * 4;
  float ls = 0.f;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int z = tid / C4; z < n; z += ZS) {
    const float* p = part_of<HDP>(a, sh, cb, z, ci & 15);
    const float f = __builtin_amdgcn_exp2f(p[0] - base);
    ls = fmaf(f, p[1], ls);
    x.x = fmaf(f, p[2 + c4], x.x);
    x.y = fmaf(f, p[3 + c4], x.y);
    x.z = fmaf(f, p[4 + c4], x.z);
    x.w = fmaf(f, p[5 + c4], x.w);
  }
  for (int w = C4; w < 64; w <<= 1) {
    ls += __shfl_xor(ls, w);
    x.x += __shfl_xor(x.x, w);
    x.y += __shfl_xor(x.y, w);
    x.z += __shfl_xor(x.z, w);
    x.w += __shfl_xor(x.w, w);
  }
  if (lane < C4) so[wave][lane] = x;
  if (lane == 0) sl[wave] = ls;
  __syncthreads();
  if (tid >= C4) return;
  ls = (sl[0] + sl[1]) + (sl[2] + sl[3]);
  const float4 y0 = so[0][tid], y1 = so[1][tid], y2 = so[2][tid], y3 = so[3][tid];
  const bool any = qi < r.count && visible(r, qi) > 0;
  const float inv = 1.f / ls;
  put4<T>(a, seq, qi, h, c4,
          any ? make_float4(((y0.x + y1.x) + (y2.x + y3.x)) * inv, ((y0.y + y1.y) + (y2.y + y3.y)) * inv,
                            ((y0.z + y1.z) + (y2.z + y3.z)) * inv, ((y0.w + y1.w) + (y2.w + y3.w)) * inv)
              : make_float4(0.f, 0.f, 0.f, 0.f));
}

constexpr int kParts = 768;  // (sequence, head, column block, split)s with partials

template <int HDP, int ND, class T>
void attend(hipStream_t s, AttnArgs& a) {
  const long heads = (long)a.c.n_seq * a.c.n_head;
  if (heads * a.cblocks >= 2048) {
    const dim3 grid((unsigned)heads, (unsigned)((a.cblocks + 3) / 4));
    q_attend_cols_kernel<HDP, ND, T><<<grid, 256, 0, s>>>(a);
    return;
  }
  const int most = (a.c.tiles + kMinTiles - 1) / kMinTiles;
  a.splits = (int)std::max<long>(1, std::min<long>(most, kParts / (heads * a.cblocks)));
  const dim3 grid((unsigned)heads, (unsigned)a.cblocks, (unsigned)a.splits);
  q_attend_split_kernel<HDP, ND, T><<<grid, 256, 0, s>>>(a);
  if (a.splits > 1)
    q_attend_join_kernel<HDP, T><<<dim3((unsigned)heads, (unsigned)(a.n_q * a.group)), 256, 0, s>>>(a);
}

template <int ND, class T>
void attend_t(hipStream_t s, AttnArgs& a) {
  const int hd = a.c.hd;
  auto vec = [&](const QRows& r) {
    return hd % 4 == 0 && r.seq % 4 == 0 && r.tok % 4 == 0 && r.head % 4 == 0 &&
           reinterpret_cast<uintptr_t>(r.p) % (4 * sizeof(T)) == 0;
  };
  a.qvec = vec(a.q);
  a.ovec = a.out.kind == QO_ROWS && vec(a.out.rows);
  if (a.c.hdp == 64) attend<64, ND, T>(s, a);
  else attend<128, ND, T>(s, a);
}

}  // namespace

size_t qattn_work_bytes(int hdp) { return (size_t)kParts * 16 * (hdp + 2) * 4; }

void launch_q_attend(hipStream_t s, const QStore& c, QLen len, int extra, QType type, const QRows& q, int n_q,
                     int n_q_head, const int* counts, float scale, const QOut& out, void* work) {
  AttnArgs a{};
  a.c = c;
  a.len = len.p;
  a.len_stride = len.stride;
  a.extra = extra;
  a.q = q;
  a.n_q = n_q;
  a.n_q_head = n_q_head;
  a.group = n_q_head / c.n_head;
  a.counts = counts;
  a.scale = scale;
  a.out = out;
  a.cblocks = (int)(((long)n_q * a.group + 15) / 16);
  a.part = static_cast<float*>(work);
  a.splits = 1;
  if (type == Q_F32) attend_t<3, float>(s, a);
  else if (type == Q_BF16) attend_t<2, __bf16>(s, a);
  else attend_t<2, _Float16>(s, a);
}

}  // namespace rtg
