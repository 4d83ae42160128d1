// Attention over the 4-bit cache (fourbit.h) for few queries, and the weights
// that queries give the cache's tokens.
//
// A wave holds 16 columns, a column being a (query, head) pair that reads one
// key/value head, and takes 32 tokens at a time:
//   scores  S[token][column] = K Q^T on v_mfma_f32_16x16x32_bf16. A lane's 16
//           bytes of codes are its matrix operands, four codes of channels to a
//           conversion with the scale in it. bf16 holds every number of the cache
//           exactly, and a query is the sum of as many bf16 parts as its type has
//           bits for (f32 three, f16 two), so that products are exact and sums f32;
//   output  O[channel][column] = V^T P^T. Scores are computed transposed: the
//           lanes of a column hold 8 of the 32 tokens each, in the order in which
//           the values' codes lie, so that a lane's probabilities are its matrix
//           operand. They are taken as two bf16 parts (16 bits) where results are
//           bf16 or f16, as three (24) where they are f32.
// The softmax's running maximum is only raised where a score passes it by 2^8: sums
// stay far within f32, and most tiles need no exchange between lanes.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "attn_core.h"
#include "fourbit_core.h"

namespace rtg {
namespace {

constexpr int kWaves = 8, kWeighWaves = 4;
constexpr int kWhole = 32, kSplitTiles = 8;  // tiles that are not split; of a split at least
constexpr float kSlack = 8.f;     // powers of two that a score may pass the maximum by

struct Args {
  FStore c;
  const int* len;
  QRows q, out;
  int n_q, n_q_head, group, cblocks;
  const int* counts;
  float query, sum;  // ScoreScale
  float* stats;
  bool qvec, ovec;
  int room;           // workgroups that the keys are split over; 0: they are not
  unsigned* tickets;  // [seq][head][cblock][kQTicketStride]
  float* parts;       // [workgroup][column][hdp + 2]
};

// What a workgroup works on: part z of n of the tiles that a sequence, head and
// block of columns have, `per` to a part.
struct Work {
  int seq, head, cb, z, n, per;
  int slot0, stride;  // workgroup of part z: slot0 + z * stride
  int ticket;
};

struct Column {
  int i, h;  // query, head within the group; i >= n_q: none
};
__device__ __forceinline__ Column column(const Args& a, int col) {
  Column r;
  r.i = a.group == 1 ? col : col / a.group;
  r.h = col - r.i * a.group;
  return r;
}
template <class T>
__device__ __forceinline__ T* row_of(const QRows& r, int seq, int i, int head) {
  return static_cast<T*>(r.p) + seq * r.seq + i * r.tok + head * r.head;
}

__device__ __forceinline__ float2& stats_of(const Args& a, int seq, int i, int head) {
  return reinterpret_cast<float2*>(a.stats)[((size_t)seq * a.n_q + i) * a.n_q_head + head];
}

// A column's query as matrix operands, this lane's quarter: channels CK g + 8 j + e.
// Loads and conversion are apart, so that loads of keys can be asked for in between.
template <int HDP, int QP, class T>
struct Query {
  static constexpr int J = HDP / 32;
  float x[J][8];
  u4v q[J][QP];
  __device__ __forceinline__ void load(const Args& a, int seq, int head, const Column& cl, int g) {
    const T* row = row_of<const T>(a.q, seq, min(cl.i, a.n_q - 1), head * a.group + cl.h);
#pragma unroll
    for (int j = 0; j < J; ++j) load8(row, HDP / 4 * g + 8 * j, a.c.hd, a.qvec, x[j]);
  }
  __device__ __forceinline__ void convert(const Args& a) {
#pragma unroll
    for (int j = 0; j < J; ++j) {
#pragma unroll
      for (int e = 0; e < 8; ++e) x[j][e] *= a.query;
      bf16_parts<QP>(x[j], q[j]);
    }
  }
};

// A tile's keys as they lie: this lane's quarter of tokens m and 16 + m.
template <int HDP>
struct Keys {
  static constexpr int J = HDP / 32;
  u4v c[HDP / 64];
  unsigned s[2];
  __device__ __forceinline__ void load(const uint8_t* k, const uint8_t* sk, int lane) {
#pragma unroll
    for (int i = 0; i < HDP / 64; ++i) c[i] = *reinterpret_cast<const u4v*>(k + i * 1024 + lane * 16);
    const int at = HDP == 128 ? lane : (lane >> 5) * 16 + (lane & 15);
    s[0] = sk[at];
    s[1] = sk[HDP / 2 + at];
  }
  // operand j of tokens b * 16 + m
  __device__ __forceinline__ u4v eight(int b, int j) const {
    return eight_bf16(HDP == 128 ? c[HDP == 128 ? b : 0][j] : c[0][b * 2 + (j & 1)], scale_of(s[b]));
  }
  // scores of tokens b * 16 + 4 g + i
  template <int QP>
  __device__ __forceinline__ f32x4 scores(int b, const u4v (&q)[J][QP]) const {
    f32x4 r = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < J; ++j) {
      const u4v k = eight(b, j);
#pragma unroll
      for (int p = 0; p < QP; ++p) r = mfma16(k, q[j][p], r);
    }
    return r;
  }
};

// A tile's values as they lie: this lane's CV channels of tokens b * 16 + 4 g + i,
// and their scales (byte b * 4 + i).
template <int HDP>
struct Values {
  static constexpr int CV = HDP / 16;
  u4v c[HDP / 64];
  unsigned s[2];
  __device__ __forceinline__ void load(const uint8_t* v, const uint8_t* sv, int lane) {
#pragma unroll
    for (int i = 0; i < HDP / 64; ++i) c[i] = *reinterpret_cast<const u4v*>(v + i * 1024 + lane * 16);
    const int g = lane >> 4, group = (lane & 15) * CV / 32;
    const uint2 x = *reinterpret_cast<const uint2*>(sv + (g * (HDP / 32) + group) * 8);
    s[0] = x.x;
    s[1] = x.y;
  }
  // o[d] += the products of channel CV m + d with the columns' probabilities
  template <int PP>
  __device__ __forceinline__ void add(const u4v (&p)[PP], f32x4 (&o)[CV]) const {
    float scale[8];
#pragma unroll
    for (int r = 0; r < 8; ++r) scale[r] = scale_of((s[r / 4] >> (r % 4 * 8)) & 255u);
    auto pairs = [&](auto pair) {  // channels CV m + 2 pair, + 1
      constexpr int PR = decltype(pair)::value;
      unsigned t[8];
      if constexpr (HDP == 128) {
#pragma unroll
        for (int r = 0; r < 8; ++r) t[r] = two_bf16<PR>(c[r / 4][r % 4], scale[r]);
      } else {  // two tokens to a word
#pragma unroll
        for (int r = 0; r < 8; r += 2) {
          t[r] = two_bf16<PR>(c[0][r / 2], scale[r]);
          t[r + 1] = two_bf16<PR + 2>(c[0][r / 2], scale[r + 1]);
        }
      }
      u4v lo, hi;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        lo[i] = low_halves(t[2 * i], t[2 * i + 1]);
        hi[i] = high_halves(t[2 * i], t[2 * i + 1]);
      }
#pragma unroll
      for (int k = 0; k < PP; ++k) {
        o[2 * PR] = mfma16(lo, p[k], o[2 * PR]);
        o[2 * PR + 1] = mfma16(hi, p[k], o[2 * PR + 1]);
      }
    };
    pairs(std::integral_constant<int, 0>{});
    pairs(std::integral_constant<int, 1>{});
    if constexpr (HDP == 128) {
      pairs(std::integral_constant<int, 2>{});
      pairs(std::integral_constant<int, 3>{});
    }
  }
  // Whether a value of this lane's reads back as NaN (or lies behind the sequence).
  __device__ __forceinline__ bool any_nan() const {
    const unsigned a = ~s[0], b = ~s[1];  // a byte of 0 in one of them
    return (((a - 0x01010101u) & ~a) | ((b - 0x01010101u) & ~b)) & 0x80808080u;
  }
  // Makes the scales of tokens from `live` on, which hold anything, and of values
  // that read back as NaN 0; the first of these tokens goes to *bad if it is lower.
  __device__ __forceinline__ void clean(int first, int live, int g, int* bad) {
#pragma unroll
    for (int r = 0; r < 8; ++r) {
      const unsigned byte = (s[r / 4] >> (r % 4 * 8)) & 255u;
      const int t = first + r / 4 * 16 + 4 * g + r % 4;
      if (t < live && byte == 255u) *bad = min(*bad, t);
      if (t >= live || byte == 255u) s[r / 4] &= ~(255u << (r % 4 * 8));
    }
  }
};

struct Seq {
  int len, count;
};
__device__ __forceinline__ Seq seq_of(const Args& a, int seq) {
  Seq r;
  r.len = a.len[seq];
  r.count = a.counts ? min(max(a.counts[seq], 0), a.n_q) : a.n_q;
  return r;
}

template <int HDP>
struct Shared {
  float m[kWaves][kCols], l[kWaves][kCols];
  __attribute__((aligned(16))) float o[kWaves][kCols][HDP + 4];
  int last;
};

// Joins the waves' results in s for the columns of a block: to the results where
// the keys were not split, else to the partials; the last of its workgroups to come
// here joins those.
template <int HDP, class T>
__device__ __forceinline__ void finish(const Args& a, Shared<HDP>& s, const Seq& r, const Work& wk) {
  const int seq = wk.seq, head = wk.head, cb = wk.cb, n = wk.n;
  constexpr int C4 = HDP / 4, STEP = 64 * kWaves / C4;
  const int tid = threadIdx.x, c4 = tid % C4 * 4;
  const int cols = min(kCols, a.n_q * a.group - cb * kCols);
  auto put = [&](int col, float m, float l, const float4& x) {
    const Column cl = column(a, cb * kCols + col);
    const bool any = keys_seen(r.len, r.count, cl.i) > 0;
    const float inv = 1.f / l;
    store4(row_of<T>(a.out, seq, cl.i, head * a.group + cl.h), c4, a.c.hd,
           any ? make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv) : make_float4(0.f, 0.f, 0.f, 0.f), a.ovec);
    if (a.stats && c4 == 0) stats_of(a, seq, cl.i, head * a.group + cl.h) = make_float2(m, any ? l : 0.f);
  };
  __syncthreads();
  for (int col = tid / C4; col < cols; col += STEP) {
    float m = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) m = fmaxf(m, s.m[w][col]);
    const float base = m == -INFINITY ? 0.f : m;
    float l = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = __builtin_amdgcn_exp2f(s.m[w][col] - base);
      const float4 y = *reinterpret_cast<const float4*>(&s.o[w][col][c4]);
      l = fmaf(f, s.l[w][col], l);
      x = make_float4(fmaf(f, y.x, x.x), fmaf(f, y.y, x.y), fmaf(f, y.z, x.z), fmaf(f, y.w, x.w));
    }
    if (n == 1) {
      put(col, m, l, x);
    } else {
      float* p = a.parts + ((size_t)(wk.slot0 + wk.z * wk.stride) * kCols + col) * (HDP + 2);
      if (c4 == 0) store2(p, m, l);
      store2(p + 2 + c4, x.x, x.y);
      store2(p + 4 + c4, x.z, x.w);
    }
  }
  if (n == 1) return;
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the stores have completed
  __syncthreads();
  if (tid == 0) {
    unsigned* count = a.tickets + (size_t)wk.ticket * kQTicketStride;
    s.last = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (unsigned)n - 1;
    if (s.last) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!s.last) return;
  // a column's splits over as many groups of C4 threads as there are, each taking every GPC-th
  int gpc = 1;
  while (gpc * 2 * cols <= STEP) gpc *= 2;
  const int group = tid / C4, zg = group % gpc;
  for (int col0 = 0; col0 < cols; col0 += STEP / gpc) {
    const int col = min(col0 + group / gpc, cols - 1);
    const float* p0 = a.parts + ((size_t)wk.slot0 * kCols + col) * (HDP + 2);
    const size_t part = (size_t)wk.stride * kCols * (HDP + 2);
    float m = -INFINITY, l = 0.f;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    constexpr int U = 8;  // (their way through memory takes over a microsecond: U at a time)
    for (int z0 = zg; z0 < n; z0 += U * gpc) {
      float2 ml[U], y[U][2];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float* p = p0 + min(z0 + u * gpc, n - 1) * part;
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
    if (gpc > 1) {  // (uniform) the groups meet in LDS: group g in row g
      __syncthreads();
      float* row = &s.o[0][0][0] + (size_t)group * (HDP + 4);
      *reinterpret_cast<float4*>(row + c4) = x;
      if (c4 == 0) {
        row[HDP] = m;
        row[HDP + 1] = l;
      }
      __syncthreads();
      if (zg != 0) continue;
      for (int g = 1; g < gpc; ++g) {
        const float* other = row + (size_t)g * (HDP + 4);
        const float m2 = other[HDP], most = fmaxf(m, m2), base = most == -INFINITY ? 0.f : most;
        const float f = __builtin_amdgcn_exp2f(m - base), f2 = __builtin_amdgcn_exp2f(m2 - base);
        const float4 y = *reinterpret_cast<const float4*>(other + c4);
        m = most;
        l = fmaf(f, l, f2 * other[HDP + 1]);
        x = make_float4(fmaf(f, x.x, f2 * y.x), fmaf(f, x.y, f2 * y.y), fmaf(f, x.z, f2 * y.z), fmaf(f, x.w, f2 * y.w));
      }
    }
    if (col0 + group / gpc < cols) put(col, m, l, x);
  }
}

// Workgroup (sequence and head, block of columns); or, where the keys are split, one
// of `room` that get about as many tiles each, so that sequences of different
// lengths are done at the same time (8 of 16000 to 32000 tokens of 8 heads of 128:
// 54 us with as many parts for each, 50 so). Blocks of padding take one each, which
// only writes zeros, and leave the others to those that read keys.
__device__ __forceinline__ Work work_of(const Args& a) {
  Work w;
  w.z = 0;
  w.n = 1;
  w.per = 0;
  if (a.room == 0) {
    w.seq = (int)blockIdx.x / a.c.n_head;
    w.head = (int)blockIdx.x - w.seq * a.c.n_head;
    w.cb = (int)blockIdx.y;
    w.slot0 = w.stride = w.ticket = 0;
    return w;
  }
  const int lane = threadIdx.x & 63, heads = a.c.n_head, inner = heads * a.cblocks;
  // the tiles, and the blocks of columns with queries in them, of the sequences s0 + lane
  auto tiles_at = [&](int s0) { return s0 + lane < a.c.n_seq ? (a.len[s0 + lane] + kFTile - 1) / kFTile : 0; };
  auto busy_at = [&](int s0) { return s0 + lane < a.c.n_seq ? (seq_of(a, s0 + lane).count * a.group + kCols - 1) / kCols : 0; };
  auto parts_of = [&](int tiles, int each) { return tiles <= kWhole ? 1 : (tiles + each - 1) / each; };
  int total = 0, idle = a.c.n_seq * inner;
  for (int s0 = 0; s0 < a.c.n_seq; s0 += 64) {
    const int busy = busy_at(s0) * heads;
    total += wave_sum(tiles_at(s0) * busy);
    idle -= wave_sum(busy);
  }
  // the fewest tiles to a part, or up to a 16th more, with which there are not too many parts
  const int room = a.room - idle;
  int each = max((total + room - 1) / room, kSplitTiles);
  for (;; each += each / 16 + 1) {
    int parts = 0;
    for (int s0 = 0; s0 < a.c.n_seq; s0 += 64) parts += wave_sum(busy_at(s0) * heads * parts_of(tiles_at(s0), each));
    if (parts <= room) break;  // (each block has one where `each` is large; there are at most half as many blocks as workgroups)
  }
  int at = (int)blockIdx.x;
  w.seq = -1;
  for (int s0 = 0; s0 < a.c.n_seq; s0 += 64) {
    const int tiles = tiles_at(s0), parts = parts_of(tiles, each), busy = busy_at(s0);
    const int mine_all = s0 + lane < a.c.n_seq ? inner + busy * heads * (parts - 1) : 0;
    const int incl = wave_scan(mine_all);
    const unsigned long long mine = __builtin_amdgcn_ballot_w64(at >= incl - mine_all && at < incl);
    if (mine) {
      const int l = __builtin_ctzll(mine), n = __builtin_amdgcn_readlane(parts, l), b = __builtin_amdgcn_readlane(busy, l);
      w.seq = s0 + l;
      const int rest = at - __builtin_amdgcn_readlane(incl - mine_all, l), split = b * heads * n;
      w.stride = b * heads;
      if (rest < split) {
        w.n = n;
        w.per = (__builtin_amdgcn_readlane(tiles, l) + n - 1) / n;
        w.z = rest / w.stride;
        const int pair = rest - w.z * w.stride;
        w.head = pair / b;
        w.cb = pair - w.head * b;
      } else {
        const int none = a.cblocks - b;
        w.head = (rest - split) / none;
        w.cb = b + rest - split - w.head * none;
      }
      w.slot0 = (int)blockIdx.x - w.z * w.stride;
      w.ticket = w.seq * inner + w.head * a.cblocks + w.cb;
      return w;
    }
    at -= __builtin_amdgcn_readlane(incl, 63);
  }
  return w;
}

template <int HDP, int QP, int PP, class T>
__global__ __launch_bounds__(64 * kWaves) void f_attend_kernel(Args a) {
  constexpr int CV = HDP / 16;
  __shared__ Shared<HDP> s;
  const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, g = lane >> 4;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const Work wk = work_of(a);
  if (wk.seq < 0) return;
  const int seq = wk.seq, head = wk.head, sh = seq * a.c.n_head + head, cb = wk.cb;
  const Column cl = column(a, cb * kCols + n);
  Query<HDP, QP, T> q;
  q.load(a, seq, head, cl, g);
  const Seq r = seq_of(a, seq);
  // keys that the block's columns see: at most, at least (columns that are none may see anything)
  // (a block of padding none: 60 queries' room for one of each of 64 sequences, 8 heads of 64
  // behind 8000 tokens in f32, takes 76 us, 303 where they all go over the keys)
  const int first_i = column(a, cb * kCols).i, last_i = min(column(a, cb * kCols + kCols - 1).i, r.count - 1);
  const int live = first_i < r.count ? keys_seen(r.len, r.count, last_i) : 0;
  const int least = keys_seen(r.len, r.count, first_i);
  const int tiles = (live + kFTile - 1) / kFTile;
  const int t0 = wk.z * wk.per, t1 = wk.n == 1 ? tiles : min(t0 + wk.per, tiles);
  const int lim = keys_seen(r.len, r.count, cl.i);
  f32x4 o[CV];
#pragma unroll
  for (int d = 0; d < CV; ++d) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;
  int bad = INT32_MAX;  // the first token whose values of this lane's group of channels are NaN
  const uint8_t *kc = a.c.k + a.c.codes(sh), *vc = a.c.v + a.c.codes(sh);
  const uint8_t *ks = a.c.sk + a.c.scales(sh), *vs = a.c.sv + a.c.scales(sh);
  Keys<HDP> k;
  Values<HDP> v;
  auto fetch = [&](int t) {
    k.load(kc + (size_t)t * 16 * HDP, ks + (size_t)t * HDP, lane);
    v.load(vc + (size_t)t * 16 * HDP, vs + (size_t)t * HDP, lane);
  };
  // (one tile of a wave ahead: two or three take registers and no time off)
  int t = t0 + wave;
  if (t < t1) fetch(t);
  q.convert(a);
  while (t < t1) {
    const Keys<HDP> k1 = k;
    Values<HDP> v1 = v;
    const int at = t * kFTile;
    t += kWaves;
    if (t < t1) fetch(t);
    float p[8];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
      const f32x4 x = k1.scores(b, q.q);
#pragma unroll
      for (int i = 0; i < 4; ++i) p[b * 4 + i] = x[i];
    }
    const bool edge = at + kFTile > least;  // (uniform)
    if (edge || __builtin_amdgcn_ballot_w64(v1.any_nan())) v1.clean(at, live, g, &bad);
    if (edge) {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (at + e / 4 * 16 + 4 * g + e % 4 >= lim) p[e] = -INFINITY;
    }
    float top = p[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) top = fmaxf(top, p[e]);
    if (__builtin_amdgcn_ballot_w64(top * a.sum > m + kSlack)) {
      top = xor32_max_k(xor16_max_k(top)) * a.sum;
      // (each column by itself: its result does not depend on its neighbours')
      const float f = top > m + kSlack ? __builtin_amdgcn_exp2f(m - top) : 1.f;
      m = top > m + kSlack ? top : m;
      l *= f;
#pragma unroll
      for (int d = 0; d < CV; ++d) o[d] *= f;
    }
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = __builtin_amdgcn_exp2f(fmaf(p[e], a.sum, -base));
    if (edge) {
#pragma unroll
      for (int e = 0; e < 8; ++e) p[e] = at + e / 4 * 16 + 4 * g + e % 4 < lim ? p[e] : 0.f;
    }
    u4v pp[PP];
    bf16_parts<PP>(p, pp);
#pragma unroll
    for (int e = 0; e < 8; ++e) l += p[e];
    v1.add(pp, o);
  }
  l = xor32_sum_k(xor16_sum_k(l));
  if (__builtin_amdgcn_ballot_w64(bad != INT32_MAX)) {
    // lane (g, m) has looked at the group of m's channels; its results are of the group of channels CV 4 g
    for (int x = 1; x < 64; x *= 2)
      if (x >= 16 || x < 32 / CV) bad = min(bad, __shfl_xor(bad, x, 64));
    bad = __shfl(bad, CV * 4 * g / 32 * (32 / CV), 64);
#pragma unroll
    for (int d = 0; d < CV; ++d)
      if (bad < lim) o[d] = f32x4{NAN, NAN, NAN, NAN};
  }
  if (g == 0) {
    s.m[wave][n] = m;
    s.l[wave][n] = l;
  }
  // o[d][e]: channel CV (4 g + e) + d of column n
#pragma unroll
  for (int e = 0; e < 4; ++e)
#pragma unroll
    for (int d = 0; d < CV; d += 4)
      *reinterpret_cast<float4*>(&s.o[wave][n][CV * (4 * g + e) + d]) = make_float4(o[d][e], o[d + 1][e], o[d + 2][e], o[d + 3][e]);
  finish<HDP, T>(a, s, r, wk);
}

// ---- weights ----

// A workgroup takes some of a head's tiles, a wave every fourth of them, and goes
// over the columns: the scores once more, and the sum of their exponentials over
// the columns' sums. Nothing but the keys is read, and each token's weight has one
// owner: no atomics, and sums in a fixed order. The queries lie in LDS as matrix
// operands, as many columns at a time as fit; a wave's next tile is loaded while it
// works on one (one token of 32 heads of 128 over 8 x 16000 in f16: 36 us with a
// tile or four to a wave and queries from memory, 17 so).
constexpr int kWeighBytes = 32 * 1024;  // of queries in LDS

template <int HDP, int QP>
struct Weigh {
  static constexpr int J = HDP / 32, BLOCKS = kWeighBytes / (J * QP * 64 * 16) < 1 ? 1 : kWeighBytes / (J * QP * 64 * 16);
  u4v q[BLOCKS][J][QP][64];
  float2 st[BLOCKS][kCols];  // a column's m, and one over its sum
  int lim[BLOCKS][kCols];    // the keys that it sees
};

template <int HDP, int QP, class T>
__global__ __launch_bounds__(256) void f_weigh_kernel(Args a, float decay) {
  typedef Weigh<HDP, QP> W;
  __shared__ W s;
  const int lane = threadIdx.x & 63, n = lane & 15, g = lane >> 4, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int sh = blockIdx.x, seq = sh / a.c.n_head, head = sh - seq * a.c.n_head;
  const Seq r = seq_of(a, seq);
  const int tiles = (r.len + kFTile - 1) / kFTile, step = (int)gridDim.y * kWeighWaves;
  if ((int)blockIdx.y * kWeighWaves >= tiles) return;
  const int cblocks = (r.count * a.group + kCols - 1) / kCols;
  const uint8_t *kc = a.c.k + a.c.codes(sh), *ks = a.c.sk + a.c.scales(sh);
  float* w = a.c.w + a.c.weights(sh);
  for (int cb0 = 0; cb0 == 0 || cb0 < cblocks; cb0 += W::BLOCKS) {
    const int blocks = min(W::BLOCKS, cblocks - cb0);
    int t = (int)blockIdx.y * kWeighWaves + wave;
    Keys<HDP> next;
    if (t < tiles) next.load(kc + (size_t)t * 16 * HDP, ks + (size_t)t * HDP, lane);
    if (cb0 > 0) __syncthreads();
    for (int b = wave; b < blocks; b += kWeighWaves) {
      const Column cl = column(a, (cb0 + b) * kCols + n);
      Query<HDP, QP, T> q;
      q.load(a, seq, head, cl, g);
      q.convert(a);
#pragma unroll
      for (int j = 0; j < W::J; ++j)
#pragma unroll
        for (int p = 0; p < QP; ++p) s.q[b][j][p][lane] = q.q[j][p];
      if (g == 0) {
        const float2 st = stats_of(a, seq, min(cl.i, a.n_q - 1), head * a.group + cl.h);
        s.st[b][n] = make_float2(st.x, 1.f / st.y);
        s.lim[b][n] = keys_seen(r.len, r.count, cl.i);
      }
    }
    __syncthreads();
    for (; t < tiles; t += step) {
      const Keys<HDP> k = next;
      if (t + step < tiles) next.load(kc + (size_t)(t + step) * 16 * HDP, ks + (size_t)(t + step) * HDP, lane);
      const int at = t * kFTile;
      u4v keys[2][W::J];
#pragma unroll
      for (int j = 0; j < W::J; ++j) {
        keys[0][j] = k.eight(0, j);
        keys[1][j] = k.eight(1, j);
      }
      float sum[8] = {};
      for (int b = 0; b < blocks; ++b) {
        f32x4 x[2] = {};
#pragma unroll
        for (int j = 0; j < W::J; ++j)
#pragma unroll
          for (int p = 0; p < QP; ++p) {
            const u4v q = s.q[b][j][p][lane];
            x[0] = mfma16(keys[0][j], q, x[0]);
            x[1] = mfma16(keys[1][j], q, x[1]);
          }
        const float2 st = s.st[b][n];
        const int lim = s.lim[b][n] - at;  // (of the tile's tokens, in this column)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float p = __builtin_amdgcn_exp2f(fmaf(x[e / 4][e % 4], a.sum, -st.x)) * st.y;
          sum[e] += e / 4 * 16 + 4 * g + e % 4 < lim ? p : 0.f;
        }
      }
      // The sums over a row's 16 lanes: of two lanes each hands half of its sums over and
      // keeps the others, until lane n has number n / 2 (22 instructions, 40 one by one).
      float four[4], two[2];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        four[e] = (n & 8 ? sum[e + 4] : sum[e]) + dpp_row<0x128>(n & 8 ? sum[e] : sum[e + 4]);  // row_ror:8
#pragma unroll
      for (int e = 0; e < 2; ++e)
        two[e] = (n & 4 ? four[e + 2] : four[e]) + dpp_row<0x141>(n & 4 ? four[e] : four[e + 2]);  // row_half_mirror
      float mine = (n & 2 ? two[1] : two[0]) + dpp_row<0x4E>(n & 2 ? two[0] : two[1]);  // quad_perm [2,3,0,1]
      mine += dpp_row<0xB1>(mine);                                                      // quad_perm [1,0,3,2]
      const int tok = at + (n >> 3) * 16 + 4 * g + (n >> 1 & 3);
      if ((n & 1) == 0 && tok < r.len) {
        const float before = cb0 > 0 ? 1.f : decay;
        w[tok] = before == 0.f ? mine : fmaf(before, w[tok], mine);
      }
    }
  }
}

Args args_of(const FAttn& f) {
  Args a;
  a.c = f.c;
  a.len = f.len;
  a.q = f.q;
  a.out = f.out;
  a.n_q = f.n_q;
  a.n_q_head = f.n_q_head;
  a.group = f.n_q_head / f.c.n_head;
  a.cblocks = (f.n_q * a.group + kCols - 1) / kCols;
  a.counts = f.counts;
  const ScoreScale sc = score_scale(f.scale);
  a.query = sc.query;
  a.sum = sc.sum;
  a.stats = f.stats;
  a.qvec = by_eights(f.q, f.c.hd, f.type);
  a.ovec = by_eights(f.out, f.c.hd, f.type);
  a.room = 0;
  a.tickets = static_cast<unsigned*>(f.work);
  a.parts = reinterpret_cast<float*>(static_cast<char*>(f.work) + 2 * kTicketBytes);
  return a;
}

template <int QP, int PP, class T>
void attend_t(hipStream_t s, const FAttn& f) {
  Args a = args_of(f);
  // Keys are split over workgroups where there are too few blocks of columns to
  // fill the device (one workgroup of eight waves a compute unit: 8 x 32000 tokens of
  // 8 heads of 128 in 49 us, with two of them or twice as many of four waves 58 and
  // 62, as the partial results take their time), and more than 32 tiles, for a join
  // takes as long as four rounds of the eight waves.
  const long blocks = (long)f.c.n_seq * f.c.n_head * a.cblocks;
  const int room = few_room(f.c.sizes());
  if (f.c.tiles > kWhole && blocks * 2 <= room) a.room = room;
  const dim3 grid = a.room ? dim3((unsigned)a.room) : dim3((unsigned)(f.c.n_seq * f.c.n_head), (unsigned)a.cblocks);
  if (f.c.hdp == 64) f_attend_kernel<64, QP, PP, T><<<grid, 64 * kWaves, 0, s>>>(a);
  else f_attend_kernel<128, QP, PP, T><<<grid, 64 * kWaves, 0, s>>>(a);
}
template <int QP, class T>
void weigh_t(hipStream_t s, const FAttn& f, float decay) {
  const Args a = args_of(f);
  // as many workgroups as the device takes at once
  const long sh = (long)f.c.n_seq * f.c.n_head, most = std::max(1l, 1024 / sh);
  const dim3 grid((unsigned)sh, (unsigned)std::min(most, (long)(f.c.tiles + kWeighWaves - 1) / kWeighWaves));
  if (f.c.hdp == 64) f_weigh_kernel<64, QP, T><<<grid, 256, 0, s>>>(a, decay);
  else f_weigh_kernel<128, QP, T><<<grid, 256, 0, s>>>(a, decay);
}

}  // namespace

size_t fattn_work_bytes(const FStore& c) { return 2 * kTicketBytes + fattn_parts_bytes(c.sizes()); }
void fattn_work_clear(hipStream_t s, void* work) { (void)hipMemsetAsync(work, 0, 2 * kTicketBytes, s); }

void launch_f_attend(hipStream_t s, const FAttn& f) {
  const int type = f.type == Q_F32 ? 0 : f.type == Q_BF16 ? 1 : 2;
  if (for_many(f.c.sizes(), type, (long)f.n_q * (f.n_q_head / f.c.n_head))) return launch_f_attend_many(s, f);
  if (f.type == Q_F32) attend_t<3, 3, float>(s, f);
  else if (f.type == Q_BF16) attend_t<1, 2, __bf16>(s, f);
  else attend_t<2, 2, _Float16>(s, f);
}
void launch_f_weigh(hipStream_t s, const FAttn& f, float decay) {
  if (f.type == Q_F32) weigh_t<3, float>(s, f, decay);
  else if (f.type == Q_BF16) weigh_t<1, __bf16>(s, f, decay);
  else weigh_t<2, _Float16>(s, f, decay);
}

}  // namespace rtg
