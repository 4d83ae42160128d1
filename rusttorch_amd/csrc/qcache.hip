// Writing the 8-bit key/value cache and reading it back; see qcache.h for what
// it holds.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "attn_core.h"
#include "qcache.h"
#include "qrows.h"
#include "qwrite.h"

namespace rtg {

void qstore_shape(QStore* c, int n_seq, int n_head, int hd, int capacity, int block) {
  c->n_seq = n_seq;
  c->n_head = n_head;
  c->hd = hd;
  c->hdp = hd <= 64 ? 64 : 128;
  c->block = block;
  c->block_shift = block == 16 ? 4 : block == 32 ? 5 : 6;
  c->capacity = capacity;
  c->tiles = (capacity + kQTile - 1) / kQTile;
}

namespace {
struct Parts {
  size_t codes, scales, tail, tail_s;
  explicit Parts(const QStore& c) {
    const size_t sh = (size_t)c.n_seq * c.n_head;
    auto up = [](size_t x) { return (x + 255) / 256 * 256; };
    codes = up(c.codes(sh));
    scales = up(c.scales(sh) * 4);
    tail = up(c.tails(sh, 0) * 4);
    tail_s = up(c.tail_scales(sh, 0) * 4);
  }
};
}  // namespace

size_t qstore_bytes(const QStore& c) {
  const Parts p(c);
  return 2 * p.codes + p.scales + p.tail + p.tail_s;
}

void qstore_place(QStore* c, void* mem) {
  const Parts p(*c);
  char* m = static_cast<char*>(mem);
  auto take = [&](size_t n) {
    char* r = m;
    m += n;
    return r;
  };
  c->k = reinterpret_cast<int8_t*>(take(p.codes));
  c->v = reinterpret_cast<int8_t*>(take(p.codes));
  c->s = reinterpret_cast<float*>(take(p.scales));
  c->tail = reinterpret_cast<float*>(take(p.tail));
  c->tail_s = reinterpret_cast<float*>(take(p.tail_s));
}

namespace {

// The workgroup's Place, read by its first thread, which then counts the
// workgroup as one that has read its sequence's length; finish() by the last of
// a sequence's workgroups (per_head of each head) writes the new one. The loads
// have returned before the barrier (their values went through LDS), so no
// workgroup can see the new length in place of the old. This saves the launch of
// a kernel for the lengths alone (3 us of the host's time, 2 of the GPU's).
class Turn {
 public:
  __device__ __forceinline__ Place begin(Place* shared, const QStore& c, int sh, const QLen& len, QTickets tickets,
                                         int n_new, const int* counts, const int* start) {
    tickets_ = tickets;
    seq_ = sh / c.n_head;
    if (threadIdx.x == 0) *shared = place(seq_, len.p, len.stride, n_new, counts, start, c.capacity);
    __syncthreads();
    mine_ = tickets.count + ((size_t)c.n_seq + sh) * kQTicketStride;
    if (threadIdx.x == 0 && tickets.count) before_ = add(mine_);
    return *shared;
  }
  __device__ __forceinline__ void finish(const Place& p, const QStore& c, const QLen& len, unsigned per_head) {
    if (threadIdx.x != 0 || !tickets_.count || before_ != per_head - 1) return;
    *mine_ = 0;
    unsigned* all = tickets_.count + (size_t)seq_ * kQTicketStride;
    if (add(all) != (unsigned)c.n_head - 1) return;
    *all = 0;
    if (p.bad) atomicMin(tickets_.err, (unsigned)seq_ * 4 + p.bad);
    else len.p[(size_t)seq_ * len.stride] = p.end;
  }

 private:
  static __device__ __forceinline__ unsigned add(unsigned* p) {
    return __hip_atomic_fetch_add(p, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  QTickets tickets_;
  unsigned* mine_ = nullptr;
  int seq_ = 0;
  unsigned before_ = 0;
};

// The integers nearest to x / s, ties to even, |x / s| <= 127, as the bytes of a
// word: r = x * (1 / s) rounded by adding 1.5 * 2^23, whose sum's low byte is r.
// That may be one off next to a border between two codes; x - r s says on which
// side x lies (it is exact there: a multiple of half s's last place below 2^24
// of those), and is looked at again where it reaches half of s, which few words do.
__device__ __forceinline__ unsigned low_bytes(unsigned a, unsigned b, unsigned c, unsigned d) {
  return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0c0c0400), __builtin_amdgcn_perm(b, a, 0x0c0c0400),
                               0x05040100);
}
__device__ __forceinline__ unsigned codes_of(const float4& x, float s, float inv) {
  if (!(s > 0.f)) return 0;
  constexpr float magic = 12582912.f;
  const float t[4] = {fmaf(x.x, inv, magic), fmaf(x.y, inv, magic), fmaf(x.z, inv, magic), fmaf(x.w, inv, magic)};
  float r[4] = {t[0] - magic, t[1] - magic, t[2] - magic, t[3] - magic};
  const float far = fmaxf(fmaxf(fabsf(fmaf(-r[0], s, x.x)), fabsf(fmaf(-r[1], s, x.y))),
                          fmaxf(fabsf(fmaf(-r[2], s, x.z)), fabsf(fmaf(-r[3], s, x.w))));
  if (far < 0.5f * s)
    return low_bytes(__float_as_uint(t[0]), __float_as_uint(t[1]), __float_as_uint(t[2]), __float_as_uint(t[3]));
  r[0] = code_of(x.x, s, r[0]);
  r[1] = code_of(x.y, s, r[1]);
  r[2] = code_of(x.z, s, r[2]);
  r[3] = code_of(x.w, s, r[3]);
  return low_bytes((unsigned)(int)r[0], (unsigned)(int)r[1], (unsigned)(int)r[2], (unsigned)(int)r[3]);
}
__device__ __forceinline__ unsigned max_abs4(const float4& x) {
  return max(max(abs_bits(x.x), abs_bits(x.y)), max(abs_bits(x.z), abs_bits(x.w)));
}

// Whether the append needs the tail that is there: it goes on in the middle of
// the block that the tail holds.
__device__ __forceinline__ bool reads_tail(const QStore& c, const Place& p) {
  return (p.from & ~(c.block - 1)) < p.at && in_tail(c, p);
}

// q[i]: byte i of x[0] .. x[3] (and the other way round).
__device__ __forceinline__ void transpose4(const unsigned (&x)[4], unsigned (&q)[4]) {
  const unsigned a = __builtin_amdgcn_perm(x[1], x[0], 0x05010400), b = __builtin_amdgcn_perm(x[3], x[2], 0x05010400);
  const unsigned c = __builtin_amdgcn_perm(x[1], x[0], 0x07030602), d = __builtin_amdgcn_perm(x[3], x[2], 0x07030602);
  q[0] = __builtin_amdgcn_perm(b, a, 0x05040100);
  q[1] = __builtin_amdgcn_perm(b, a, 0x07060302);
  q[2] = __builtin_amdgcn_perm(d, c, 0x05040100);
  q[3] = __builtin_amdgcn_perm(d, c, 0x07060302);
}

// The tail of an append that reads the old one and whose last block starts behind
// its first tile: written by the first tile's workgroup, which has read the old
// tail by then.
template <int HDP, class T>
__device__ void append_tail(const QStore& c, const Place& p, size_t sh, int which, const T* src, long tok_stride,
                            bool vec) {
  constexpr int LPR = HDP / 4, TPP = 256 / LPR, ROWS = 64 / TPP;
  const int c4 = (threadIdx.x % LPR) * 4, trow = threadIdx.x / LPR;
  const int last = (p.end - 1) & ~(c.block - 1);
  float* tail = c.tail + c.tails(sh, which);
  float* tail_s = c.tail_s + c.tail_scales(sh, which);
  float4 x[ROWS];
  // (all rows in flight, those behind the end as the last one: one after the
  // other they took most of a short append's time, 18.9 us against 10)
#pragma unroll
  for (int i = 0; i < ROWS; ++i)
    x[i] = load4(src + (long)(min(last + i * TPP + trow, p.end - 1) - p.at) * tok_stride, c4, c.hd, vec);
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int t = i * TPP + trow;
    const float amax = __uint_as_float(row_max_bits<HDP>(max_abs4(x[i])));
    if (last + t < p.end) {  // (t < block)
      *reinterpret_cast<float4*>(tail + (size_t)t * HDP + c4) = x[i];
      if (c4 == 0) tail_s[t] = __uint_as_float(token_scale(amax));
    }
  }
}

// One tile (64 tokens) of one (sequence, head) of an append, keys (which = 0)
// or values: the y-th tile that the new tokens touch. A thread has 4 columns of
// 4 neighbouring tokens (a quad), a quad's columns lie on 16 or 32 neighbouring
// lanes. The first tile's workgroup also quantises the block's earlier tokens
// anew; the last block's writes the tail.
template <int HDP, class T>
__device__ __forceinline__ void append_tile(const QStore& c, const Place& p, size_t sh, int y, int which, const T* src,
                                            long tok_stride, bool vec, unsigned* blkmax, unsigned* image) {
  constexpr int LPR = HDP / 4, QPP = 256 / LPR, PASSES = 16 / QPP;  // lanes per quad, quads per pass
  const int tid = threadIdx.x, c4 = (tid % LPR) * 4, qrow = tid / LPR;
  const int tile0 = (p.from / kQTile + y) * kQTile;  // first token of the tile
  const int blk0 = p.from & ~(c.block - 1);
  const int first = y == 0 ? blk0 : tile0, hi = min(p.end, tile0 + kQTile);
  const bool tailed = in_tail(c, p);
  float* tail = c.tail + c.tails(sh, which);
  float* tail_s = c.tail_s + c.tail_scales(sh, which);
  int8_t* codes = (which ? c.v : c.k) + c.codes(sh);
  float* scales = c.s + c.scales(sh) + which;

  // the block's earlier tokens (uniform; y == 0), rows outside as the nearest of
  // them: asked for before the new rows, so that both are in flight together
  const bool earlier = first < p.at;
  auto old = [&](int i, int e) { return min(max(tile0 + (i * QPP + qrow) * 4 + e, first), p.at - 1); };
  float4 o[PASSES][4];        // tailed: values
  unsigned os[PASSES][4];     // and their tokens' scales; else words of codes: a token's, or a quad's by column
  float old_s;
  if (earlier && tailed) {
#pragma unroll
    for (int i = 0; i < PASSES; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        o[i][e] = *reinterpret_cast<const float4*>(tail + (size_t)(old(i, e) - blk0) * HDP + c4);
        os[i][e] = __float_as_uint(tail_s[old(i, e) - blk0]);
      }
  } else if (earlier) {
    old_s = scales[2 * (blk0 >> c.block_shift)];
#pragma unroll
    for (int i = 0; i < PASSES; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        os[i][e] = *reinterpret_cast<const unsigned*>(codes + (which ? value_byte(old(i, 0) & ~3, c4 + e, HDP)
                                                                     : (size_t)old(i, e) * HDP + c4));
  }
  float4 x[PASSES][4];
  unsigned ts[PASSES][4];
#pragma unroll
  for (int i = 0; i < PASSES; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) x[i][e] = make_float4(0.f, 0.f, 0.f, 0.f);
  if (p.end > p.at) {
    // (rows outside are read as the nearest inside, so that no load waits for a branch)
#pragma unroll
    for (int i = 0; i < PASSES; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int tok = tile0 + (i * QPP + qrow) * 4 + e;
        x[i][e] = load4(src + (long)(min(max(tok, p.at), hi - 1) - p.at) * tok_stride, c4, c.hd, vec);
      }
  }
  if (tid < 4) blkmax[tid] = 0;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < PASSES; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const int tok = tile0 + (i * QPP + qrow) * 4 + e;
      ts[i][e] = token_scale(__uint_as_float(row_max_bits<HDP>(max_abs4(x[i][e]))));
      if (tok < p.at || tok >= hi) {
        x[i][e] = make_float4(0.f, 0.f, 0.f, 0.f);
        ts[i][e] = 0;
      }
    }
  if (earlier) {
    if (!tailed) {
#pragma unroll
      for (int i = 0; i < PASSES; ++i) {
        unsigned q[4] = {os[i][0], os[i][1], os[i][2], os[i][3]};
        if (which) transpose4(os[i], q);  // (a quad's four tokens lie side by side, by column)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          o[i][e] = make_float4(code_value((int8_t)q[e], old_s), code_value((int8_t)(q[e] >> 8), old_s),
                                code_value((int8_t)(q[e] >> 16), old_s), code_value((int8_t)(q[e] >> 24), old_s));
      }
#pragma unroll
      for (int i = 0; i < PASSES; ++i)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          os[i][e] = read_back_scale(__uint_as_float(row_max_bits<HDP>(max_abs4(o[i][e]))), old_s);
    }
#pragma unroll
    for (int i = 0; i < PASSES; ++i)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int tok = tile0 + (i * QPP + qrow) * 4 + e;
        if (tok >= first && tok < p.at) {
          x[i][e] = o[i][e];
          ts[i][e] = os[i][e];
        }
      }
  }
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const unsigned m = max(max(ts[i][0], ts[i][1]), max(ts[i][2], ts[i][3]));
    if (c4 == 0) atomicMax(&blkmax[((i * QPP + qrow) * 4) >> c.block_shift], m);
  }
  __syncthreads();  // (also: every read of the tail, the scales and the codes is done)
  const int last = (p.end - 1) >> c.block_shift;  // the block that the tail is to hold
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int quad = i * QPP + qrow, tok0 = tile0 + quad * 4;
    const float s = __uint_as_float(blkmax[(quad * 4) >> c.block_shift]), inv = scale_inv(s);
    unsigned q[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) q[e] = codes_of(x[i][e], s, inv);
    if (which == 0) {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (tok0 + e >= first && tok0 + e < hi) *reinterpret_cast<unsigned*>(codes + (size_t)(tok0 + e) * HDP + c4) = q[e];
    } else {
      // the quad's bytes by column; they leave in order of the image
      unsigned r[4];
      transpose4(q, r);
      unsigned* im = image + ((quad & 3) * HDP + c4) * 4 + (quad >> 2);
#pragma unroll
      for (int e = 0; e < 4; ++e) im[4 * e] = r[e];
    }
    if (c4 == 0 && (tok0 & (c.block - 1)) == 0 && tok0 >= first && tok0 < hi) scales[2 * (tok0 >> c.block_shift)] = s;
    // the tail, unless the first tile's workgroup may still be reading the old one (then: append_tail)
    if (tok0 >> c.block_shift == last && (y == 0 || !reads_tail(c, p))) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int tok = tok0 + e;
        if (tok >= first && tok < hi && !(tailed && tok < p.at)) {
          *reinterpret_cast<float4*>(tail + (size_t)(tok & (c.block - 1)) * HDP + c4) = x[i][e];
          if (c4 == 0) tail_s[tok & (c.block - 1)] = __uint_as_float(ts[i][e]);
        }
      }
    }
  }
  if (which == 1) {
    // the values leave in whole quads (bytes of tokens behind the end are not part of the cache)
    __syncthreads();
    for (int j = tid; j < 4 * HDP; j += 256) {
      const int g = j / HDP;
      const uint4 im = *reinterpret_cast<const uint4*>(image + j * 4);
      unsigned* dst = reinterpret_cast<unsigned*>(codes + (size_t)tile0 * HDP + (size_t)j * 16);
      if (first <= tile0 && hi == tile0 + kQTile) {
        *reinterpret_cast<uint4*>(dst) = im;
      } else {
        const unsigned w[4] = {im.x, im.y, im.z, im.w};
#pragma unroll
        for (int t = 0; t < 4; ++t) {
          const int tok = tile0 + t * 16 + g * 4;
          if (tok >= first && tok < hi) dst[t] = w[t];
        }
      }
    }
  }
}

// A workgroup per (sequence, head, tile) and side (keys, values). Any such append
// takes 5.6 us of latency (two tokens of 8 x 12 heads of 64: launch, length, rows,
// stores; one that goes on in a block of 128 columns 8.9: its earlier tokens too);
// behind that memory bounds it (8 x 1000 tokens in f32: 14.8 to 17 us; 4000 take 36.6
// us more, 5.0 TB/s), unless the workgroups do not fill the device (4 x 517 of 8
// heads of 128 in bf16: 640 of them, 12.6 us, 3.4 TB/s behind its 8.9).
template <int HDP, class T>
__global__ __launch_bounds__(256) void q_append_kernel(QStore c, QLen len, QTickets tickets, QRows k, QRows v, int n_new,
                                                       const int* __restrict__ counts, const int* __restrict__ start,
                                                       bool vec) {
  __shared__ unsigned blkmax[4];
  __shared__ Place shared;
  __shared__ __attribute__((aligned(16))) unsigned image[kQTile * HDP / 4];
  const int sh = blockIdx.x, seq = sh / c.n_head, head = sh - seq * c.n_head, y = blockIdx.y, which = blockIdx.z;
  Turn turn;
  const Place p = turn.begin(&shared, c, sh, len, tickets, n_new, counts, start);
  const int tile0 = (p.from / kQTile + y) * kQTile;
  if (!p.bad && (p.end > p.at || p.at < p.len) && (y == 0 || tile0 < p.end)) {
    const QRows& r = which ? v : k;
    const T* src = static_cast<const T*>(r.p) + seq * r.seq + head * r.head;
    append_tile<HDP, T>(c, p, sh, y, which, src, r.tok, vec, blkmax, image);
    if (y == 0 && p.end > tile0 + kQTile && reads_tail(c, p)) append_tail<HDP, T>(c, p, sh, which, src, r.tok, vec);
  }
  turn.finish(p, c, len, gridDim.y * 2);
}

// One new token (or only a cut) for each sequence: a workgroup per (sequence, head).
// Latency bounds it: 3.8 us for 16 sequences of 25 heads, 400 workgroups, where no
// token raises its block's scale. Among so many one nearly always does, and its
// block is written anew, two waves taking its tokens by turns: 5.8 us a token on
// average over a block of 32, 7.7 of 64 (128 columns, 8 x 8 heads: 7.9 and 10.9).
template <int HDP, class T>
__global__ __launch_bounds__(256) void q_append_one_kernel(QStore c, QLen len, QTickets tickets, QRows k, QRows v,
                                                           int n_new, const int* __restrict__ counts,
                                                           const int* __restrict__ start) {
  __shared__ Place shared;
  const int sh = blockIdx.x, seq = sh / c.n_head, head = sh - seq * c.n_head;
  const OneToken<HDP, T, 4> token(c, seq, head, k, v, n_new > 0);
  Turn turn;
  const Place p = turn.begin(&shared, c, sh, len, tickets, n_new, counts, start);
  if (!p.bad && (p.end > p.at || p.at < p.len)) token.write(c, p, sh);
  turn.finish(p, c, len, 1);
}

// code * s rounded to f32 before anything else is done with it: without the
// empty asm the compiler makes one instruction of the product and its conversion
// to f16, which then differs from a cut's values in the last place now and then.
__device__ __forceinline__ float value_of(int code, float s) {
  float x = (float)code * s;
  asm("" : "+v"(x));
  return x;
}

// A row's CPL columns from c on.
template <class T, int CPL>
__device__ __forceinline__ void put_cols(T* row, int c, int n, const float (&x)[CPL], bool vec) {
  if (vec) {
    if (c >= n) return;
    typedef T TV __attribute__((ext_vector_type(CPL)));
    TV v;
#pragma unroll
    for (int e = 0; e < CPL; ++e) v[e] = (T)x[e];  // to nearest even
    *reinterpret_cast<TV*>(row + c) = v;
  } else {
#pragma unroll
    for (int e = 0; e < CPL; ++e)
      if (c + e < n) row[c + e] = (T)x[e];
  }
}

// A wave per (sequence, head), side and so many 64-token tiles of the cache that
// its lanes have 4 * TPL tokens each: CPL columns (16 bytes of T, one store) of the
// tokens (t0 + t) * 16 + group * 4 + e. Values come as 4 * TPL bytes of a column and
// are transposed in registers, 4 x 4 bytes at a time. Few workgroups are latency and
// take TPL = 1 (333 tokens of 12 heads of 64: 3.9 us against 5.7 in f32, 4.6 against
// 8.0 in bf16; 4 x 580 of 8 of 128 in bf16: 6.9 against 9.1), many are memory and
// take 4 (16 x 1000 of 16 heads of 128: 61.8 against 68.0, 32.4 against 36.5; equal
// at 600 workgroups). Codes and scales of short reads are loaded before the
// sequence's length is known (they lie within the capacity): 0.2 to 0.35 us less for
// 333 and 1000 tokens, but 4 x 20000 and 16 x 2000 of different lengths took 103.6 and
// 36.5 us where 101.2 (4.5 TB/s) and 34.6 do without what lies behind.
constexpr int kLongRead = 1500;
constexpr long kFewReads = 600;  // workgroups of TPL = 4
template <int HDP, class T, int CPL, int TPL>
__global__ __launch_bounds__(256) void q_read_kernel(QStore c, const int* __restrict__ len, int len_stride, QRows k,
                                                     QRows v, int n, const int* __restrict__ first, bool vec) {
  constexpr int LPG = HDP / CPL;             // lanes per group of 16 tokens
  constexpr int GPW = 64 / LPG;              // groups per wave and step
  const int sh = blockIdx.x, seq = sh / c.n_head, head = sh - seq * c.n_head, which = blockIdx.z;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = (lane % LPG) * CPL;
  const QRows& o = which ? v : k;
  if (!o.p) return;
  const int f = first ? first[seq] : 0;
  // tiles before 0 (a first below 0) are counted too
  const long tile_f = f >= 0 ? f / kQTile : -((-(long)f + kQTile - 1) / kQTile);
  const long unit = ((long)blockIdx.y * 4 + wave) * GPW + lane / LPG;  // groups of 4 * TPL tokens from tile_f's first on
  const long tile = tile_f + unit / (16 / TPL);
  const int group = (int)(unit & 3), t0 = TPL == 4 ? 0 : (int)(unit >> 2) & 3;
  if (tile * kQTile >= (long)f + n) return;
  const int l = min(len[(size_t)seq * len_stride], c.capacity);
  const bool there = tile >= 0 && tile * kQTile < (n >= kLongRead ? l : c.tiles * kQTile);
  const int8_t* codes = (which ? c.v : c.k) + c.codes(sh) + (there ? tile : 0) * (long)kQTile * HDP;
  const float* scales = c.s + c.scales(sh) + which + 2 * ((there ? tile : 0) * kQTile >> c.block_shift);
  unsigned q[TPL][4][CPL / 4];  // [t][token][columns / 4]
  float s[TPL];
#pragma unroll
  for (int t = 0; t < TPL; ++t) {
    s[t] = 0.f;
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int w = 0; w < CPL / 4; ++w) q[t][e][w] = 0;
  }
  if (there && which) {
    unsigned raw[CPL][TPL];
#pragma unroll
    for (int e = 0; e < CPL; ++e) {
      typedef unsigned UV __attribute__((ext_vector_type(TPL)));
      const UV r = *reinterpret_cast<const UV*>(codes + (group * HDP + col + e) * 16 + t0 * 4);
      for (int t = 0; t < TPL; ++t) raw[e][t] = r[t];
    }
#pragma unroll
    for (int w = 0; w < CPL / 4; ++w)
#pragma unroll
      for (int t = 0; t < TPL; ++t) {
        const unsigned x[4] = {raw[4 * w][t], raw[4 * w + 1][t], raw[4 * w + 2][t], raw[4 * w + 3][t]};
        unsigned r[4];
        transpose4(x, r);
#pragma unroll
        for (int e = 0; e < 4; ++e) q[t][e][w] = r[e];
      }
  } else if (there) {
#pragma unroll
    for (int t = 0; t < TPL; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int8_t* p = codes + ((t0 + t) * 16 + group * 4 + e) * HDP + col;
#pragma unroll
        for (int w = 0; w < CPL / 4; ++w) q[t][e][w] = reinterpret_cast<const unsigned*>(p)[w];
      }
  }
  if (there) {
#pragma unroll
    for (int t = 0; t < TPL; ++t) s[t] = scales[2 * ((t0 + t) * 16 >> c.block_shift)];
  }
  T* out = static_cast<T*>(o.p) + seq * o.seq + head * o.head;
#pragma unroll
  for (int t = 0; t < TPL; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const long tok = tile * kQTile + (t0 + t) * 16 + group * 4 + e, r = tok - f;
      if (r < 0 || r >= n) continue;
      const bool in = there && tok < l;
      float x[CPL];
#pragma unroll
      for (int j = 0; j < CPL; ++j) x[j] = in ? value_of((int8_t)(q[t][e][j / 4] >> (8 * (j & 3))), s[t]) : 0.f;
      put_cols<T, CPL>(out + r * o.tok, col, c.hd, x, vec);
    }
}

// Whether rows of hd elements are made of aligned vectors of N.
template <class T, int N>
bool vec_ok(const QRows& r, int hd) {
  return !r.p || (hd % N == 0 && r.seq % N == 0 && r.tok % N == 0 && r.head % N == 0 &&
                  reinterpret_cast<uintptr_t>(r.p) % (N * sizeof(T)) == 0);
}

template <class T>
void append_t(hipStream_t s, const QStore& c, QLen len, QTickets tickets, const QRows& k, const QRows& v, int n_new, const int* counts,
              const int* start) {
  if (n_new <= 1) {
    const unsigned n = (unsigned)(c.n_seq * c.n_head);
    if (c.hdp == 64)
      q_append_one_kernel<64, T><<<n, 256, 0, s>>>(c, len, tickets, k, v, n_new, counts, start);
    else
      q_append_one_kernel<128, T><<<n, 256, 0, s>>>(c, len, tickets, k, v, n_new, counts, start);
    return;
  }
  // (n_new tokens touch at most this many tiles, whatever the first one's offset)
  const dim3 grid((unsigned)(c.n_seq * c.n_head), (unsigned)((n_new + kQTile - 2) / kQTile + 1), 2);
  const bool vec = vec_ok<T, 4>(k, c.hd) && vec_ok<T, 4>(v, c.hd);
  if (c.hdp == 64)
    q_append_kernel<64, T><<<grid, 256, 0, s>>>(c, len, tickets, k, v, n_new, counts, start, vec);
  else
    q_append_kernel<128, T><<<grid, 256, 0, s>>>(c, len, tickets, k, v, n_new, counts, start, vec);
}

template <int HDP, class T, int CPL>
void read_rows(hipStream_t s, const QStore& c, QLen len, const QRows& k, const QRows& v, int n, const int* first,
               bool vec) {
  const unsigned heads = (unsigned)(c.n_seq * c.n_head);
  const int tiles = (n + kQTile - 2) / kQTile + 1;  // (whatever the first token's offset in its tile)
  constexpr int per = 4 * (64 / (HDP / CPL));       // units of 4 * TPL tokens that a workgroup takes
  const dim3 grid(heads, (unsigned)((tiles * 4 + per - 1) / per), 2);
  if ((long)grid.x * grid.y * 2 <= kFewReads) {
    const dim3 fine(heads, (unsigned)((tiles * 16 + per - 1) / per), 2);
    q_read_kernel<HDP, T, CPL, 1><<<fine, 256, 0, s>>>(c, len.p, len.stride, k, v, n, first, vec);
  } else {
    q_read_kernel<HDP, T, CPL, 4><<<grid, 256, 0, s>>>(c, len.p, len.stride, k, v, n, first, vec);
  }
}

template <class T>
void read_t(hipStream_t s, const QStore& c, QLen len, const QRows& k, const QRows& v, int n, const int* first) {
  constexpr int CPL = 16 / sizeof(T);
  const bool vec = vec_ok<T, CPL>(k, c.hd) && vec_ok<T, CPL>(v, c.hd);
  if (c.hdp == 64) read_rows<64, T, CPL>(s, c, len, k, v, n, first, vec);
  else read_rows<128, T, CPL>(s, c, len, k, v, n, first, vec);
}

}  // namespace

void launch_q_append(hipStream_t s, const QStore& c, QLen len, QTickets tickets, QType type, const QRows& k,
                     const QRows& v, int n_new, const int* counts, const int* start) {
  if (type == Q_F32) append_t<float>(s, c, len, tickets, k, v, n_new, counts, start);
  else if (type == Q_BF16) append_t<__bf16>(s, c, len, tickets, k, v, n_new, counts, start);
  else append_t<_Float16>(s, c, len, tickets, k, v, n_new, counts, start);
}

void launch_q_read(hipStream_t s, const QStore& c, QLen len, QType type, const QRows& k, const QRows& v, int n,
                   const int* first) {
  if (n <= 0) return;
  if (type == Q_F32) read_t<float>(s, c, len, k, v, n, first);
  else if (type == Q_BF16) read_t<__bf16>(s, c, len, k, v, n, first);
  else read_t<_Float16>(s, c, len, k, v, n, first);
}

}  // namespace rtg
