// Writing the 8-bit key/value cache and reading it back; see qcache.h for what
// it holds.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "attn_core.h"
#include "qcache.h"
#include "qrows.h"

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
  return 2 * p.codes + 2 * p.scales + p.tail + p.tail_s;
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
  c->ks = reinterpret_cast<float*>(take(p.scales));
  c->vs = reinterpret_cast<float*>(take(p.scales));
  c->tail = reinterpret_cast<float*>(take(p.tail));
  c->tail_s = reinterpret_cast<float*>(take(p.tail_s));
}

namespace {

// Where an append of a sequence goes: tokens [at, end) over a length of len.
struct Place {
  int len, at, end;
  int bad;  // 0, or why it is refused (launch_q_advance)
};
__device__ __forceinline__ Place place(int seq, const int* len, int len_stride, int n_new, const int* counts,
                                       const int* start, int capacity) {
  Place p;
  p.len = len[(size_t)seq * len_stride];
  p.at = start ? start[seq] : p.len;
  const int n = counts ? min(max(counts[seq], 0), n_new) : n_new;
  p.bad = p.at < 0 || p.at > p.len ? 1 : n > capacity - p.at ? 2 : 0;
  p.end = p.bad ? p.at : p.at + n;
  return p;
}

constexpr unsigned kNanBits = 0x7FC00000u;

// fl(amax / 127) of a token, as bits (which order like the values): 0 below
// 127 * 2^-126 (so that a scale is never subnormal), NaN for what is not finite.
__device__ __forceinline__ unsigned token_scale(float amax) {
  if (!(amax <= 3.402823466e38f)) return kNanBits;
  if (amax < 127.f * 1.17549435e-38f) return 0;
  return __float_as_uint(__fdiv_rn(amax, 127.f));
}

// The integer nearest to x / s, ties to even, |x / s| <= 127: r = rint(x * (1 /
// s)) may be one off next to a border between two codes; x - r s says on which
// side x lies (it is exact there: a multiple of half s's last place below 2^24
// of those).
__device__ __forceinline__ int code_of(float x, float s, float inv) {
  float r = rintf(x * inv);
  const float res = fmaf(-r, s, x), half = 0.5f * s;
  const bool odd = ((int)r & 1) != 0;
  if (res > half || (res == half && odd)) r += 1.f;
  else if (res < -half || (res == -half && odd)) r -= 1.f;
  return (int)r;
}
__device__ __forceinline__ float scale_inv(float s) { return s > 0.f ? __fdiv_rn(1.f, s) : 0.f; }

// Largest of a value >= 0 over the lanes of a row (16 lanes for hdp 64, 32 for
// hdp 128), NaN being larger than all: on the bits, which order like the values.
template <int HDP>
__device__ __forceinline__ unsigned row_max_bits(unsigned v) {
#define RTG_STEP(ctrl) v = max(v, (unsigned)__builtin_amdgcn_update_dpp(0, (int)v, ctrl, 0xF, 0xF, false))
  RTG_STEP(0xB1);   // quad_perm [1,0,3,2]
  RTG_STEP(0x4E);   // quad_perm [2,3,0,1]
  RTG_STEP(0x124);  // row_ror:4
  RTG_STEP(0x128);  // row_ror:8
#undef RTG_STEP
  if (HDP == 128) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    v = max(r[0], r[1]);
  }
  return v;
}
__device__ __forceinline__ unsigned abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }
__device__ __forceinline__ unsigned max_abs4(const float4& x) {
  return max(max(abs_bits(x.x), abs_bits(x.y)), max(abs_bits(x.z), abs_bits(x.w)));
}

// Byte of a value's code within its (sequence, head): tile, then [4][hdp][16].
__device__ __forceinline__ size_t value_byte(int tok, int col, int hdp) {
  return (size_t)(tok >> 6) * kQTile * hdp + ((size_t)((tok >> 2) & 3) * hdp + col) * 16 + ((tok >> 4) & 3) * 4 +
         (tok & 3);
}

// One tile (64 tokens) of one (sequence, head) of an append, keys (which = 0)
// or values. Workgroup y takes the y-th tile that the new tokens touch; tokens
// and groups of 4 columns go over the threads, a token's row over 16 or 32
// neighbouring lanes. The first tile's workgroup also quantises the open block's
// earlier tokens anew and writes the tail.
template <int HDP, class T>
__device__ void append_tile(const QStore& c, const Place& p, size_t sh, int y, int which, const T* src, long tok_stride,
                            bool vec, unsigned* blkmax, unsigned char* image) {
  constexpr int LPR = HDP / 4, TPP = 256 / LPR, PASSES = kQTile / TPP;  // lanes per row, tokens per pass
  const int tid = threadIdx.x, c4 = (tid % LPR) * 4, trow = tid / LPR;
  const int block = c.block;
  const int tile0 = (p.at / kQTile + y) * kQTile;  // first token of the tile
  const int blk0 = p.at / block * block;
  const int first = y == 0 ? blk0 : tile0, hi = min(p.end, tile0 + kQTile);
  // earlier tokens of the block that `at` lies in: from the tail while it is
  // the open block, else as they read back
  const bool open = p.at / block == p.len / block;
  float* tail = c.tail + c.tails(sh, which);
  float* tail_s = c.tail_s + c.tail_scales(sh, which);
  int8_t* codes = (which ? c.v : c.k) + c.codes(sh);
  float* scales = (which ? c.vs : c.ks) + c.scales(sh);

  if (tid < 4) blkmax[tid] = 0;
  __syncthreads();
  float4 x[PASSES];
  unsigned ts[PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int tok = tile0 + i * TPP + trow;
    x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    ts[i] = 0;
    if (tok >= first && tok < hi) {
      if (tok >= p.at) {
        x[i] = load4(src + (long)(tok - p.at) * tok_stride, c4, c.hd, vec);
      } else if (open) {
        x[i] = *reinterpret_cast<const float4*>(tail + (size_t)(tok - blk0) * HDP + c4);
      } else {
        const float s = scales[tok >> c.block_shift];
        float* xe = &x[i].x;
        for (int e = 0; e < 4; ++e)
          xe[e] = (float)codes[which ? value_byte(tok, c4 + e, HDP) : (size_t)tok * HDP + c4 + e] * s;
      }
    }
    const float amax = __uint_as_float(row_max_bits<HDP>(max_abs4(x[i])));
    if (tok >= first && tok < hi) {
      if (tok >= p.at) {
        ts[i] = token_scale(amax);
      } else if (open) {
        ts[i] = __float_as_uint(tail_s[tok - blk0]);
      } else {
        // (a token that holds code 127 had the block's scale: amax / 127 may round otherwise)
        const float s = scales[tok >> c.block_shift];
        ts[i] = amax == 127.f * s ? __float_as_uint(s) : token_scale(amax);
      }
      if (c4 == 0) atomicMax(&blkmax[(tok - tile0) >> c.block_shift], ts[i]);
    }
  }
  __syncthreads();  // (also: every read of the tail and of the codes is done)
#pragma unroll
  for (int i = 0; i < PASSES; ++i) {
    const int tok = tile0 + i * TPP + trow;
    if (tok < first || tok >= hi) continue;
    const float s = __uint_as_float(blkmax[(tok - tile0) >> c.block_shift]);
    const float inv = scale_inv(s);
    const float* xe = &x[i].x;
    unsigned q = 0;
    int qe[4];
    for (int e = 0; e < 4; ++e) {
      qe[e] = s > 0.f ? code_of(xe[e], s, inv) : 0;
      q |= (unsigned)(qe[e] & 255) << (8 * e);
    }
    if (which == 0) {
      *reinterpret_cast<unsigned*>(codes + (size_t)tok * HDP + c4) = q;
    } else {
      for (int e = 0; e < 4; ++e) image[value_byte(tok - tile0, c4 + e, HDP)] = (unsigned char)qe[e];
    }
    if (c4 == 0 && (tok & (block - 1)) == 0) scales[tok >> c.block_shift] = s;
    // the tail, where the first tile's block stays open (later tiles': append_tail)
    if (y == 0 && tok / block == p.end / block && !(open && tok < p.at)) {
      *reinterpret_cast<float4*>(tail + (size_t)(tok & (block - 1)) * HDP + c4) = x[i];
      if (c4 == 0) tail_s[tok & (block - 1)] = __uint_as_float(ts[i]);
    }
  }
  if (which == 1) {
    // the tile's values leave in whole groups of 4 tokens (bytes of tokens
    // behind the end are not part of the cache)
    __syncthreads();
    for (int j = tid; j < 4 * HDP; j += 256) {
      const int g = j / HDP;
      unsigned* dst = reinterpret_cast<unsigned*>(codes + (size_t)tile0 * HDP + (size_t)j * 16);
      const unsigned* im = reinterpret_cast<const unsigned*>(image + (size_t)j * 16);
      for (int t = 0; t < 4; ++t) {
        const int tok = tile0 + t * 16 + g * 4;
        if (tok >= first && tok < hi) dst[t] = im[t];
      }
    }
  }
  __syncthreads();
}

// The tail of an append whose open block starts behind its first tile: written
// by the first tile's workgroup, which has read the old tail by then.
template <int HDP, class T>
__device__ void append_tail(const QStore& c, const Place& p, size_t sh, int which, const T* src, long tok_stride,
                            bool vec) {
  constexpr int LPR = HDP / 4, TPP = 256 / LPR;
  const int c4 = (threadIdx.x % LPR) * 4, trow = threadIdx.x / LPR;
  const int ob = p.end / c.block * c.block;
  float* tail = c.tail + c.tails(sh, which);
  float* tail_s = c.tail_s + c.tail_scales(sh, which);
  for (int t0 = 0; t0 < c.block; t0 += TPP) {  // (whole rows of lanes for row_max_bits)
    const int t = t0 + trow;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (ob + t < p.end) x = load4(src + (long)(ob + t - p.at) * tok_stride, c4, c.hd, vec);
    const float amax = __uint_as_float(row_max_bits<HDP>(max_abs4(x)));
    if (ob + t < p.end) {
      *reinterpret_cast<float4*>(tail + (size_t)t * HDP + c4) = x;
      if (c4 == 0) tail_s[t] = __uint_as_float(token_scale(amax));
    }
  }
}

// A workgroup per (sequence, head, tile).
template <int HDP, class T>
__global__ __launch_bounds__(256) void q_append_kernel(QStore c, const int* __restrict__ len, int len_stride, QRows k,
                                                       QRows v, int n_new, const int* __restrict__ counts,
                                                       const int* __restrict__ start, bool vec) {
  __shared__ unsigned blkmax[4];
  __shared__ __attribute__((aligned(16))) unsigned char image[kQTile * HDP];
  const int sh = blockIdx.x, seq = sh / c.n_head, head = sh - seq * c.n_head, y = blockIdx.y;
  const Place p = place(seq, len, len_stride, n_new, counts, start, c.capacity);
  if (p.bad || (p.at == p.end && p.at == p.len)) return;
  const int tile0 = (p.at / kQTile + y) * kQTile;
  if (y > 0 && tile0 >= p.end) return;
  const T* ks = static_cast<const T*>(k.p) + seq * k.seq + head * k.head;
  const T* vs = static_cast<const T*>(v.p) + seq * v.seq + head * v.head;
  append_tile<HDP, T>(c, p, sh, y, 0, ks, k.tok, vec, blkmax, image);
  append_tile<HDP, T>(c, p, sh, y, 1, vs, v.tok, vec, blkmax, image);
  if (y == 0 && p.end / kQTile * kQTile > tile0 && p.end % c.block != 0) {
    append_tail<HDP, T>(c, p, sh, 0, ks, k.tok, vec);
    append_tail<HDP, T>(c, p, sh, 1, vs, v.tok, vec);
  }
}

__global__ __launch_bounds__(256) void q_advance_kernel(int n_seq, int capacity, int* len, int n_new,
                                                        const int* __restrict__ counts,
                                                        const int* __restrict__ start, unsigned* err) {
  const int seq = blockIdx.x * 256 + threadIdx.x;
  if (seq >= n_seq) return;
  const Place p = place(seq, len, 1, n_new, counts, start, capacity);
  if (p.bad) atomicMin(err, (unsigned)seq * 4 + p.bad);
  else len[seq] = p.end;
}

// code * s rounded to f32 before anything else is done with it: without the
// empty asm the compiler makes one instruction of the product and its conversion
// to f16, which then differs from a cut's values in the last place now and then.
__device__ __forceinline__ float value_of(int code, float s) {
  float x = (float)code * s;
  asm("" : "+v"(x));
  return x;
}

// A workgroup per (sequence, head) and 64 tokens of the cache: keys 4 columns
// of a token per lane; values 16 tokens of a column per lane.
template <int HDP, class T>
__global__ __launch_bounds__(256) void q_read_kernel(QStore c, const int* __restrict__ len, int len_stride, QRows k,
                                                     QRows v, int n, const int* __restrict__ first, bool vec) {
  constexpr int LPR = HDP / 4, TPP = 256 / LPR;
  const int sh = blockIdx.x, seq = sh / c.n_head, head = sh - seq * c.n_head, tid = threadIdx.x;
  const int f = first ? first[seq] : 0, l = min(len[(size_t)seq * len_stride], c.capacity);
  // rows [r0, r1) of the result are tokens [tile0, tile0 + 64)
  const long tile0 = (long)(f >= 0 ? f / kQTile : -((-(long)f + kQTile - 1) / kQTile)) * kQTile + (long)blockIdx.y * kQTile;
  if (tile0 >= (long)f + n) return;
  if (k.p) {
    T* out = static_cast<T*>(k.p) + seq * k.seq + head * k.head;
    const int c4 = (tid % LPR) * 4;
    for (int t = tid / LPR; t < kQTile; t += TPP) {
      const long tok = tile0 + t, r = tok - f;
      if (r < 0 || r >= n || c4 >= c.hd) continue;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (tok >= 0 && tok < l) {
        const int q = *reinterpret_cast<const int*>(c.k + c.codes(sh) + (size_t)tok * HDP + c4);
        const float s = c.ks[c.scales(sh) + (tok >> c.block_shift)];
        x = make_float4(value_of((int8_t)q, s), value_of((int8_t)(q >> 8), s), value_of((int8_t)(q >> 16), s),
                        value_of((int8_t)(q >> 24), s));
      }
      store4(out + r * k.tok, c4, c.hd, x, vec);
    }
  }
  if (v.p) {
    T* out = static_cast<T*>(v.p) + seq * v.seq + head * v.head;
    for (int j = tid; j < 4 * HDP; j += 256) {
      const int g = j / HDP, col = j - g * HDP;
      if (col >= c.hd) continue;
      int4 q = make_int4(0, 0, 0, 0);
      if (tile0 >= 0 && tile0 < l)
        q = *reinterpret_cast<const int4*>(c.v + c.codes(sh) + (size_t)tile0 * HDP + (size_t)j * 16);
      const int qe[4] = {q.x, q.y, q.z, q.w};
      for (int t = 0; t < 4; ++t)
        for (int e = 0; e < 4; ++e) {
          const long tok = tile0 + t * 16 + g * 4 + e, r = tok - f;
          if (r < 0 || r >= n) continue;
          float x = 0.f;
          if (tok >= 0 && tok < l)
            x = value_of((int8_t)(qe[t] >> (8 * e)), c.vs[c.scales(sh) + (tok >> c.block_shift)]);
          store1(out + r * v.tok + col, x);
        }
    }
  }
}

template <class T>
bool vec_ok(const QRows& r, int hd) {
  const long a = sizeof(T) == 4 ? 4 : 4;  // 4 elements at a time
  return !r.p || (hd % 4 == 0 && r.seq % a == 0 && r.tok % a == 0 && r.head % a == 0 &&
                  reinterpret_cast<uintptr_t>(r.p) % (4 * sizeof(T)) == 0);
}

template <class T>
void append_t(hipStream_t s, const QStore& c, QLen len, const QRows& k, const QRows& v, int n_new, const int* counts,
              const int* start) {
  // (n_new tokens touch at most this many tiles, whatever the first one's offset)
  const dim3 grid((unsigned)(c.n_seq * c.n_head), (unsigned)((n_new + kQTile - 2) / kQTile + 1));
  const bool vec = vec_ok<T>(k, c.hd) && vec_ok<T>(v, c.hd);
  if (c.hdp == 64)
    q_append_kernel<64, T><<<grid, 256, 0, s>>>(c, len.p, len.stride, k, v, n_new, counts, start, vec);
  else
    q_append_kernel<128, T><<<grid, 256, 0, s>>>(c, len.p, len.stride, k, v, n_new, counts, start, vec);
}

template <class T>
void read_t(hipStream_t s, const QStore& c, QLen len, const QRows& k, const QRows& v, int n, const int* first) {
  const dim3 grid((unsigned)(c.n_seq * c.n_head), (unsigned)((n + kQTile - 2) / kQTile + 1));
  const bool vec = vec_ok<T>(k, c.hd) && vec_ok<T>(v, c.hd);
  if (c.hdp == 64)
    q_read_kernel<64, T><<<grid, 256, 0, s>>>(c, len.p, len.stride, k, v, n, first, vec);
  else
    q_read_kernel<128, T><<<grid, 256, 0, s>>>(c, len.p, len.stride, k, v, n, first, vec);
}

}  // namespace

void launch_q_append(hipStream_t s, const QStore& c, QLen len, QType type, const QRows& k, const QRows& v, int n_new,
                     const int* counts, const int* start) {
  if (type == Q_F32) append_t<float>(s, c, len, k, v, n_new, counts, start);
  else if (type == Q_BF16) append_t<__bf16>(s, c, len, k, v, n_new, counts, start);
  else append_t<_Float16>(s, c, len, k, v, n_new, counts, start);
}

void launch_q_advance(hipStream_t s, const QStore& c, int* len, int n_new, const int* counts, const int* start,
                      unsigned* err) {
  q_advance_kernel<<<(unsigned)((c.n_seq + 255) / 256), 256, 0, s>>>(c.n_seq, c.capacity, len, n_new, counts, start,
                                                                     err);
}

void launch_q_read(hipStream_t s, const QStore& c, QLen len, QType type, const QRows& k, const QRows& v, int n,
                   const int* first) {
  if (n <= 0) return;
  if (type == Q_F32) read_t<float>(s, c, len, k, v, n, first);
  else if (type == Q_BF16) read_t<__bf16>(s, c, len, k, v, n, first);
  else read_t<_Float16>(s, c, len, k, v, n, first);
}

}  // namespace rtg
