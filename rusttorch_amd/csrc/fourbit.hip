// Writing the 4-bit key/value cache, reading it back, and cutting it to the
// tokens that have got most attention; see fourbit.h for what it holds.
#include "fourbit.h"

#include <algorithm>

#include "fourbit_core.h"
#include "qwrite.h"

namespace rtg {

void fstore_shape(FStore* c, int n_seq, int n_head, int hd, int capacity) {
  c->n_seq = n_seq;
  c->n_head = n_head;
  c->hd = hd;
  c->hdp = hd <= 64 ? 64 : 128;
  c->capacity = capacity;
  c->tiles = (capacity + kFTile - 1) / kFTile;
}

namespace {
size_t up256(size_t x) { return (x + 255) / 256 * 256; }
}  // namespace

size_t fstore_bytes(const FStore& c) {
  const size_t sh = (size_t)c.n_seq * c.n_head;
  return 2 * up256(c.codes(sh)) + 2 * up256(c.scales(sh)) + up256(c.weights(sh) * 4);
}

void fstore_place(FStore* c, void* mem) {
  const size_t sh = (size_t)c->n_seq * c->n_head, codes = up256(c->codes(sh)), scales = up256(c->scales(sh));
  uint8_t* m = static_cast<uint8_t*>(mem);
  c->k = m;
  c->v = c->k + codes;
  c->sk = c->v + codes;
  c->sv = c->sk + scales;
  c->w = reinterpret_cast<float*>(c->sv + scales);
}

namespace {

// Where a token's parts lie within its tile: `tok` its number in the tile.
template <int HDP>
struct At {
  static constexpr int CK = HDP / 4, CV = HDP / 16;
  // 4 bytes: the codes of channels c8 .. c8 + 7 of a key
  static __device__ __forceinline__ int k(int tok, int c8) {
    const int b = tok >> 4, lane = c8 / CK * 16 + (tok & 15), byte = c8 % CK / 2;
    return HDP == 128 ? b * 1024 + lane * 16 + byte : lane * 16 + b * 8 + byte;
  }
  static __device__ __forceinline__ int k_scale(int tok, int group) {
    return (tok >> 4) * (HDP / 2) + group * 16 + (tok & 15);
  }
  // CV / 2 bytes: the codes of channels CV m .. of a value
  static __device__ __forceinline__ int v(int tok, int m) {
    const int b = tok >> 4, lane = ((tok >> 2) & 3) * 16 + m, i = tok & 3;
    return HDP == 128 ? b * 1024 + lane * 16 + i * 4 : lane * 16 + b * 8 + i * 2;
  }
  static __device__ __forceinline__ int v_scale(int tok, int group) {
    return (((tok >> 2) & 3) * (HDP / 32) + group) * 8 + (tok >> 4) * 4 + (tok & 3);
  }
};

// The last of a sequence's n workgroups to have read its length writes the new
// one, which saves the launch of a kernel for it. The first thread counts the
// workgroup (read) once the length has gone through LDS and looks at the count
// when it is done with the rest (last).
class Readers {
 public:
  __device__ __forceinline__ void read(QTickets t, int seq) {
    count_ = t.count + (size_t)seq * kQTicketStride;
    if (threadIdx.x == 0) before_ = __hip_atomic_fetch_add(count_, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __device__ __forceinline__ bool last(unsigned n) {
    if (threadIdx.x != 0 || before_ != n - 1) return false;
    *count_ = 0;
    return true;
  }

 private:
  unsigned *count_ = nullptr, before_ = 0;
};

// Eight channels of a row: the byte of the 32 that the lanes 4q .. 4q + 3 hold
// together, and this lane's codes.
__device__ __forceinline__ unsigned encode8(const float (&x)[8], unsigned* byte) {
  unsigned top = 0;  // (bits order like the values, NaN above infinity)
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(x[e]) & 0x7FFFFFFFu);
  top = max(top, (unsigned)__shfl_xor((int)top, 1, 64));
  top = max(top, (unsigned)__shfl_xor((int)top, 2, 64));
  // 0x1FFFFF carries into the exponent where the fraction is over 0.75
  const int b = min(max((int)((top + 0x1FFFFFu) >> 23) - 2, 27), 252);
  const float scale = scale_of((unsigned)b);
  unsigned w = 0;
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[0], x[1], scale, 0);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[2], x[3], scale, 1);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[4], x[5], scale, 2);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x[6], x[7], scale, 3);
  *byte = top >= 0x7F800000u ? 255u : (unsigned)b;
  return w;
}

// Wave by wave, the waves of a sequence's workgroups take every so many'th 64
// units of it; a unit is eight channels of a new token's key and value. 64 units
// are 4 or 8 tokens of one head, a workgroup's are 16 or 32: rows are read whole
// and a tile's bytes are written by neighbours.
template <int HDP, class T>
__global__ __launch_bounds__(256) void f_append_kernel(FStore c, int* len, QTickets tickets, QRows k, QRows v, int n_new,
                                                       const int* counts, const int* start, bool vec) {
  constexpr int U = HDP / 8;
  __shared__ Place shared;
  const int seq = blockIdx.x, tid = threadIdx.x;
  if (tid == 0) shared = place(seq, len, 1, n_new, counts, start, c.capacity);
  __syncthreads();
  const Place p = shared;
  Readers readers;
  readers.read(tickets, seq);
  const int n = p.bad ? 0 : p.end - p.at;
  const unsigned per_head = (unsigned)((n + 64 / U - 1) / (64 / U));  // waves' worth of units of a head
  unsigned at = blockIdx.y * 4 + (tid >> 6);
  int head = 0;
  while (n > 0) {
    head += (int)(at / per_head);
    at %= per_head;
    if (head >= c.n_head) break;
    const int row = (int)at * (64 / U) + (tid & 63) / U, i = min(row, n - 1), c8 = tid % U * 8;
    at += gridDim.y * 4;
    float x[8], y[8];
    load8(static_cast<const T*>(k.p) + seq * k.seq + i * k.tok + head * k.head, c8, c.hd, vec, x);
    load8(static_cast<const T*>(v.p) + seq * v.seq + i * v.tok + head * v.head, c8, c.hd, vec, y);
    unsigned kb, vb;
    const unsigned kw = encode8(x, &kb), vw = encode8(y, &vb);
    if (row >= n) continue;
    const size_t sh = (size_t)seq * c.n_head + head;
    const int t = p.at + i, tile = t / kFTile, tok = t % kFTile;
    uint8_t *kt = c.k + c.codes(sh) + (size_t)tile * 16 * HDP, *vt = c.v + c.codes(sh) + (size_t)tile * 16 * HDP;
    *reinterpret_cast<unsigned*>(kt + At<HDP>::k(tok, c8)) = kw;
    if constexpr (HDP == 128) {
      *reinterpret_cast<unsigned*>(vt + At<HDP>::v(tok, c8 / 8)) = vw;
    } else {
      *reinterpret_cast<uint16_t*>(vt + At<HDP>::v(tok, c8 / 4)) = (uint16_t)vw;
      *reinterpret_cast<uint16_t*>(vt + At<HDP>::v(tok, c8 / 4 + 1)) = (uint16_t)(vw >> 16);
    }
    if (c8 % 32 == 0) {
      const size_t st = c.scales(sh) + (size_t)tile * HDP;
      c.sk[st + At<HDP>::k_scale(tok, c8 / 32)] = (uint8_t)kb;
      c.sv[st + At<HDP>::v_scale(tok, c8 / 32)] = (uint8_t)vb;
      if (c8 == 0) c.w[c.weights(sh) + t] = 0.f;
    }
  }
  if (readers.last(gridDim.y)) {
    if (p.bad) atomicMin(tickets.err, (unsigned)seq * 4 + p.bad);
    else len[seq] = p.end;
  }
}

__device__ __forceinline__ void decode8(unsigned w, unsigned byte, float (&x)[8]) {
  const u4v p = eight_bf16(w, scale_of(byte));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(p[i] << 16);
    x[2 * i + 1] = __uint_as_float(p[i] & 0xffff0000u);
  }
}

// A thread has eight channels of a token's key and value.
template <int HDP, class T>
__global__ __launch_bounds__(256) void f_read_kernel(FStore c, const int* len, QRows k, QRows v, int n, const int* first,
                                                     bool vec) {
  constexpr int U = HDP / 8;
  const size_t sh = blockIdx.x;
  const int seq = (int)(sh / c.n_head), head = (int)(sh % c.n_head);
  const int l = len[seq];
  const long from = first ? first[seq] : 0;
  for (long u = (long)blockIdx.y * 256 + threadIdx.x; u < (long)n * U; u += (long)gridDim.y * 256) {
    const int i = (int)(u / U), c8 = (int)(u % U) * 8;
    const long t = from + i;
    float x[8] = {}, y[8] = {};
    if (t >= 0 && t < l) {
      const int tile = (int)(t / kFTile), tok = (int)(t % kFTile);
      const uint8_t *kt = c.k + c.codes(sh) + (size_t)tile * 16 * HDP, *vt = c.v + c.codes(sh) + (size_t)tile * 16 * HDP;
      const size_t st = c.scales(sh) + (size_t)tile * HDP;
      const unsigned kw = *reinterpret_cast<const unsigned*>(kt + At<HDP>::k(tok, c8));
      unsigned vw;
      if constexpr (HDP == 128)
        vw = *reinterpret_cast<const unsigned*>(vt + At<HDP>::v(tok, c8 / 8));
      else
        vw = *reinterpret_cast<const uint16_t*>(vt + At<HDP>::v(tok, c8 / 4)) |
             (unsigned)*reinterpret_cast<const uint16_t*>(vt + At<HDP>::v(tok, c8 / 4 + 1)) << 16;
      decode8(kw, c.sk[st + At<HDP>::k_scale(tok, c8 / 32)], x);
      decode8(vw, c.sv[st + At<HDP>::v_scale(tok, c8 / 32)], y);
    }
    if (k.p) store8(static_cast<T*>(k.p) + seq * k.seq + i * k.tok + head * k.head, c8, c.hd, x, vec);
    if (v.p) store8(static_cast<T*>(v.p) + seq * v.seq + i * v.tok + head * v.head, c8, c.hd, y, vec);
  }
}

__global__ __launch_bounds__(256) void f_weights_kernel(FStore c, const int* len, float* out, int n) {
  const size_t sh = blockIdx.x;
  const int l = len[sh / c.n_head];
  for (long t = (long)blockIdx.y * 256 + threadIdx.x; t < n; t += (long)gridDim.y * 256)
    out[sh * n + t] = t < l ? c.w[c.weights(sh) + t] : 0.f;
}
__global__ __launch_bounds__(256) void f_add_weights_kernel(FStore c, const int* len, const float* x, int n) {
  const size_t sh = blockIdx.x;
  const long l = min(n, len[sh / c.n_head]);
  for (long t = (long)blockIdx.y * 256 + threadIdx.x; t < l; t += (long)gridDim.y * 256)
    c.w[c.weights(sh) + t] += x[sh * n + t];
}

// ---- eviction ----

constexpr int kPickWaves = 16;

// Weights in the order in which they are kept: larger is later. -0 and 0 are the
// same; NaN is larger than infinity.
__device__ __forceinline__ unsigned pick_key(float x) {
  if (x != x) return 0xFFFFFFFFu;
  const unsigned b = __float_as_uint(x + 0.f);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}

// One workgroup per (sequence, head) finds the key of the last token to be kept,
// eight bits at a time, and how many of those that have just this key; then each
// wave lists what is kept of its stretch of the sequence, behind what the waves
// before it keep.
__global__ __launch_bounds__(64 * kPickWaves) void f_pick_kernel(FStore c, const int* len, int keep, int recent,
                                                                int* kept) {
  constexpr int NT = 64 * kPickWaves, COPIES = 16;
  __shared__ unsigned hist[COPIES][257];  // (copies: lanes that count the same bin take turns)
  __shared__ unsigned found[2];
  __shared__ int above[kPickWaves], equal[kPickWaves];
  const size_t sh = blockIdx.x;
  const int l = len[sh / c.n_head], tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  int* to = kept + sh * keep;
  if (l <= keep) {
    for (int j = tid; j < keep; j += NT) to[j] = j < l ? j : -1;
    return;
  }
  const float* w = c.w + c.weights(sh);
  const int old = l - recent, some = keep - recent;  // `some` of the `old` first ones; the others are kept
  unsigned top = 0, left = (unsigned)some;  // the key's bits so far; how many of those with these bits are kept
  for (int shift = 24; shift >= 0 && some > 0; shift -= 8) {
    for (int j = tid; j < COPIES * 257; j += NT) (&hist[0][0])[j] = 0;
    __syncthreads();
    for (int t = tid; t < old; t += NT) {
      const unsigned key = pick_key(w[t]);
      if (shift == 24 || key >> (shift + 8) == top >> (shift + 8)) atomicAdd(&hist[lane & (COPIES - 1)][(key >> shift) & 255], 1u);
    }
    __syncthreads();
    if (wave == 0) {
      unsigned n[4], sum = 0;  // bins 255 - 4 lane - i, from the top
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        n[i] = 0;
        for (int k = 0; k < COPIES; ++k) n[i] += hist[k][255 - 4 * lane - i];
        sum += n[i];
      }
      unsigned incl = sum;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const unsigned u = __shfl_up(incl, o, 64);
        if (lane >= o) incl += u;
      }
      unsigned before = incl - sum;
      if (before < left && left <= incl) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (before < left && left <= before + n[i]) {
            found[0] = (unsigned)(255 - 4 * lane - i);
            found[1] = left - before;
          }
          before += n[i];
        }
      }
    }
    __syncthreads();
    top |= found[0] << shift;
    left = found[1];
  }
  // a wave's stretch of the old tokens
  const int per = (old + kPickWaves - 1) / kPickWaves, lo = min(wave * per, old), hi = min(lo + per, old);
  if (some > 0) {
    int a = 0, e = 0;
    for (int t = lo + lane; t < hi; t += 64) {
      const unsigned key = pick_key(w[t]);
      a += key > top;
      e += key == top;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
      a += __shfl_xor(a, o, 64);
      e += __shfl_xor(e, o, 64);
    }
    if (lane == 0) {
      above[wave] = a;
      equal[wave] = e;
    }
    __syncthreads();
    int at = 0, ties = 0;
    for (int i = 0; i < wave; ++i) {
      at += above[i];
      ties += equal[i];
    }
    at += min(ties, (int)left);
    for (int t0 = lo; t0 < hi; t0 += 64) {
      const int t = t0 + lane;
      const unsigned key = t < hi ? pick_key(w[t]) : 0;
      const bool tie = t < hi && key == top;
      const unsigned long long eq = __ballot(tie), below = (1ull << lane) - 1;
      const bool take = t < hi && (key > top || (tie && ties + __popcll(eq & below) < (int)left));
      const unsigned long long got = __ballot(take);
      if (take) to[at + __popcll(got & below)] = t;
      at += __popcll(got);
      ties += __popcll(eq);
    }
  }
  for (int j = tid; j < recent; j += NT) to[some + j] = old + j;
}

// Moves what is kept to the front, in place. A workgroup goes over the kept
// tokens in order, STEP at a time: all of them are read before any is written
// (all_have_read), and those of later steps lie behind everything that is written
// by then, since token j of the kept ones was never before j. Two workgroups have
// half of the keys' bytes each, two of the values'.
__device__ __forceinline__ void all_have_read() {
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
}
template <int HDP>
__device__ __forceinline__ void move_keys(const FStore& c, size_t sh, int half, int keep, const int* from) {
  // a thread has 16 channels of a token
  constexpr int U = HDP / 32, STEP = 256 / U;
  uint8_t *codes = c.k + c.codes(sh), *scales = c.sk + c.scales(sh);
  float* w = c.w + c.weights(sh);
  const int c16 = (half * U + (int)threadIdx.x % U) * 16;
  const bool scaled = c16 % 32 == 0;
  for (int j0 = 0; j0 < keep; j0 += STEP) {
    const int j = j0 + (int)threadIdx.x / U, t = from[min(j, keep - 1)], tile = t / kFTile, tok = t % kFTile;
    const uint2 x = *reinterpret_cast<const uint2*>(codes + (size_t)tile * 16 * HDP + At<HDP>::k(tok, c16));
    const uint8_t s = scaled ? scales[(size_t)tile * HDP + At<HDP>::k_scale(tok, c16 / 32)] : 0;
    const float weight = c16 == 0 ? w[t] : 0.f;
    all_have_read();
    if (j >= keep) break;
    const int to = j / kFTile, tj = j % kFTile;
    *reinterpret_cast<uint2*>(codes + (size_t)to * 16 * HDP + At<HDP>::k(tj, c16)) = x;
    if (scaled) scales[(size_t)to * HDP + At<HDP>::k_scale(tj, c16 / 32)] = s;
    if (c16 == 0) w[j] = weight;
  }
}
template <int HDP>
__device__ __forceinline__ void move_values(const FStore& c, size_t sh, int half, int keep, const int* from) {
  // a thread has one lane's part of a token
  constexpr int STEP = 256 / 8;
  uint8_t *codes = c.v + c.codes(sh), *scales = c.sv + c.scales(sh);
  const int m = half * 8 + (int)threadIdx.x % 8, channel = m * (HDP / 16);
  const bool scaled = channel % 32 == 0;
  for (int j0 = 0; j0 < keep; j0 += STEP) {
    const int j = j0 + (int)threadIdx.x / 8, t = from[min(j, keep - 1)], tile = t / kFTile, tok = t % kFTile;
    const uint8_t* p = codes + (size_t)tile * 16 * HDP + At<HDP>::v(tok, m);
    const unsigned x = HDP == 128 ? *reinterpret_cast<const unsigned*>(p) : *reinterpret_cast<const uint16_t*>(p);
    const uint8_t s = scaled ? scales[(size_t)tile * HDP + At<HDP>::v_scale(tok, channel / 32)] : 0;
    all_have_read();
    if (j >= keep) break;
    const int to = j / kFTile, tj = j % kFTile;
    uint8_t* o = codes + (size_t)to * 16 * HDP + At<HDP>::v(tj, m);
    if (HDP == 128) *reinterpret_cast<unsigned*>(o) = x;
    else *reinterpret_cast<uint16_t*>(o) = (uint16_t)x;
    if (scaled) scales[(size_t)to * HDP + At<HDP>::v_scale(tj, channel / 32)] = s;
  }
}

template <int HDP>
__global__ __launch_bounds__(256) void f_move_kernel(FStore c, int* len, QTickets tickets, int keep, const int* kept) {
  __shared__ int length;
  const size_t sh = blockIdx.x / 4;
  const int seq = (int)(sh / c.n_head), part = blockIdx.x % 4;
  if (threadIdx.x == 0) length = len[seq];
  __syncthreads();
  const int l = length;
  Readers readers;
  readers.read(tickets, seq);
  if (l > keep) {
    if (part < 2) move_keys<HDP>(c, sh, part, keep, kept + sh * keep);
    else move_values<HDP>(c, sh, part - 2, keep, kept + sh * keep);
  }
  if (readers.last((unsigned)c.n_head * 4) && l > keep) len[seq] = keep;
}

template <class T>
void append_t(hipStream_t s, const FStore& c, int* len, QTickets tickets, const QRows& k, const QRows& v, int n_new,
              const int* counts, const int* start, bool vec) {
  // units of 256 threads; at most 64 workgroups of a sequence count themselves on one word
  const long units = ((long)n_new * (c.hdp / 8) + 63) / 64 * 64 * c.n_head;
  const dim3 grid((unsigned)c.n_seq, (unsigned)std::max(1l, std::min(64l, (units + 255) / 256)));
  if (c.hdp == 64) f_append_kernel<64, T><<<grid, 256, 0, s>>>(c, len, tickets, k, v, n_new, counts, start, vec);
  else f_append_kernel<128, T><<<grid, 256, 0, s>>>(c, len, tickets, k, v, n_new, counts, start, vec);
}
template <class T>
void read_t(hipStream_t s, const FStore& c, const int* len, const QRows& k, const QRows& v, int n, const int* first,
            bool vec) {
  const long blocks = ((long)n * (c.hdp / 8) + 255) / 256;
  const dim3 grid((unsigned)(c.n_seq * c.n_head), (unsigned)std::min(blocks, 65535l));
  if (c.hdp == 64) f_read_kernel<64, T><<<grid, 256, 0, s>>>(c, len, k, v, n, first, vec);
  else f_read_kernel<128, T><<<grid, 256, 0, s>>>(c, len, k, v, n, first, vec);
}

}  // namespace

void launch_f_append(hipStream_t s, const FStore& c, int* len, QTickets tickets, QType type, const QRows& k,
                     const QRows& v, int n_new, const int* counts, const int* start) {
  const bool vec = by_eights(k, c.hd, type) && by_eights(v, c.hd, type);
  if (type == Q_F32) append_t<float>(s, c, len, tickets, k, v, n_new, counts, start, vec);
  else if (type == Q_BF16) append_t<__bf16>(s, c, len, tickets, k, v, n_new, counts, start, vec);
  else append_t<_Float16>(s, c, len, tickets, k, v, n_new, counts, start, vec);
}

void launch_f_read(hipStream_t s, const FStore& c, const int* len, QType type, const QRows& k, const QRows& v, int n,
                   const int* first) {
  const bool vec = (!k.p || by_eights(k, c.hd, type)) && (!v.p || by_eights(v, c.hd, type));
  if (type == Q_F32) read_t<float>(s, c, len, k, v, n, first, vec);
  else if (type == Q_BF16) read_t<__bf16>(s, c, len, k, v, n, first, vec);
  else read_t<_Float16>(s, c, len, k, v, n, first, vec);
}

void launch_f_weights(hipStream_t s, const FStore& c, const int* len, float* out, int n) {
  const dim3 grid((unsigned)(c.n_seq * c.n_head), (unsigned)std::min((n + 255) / 256, 1024));
  f_weights_kernel<<<grid, 256, 0, s>>>(c, len, out, n);
}
void launch_f_add_weights(hipStream_t s, const FStore& c, const int* len, const float* x, int n) {
  const dim3 grid((unsigned)(c.n_seq * c.n_head), (unsigned)std::min((n + 255) / 256, 1024));
  f_add_weights_kernel<<<grid, 256, 0, s>>>(c, len, x, n);
}

void launch_f_evict(hipStream_t s, const FStore& c, int* len, QTickets tickets, int keep, int recent, int* kept) {
  f_pick_kernel<<<(unsigned)(c.n_seq * c.n_head), 64 * kPickWaves, 0, s>>>(c, len, keep, recent, kept);
  const unsigned grid = (unsigned)(c.n_seq * c.n_head) * 4;
  if (c.hdp == 64) f_move_kernel<64><<<grid, 256, 0, s>>>(c, len, tickets, keep, kept);
  else f_move_kernel<128><<<grid, 256, 0, s>>>(c, len, tickets, keep, kept);
}

}  // namespace rtg
