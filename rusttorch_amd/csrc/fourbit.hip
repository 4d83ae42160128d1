// Writing the 4-bit key/value cache, reading it back, and cutting it to the
// tokens that have got most attention; see fourbit.h for what it holds.
#include "fourbit.h"

#include <algorithm>
#include <type_traits>

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

void fstore_place(FStore* c, void* mem) {
  const FSizes size = c->sizes();
  c->k = static_cast<uint8_t*>(mem);
  c->v = c->k + size.code_bytes();
  c->sk = c->v + size.code_bytes();
  c->sv = c->sk + size.scale_bytes();
  c->w = reinterpret_cast<float*>(c->sv + size.scale_bytes());
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
  top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0xB1, 0xF, 0xF, false));  // quad_perm [1,0,3,2]
  top = max(top, (unsigned)__builtin_amdgcn_update_dpp(0, (int)top, 0x4E, 0xF, 0xF, false));  // quad_perm [2,3,0,1]
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

// A unit is 64 times eight channels of a new token's key and value: 4 or 8 tokens of
// one head. A workgroup's four are behind each other (`wide`), so that lines of the
// cache are written by one of them, or where there are few tokens of different
// heads; the heads of the same tokens are the next workgroups', so that rows are
// read whole at about the same time. 4 x 10000 to 20000 tokens of 8 heads of 128 in
// bf16 take 74 us (4.2 TB/s in and out; a kernel with branches for rows that are not
// aligned, and twice as many units in flight, took 95).
template <int HDP, class T, bool VEC>
__global__ __launch_bounds__(256) void f_append_kernel(FStore c, int* len, QTickets tickets, QRows k, QRows v, int n_new,
                                                       const int* counts, const int* start) {
  constexpr int U = HDP / 8;
  __shared__ Place shared;
  const int seq = blockIdx.x, tid = threadIdx.x;
  if (tid == 0) shared = place(seq, len, 1, n_new, counts, start, c.capacity);
  __syncthreads();
  const Place p = shared;
  Readers readers;
  readers.read(tickets, seq);
  const int n = p.bad ? 0 : p.end - p.at;
  const bool wide = n_new > 2 * (64 / U);
  const unsigned heads = (unsigned)c.n_head, units = (unsigned)((n + 64 / U - 1) / (64 / U));  // of a head
  const unsigned wave = (unsigned)tid >> 6, step = wide ? gridDim.y : gridDim.y * 4;
  unsigned at = wide ? blockIdx.y : blockIdx.y * 4 + wave;
  const int c8 = tid % U * 8;
  // A wave's next unit: its head (n_head behind the last) and the row of this lane's.
  auto next = [&](int& h, int& row) {
    const unsigned group = at / heads, unit = wide ? group * 4 + wave : group;
    h = (int)(unit < units ? at - group * heads : heads);
    row = (int)unit * (64 / U) + (tid & 63) / U;
    at += step;
  };
  constexpr int AHEAD = 2;  // loads of so many units are in flight together
  for (;;) {
    float x[AHEAD][8], y[AHEAD][8];
    int h[AHEAD], row[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      row[u] = 0;
      next(h[u], row[u]);
      if (h[u] >= c.n_head) continue;
      const int i = min(row[u], n - 1);
      load8(static_cast<const T*>(k.p) + seq * k.seq + i * k.tok + h[u] * k.head, c8, c.hd, VEC, x[u]);
      load8(static_cast<const T*>(v.p) + seq * v.seq + i * v.tok + h[u] * v.head, c8, c.hd, VEC, y[u]);
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (h[u] >= c.n_head) continue;
      unsigned kb, vb;
      const unsigned kw = encode8(x[u], &kb), vw = encode8(y[u], &vb);
      if (row[u] >= n) continue;
      const size_t sh = (size_t)seq * c.n_head + h[u];
      const int t = p.at + row[u], tile = t / kFTile, tok = t % kFTile;
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
    if (at / heads * (wide ? 4u : 1u) >= units) break;
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
constexpr int kPickHeld = 24 * 1024;  // weights that stay in LDS between the passes

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
// before it keep. The first pass takes the weights to LDS, eight loads of a thread
// at a time; longer sequences' are read from memory in every pass (20000 tokens of
// 32 heads: 30 us that way, 20 from LDS).
__global__ __launch_bounds__(64 * kPickWaves) void f_pick_kernel(FStore c, const int* len, int keep, int recent,
                                                                int* kept) {
  constexpr int NT = 64 * kPickWaves, AHEAD = 8;
  // A copy for each lane (lanes that count the same bin would take turns, and most
  // weights share a few), two bins to a word: a copy counts 4000000 / 64 at most.
  __shared__ unsigned hist[64][129];
  __shared__ unsigned totals[256];
  __shared__ unsigned held[kPickHeld];
  __shared__ unsigned found[3];
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
  const bool inside = old <= kPickHeld;
  auto key_of = [&](int t) { return inside ? held[t] : pick_key(w[t]); };
  auto count = [&](unsigned key, int shift) {
    const unsigned bin = (key >> shift) & 255;
    atomicAdd(&hist[lane][bin >> 1], 1u << (16 * (bin & 1)));
  };
  unsigned top = 0, left = (unsigned)some;  // the key's bits so far; how many of those with these bits are kept
  for (int shift = 24; shift >= 0 && some > 0; shift -= 8) {
    for (int j = tid; j < 64 * 129; j += NT) (&hist[0][0])[j] = 0;
    if (tid < 256) totals[tid] = 0;
    __syncthreads();
    if (shift == 24) {
      for (int t0 = tid; t0 < old; t0 += AHEAD * NT) {
        float x[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) x[u] = t0 + u * NT < old ? w[t0 + u * NT] : 0.f;
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
          const int t = t0 + u * NT;
          if (t >= old) break;
          const unsigned key = pick_key(x[u]);
          if (inside) held[t] = key;
          count(key, shift);
        }
      }
    } else {
      for (int t = tid; t < old; t += NT) {
        const unsigned key = key_of(t);
        if (key >> (shift + 8) == top >> (shift + 8)) count(key, shift);
      }
    }
    __syncthreads();
    {
      const int word = tid & 127, part = tid >> 7;  // eight copies of two bins
      unsigned low = 0, high = 0;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const unsigned x = hist[part * 8 + k][word];
        low += x & 0xFFFFu;
        high += x >> 16;
      }
      if (low) atomicAdd(&totals[2 * word], low);
      if (high) atomicAdd(&totals[2 * word + 1], high);
    }
    __syncthreads();
    if (wave == 0) {
      unsigned n[4], sum = 0;  // bins 255 - 4 lane - i, from the top
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        n[i] = totals[255 - 4 * lane - i];
        sum += n[i];
      }
      const unsigned incl = (unsigned)wave_scan((int)sum);
      unsigned before = incl - sum;
      if (before < left && left <= incl) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (before < left && left <= before + n[i]) {
            found[0] = (unsigned)(255 - 4 * lane - i);
            found[1] = left - before;
            found[2] = n[i] == left - before;
          }
          before += n[i];
        }
      }
    }
    __syncthreads();
    top |= found[0] << shift;
    left = found[1];
    if (found[2]) {  // all with these bits are kept: the others do not matter
      left = INT32_MAX;
      break;
    }
  }
  // a wave's stretch of the old tokens
  const int per = (old + kPickWaves - 1) / kPickWaves, lo = min(wave * per, old), hi = min(lo + per, old);
  if (some > 0) {
    int a = 0, e = 0;
    for (int t = lo + lane; t < hi; t += 64) {
      const unsigned key = key_of(t);
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
      const unsigned key = t < hi ? key_of(t) : 0;
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

// A thread's part of a token that is moved: 16 channels of a key, or one lane's of a value.
template <int HDP>
struct KeyPiece {
  static constexpr int U = HDP / 32;  // pieces of a token in a half
  uint2 x;
  uint8_t s;
  float w;
  static __device__ __forceinline__ int channel(int half, int p) { return (half * U + p) * 16; }
  __device__ __forceinline__ void read(const FStore& c, size_t sh, int t, int ch) {
    x = *reinterpret_cast<const uint2*>(c.k + c.codes(sh) + (size_t)(t / kFTile) * 16 * HDP + At<HDP>::k(t % kFTile, ch));
    if (ch % 32 == 0) s = c.sk[c.scales(sh) + (size_t)(t / kFTile) * HDP + At<HDP>::k_scale(t % kFTile, ch / 32)];
    if (ch == 0) w = c.w[c.weights(sh) + t];
  }
  __device__ __forceinline__ void write(const FStore& c, size_t sh, int t, int ch) const {
    *reinterpret_cast<uint2*>(c.k + c.codes(sh) + (size_t)(t / kFTile) * 16 * HDP + At<HDP>::k(t % kFTile, ch)) = x;
    if (ch % 32 == 0) c.sk[c.scales(sh) + (size_t)(t / kFTile) * HDP + At<HDP>::k_scale(t % kFTile, ch / 32)] = s;
    if (ch == 0) c.w[c.weights(sh) + t] = w;
  }
};
template <int HDP>
struct ValuePiece {
  static constexpr int U = 8, CV = HDP / 16;
  unsigned x;
  uint8_t s;
  static __device__ __forceinline__ int channel(int half, int p) { return (half * U + p) * CV; }
  __device__ __forceinline__ void read(const FStore& c, size_t sh, int t, int ch) {
    const uint8_t* p = c.v + c.codes(sh) + (size_t)(t / kFTile) * 16 * HDP + At<HDP>::v(t % kFTile, ch / CV);
    x = HDP == 128 ? *reinterpret_cast<const unsigned*>(p) : *reinterpret_cast<const uint16_t*>(p);
    if (ch % 32 == 0) s = c.sv[c.scales(sh) + (size_t)(t / kFTile) * HDP + At<HDP>::v_scale(t % kFTile, ch / 32)];
  }
  __device__ __forceinline__ void write(const FStore& c, size_t sh, int t, int ch) const {
    uint8_t* p = c.v + c.codes(sh) + (size_t)(t / kFTile) * 16 * HDP + At<HDP>::v(t % kFTile, ch / CV);
    if (HDP == 128) *reinterpret_cast<unsigned*>(p) = x;
    else *reinterpret_cast<uint16_t*>(p) = (uint16_t)x;
    if (ch % 32 == 0) c.sv[c.scales(sh) + (size_t)(t / kFTile) * HDP + At<HDP>::v_scale(t % kFTile, ch / 32)] = s;
  }
};

// Moves what is kept to the front, in place, in order, STEP tokens at a time: all
// of a step's are read before any is written (the wait and the barrier), and those
// of later steps lie behind everything that is written by then, since token j of
// the kept ones was never before j; so the next step is read meanwhile, and which
// tokens the one after it has (32 heads' 2048 of 20000: 53 us without, 16 with, a thousand threads a workgroup in the latter).
// Two workgroups have half of the keys' bytes each, two of the values'.
constexpr int kMoveThreads = 1024;

template <class Piece>
__device__ __forceinline__ void move(const FStore& c, size_t sh, int half, int keep, const int* from) {
  constexpr int UN = 4, ROWS = kMoveThreads / Piece::U, STEP = UN * ROWS;
  const int r = (int)threadIdx.x / Piece::U, ch = Piece::channel(half, (int)threadIdx.x % Piece::U);
  Piece x[UN];
  int at[UN];
  auto which = [&](int j0) {
#pragma unroll
    for (int u = 0; u < UN; ++u) at[u] = from[min(j0 + u * ROWS + r, keep - 1)];
  };
  auto read = [&](Piece (&p)[UN]) {
#pragma unroll
    for (int u = 0; u < UN; ++u) p[u].read(c, sh, at[u], ch);
  };
  which(0);
  read(x);
  which(STEP);
  for (int j0 = 0; j0 < keep; j0 += STEP) {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    Piece y[UN];
    read(y);  // (behind the last step: the last token once more)
    which(j0 + 2 * STEP);
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int j = j0 + u * ROWS + r;
      if (j < keep) x[u].write(c, sh, j, ch);
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) x[u] = y[u];
  }
}

template <int HDP>
__global__ __launch_bounds__(kMoveThreads) void f_move_kernel(FStore c, int* len, QTickets tickets, int keep, const int* kept) {
  __shared__ int length;
  const size_t sh = blockIdx.x / 4;
  const int seq = (int)(sh / c.n_head), part = blockIdx.x % 4;
  if (threadIdx.x == 0) length = len[seq];
  __syncthreads();
  const int l = length;
  Readers readers;
  readers.read(tickets, seq);
  if (l > keep) {
    if (part < 2) move<KeyPiece<HDP>>(c, sh, part, keep, kept + sh * keep);
    else move<ValuePiece<HDP>>(c, sh, part - 2, keep, kept + sh * keep);
  }
  if (readers.last((unsigned)c.n_head * 4) && l > keep) len[seq] = keep;
}

template <class T>
void append_t(hipStream_t s, const FStore& c, int* len, QTickets tickets, const QRows& k, const QRows& v, int n_new,
              const int* counts, const int* start, bool vec) {
  // Four units a workgroup; enough of them to fill the device three times (768), as
  // sequences differ in length, but few of a sequence's, which count themselves on
  // one word, 8.6 ns each (20000 tokens of 8 heads of 128, one sequence: 2048
  // workgroups 40 us, 768 of them 30; four of 10000 to 20000: 512 77, 768 74).
  const int rows = 512 / c.hdp;  // of a unit
  const long units = n_new > 2 * rows ? (long)c.n_head * ((n_new + 4 * rows - 1) / (4 * rows))
                                      : ((long)c.n_head * ((n_new + rows - 1) / rows) + 3) / 4;
  const long most = std::max(64l, std::min(768l, 4 * 768l / c.n_seq));
  const dim3 grid((unsigned)c.n_seq, (unsigned)std::max(1l, std::min(most, units)));
  auto run = [&](auto width) {
    constexpr int HDP = decltype(width)::value;
    if (vec) f_append_kernel<HDP, T, true><<<grid, 256, 0, s>>>(c, len, tickets, k, v, n_new, counts, start);
    else f_append_kernel<HDP, T, false><<<grid, 256, 0, s>>>(c, len, tickets, k, v, n_new, counts, start);
  };
  if (c.hdp == 64) run(std::integral_constant<int, 64>{});
  else run(std::integral_constant<int, 128>{});
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
  if (c.hdp == 64) f_move_kernel<64><<<grid, kMoveThreads, 0, s>>>(c, len, tickets, keep, kept);
  else f_move_kernel<128><<<grid, kMoveThreads, 0, s>>>(c, len, tickets, keep, kept);
}

}  // namespace rtg
