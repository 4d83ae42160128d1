// Attention for many queries: packed prompts over their own keys, and the 4-bit
// cache's (fourbit.h) chunks and prompts.
//
// Four waves share the keys and values of one head, 64 at a time in LDS; a wave
// has 32 rows, a row being a (query, head) pair that reads this key/value head
// (the heads of a group side by side, so a tile of 128 rows is 128 / group
// positions and little of it lies above the diagonal).
//   scores  S[key][row] = K Q^T on v_mfma_f32_32x32x16, computed transposed: a
//           row's lanes hold 16 of 32 keys each, maximum and sum of the softmax
//           need the lane 32 further on only, and the probabilities are the
//           matrix operand of the second product as they lie;
//   output  O[channel][row] = V^T P^T. Values lie in LDS as rows, like keys; the
//           operand is read with ds_read_b64_tr_b16, which gives a lane four keys
//           of one channel.
// f16 rows are taken as they are by the f16 instructions, bf16 rows by the bf16
// ones. f32 numbers are the sum of three bf16 parts (24 bits): of the products
// of parts the six that reach f32's last bits are computed. Over the 4-bit cache
// keys and values are bf16 exactly, f16 queries two parts. Probabilities have two parts for
// 16-bit results, three for f32: bf16's to 2^-16 of each over the cache and of packed bf16
// rows, as in the kernel of few columns (a result's bits must not hang on the capacity that
// chooses between the two); f16's of packed f16 rows, from 2^14 to 2^-24 of 2^6, to 2^-22.
// (One part takes 393 us instead of 525 for 2047 bf16 tokens behind 12001, 1751 instead of
// 2380 for 16000 packed ones of 32 heads over 8 of 128, 154 instead of 216 for 8000 in f16 of
// 16 heads of 64, and is off by 2^-9 of each probability, 2^-11 in f16: a result whose values
// cancel by many times its own rounding.) Sums are f32.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "attn_core.h"
#include "f16_pair.h"
#include "fourbit_core.h"
#include "lds_direct.h"

namespace rtg {
namespace {

constexpr int kKeys = 64;      // of a stage in LDS
constexpr float kSlack = 8.f;  // powers of two that a score may pass the running maximum by

struct Args {
  QRows q, k, v, out;  // k, v: packed prompts only
  FStore c;            // the cache, else
  const int* len;
  const int* counts;
  const int* offsets;
  int n_rows, n_seq, n_head, n_q, n_q_head, group, hd;
  float query, sum;  // ScoreScale
  float* stats;
  bool qvec, kvec, ovec;
  int min_stages;     // of a split of the keys
  unsigned* tickets;  // [tile][kQTicketStride], a word for each wave
  float* parts;       // [tile][split][wave][value][lane]
};

// What a workgroup of NT threads works on: NT / 2 rows of the (query, head) pairs of
// a sequence and key/value head, `tile` times as many before them.
struct Job {
  int seq, head, tile;
  int len, count;  // keys, queries
  int base;        // packed: the sequence's first row
  int z = 0, zs = 1;  // which of how many parts of the keys, where they are split
  int slot = 0;       // where split parts meet: number of the tile among all
};
__device__ __forceinline__ int seen(const Job& j, int i) { return keys_seen(j.len, j.count, i); }

struct Bf16 {
  typedef __bf16 V2 __attribute__((ext_vector_type(2)));
  static constexpr float kUp = 0.f;  // probabilities are taken 2^kUp times as large
  static __device__ __forceinline__ f32x16 mfma(const u4v& a, const u4v& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf16x8(a), as_bf16x8(b), c, 0, 0, 0);
  }
  static constexpr unsigned kExponents = 0x7F807F80u, kLowest = 0x00800080u;
};
struct F16 {
  typedef _Float16 V2 __attribute__((ext_vector_type(2)));
  static constexpr float kUp = 6.f;
  static __device__ __forceinline__ f32x16 mfma(const u4v& a, const u4v& b, const f32x16& c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ unsigned two(float x, float y) {
    const V2 v = {(_Float16)x, (_Float16)y};
    return __builtin_bit_cast(unsigned, v);
  }
  static constexpr unsigned kExponents = 0x7C007C00u, kLowest = 0x04000400u;
};

// Eight f32 as N parts of M's type.
template <class M, int N>
__device__ __forceinline__ void parts_of(const float (&x)[8], u4v (&p)[N]) {
  if constexpr (std::is_same_v<M, F16>) {
    static_assert(N <= 2, "f16 rows are one part, probabilities two");
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const typename M::V2 hi = {(_Float16)x[2 * i], (_Float16)x[2 * i + 1]};
      p[0][i] = __builtin_bit_cast(unsigned, hi);
      if constexpr (N == 2) p[1][i] = M::two(x[2 * i] - (float)hi[0], x[2 * i + 1] - (float)hi[1]);
    }
  } else {
    bf16_parts<N>(x, p);
  }
}

// Keys and values of a stage in LDS: rows of HD, 16-byte chunks xor'ed so that the
// reads below fall on all banks. A matrix operand of keys takes the same chunk of
// 32 rows; one of values takes four rows of 64 bytes and four rows 4 further on.
template <int HD, int KP>
struct Buffer {
  static constexpr int CH = HD / 8;  // chunks of a row
  static __device__ __forceinline__ int k_swizzle(int key) { return HD == 128 ? key & 15 : (key >> 1) & 7; }
  static __device__ __forceinline__ int v_swizzle(int key) {
    return HD == 128 ? (key & 3) << 2 | ((key >> 2) & 3) : (key & 2) << 1 | ((key >> 2) & 3);
  }
  static __device__ __forceinline__ int k_at(int key, int chunk) { return key * CH + (chunk ^ k_swizzle(key)); }
  static __device__ __forceinline__ int v_at(int key, int chunk) { return key * CH + (chunk ^ v_swizzle(key)); }
  u4v k[KP][kKeys * CH], v[KP][kKeys * CH];
};
// The first key whose value in a channel is not finite (and was taken as 0).
template <int HD>
struct Bad {
  int key[HD];
  int any;
};
// KG groups of waves, each with NB buffers of its own.
template <int HD, int KP, int NB, int KG>
struct Shared {
  Buffer<HD, KP> b[KG][NB];
  Bad<HD> bad;
};

// Whether one of the 16-bit numbers of x is not finite: its exponent's carry.
template <class M>
__device__ __forceinline__ bool any_odd(const u4v& x) {
  unsigned r = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) r |= (x[i] & M::kExponents) + M::kLowest;
  return r & 0x80008000u;
}
// The numbers of a chunk of values (of key `key`) that are not finite become 0,
// and are remembered: a value times a probability of 0 has to be 0 for the rows
// that do not see it.
template <class M, int HD>
__device__ __forceinline__ void clean(u4v& x, Bad<HD>& bad, int channel, int key) {
  bad.any = 1;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const unsigned half = 0xFFFFu << (16 * h);
      if ((((x[i] & M::kExponents) + M::kLowest) & 0x80008000u & half) == 0) continue;
      atomicMin(&bad.key[channel + 2 * i + h], key);
      x[i] &= ~half;
    }
}

// Rows of 16 bits, aligned, straight to LDS: a wave's load is 1 KB of LDS, each
// lane picking the chunk that belongs there.
template <class M, int HD, int NW>
struct DirectStage {
  static constexpr int KP = 1, NB = 2, NT = 64 * NW, CH = HD / 8, N = kKeys * CH / NT;
  static constexpr bool kDirect = true;
  typedef Buffer<HD, 1> Buf;
  const char *k, *v;
  unsigned kv[N], vv[N];  // this lane's bytes of unit u, keys and values
  unsigned kstep, vstep;  // bytes of a stage
  int key[N], wave;
  bool in[N];  // whether the chunk belongs to the row (of keys', values')
  bool vin[N];

  int tid;

  __device__ __forceinline__ void init(const Args& a, const Job& j, Buf (&b)[NB], int thread) {
    tid = thread;
    wave = __builtin_amdgcn_readfirstlane(thread >> 6);
    k = static_cast<const char*>(a.k.p) + ((long)j.base * a.k.tok + j.head * a.k.head) * 2;
    v = static_cast<const char*>(a.v.p) + ((long)j.base * a.v.tok + j.head * a.v.head) * 2;
    kstep = (unsigned)a.k.tok * 2 * kKeys;
    vstep = (unsigned)a.v.tok * 2 * kKeys;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int unit = u * NT + tid, pos = unit % CH;
      key[u] = unit / CH;
      const int kc = pos ^ Buf::k_swizzle(key[u]), vc = pos ^ Buf::v_swizzle(key[u]);
      kv[u] = (unsigned)key[u] * (unsigned)a.k.tok * 2 + kc * 16;
      vv[u] = (unsigned)key[u] * (unsigned)a.v.tok * 2 + vc * 16;
      in[u] = kc * 8 < a.hd;
      vin[u] = vc * 8 < a.hd;
    }
    if (a.hd < HD) {  // the channels behind the rows' stay 0
      u4v* p = &b[0].k[0][0];
      for (int i = tid; i < (int)(sizeof(b) / 16); i += NT) p[i] = u4v{0, 0, 0, 0};
      __syncthreads();
    }
  }
  // keys at .. + 63 (as far as they are below live) on their way to b
  __device__ __forceinline__ void issue(Buf& b, int at, int live, bool whole) {
    const unsigned lk = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)b.k + wave * 1024;
    const unsigned lv = (unsigned)(uintptr_t)(__attribute__((address_space(3))) char*)b.v + wave * 1024;
    const size_t stage = (size_t)(at / kKeys);
    const char *kp = k + stage * kstep, *vp = v + stage * vstep;
    if (whole) {
#pragma unroll
      for (int u = 0; u < N; ++u) load_lds16(kv[u], kp, lk + u * NT * 16);
#pragma unroll
      for (int u = 0; u < N; ++u) load_lds16(vv[u], vp, lv + u * NT * 16);
    } else {
#pragma unroll
      for (int u = 0; u < N; ++u) {
        if (in[u] && at + key[u] < live) load_lds16(kv[u], kp, lk + u * NT * 16);
        if (vin[u] && at + key[u] < live) load_lds16(vv[u], vp, lv + u * NT * 16);
      }
    }
  }
  // for a stage that not every row sees whole, once it is there
  __device__ __forceinline__ void check(Buf& b, Bad<HD>& bad, int at, int live) {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      u4v& x = b.v[0][u * NT + tid];
      if (at + key[u] >= live) x = u4v{0, 0, 0, 0};
      u4v y = x;
      if (any_odd<M>(y)) {
        clean<M>(y, bad, ((tid % CH) ^ Buf::v_swizzle(key[u])) * 8, at + key[u]);
        x = y;
      }
    }
  }
};

// Rows through registers, NW waves sharing a stage: aligned ones (VEC), or any.
template <class M, int HD, int P, class T, bool VEC, int NW, int BUFFERS>
struct RowStage {
  static constexpr int KP = P, NB = BUFFERS, CH = HD / 8, NT = 64 * NW, N = kKeys * CH / NT;
  static constexpr bool kDirect = false;
  typedef T T8 __attribute__((ext_vector_type(8)));
  typedef T Aligned8 __attribute__((ext_vector_type(8), aligned(16)));  // (eight f32 are not aligned to their size)
  typedef Buffer<HD, P> Buf;
  T8 k[N], v[N];
  int tid;

  __device__ __forceinline__ void init(const Args&, const Job&, Buf (&)[NB], int thread) { tid = thread; }
  static __device__ __forceinline__ void load1(const T* row, int c8, int n, T8& x) {
    if constexpr (VEC) {
      x = *reinterpret_cast<const Aligned8*>(row + c8);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (c8 + e < n) x[e] = row[c8 + e];
    }
  }
  __device__ __forceinline__ void load(const Args& a, const Job& j, int at, int live) {
    const bool whole = VEC && at + kKeys <= live && a.hd == HD;  // (uniform)
    const T* kp = static_cast<const T*>(a.k.p) + (j.base + (long)at) * a.k.tok + j.head * a.k.head;
    const T* vp = static_cast<const T*>(a.v.p) + (j.base + (long)at) * a.v.tok + j.head * a.v.head;
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int unit = u * NT + tid, key = unit / CH, c8 = unit % CH * 8;
      if (!whole) {
        k[u] = T8{};
        v[u] = T8{};
        if (at + key >= live || c8 >= a.hd) continue;
      }
      load1(kp + key * a.k.tok, c8, a.hd, k[u]);
      load1(vp + key * a.v.tok, c8, a.hd, v[u]);
    }
  }
  static __device__ __forceinline__ void parts(const T8& x, u4v (&p)[P]) {
    if constexpr (sizeof(T) == 2) {
      p[0] = __builtin_bit_cast(u4v, x);
    } else {
      float f[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] = x[e];
      bf16_parts<P>(f, p);
    }
  }
  __device__ __forceinline__ void store(Buf& s, Bad<HD>& bad, int at, int, bool edge) {
#pragma unroll
    for (int u = 0; u < N; ++u) {
      const int unit = u * NT + tid, key = unit / CH, chunk = unit % CH;
      u4v p[P];
      parts(k[u], p);
#pragma unroll
      for (int i = 0; i < P; ++i) s.k[i][Buf::k_at(key, chunk)] = p[i];
      parts(v[u], p);
      // (the first part of what is not finite is not finite: it is cut or the number itself)
      if (edge && any_odd<M>(p[0])) {
        const u4v first = p[0];
        clean<M>(p[0], bad, chunk * 8, at + key);
#pragma unroll
        for (int i = 1; i < P; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const unsigned kept = ~(first[e] ^ p[0][e]);  // halves that clean() has left alone, and zeros
            p[i][e] &= ((kept & 0x7F80u) == 0x7F80u ? 0xFFFFu : 0u) | ((kept & 0x7F800000u) == 0x7F800000u ? 0xFFFF0000u : 0u);
          }
      }
#pragma unroll
      for (int i = 0; i < P; ++i) s.v[i][Buf::v_at(key, chunk)] = p[i];
    }
  }
};

// Two tiles of the 4-bit cache as a stage: a thread has HD / 8 bytes of codes of
// one key, and of four values.
template <int HD>
struct CodeStage {
  static constexpr int KP = 1, NB = 2, NT = 256;
  static constexpr bool kDirect = false;
  typedef unsigned W __attribute__((ext_vector_type(HD / 32)));
  typedef Buffer<HD, 1> Buf;
  W k, v;
  unsigned ks, vs;
  int tid;

  __device__ __forceinline__ void init(const Args&, const Job&, Buf (&)[NB], int thread) { tid = thread; }
  __device__ __forceinline__ void load(const Args& a, const Job& j, int at, int) {
    const int unit = tid & 127, lane = HD == 128 ? unit & 63 : unit >> 1, b = HD == 128 ? unit >> 6 : unit & 1;
    // (a second tile behind the capacity is the first once more: no key of it is seen)
    const int tile = min(at / kFTile + (tid >> 7), a.c.tiles - 1), g = lane >> 4, m = lane & 15;
    const size_t sh = (size_t)j.seq * a.c.n_head + j.head, codes = a.c.codes(sh) + (size_t)tile * 16 * HD + unit * (HD / 8);
    const size_t scales = a.c.scales(sh) + (size_t)tile * HD;
    k = *reinterpret_cast<const W*>(a.c.k + codes);
    v = *reinterpret_cast<const W*>(a.c.v + codes);
    ks = a.c.sk[scales + b * (HD / 2) + (HD == 128 ? lane : (g >> 1) * 16 + m)];
    vs = *reinterpret_cast<const unsigned*>(a.c.sv + scales + (g * (HD / 32) + m * (HD / 16) / 32) * 8 + b * 4);
  }
  __device__ __forceinline__ void store(Buf& s, Bad<HD>& bad, int at, int live, bool edge) {
    const int unit = tid & 127, lane = HD == 128 ? unit & 63 : unit >> 1, b = HD == 128 ? unit >> 6 : unit & 1;
    const int g = lane >> 4, m = lane & 15, first = (tid >> 7) * kFTile + b * 16;
    const float kscale = scale_of(ks);
#pragma unroll
    for (int i = 0; i < HD / 32; ++i) s.k[0][Buf::k_at(first + m, g * (HD / 32) + i)] = eight_bf16(k[i], kscale);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int key = first + 4 * g + i;
      unsigned byte = (vs >> (8 * i)) & 255u;
      if (edge && at + key >= live) byte = 0;  // (what lies there is anything)
      if (byte == 255u) {
        bad.any = 1;
        for (int e = 0; e < HD / 16; ++e) atomicMin(&bad.key[m * (HD / 16) + e], at + key);
        byte = 0;
      }
      if constexpr (HD == 128) {
        s.v[0][Buf::v_at(key, m)] = eight_bf16(v[i], scale_of(byte));
      } else {
        const unsigned w = v[i / 2];
        uint2* to = reinterpret_cast<uint2*>(&s.v[0][Buf::v_at(key, m >> 1)]) + (m & 1);
        *to = i & 1 ? make_uint2(two_bf16<2>(w, scale_of(byte)), two_bf16<3>(w, scale_of(byte)))
                    : make_uint2(two_bf16<0>(w, scale_of(byte)), two_bf16<1>(w, scale_of(byte)));
      }
    }
  }
};

typedef short s4v __attribute__((ext_vector_type(4)));
typedef const u4v __attribute__((address_space(3))) * LdsChunk;
typedef s4v __attribute__((address_space(3))) * LdsFour;
__device__ __forceinline__ unsigned lds_address(const void* p) {
  return (unsigned)(uintptr_t)(__attribute__((address_space(3))) const char*)p;
}
// Four values of 16 bits of one channel, of the rows whose chunks the 16 lanes point at.
__device__ __forceinline__ uint2 read_tr(unsigned at) {
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((LdsFour)(uintptr_t)at));
}

// Of READS reads of LDS in this stretch, the first AHEAD before the first matrix
// instruction, then STEP of them behind every MFMAS: left to itself the compiler
// reads each operand right before its use and waits for it, 100 cycles a time.
template <int READS, int AHEAD, int STEP, int MFMAS>
__device__ __forceinline__ void reads_ahead() {
  constexpr int kRead = 0x100, kMfma = 0x8;
  __builtin_amdgcn_sched_group_barrier(kRead, AHEAD, 0);
#pragma unroll
  for (int i = AHEAD; i < READS; i += STEP) {
    __builtin_amdgcn_sched_group_barrier(kMfma, MFMAS, 0);
    __builtin_amdgcn_sched_group_barrier(kRead, STEP, 0);
  }
  __builtin_amdgcn_sched_group_barrier(kMfma, (AHEAD + STEP - 1) / STEP * MFMAS, 0);
}

template <class M, int HD, int QP, int PP, class T, class Stage, int KG>
__device__ __forceinline__ void attend(const Args& a, const Job& job, Shared<HD, Stage::KP, Stage::NB, KG>& s) {
  constexpr int KS = HD / 16, DT = HD / 32, KP = Stage::KP, NB = Stage::NB, ROWS = Stage::NT / 2;
  typedef Buffer<HD, KP> Buf;
  constexpr int SPAN = KG * kKeys;  // keys of a step: a stage for each group
  const int tid = threadIdx.x % Stage::NT, lane = tid & 63, n = lane & 31, half = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int group = __builtin_amdgcn_readfirstlane((int)threadIdx.x / Stage::NT);
  Buf(&bufs)[NB] = s.b[group];
  const int first = job.tile * ROWS, rows = job.count * a.group;
  // this lane's row: query i of head h
  const int row = first + wave * 32 + n, i = row / a.group, head = job.head * a.group + row % a.group;
  const int lim = seen(job, i);
  // keys that the workgroup's rows see: at most, and at least but for padding
  const int all = rows > first ? seen(job, (min(first + ROWS, rows) - 1) / a.group) : 0, least = seen(job, first / a.group);
  // this workgroup's part of them
  const int stages = (all + kKeys - 1) / kKeys, splits = job.zs == 1 ? 1 : max(min((stages + a.min_stages - 1) / a.min_stages, job.zs), 1);
  if (job.z >= splits) return;
  const int per = splits == 1 ? stages : (stages + splits - 1) / splits;
  const int begin = job.z * per * kKeys, live = min(all, begin + per * kKeys);
  const int end = min(first + wave * 32 + 32, rows);  // of this wave's rows
  const int mine = end > first + wave * 32 ? min(seen(job, (end - 1) / a.group), live) : 0;
  Stage st;
  st.init(a, job, bufs, tid);
  for (int c = threadIdx.x; c < HD; c += KG * Stage::NT) s.bad.key[c] = INT32_MAX;
  if (threadIdx.x == 0) s.bad.any = 0;
  const int whole_to = min(least, live);
  auto edge_at = [&](int at) { return at + SPAN > whole_to; };  // (uniform)
  const int own = begin + group * kKeys;  // of the first step's keys, this group's
  auto fetch = [&](int at, Buf& b) {
    if (at >= live) return;
    if constexpr (Stage::kDirect) st.issue(b, at, live, at + kKeys <= live && a.hd == HD);
    else st.load(a, job, at, live);
  };
  fetch(own, bufs[0]);
  u4v q[KS][QP];
  {
    const T* p = static_cast<const T*>(a.q.p) + job.seq * a.q.seq + (job.base + (long)min(i, max(job.count - 1, 0))) * a.q.tok + head * a.q.head;
    bool raw = false;
    if constexpr (QP == 1 && sizeof(T) == 2) {
      if (a.qvec && a.query == 1.f) {  // (uniform) as they are
        raw = true;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const int c8 = k * 16 + half * 8;
          q[k][0] = u4v{0, 0, 0, 0};
          if (c8 < a.hd) q[k][0] = *reinterpret_cast<const u4v*>(p + c8);
        }
      }
    }
    if (!raw)
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      float x[8];
      load8(p, k * 16 + half * 8, a.hd, a.qvec, x);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= a.query;
      parts_of<M, QP>(x, q[k]);
    }
  }
  // Where this lane's operands lie in the first buffer, but for multiples of 16 keys
  // (which the swizzles do not see, and instructions hold as their offsets).
  unsigned ka[KS], va[DT][2];
  {
    const unsigned at_k = lds_address(&bufs[0].k[0][0]), at_v = lds_address(&bufs[0].v[0][0]);
    const int key = half * 4 + ((lane & 15) >> 2), chan = (lane >> 4 & 1) * 16 + (lane & 3) * 4;
#pragma unroll
    for (int k = 0; k < KS; ++k) ka[k] = at_k + Buf::k_at(n, k * 2 + half) * 16;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int r = 0; r < 2; ++r) va[d][r] = at_v + Buf::v_at(key + 8 * r, d * 4 + chan / 8) * 16 + (chan & 7) * 2;
  }
  f32x16 o[DT];
#pragma unroll
  for (int d = 0; d < DT; ++d) o[d] = f32x16{};
  float m = -INFINITY, l = 0.f;
  if constexpr (!Stage::kDirect && NB == 2) {
    __syncthreads();
    if (own < live) st.store(bufs[0], s.bad, own, live, edge_at(begin));
    fetch(own + SPAN, bufs[0]);
  }
  // Between their matrix instructions a SIMD's two waves leave each other room, so the
  // one that is at its products goes first (2047 tokens behind 12001 in bf16: 559 us
  // without, 532 with; 16000 packed 2547 and 2519). With f32's six products it does
  // not pay (500 behind 4 x 4000: 89 us, 95 with).
  auto in_products = [](bool yes) {
    if constexpr (QP < 3) {
      if (yes) __builtin_amdgcn_s_setprio(1);
      else __builtin_amdgcn_s_setprio(0);
    }
  };
  // (two forms of the step: the compiler would else select for every score of every stage)
  auto step = [&](int from, auto edge_stage, auto in_buffer) {
    constexpr bool edge = decltype(edge_stage)::value;
    const int at = from + group * kKeys, next = at + SPAN;
    const unsigned which = in_buffer;  // (a constant but at the edge)
    Buf& b = bufs[which];
    Buf& other = bufs[NB - 1 - which];
    const unsigned boff = which * (unsigned)sizeof(Buf);
    if constexpr (Stage::kDirect) {
      wait_and_sync();  // the stage is there, and nobody reads the other one any more
      if (edge) {
        if (at < live) st.check(b, s.bad, at, live);
        __syncthreads();
      }
      fetch(next, other);
    } else if constexpr (NB == 2) {
      __syncthreads();
      if (next < live) st.store(other, s.bad, next, live, edge_at(from + SPAN));
      fetch(next + SPAN, other);
    } else {
      __syncthreads();
      if (at < live) st.store(b, s.bad, at, live, edge);
      __syncthreads();
      fetch(next, b);
    }
    if (edge && at >= mine) return;  // (no row of this wave sees one of these keys)
    in_products(true);
    const bool short_of = edge && at + 32 >= mine;  // the second 32 keys are seen by no row of this wave
    float p[2][16];  // keys at + sub * 32 + e / 4 * 8 + half * 4 + e % 4
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
      if (sub == 1 && short_of) {
#pragma unroll
        for (int e = 0; e < 16; ++e) p[1][e] = -INFINITY;
        break;
      }
      f32x16 x = {};
#pragma unroll
      for (int k = 0; k < KS; ++k)
#pragma unroll
        for (int kp = KP - 1; kp >= 0; --kp) {
          const u4v f = *(LdsChunk)(uintptr_t)(ka[k] + (boff + kp * (unsigned)sizeof(b.k[0]) + sub * 512 * Buf::CH));
#pragma unroll
          for (int qp = QP - 1; qp >= 0; --qp)
            if (kp + qp < 3) x = M::mfma(f, q[k][qp], x);
        }
#pragma unroll
      for (int e = 0; e < 16; ++e) p[sub][e] = x[e];
    }
    reads_ahead<2 * KS * KP, 6, 1, KP == 1 ? QP : 2>();
    in_products(false);
    if constexpr (edge) {
#pragma unroll
      for (int e = 0; e < 32; ++e)
        if (at + e / 16 * 32 + e % 16 / 4 * 8 + half * 4 + e % 4 >= lim) p[e / 16][e % 16] = -INFINITY;
    }
    float top = p[0][0];
#pragma unroll
    for (int e = 1; e < 32; ++e) top = fmaxf(top, p[e / 16][e % 16]);
    if (__builtin_amdgcn_ballot_w64(top * a.sum > m + kSlack)) {
      top = xor32_max_k(top) * a.sum;
      // (each row by itself: its result does not depend on its neighbours')
      const float f = top > m + kSlack ? __builtin_amdgcn_exp2f(m - top) : 1.f;
      m = top > m + kSlack ? top : m;
      l *= f;
#pragma unroll
      for (int d = 0; d < DT; ++d) o[d] *= f;
    }
    const float base = (m == -INFINITY ? 0.f : m) - M::kUp;
#pragma unroll
    for (int e = 0; e < 32; ++e) p[e / 16][e % 16] = __builtin_amdgcn_exp2f(fmaf(p[e / 16][e % 16], a.sum, -base));
    if constexpr (edge) {
#pragma unroll
      for (int e = 0; e < 32; ++e)
        if (at + e / 16 * 32 + e % 16 / 4 * 8 + half * 4 + e % 4 >= lim) p[e / 16][e % 16] = 0.f;
    }
    in_products(true);
#pragma unroll
    for (int sub = 0; sub < 2; ++sub) {
      if (sub == 1 && short_of) break;
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        // keys sub * 32 + u * 16 + e / 4 * 8 + half * 4 + e % 4, e < 8
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = p[sub][u * 8 + e];
        u4v pp[PP];
        parts_of<M, PP>(x, pp);
#pragma unroll
        for (int e = 0; e < 8; ++e) l += x[e];
#pragma unroll
        for (int d = 0; d < DT; ++d)
#pragma unroll
          for (int kp = KP - 1; kp >= 0; --kp) {
            u4v f;
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const uint2 w = read_tr(va[d][r] + (boff + kp * (unsigned)sizeof(b.v[0]) + (sub * 32 + u * 16) * 16 * Buf::CH));
              f[2 * r] = w.x;
              f[2 * r + 1] = w.y;
            }
#pragma unroll
            for (int k = PP - 1; k >= 0; --k)
              if (kp + k < 3) o[d] = M::mfma(f, pp[k], o[d]);
          }
      }
    }
    reads_ahead<8 * DT * KP, 8, 2, KP == 1 ? PP : 2>();
    in_products(false);
  };
  int at = begin;
  if constexpr (NB == 1) {
    for (; at < live && !edge_at(at); at += SPAN) step(at, std::false_type{}, std::integral_constant<unsigned, 0>{});
  } else {
    for (; at < live && !edge_at(at + SPAN); at += 2 * SPAN) {
      step(at, std::false_type{}, std::integral_constant<unsigned, 0>{});
      step(at + SPAN, std::false_type{}, std::integral_constant<unsigned, 1>{});
    }
  }
  for (; at < live; at += SPAN) step(at, std::true_type{}, NB == 1 ? 0u : (unsigned)((at - begin) / SPAN) & 1u);
  if constexpr (KG > 1) {
    // the groups' results meet in LDS, value by value with the lanes side by side
    constexpr int N = DT * 16 + 2;
    static_assert(sizeof(s.b) >= (KG - 1) * (Stage::NT / 64) * N * 64 * 4, "room for the results");
    __syncthreads();
    float* to = reinterpret_cast<float*>(&s.b) + ((group - 1) * (Stage::NT / 64) + wave) * N * 64 + lane;
    if (group > 0) {
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) to[(d * 16 + e) * 64] = o[d][e];
      to[(N - 2) * 64] = m;
      to[(N - 1) * 64] = l;
    }
    __syncthreads();
    if (group > 0) return;
    for (int g = 1; g < KG; ++g) {
      const float* x = reinterpret_cast<const float*>(&s.b) + ((g - 1) * (Stage::NT / 64) + wave) * N * 64 + lane;
      const float m2 = x[(N - 2) * 64], most = fmaxf(m, m2), base = most == -INFINITY ? 0.f : most;
      const float f = __builtin_amdgcn_exp2f(m - base), f2 = __builtin_amdgcn_exp2f(m2 - base);
      m = most;
      l = fmaf(f, l, f2 * x[(N - 1) * 64]);
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; ++e) o[d][e] = fmaf(f, o[d][e], f2 * x[(d * 16 + e) * 64]);
    }
  }
  if (all > 0 && s.bad.any) {
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        if (s.bad.key[d * 32 + e / 4 * 8 + half * 4 + e % 4] < lim) o[d][e] = NAN;
  }
  if (splits > 1) {
    // Every wave's results, in pairs with the lanes side by side, past the L2 caches;
    // the last of a tile's waves of one number to come here joins theirs, in order.
    constexpr int N = DT * 16 + 2;
    float* p = a.parts + ((size_t)(job.slot * job.zs + job.z) * (Stage::NT / 64) + wave) * N * 64 + lane * 2;
#pragma unroll
    for (int d = 0; d < DT; ++d)
#pragma unroll
      for (int e = 0; e < 16; e += 2) store2(p + (d * 16 + e) * 64, o[d][e], o[d][e + 1]);
    store2(p + (N - 2) * 64, m, l);
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the stores have completed
    unsigned before = 0, *count = a.tickets + (size_t)job.slot * kQTicketStride + wave;
    if (lane == 0) before = __hip_atomic_fetch_add(count, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    if (__builtin_amdgcn_readfirstlane(before) != (unsigned)splits - 1) return;
    if (lane == 0) __hip_atomic_store(count, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int d = 0; d < DT; ++d) o[d] = f32x16{};
    for (int z = 0; z < splits; ++z) {
      const float* x = a.parts + ((size_t)(job.slot * job.zs + z) * (Stage::NT / 64) + wave) * N * 64 + lane * 2;
      const float2 ml = load2(x + (N - 2) * 64);
      const float most = fmaxf(m, ml.x), base = most == -INFINITY ? 0.f : most;
      const float f = __builtin_amdgcn_exp2f(m - base), f2 = __builtin_amdgcn_exp2f(ml.x - base);
      m = most;
      l = fmaf(f, l, f2 * ml.y);
#pragma unroll
      for (int d = 0; d < DT; ++d)
#pragma unroll
        for (int e = 0; e < 16; e += 2) {
          const float2 y = load2(x + (d * 16 + e) * 64);
          o[d][e] = fmaf(f, o[d][e], f2 * y.x);
          o[d][e + 1] = fmaf(f, o[d][e + 1], f2 * y.y);
        }
    }
  }
  if (row >= a.n_q * a.group) return;
  l = xor32_sum_k(l);
  const bool any = lim > 0;
  const float inv = 1.f / l;
  T* out = static_cast<T*>(a.out.p) + job.seq * a.out.seq + (job.base + (long)i) * a.out.tok + head * a.out.head;
#pragma unroll
  for (int d = 0; d < DT; ++d)
#pragma unroll
    for (int e = 0; e < 16; e += 4) {
      float x[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) x[r] = any ? o[d][e + r] * inv : 0.f;
      store4(out, d * 32 + e / 4 * 8 + half * 4, a.hd, make_float4(x[0], x[1], x[2], x[3]), a.ovec);
    }
  if (a.stats && half == 0)
    reinterpret_cast<float2*>(a.stats)[((size_t)job.seq * a.n_q + i) * a.n_q_head + head] = make_float2(m - M::kUp, any ? l : 0.f);
}

template <int HD, int QP, int PP, class T, int KG>
__global__ __launch_bounds__(256 * KG, KG > 1 || HD == 64 || sizeof(T) == 2 ? 2 : 1) void f_attend_many_kernel(Args a) {
  __shared__ Shared<HD, 1, 2, KG> s;
  Job j;
  j.seq = (int)blockIdx.x / a.n_head;
  j.head = (int)blockIdx.x % a.n_head;
  j.tile = (int)(gridDim.y - 1 - blockIdx.y);  // the longest first
  j.len = a.len[j.seq];
  j.count = a.counts ? min(max(a.counts[j.seq], 0), a.n_q) : a.n_q;
  j.base = 0;
  j.z = (int)blockIdx.z;
  j.zs = (int)gridDim.z;
  j.slot = (int)(blockIdx.x * gridDim.y + blockIdx.y);
  attend<Bf16, HD, QP, PP, T, CodeStage<HD>, KG>(a, j, s);
}

// The workgroups of a packed batch: the tiles of all sequences, each for all heads
// in turn; those behind the last tile clear the rows that no sequence has. There
// is one at least: the sum of the sequences' tiles, rounded up each, is less than
// the rows' tiles and the number of sequences.
// Up to 64 sequences are taken by their lengths, a sequence's tiles by the keys they
// see, so that what runs last is short (8 x up to 1500 tokens of 32 heads of 128 over
// 8 in bf16: 142 us; the longest tiles of all sequences first would be shorter still
// at the end, but the keys of 8 sequences do not fit the caches that one's do: 128 us
// instead of 117 with one part of probabilities). More are taken in their order.
// Where all workgroups are on the device at once, RESIDENT of them on each of its 256
// compute units, every second 256 go the other way, so that those of a compute unit
// have about the same to do between them.
template <class M, int HD, int P, class T, class Stage, int KG, int RESIDENT>
__global__ __launch_bounds__(Stage::NT * KG, KG > 1 || HD == 64 || P == 1 ? 2 : 1) void packed_attend_kernel(Args a) {
  constexpr int ROWS = Stage::NT / 2;
  __shared__ Shared<HD, Stage::KP, Stage::NB, KG> s;
  const int lane = threadIdx.x & 63;
  int block = (int)blockIdx.x, end = 0;
  Job j;
  j.seq = 0;  // (packed rows have no stride of sequences)
  j.tile = -1;
  // The 64 sequences from s0 on, one per lane. An offset that descends counts as the
  // largest before it: whatever they hold, sequences lie behind each other within the rows.
  int lo = 0, hi = 0;
  end = min(max(a.offsets[0], 0), a.n_rows);
  auto sequences = [&](int s0) {
    const int seq = s0 + lane;
    hi = max(wave_max_scan(seq < a.n_seq ? min(max(a.offsets[seq + 1], 0), a.n_rows) : 0), end);
    lo = __shfl_up(hi, 1, 64);
    if (lane == 0) lo = end;
    end = __builtin_amdgcn_readlane(hi, 63);
    return ((hi - lo) * a.group + ROWS - 1) / ROWS;
  };
  auto take = [&](int lane_of, int tile) {
    j.base = __builtin_amdgcn_readlane(lo, lane_of);
    j.len = j.count = __builtin_amdgcn_readlane(hi, lane_of) - j.base;
    j.tile = tile;
  };
  int at, index;  // of this tile among those not yet looked at, among all
  if (a.n_seq <= 64) {
    const int tiles = sequences(0), total = wave_sum(tiles), busy = total * a.n_head;
    if (busy <= 256 * RESIDENT && block < busy && block & 256) {
      const int row = block & ~255;
      block = row + min(256, busy - row) - 1 - (block - row);
    }
    index = block / a.n_head;
    j.head = block - index * a.n_head;
    at = index - total;
    if (at < 0) {
      int before = 0;  // tiles of the sequences before this lane's
      for (int i = 0; i < a.n_seq; ++i) {
        const int t = __builtin_amdgcn_readlane(tiles, i);
        before += t > tiles || (t == tiles && i < lane) ? t : 0;
      }
      const int l = __builtin_ctzll(__builtin_amdgcn_ballot_w64(index >= before && index < before + tiles));
      take(l, __builtin_amdgcn_readlane(before + tiles, l) - 1 - index);
    }
  } else {
    index = block / a.n_head;
    j.head = block - index * a.n_head;
    at = index;
    int s0 = 0;
    // Sequences that end before this tile, 256 N at a time: a lane has four in a row of
    // each 256, the next ones' offsets are on their way (10000 sequences of 20 tokens, 12
    // heads of 64 in f32: 3.4 ms, 13.3 by 64 at a time).
    auto skip = [&](auto chunks) {
      constexpr int N = decltype(chunks)::value, SPAN = 256 * N;
      typedef int I4 __attribute__((ext_vector_type(4), aligned(4)));
      I4 next[N];
      auto load = [&](int s) {
#pragma unroll
        for (int u = 0; u < N; ++u) next[u] = *reinterpret_cast<const I4*>(a.offsets + s + 1 + u * 256 + lane * 4);
      };
      if (s0 + SPAN <= a.n_seq) load(s0);
      for (; s0 + SPAN <= a.n_seq; s0 += SPAN) {
        I4 o[N];
#pragma unroll
        for (int u = 0; u < N; ++u) o[u] = next[u];
        if (s0 + 2 * SPAN <= a.n_seq) load(s0 + SPAN);
        int last = end, tiles = 0;
#pragma unroll
        for (int u = 0; u < N; ++u) {
          int h[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) h[i] = max(min(max(o[u][i], 0), a.n_rows), i ? h[i ? i - 1 : 0] : 0);
          const int upto = max(wave_max_scan(h[3]), last);
          int from = __shfl_up(upto, 1, 64);
          if (lane == 0) from = last;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int to = max(h[i], from);
            tiles += ((to - from) * a.group + ROWS - 1) / ROWS;
            from = to;
          }
          last = __builtin_amdgcn_readlane(upto, 63);
        }
        const int sum = wave_sum(tiles);
        if (at < sum) return;
        at -= sum;
        end = last;
      }
    };
    skip(std::integral_constant<int, 4>{});
    skip(std::integral_constant<int, 1>{});
    for (; s0 < a.n_seq; s0 += 64) {
      const int tiles = sequences(s0);
      int incl = tiles;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const int u = __shfl_up(incl, o, 64);
        if (lane >= o) incl += u;
      }
      const unsigned long long mine = __builtin_amdgcn_ballot_w64(at >= incl - tiles && at < incl);
      if (mine) {
        const int l = __builtin_ctzll(mine);
        take(l, __builtin_amdgcn_readlane(incl, l) - 1 - at);
        break;
      }
      at -= __builtin_amdgcn_readlane(incl, 63);
    }
  }
  if (j.tile >= 0) {
    a.n_q = j.count;
    return attend<M, HD, P, P == 1 ? 2 : P, T, Stage, KG>(a, j, s);
  }
  // `at` workgroups of this head are before this one among those that are left
  const int start = min(max(a.offsets[0], 0), a.n_rows), spare = start + a.n_rows - end;
  const int step = (int)(gridDim.x / a.n_head) - (index - at), per = a.group * a.hd;
  for (int r = at; r < spare; r += step) {
    const long row = r < start ? r : end + (r - start);
    for (int c = threadIdx.x; c < per; c += Stage::NT * KG)
      static_cast<T*>(a.out.p)[row * a.out.tok + (long)(j.head * a.group + c / a.hd) * a.out.head + c % a.hd] = (T)0.f;
  }
}

template <int QP, int PP, class T>
void many_t(hipStream_t s, Args a) {
  dim3 grid((unsigned)(a.n_seq * a.n_head), (unsigned)((a.n_q * a.group + 127) / 128));
  const long tiles = (long)grid.x * grid.y;
  if (tiles <= kSplits) {
    // eight waves a workgroup, one workgroup a compute unit; the keys are split where there are fewer
    a.min_stages = kMinStages;
    grid.z = (unsigned)fmany_parts(tiles, a.c.sizes());
    constexpr int KG = QP == 3 ? 1 : 2;  // (f32 queries of 128 columns leave registers for four)
    if (a.c.hdp == 64) f_attend_many_kernel<64, QP, PP, T, 2><<<grid, 512, 0, s>>>(a);
    else f_attend_many_kernel<128, QP, PP, T, KG><<<grid, 256 * KG, 0, s>>>(a);
  } else {
    if (a.c.hdp == 64) f_attend_many_kernel<64, QP, PP, T, 1><<<grid, 256, 0, s>>>(a);
    else f_attend_many_kernel<128, QP, PP, T, 1><<<grid, 256, 0, s>>>(a);
  }
}
template <class M, int HD, int P, class T, class Stage, int KG, int RESIDENT>
void packed_run(hipStream_t s, const Args& a) {
  constexpr int ROWS = Stage::NT / 2;
  const unsigned tiles = (unsigned)((a.n_rows * (long)a.group + ROWS - 1) / ROWS + a.n_seq);
  packed_attend_kernel<M, HD, P, T, Stage, KG, RESIDENT><<<tiles * (unsigned)a.n_head, Stage::NT * KG, 0, s>>>(a);
}
template <class M, int HD, class T>
void packed_t(hipStream_t s, const Args& a) {
  // Where all tiles are on the device at once, the time is that of the tile with most
  // keys: two groups of waves have every second stage of its keys each, if it has many
  // of them (4001 tokens of 12 heads of 64 in f32: 171 us, 198 with one group; of 16
  // in f16: 73 and 79; 16 x up to 1023 of 20 in f32: 191 and 161). (Rows of 16 bits that
  // are not aligned, in heads above 64: all registers are taken, and two to four that the
  // results need at the end wait in scratch meanwhile.)
  const bool two = a.n_rows * (long)a.group / 128 * a.n_head <= 512 && a.n_rows >= 512L * a.n_seq;
  if constexpr (sizeof(T) == 4) {
    // (one buffer: with two, 64 columns take 96 KB, which leaves a compute unit one
    // workgroup, of four waves or eight; 128 columns do so in any case)
    constexpr int KG = HD == 64 ? 2 : 1, RES = HD == 64 ? 2 : 1;
    if (a.kvec && two) packed_run<M, HD, 3, T, RowStage<M, HD, 3, T, true, 4, 1>, KG, 1>(s, a);
    else if (a.kvec) packed_run<M, HD, 3, T, RowStage<M, HD, 3, T, true, 4, 1>, 1, RES>(s, a);
    else if (two) packed_run<M, HD, 3, T, RowStage<M, HD, 3, T, false, 4, 1>, KG, 1>(s, a);
    else packed_run<M, HD, 3, T, RowStage<M, HD, 3, T, false, 4, 1>, 1, RES>(s, a);
  } else {
    // (a lane's offset within a stage of 64 rows is 32 bits, unsigned)
    auto near = [](const QRows& r) { return r.tok >= 0 && r.tok < 1 << 22; };
    const bool direct = a.kvec && near(a.k) && near(a.v);
    if (direct && two) packed_run<M, HD, 1, T, DirectStage<M, HD, 4>, 2, 1>(s, a);
    else if (direct) packed_run<M, HD, 1, T, DirectStage<M, HD, 4>, 1, 2>(s, a);
    else if (two) packed_run<M, HD, 1, T, RowStage<M, HD, 1, T, false, 4, 2>, 2, 1>(s, a);
    else packed_run<M, HD, 1, T, RowStage<M, HD, 1, T, false, 4, 2>, 1, 2>(s, a);
  }
}
template <class M, class T>
void packed(hipStream_t s, const Args& a) {
  if (a.hd <= 64) packed_t<M, 64, T>(s, a);
  else packed_t<M, 128, T>(s, a);
}

}  // namespace

void launch_f_attend_many(hipStream_t s, const FAttn& f) {
  Args a = {};
  a.tickets = reinterpret_cast<unsigned*>(static_cast<char*>(f.work) + kTicketBytes);
  a.parts = reinterpret_cast<float*>(static_cast<char*>(f.work) + 2 * kTicketBytes);
  a.q = f.q;
  a.out = f.out;
  a.c = f.c;
  a.len = f.len;
  a.counts = f.counts;
  a.n_seq = f.c.n_seq;
  a.n_head = f.c.n_head;
  a.n_q = f.n_q;
  a.n_q_head = f.n_q_head;
  a.group = f.n_q_head / f.c.n_head;
  a.hd = f.c.hd;
  const ScoreScale sc = score_scale(f.scale);
  a.query = sc.query;
  a.sum = sc.sum;
  a.stats = f.stats;
  a.qvec = by_eights(f.q, a.hd, f.type);
  a.ovec = by_eights(f.out, a.hd, f.type);
  if (f.type == Q_F32) many_t<3, 3, float>(s, a);
  else if (f.type == Q_BF16) many_t<1, 2, __bf16>(s, a);
  else many_t<2, 2, _Float16>(s, a);
}

void launch_packed_attend(hipStream_t s, const PAttn& p) {
  Args a = {};
  a.q = p.q;
  a.k = p.k;
  a.v = p.v;
  a.out = p.out;
  a.offsets = p.offsets;
  a.n_rows = p.n_rows;
  a.n_seq = p.n_seq;
  a.n_head = p.n_head;
  a.n_q_head = p.n_q_head;
  a.group = p.n_q_head / p.n_head;
  a.hd = p.hd;
  ScoreScale sc = score_scale(p.scale);
  if (p.type == Q_F16) {
    // (f16 does not hold the queries times any power of two)
    sc.sum = (float)std::min(std::max(fabs((double)p.scale) * 1.4426950408889634074, 1.2e-38), 3.4e38);
    sc.query = p.scale == 0.f ? 0.f : copysignf(1.f, p.scale);
  }
  a.query = sc.query;
  a.sum = sc.sum;
  a.qvec = by_eights(p.q, a.hd, p.type);
  a.kvec = by_eights(p.k, a.hd, p.type) && by_eights(p.v, a.hd, p.type);
  a.ovec = by_eights(p.out, a.hd, p.type);
  if (p.type == Q_F32) packed<Bf16, float>(s, a);
  else if (p.type == Q_BF16) packed<Bf16, __bf16>(s, a);
  else packed<F16, _Float16>(s, a);
}

}  // namespace rtg
