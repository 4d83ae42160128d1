// What an append of tokens to the 8-bit cache is made of (qcache.h): where it goes,
// scales and codes, and one token's append as a part of a kernel.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "qcache.h"

namespace rtg {

// Where an append of a sequence goes: tokens [at, end) over a length of len.
struct Place {
  int len, at, end;
  int from;  // a token of the first block to be written: of the last one left where nothing is new
  int bad;   // 0, or why it is refused (QTickets)
};
__device__ __forceinline__ Place place(int seq, const int* len, int len_stride, int n_new, const int* counts,
                                       const int* start, int capacity) {
  Place p;
  p.len = len[(size_t)seq * len_stride];
  p.at = start ? start[seq] : p.len;
  const int n = counts ? min(max(counts[seq], 0), n_new) : n_new;
  p.bad = p.at < 0 || p.at > p.len ? 1 : n > capacity - p.at ? 2 : 0;
  p.end = p.bad ? p.at : p.at + n;
  p.from = p.end > p.at || p.at == 0 ? p.at : p.at - 1;
  return p;
}

// Byte of a value's code within its (sequence, head): tile, then [4][hdp][16].
__device__ __forceinline__ size_t value_byte(int tok, int col, int hdp) {
  return (size_t)(tok >> 6) * kQTile * hdp + ((size_t)((tok >> 2) & 3) * hdp + col) * 16 + ((tok >> 4) & 3) * 4 +
         (tok & 3);
}

// Whether the first block to be written is the one that the tail holds: the block
// of the last token.
__device__ __forceinline__ bool in_tail(const QStore& c, const Place& p) {
  return p.len > 0 && p.from >> c.block_shift == (p.len - 1) >> c.block_shift;
}

constexpr unsigned kNanBits = 0x7FC00000u;

// fl(amax / 127) of a token, as bits (which order like the values): 0 below
// 127 * 2^-126 (so that a scale is never subnormal), NaN for what is not finite.
__device__ __forceinline__ unsigned token_scale(float amax) {
  if (!(amax <= 3.402823466e38f)) return kNanBits;
  if (amax < 127.f * 1.17549435e-38f) return 0;
  return __float_as_uint(__fdiv_rn(amax, 127.f));
}

// The integer nearest to x / s, ties to even, from one that is off by one at most: r.
__device__ __forceinline__ float code_of(float x, float s, float r) {
  const float res = fmaf(-r, s, x), half = 0.5f * s;
  const bool odd = ((int)r & 1) != 0;
  if (res > half || (res == half && odd)) return r + 1.f;
  if (res < -half || (res == -half && odd)) return r - 1.f;
  return r;
}
__device__ __forceinline__ float scale_inv(float s) { return s > 0.f ? __fdiv_rn(1.f, s) : 0.f; }

// A value of a full block as it reads back, and its token's own scale: a token
// that holds code 127 had the block's scale (amax / 127 may round otherwise).
__device__ __forceinline__ float code_value(int8_t code, float s) { return (float)code * s; }
__device__ __forceinline__ unsigned read_back_scale(float amax, float s) {
  return amax == 127.f * s ? __float_as_uint(s) : token_scale(amax);
}

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
// Largest bits over the wave.
__device__ __forceinline__ unsigned wave_max_bits(unsigned v) {
  v = row_max_bits<128>(v);
  const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return max(r[0], r[1]);
}

// One new token (or only a cut) of one (sequence, head) by the first four of a
// workgroup's WAVES: 0 and 1 write the keys, 2 and 3 the values, a lane a column
// (two for hdp 128). The new scale follows from the tokens' own scales; only
// where it differs from the block's are the block's codes written anew, the two
// waves taking every other token.
template <int HDP, class T, int WAVES>
class OneToken {
 public:
  // The token's row, if there is one (it does not depend on the place: the load
  // is in flight while that is found).
  __device__ __forceinline__ OneToken(const QStore& c, int seq, int head, const QRows& k, const QRows& v, bool any)
      : lane(threadIdx.x & 63), which(threadIdx.x >> 7), part((threadIdx.x >> 6) & 1) {
    const QRows& src = which ? v : k;
#pragma unroll
    for (int e = 0; e < CL; ++e) {
      const int col = lane + e * 64;
      x[e] = any && active() && col < c.hd
                 ? (float)(static_cast<const T*>(src.p) + seq * src.seq + head * src.head)[col] : 0.f;
    }
  }

  // By the whole workgroup, where p moves the sequence's end.
  __device__ __forceinline__ void write(const QStore& c, const Place& p, int sh) const {
    const bool has = p.end > p.at;
    const int blk = p.from >> c.block_shift, in = p.at - (blk << c.block_shift);  // `in` earlier tokens in the block
    const bool tailed = in_tail(c, p);
    float* tail = c.tail + c.tails(sh, which);
    float* tail_s = c.tail_s + c.tail_scales(sh, which);
    int8_t* codes = (which ? c.v : c.k) + c.codes(sh);
    float* scale = c.s + c.scales(sh) + 2 * blk + which;
    auto code_at = [&](int tok, int col) { return which ? value_byte(tok, col, HDP) : (size_t)tok * HDP + col; };
    const int blk0 = blk << c.block_shift;
    unsigned mine = 0, all = 0;
    float old = 0.f;
    // an earlier token's own scale, where the block was full: from its codes
    auto own_scale = [&](int t) {
      unsigned m = 0;
#pragma unroll
      for (int e = 0; e < CL; ++e) m = max(m, abs_bits(code_value(codes[code_at(blk0 + t, lane + e * 64)], old)));
      return read_back_scale(__uint_as_float(wave_max_bits(m)), old);
    };
    if (active()) {
      unsigned top = 0;
#pragma unroll
      for (int e = 0; e < CL; ++e) top = max(top, abs_bits(x[e]));
      mine = has ? token_scale(__uint_as_float(wave_max_bits(top))) : 0;
      old = in > 0 ? *scale : 0.f;
      all = mine;
      if (tailed) {
        all = max(all, wave_max_bits(lane < in ? __float_as_uint(tail_s[lane]) : 0));
      } else {
        for (int t = 0; t < in; ++t) all = max(all, own_scale(t));
      }
    }
    __syncthreads();  // both waves have read the scale, the tail's scales and the codes
    if (!active()) return;
    const float s = __uint_as_float(all), inv = scale_inv(s);
    const bool anew = in > 0 && __float_as_uint(old) != all;
    auto put = [&](int tok, int col, float value) {
      codes[code_at(tok, col)] = (int8_t)(s > 0.f ? (int)code_of(value, s, rintf(value * inv)) : 0);
    };
    if (anew || !tailed) {
      constexpr int U = 8;  // tokens in flight
      for (int t0 = part; t0 < in; t0 += 2 * U) {
        float y[U][CL];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int e = 0; e < CL; ++e) {
            const int t = min(t0 + 2 * u, in - 1), col = lane + e * 64;
            y[u][e] = tailed ? tail[t * HDP + col] : code_value(codes[code_at(blk0 + t, col)], old);
          }
#pragma unroll
        for (int u = 0; u < U; ++u) {
          const int t = t0 + 2 * u;
          if (t >= in) break;
          if (!tailed) {
            const unsigned ts = own_scale(t);
            if (lane == 0) tail_s[t] = __uint_as_float(ts);
          }
#pragma unroll
          for (int e = 0; e < CL; ++e) {
            const int col = lane + e * 64;
            if (!tailed) tail[t * HDP + col] = y[u][e];
            if (anew) put(blk0 + t, col, y[u][e]);
          }
        }
      }
    }
    if (part == 0) {
      if (has) {
#pragma unroll
        for (int e = 0; e < CL; ++e) {
          const int col = lane + e * 64;
          put(p.at, col, x[e]);
          tail[in * HDP + col] = x[e];
        }
        if (lane == 0) tail_s[in] = __uint_as_float(mine);
      }
      if (lane == 0 && (has || in > 0)) *scale = s;
    }
  }

 private:
  static constexpr int CL = HDP / 64;
  __device__ __forceinline__ bool active() const { return WAVES <= 4 || which < 2; }
  const int lane, which, part;
  float x[CL];
};

}  // namespace rtg
