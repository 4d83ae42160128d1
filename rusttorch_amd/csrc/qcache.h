// The 8-bit key/value cache: layout and launchers (qcache.hip, qattn.hip).
//
// For each (sequence, head) keys and values are codes of 8 bits, x ~ code * s,
// with one scale s for each block of `block` consecutive tokens:
//   s = max over the block's tokens of fl(amax(token) / 127)  (fl: f32 rounding)
//       (a token whose amax is below 127 * 2^-126 counts as 0, one with a value
//       that is not finite as NaN, and NaN is the largest)
//   code = the integer nearest to x / s, ties to even; 0 where s is 0 or NaN.
// The block of the last token is quantised anew from its tokens' f32 values,
// kept in `tail`, whenever a token raises its scale, so the cache depends on the
// tokens only and not on how they were split over calls.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kernels.h"

namespace rtg {

constexpr int kQTile = 64;  // tokens that the attention takes at a time: one i8 MFMA's depth

// Rows are padded to hdp = 64 or 128 columns of code 0 (one or two i8 MFMAs).
// Keys [seq][head][token][hdp]. Values in tiles of 64 tokens, each as
// [4][hdp][16]: token t of a tile is byte ((t >> 4) & 3) * 4 + (t & 3) of the
// 16 at [(t >> 2) & 3][column], the order in which the lanes that compute a
// tile's probabilities hold them (qattn.hip), 4 consecutive tokens side by side.
struct QStore {
  int n_seq = 0, n_head = 0, hd = 0, hdp = 0;
  int block = 0, block_shift = 0;
  int capacity = 0, tiles = 0;  // tokens; tiles per (sequence, head)
  int8_t *k = nullptr, *v = nullptr;
  float* s = nullptr;       // scales [seq][head][tiles * 64 / block][2]: keys', values'
  float* tail = nullptr;    // the last block's values [seq][head][2][block][hdp]
  float* tail_s = nullptr;  // and its tokens' own scales [seq][head][2][block]

  __host__ __device__ size_t codes(size_t sh) const { return sh * tiles * (size_t)kQTile * hdp; }
  __host__ __device__ size_t scales(size_t sh) const { return sh * 2 * ((size_t)tiles * kQTile >> block_shift); }
  __host__ __device__ size_t tails(size_t sh, int which) const { return (sh * 2 + which) * (size_t)block * hdp; }
  __host__ __device__ size_t tail_scales(size_t sh, int which) const { return (sh * 2 + which) * (size_t)block; }
  // The sequences from `first` on as a store of their own (a layer of a model's cache).
  QStore from(size_t first, int n) const {
    QStore r = *this;
    const size_t sh = first * n_head;
    r.n_seq = n;
    r.k += codes(sh);
    r.v += codes(sh);
    r.s += scales(sh);
    r.tail += tails(sh, 0);
    r.tail_s += tail_scales(sh, 0);
    return r;
  }
};

// Element types of rows in device memory.
enum QType { Q_F32 = 0, Q_BF16 = 1, Q_F16 = 2 };

// Rows [seq][token][head][hd] in device memory, strides in elements, the
// columns of a row contiguous.
struct QRows {
  void* p = nullptr;
  long seq = 0, tok = 0, head = 0;
};

// Bytes of the parts of a store (n_seq, n_head, hd, hdp, block, capacity, tiles set).
size_t qstore_bytes(const QStore& c);
// Shapes and then pointers into mem (qstore_bytes bytes, 256-byte aligned).
void qstore_shape(QStore* c, int n_seq, int n_head, int hd, int capacity, int block);
void qstore_place(QStore* c, void* mem);

// Where the sequences' lengths are: len[seq * stride] (stride 0: one for all).
struct QLen {
  int* p = nullptr;
  int stride = 1;
};

// For appends that move the lengths: how many workgroups of the append in flight
// have read their sequence's length, counted per (sequence, head) and, as the
// heads are through, per sequence (0 between appends; a counter per cache line:
// atomics on one line take turns, 8.6 ns each); and *err = min(*err,
// seq * 4 + 1 or 2) where a sequence's start (1) or its number of tokens (2) is refused.
struct QTickets {
  unsigned* count = nullptr;  // [n_seq * (n_head + 1)][kQTicketStride]
  unsigned* err = nullptr;
};
constexpr int kQTicketStride = 32;

// New tokens k, v (at most n_new for a sequence; counts[seq] of them where
// counts is given, clamped to 0 .. n_new) behind the length, or from start[seq]
// on where start is given. A sequence whose start is negative or behind its
// length, or whose tokens would pass the capacity, is left as it is. With
// tickets the lengths are the new ones afterwards, else as they were.
void launch_q_append(hipStream_t s, const QStore& c, QLen len, QTickets tickets, QType type, const QRows& k,
                     const QRows& v, int n_new, const int* counts, const int* start);
// Tokens first[seq] (0 without first) .. + n of every sequence as values; rows
// that hold no token are set to 0. k or v may have no p.
void launch_q_read(hipStream_t s, const QStore& c, QLen len, QType type, const QRows& k, const QRows& v, int n,
                   const int* first);

// Attention results: rows (QRows), or the layouts of the model's next GEMM, for
// f32 queries and head dims up to 64: the pair GEMM's input scaled per column
// (as many query heads as the cache has), or the batched decode GEMV's
// (launch_q_step; xt_index with n_seq rows).
enum QOutKind { QO_ROWS = 0, QO_PAIR = 1, QO_XT = 2 };
struct QOut {
  QOutKind kind = QO_ROWS;
  QRows rows;
  uint16_t* pair = nullptr;      // row seq * n_q + query of 2 d f16, d = n_q_head * hd
  const float* scale = nullptr;  // [d]
  float* xt = nullptr;
  int tk = 0;
};

// Attention of each sequence's last counts[seq] (n_q without counts) tokens
// over the cache: query i sits at position len - count + i and sees the keys up
// to its own position. extra is added to the lengths. scale: of the dot products.
// Rows of queries that see no key, and of i >= count, are set to 0.
// work: qattn_work_bytes() bytes, cleared once (qattn_work_clear).
void launch_q_attend(hipStream_t s, const QStore& c, QLen len, int extra, QType type, const QRows& q, int n_q,
                     int n_q_head, const int* counts, float scale, const QOut& out, void* work);
// A model's decode step: one f32 token k, v behind the length of every sequence
// (which is below the capacity, and stays as it is), and its query's attention
// over them all. Head dims up to 64, as many query heads as the cache has.
void launch_q_step(hipStream_t s, const QStore& c, QLen len, const QRows& k, const QRows& v, const QRows& q,
                   float scale, const QOut& out, void* work);
size_t qattn_work_bytes(int hdp);
void qattn_work_clear(hipStream_t s, void* work, int hdp);

}  // namespace rtg
