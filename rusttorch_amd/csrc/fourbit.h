// The 4-bit key/value cache: layout and launchers (fourbit.hip, fourbit_attn.hip,
// attn_tile.hip).
//
// For each (sequence, head) and token, keys and values apart, 32 consecutive
// channels are numbers of 4 bits (E2M1: a sign and 0, 0.5, 1, 1.5, 2, 3, 4, 6)
// times one power of two, kept as its biased exponent in a byte:
//   byte = exponent of max |x|, one more where max |x| is over 1.75 times its
//          power of two, less 2; within 27 .. 252; 255 (NaN) where a value is
//          not finite
//   number = the nearest to x / 2^(byte - 127), ties to the even code, at most 6.
// A token's codes depend on its own values alone, so tokens can be moved and
// dropped without rounding anything anew. The format is the one that the matrix
// unit's conversions take (v_cvt_scalef32_pk_*_fp4): two codes and a scale become
// two bf16 in one instruction, exactly.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fourbit_choice.h"
#include "qcache.h"

namespace rtg {

constexpr int kFTile = 32;  // tokens: the depth of one bf16 MFMA

// Heads are padded to hdp = 64 or 128 channels of code 0 (CK = hdp / 4 channels
// are a quarter, CV = hdp / 16 a sixteenth). Codes lie in tiles of 32 tokens in
// the order in which the lanes of a wave take them as matrix operands; lane
// (g, m) = g * 16 + m.
//   keys    lane (g, m) has channels CK g .. of tokens m and 16 + m:
//           hdp 128 [2 b][64 lanes][16 bytes], token 16 b + m; hdp 64
//           [64 lanes][2 b][8 bytes]. Their scales: hdp 128 [2 b][4 g][16 m],
//           hdp 64 [2 b][2][16 m].
//   values  lane (g, m) has channels CV m .. of the tokens b * 16 + 4 g + i,
//           b < 2, i < 4 (those whose scores it computes): hdp 128
//           [2 b][64 lanes][4 i][4 bytes], hdp 64 [64 lanes][2 b][4 i][2 bytes].
//           Their scales: [4 g][hdp / 32][2 b][4 i].
struct FStore {
  int n_seq = 0, n_head = 0, hd = 0, hdp = 0;
  int capacity = 0, tiles = 0;  // tokens; tiles of each (sequence, head)
  uint8_t *k = nullptr, *v = nullptr;    // codes [seq][head][tile][16 * hdp]
  uint8_t *sk = nullptr, *sv = nullptr;  // scales [seq][head][tile][hdp]
  float* w = nullptr;  // what attention the tokens have got [seq][head][tiles * 32]

  FSizes sizes() const { return {n_seq, n_head, hdp, tiles}; }
  __host__ __device__ size_t codes(size_t sh) const { return sh * tiles * (size_t)(16 * hdp); }
  __host__ __device__ size_t scales(size_t sh) const { return sh * tiles * (size_t)hdp; }
  __host__ __device__ size_t weights(size_t sh) const { return sh * tiles * (size_t)kFTile; }
};

void fstore_shape(FStore* c, int n_seq, int n_head, int hd, int capacity);
void fstore_place(FStore* c, void* mem);

// As launch_q_append and launch_q_read (qcache.h). Tickets: [n_seq][kQTicketStride].
void launch_f_append(hipStream_t s, const FStore& c, int* len, QTickets tickets, QType type, const QRows& k,
                     const QRows& v, int n_new, const int* counts, const int* start);
void launch_f_read(hipStream_t s, const FStore& c, const int* len, QType type, const QRows& k, const QRows& v, int n,
                   const int* first);

// The weights of tokens 0 .. n - 1 of every (sequence, head) to out [sh][n], 0
// where there is no token; and x [sh][n] added to those that are there.
void launch_f_weights(hipStream_t s, const FStore& c, const int* len, float* out, int n);
void launch_f_add_weights(hipStream_t s, const FStore& c, const int* len, const float* x, int n);
// Sequences longer than `keep` are cut to it; kept [sh][keep]: which tokens
// (ascending), -1 behind a shorter sequence's.
void launch_f_evict(hipStream_t s, const FStore& c, int* len, QTickets tickets, int keep, int recent, int* kept);

// Attention as launch_q_attend, results as rows; stats [seq][n_q][n_q_head][2] (may
// be null): for each query's scores x (times log2 e) an m and the sum of 2^(x - m),
// 0 where it sees no key. work: fattn_work_bytes() bytes, cleared once (fattn_work_clear):
// tickets of the kernels of few columns and of many rows, kSplits of each, then partial
// results of either (one call at a time works on a cache).
struct FAttn {
  FStore c;
  const int* len = nullptr;
  QType type = Q_F32;
  QRows q, out;
  int n_q = 0, n_q_head = 0;
  const int* counts = nullptr;
  float scale = 0.f;
  float* stats = nullptr;
  void* work = nullptr;
};
void launch_f_attend(hipStream_t s, const FAttn& a);
// for many queries (launch_f_attend chooses)
void launch_f_attend_many(hipStream_t s, const FAttn& a);
// w = decay * w + the probabilities that the queries (as in launch_f_attend, whose
// stats it takes) give a token, summed over the counted queries and the heads of
// the token's head; decay 0: w as it was is not read.
void launch_f_weigh(hipStream_t s, const FAttn& a, float decay);
size_t fattn_work_bytes(const FStore& c);
void fattn_work_clear(hipStream_t s, void* work);
constexpr size_t kTicketBytes = (size_t)kSplits * kQTicketStride * 4;

// Causal attention of packed sequences, each over itself: rows [n_rows][head][hd]
// (the rows' seq strides are not used), sequence s at rows offsets[s] ..
// offsets[s + 1] (clamped to the rows there are). Rows of no sequence are 0.
struct PAttn {
  QType type = Q_F32;
  QRows q, k, v, out;
  int n_rows = 0, n_seq = 0, n_head = 0, n_q_head = 0, hd = 0;
  const int* offsets = nullptr;
  float scale = 0.f;
};
void launch_packed_attend(hipStream_t s, const PAttn& a);

}  // namespace rtg
