// Sizes of the 4-bit cache, and which of the two kernels attends over it
// (fourbit_attn.hip, attn_tile.hip); host code without HIP, so that a test can check
// what the dispatch reaches.
#pragma once
#include <stddef.h>

#include <algorithm>

namespace rtg {

struct FSizes {
  int n_seq, n_head, hdp, tiles;  // hdp: head_dim padded to 64 or 128; tiles of 32 tokens
  size_t pairs() const { return (size_t)n_seq * n_head; }
  size_t code_bytes() const { return up256(pairs() * tiles * 16 * hdp); }  // of keys; of values
  size_t scale_bytes() const { return up256(pairs() * tiles * hdp); }
  size_t weight_bytes() const { return up256(pairs() * tiles * 32 * 4); }
  size_t bytes() const { return 2 * code_bytes() + 2 * scale_bytes() + weight_bytes(); }

 private:
  static size_t up256(size_t x) { return (x + 255) / 256 * 256; }
};

constexpr int kCols = 16, kRows = 128;  // (query, head) pairs: of a block of the one kernel, of a tile of the other

// Workgroups at most where the keys are split, and how many of them there is room for.
// One's results take 4 KB (16 columns) or 34 (128 rows) for heads up to 64 channels,
// twice that above: room for all of them, 9 or 17 MB, would be more than the keys and
// values of a cache of up to 10000 tokens of 12 heads, and there is one for each layer;
// so there is room for half as many bytes as the cache holds.
constexpr int kSplits = 256;
inline size_t few_part_bytes(const FSizes& c) { return kCols * (size_t)(c.hdp + 2) * 4; }
inline size_t many_part_bytes(const FSizes& c) { return kRows * (size_t)(c.hdp + 4) * 4; }
inline size_t fattn_parts_bytes(const FSizes& c) {
  return std::min(c.bytes() / 2 / 256 * 256, kSplits * many_part_bytes(c));
}
inline int few_room(const FSizes& c) { return (int)std::min((size_t)kSplits, fattn_parts_bytes(c) / few_part_bytes(c)); }
inline int many_room(const FSizes& c) { return (int)(fattn_parts_bytes(c) / many_part_bytes(c)); }

constexpr int kMinStages = 8;  // of 64 keys, of a part at least in the kernel of many rows
// Parts that it splits the keys into, for up to kSplits tiles of rows.
inline long fmany_parts(long row_tiles, const FSizes& c) {
  return std::max(1l, std::min(many_room(c) / row_tiles, ((long)c.tiles / 2 + kMinStages - 1) / kMinStages));
}

// What the two kernels take, in us, fitted to 816 calls (24 to 3200 columns of 2 to 320
// sequences' heads, 40 to 16400 tokens) within 10 and 5 % on average: by blocks of 16
// columns, tiles of 128 rows, and the keys' tiles that a sequence may have, as the host
// does not know the lengths (both take less where they are shorter). The kernel that is
// chosen so takes 0.8 % longer than the better one on average, at most 38 % (80 queries of
// 24 sequences' 8 heads of 128 behind 40 tokens in f32: 21 and 15 us); the one of few
// columns alone 6.6 % and 129 %, the other alone 58 % and 488 %. Where a sequence is much
// shorter than the capacity the other kernel may be the better one, and results may differ
// in their last place with the capacity, as sums in another order do.
struct FCosts {
  float few, few_block, few_tile;        // a call; 256 blocks; 256 blocks of 32 tiles of keys
  float many, many_join, many_split;     // up to 256 tiles of rows: a call; parts to join; 32 tiles of keys of a part
  float many_block, many_tile;           // more: 512 of them; 512 of 32 tiles of keys
};
constexpr FCosts kFCosts[3][2] = {
    {{9.0f, 0.2f, 3.4f, 9.5f, 3.9f, 18.9f, 0.9f, 45.5f}, {7.9f, 2.6f, 6.0f, 10.6f, 5.1f, 39.5f, 16.5f, 86.0f}},  // f32
    {{9.0f, 0.1f, 2.7f, 8.5f, 3.9f, 13.3f, 0.1f, 28.8f}, {8.1f, 1.8f, 4.5f, 9.9f, 7.8f, 19.2f, 1.1f, 48.8f}},    // bf16
    {{8.9f, 0.2f, 2.8f, 8.7f, 4.1f, 16.2f, 0.8f, 32.1f}, {7.9f, 2.0f, 4.9f, 11.1f, 7.8f, 22.0f, 1.6f, 55.5f}},   // f16
};
// Whether the kernel of many rows takes `columns` pairs of query and head of each
// sequence's key/value heads; type: 0 f32, 1 bf16, 2 f16.
inline bool for_many(const FSizes& f, int type, long columns) {
  const long blocks = (columns + kCols - 1) / kCols;
  if (columns <= 32) return false;   // (a quarter of the rows at most)
  if (blocks > 65535) return true;   // (what a grid holds)
  const long heads = (long)f.n_seq * f.n_head, rows = heads * ((columns + kRows - 1) / kRows), keys = f.tiles;
  const FCosts& c = kFCosts[type][f.hdp == 128];
  const float b = heads * blocks / 256.f, few = c.few + b * (c.few_block + c.few_tile * (keys / 32.f));
  if (rows > kSplits) return few > c.many + rows / 512.f * (c.many_block + c.many_tile * (keys / 32.f));
  const long parts = fmany_parts(rows, f);
  return few > c.many + (parts > 1 ? c.many_join : 0.f) + c.many_split * ((keys + parts - 1) / parts / 32.f);
}

}  // namespace rtg
