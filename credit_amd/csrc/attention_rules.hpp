// How attention over a paged cache (attention.hip) cuts its work, and the
// workspace that takes.  Host arithmetic alone, so that the CPU tests build it
// with g++ (tests/cpp/heads_rules_query.cpp).
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <algorithm>

namespace credit {
namespace attention {

constexpr int kMaxDim = 256;
constexpr int kFew = 32;     // query rows (tokens times heads of a group) of a small tile
constexpr int kMany = 128;   // of a large one
constexpr int kKeys = 64;    // positions of a step of large tiles
constexpr int kFewKeys = 32; // of small ones
constexpr int kMaxParts = 128;
constexpr int kMaxBatch = 1024;     // sequences that a wave counts through

// Small tiles serve where a sequence has no more rows than one.
inline int tile_rows(int64_t tokens, int64_t batch, int64_t group) {
  return tokens * group <= kFew * batch ? kFew : kMany;
}

// Tiles of a call whose sequences may lie anywhere: sequence b's begin at slot
// floor(first row of b / rows) + b, which leaves it at least as many as its rows
// fill whatever the lengths are.
inline int64_t tiles(int64_t tokens, int64_t batch, int64_t group, int rows) {
  return tokens * group / rows + batch;
}

// Parts that the positions of tiles are cut into: all tiles' steps, as they turn
// out on the device, are dealt to about `share` units (of each key head) of one
// length, at least least_steps, a tile to at most `most` of them; `units` bounds
// their number.  most 1: none are cut.
struct Parts {
  int most, least_steps, share, units;
};
inline Parts parts(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads,
                   int64_t positions) {
  const int64_t group = heads / kv_heads;
  const int rows = tile_rows(tokens, batch, group);
  const int64_t all = tiles(tokens, batch, group, rows);
  const int keys = rows == kFew ? kFewKeys : kKeys;
  const int64_t least = rows == kFew ? 8 : 16;
  const int64_t longest = (positions + keys - 1) / keys;
  const int64_t share = rows == kFew ? std::max<int64_t>(1, (2048 + kv_heads - 1) / kv_heads)
                                     : std::max<int64_t>(1, 512 / kv_heads - all);
  const int64_t most = std::min<int64_t>({rows == kFew ? kMaxParts : kMaxParts / 4,
                                          (longest + least - 1) / least, share});
  if (most < 2 || batch > kMaxBatch || all > 4 * share) return {1, 0, 0, 0};
  return {static_cast<int>(most), static_cast<int>(least), static_cast<int>(share),
          static_cast<int>(share + all)};
}

inline int padded_dim(int dim) { return dim <= 64 ? 64 : dim <= 128 ? 128 : 256; }

// Floats that a part of a tile leaves: its rows' outputs, maxima and sums.
inline int64_t part_floats(int rows, int dim) {
  return static_cast<int64_t>(rows) * (padded_dim(dim) + 2);
}

inline size_t workspace(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int dim,
                        int64_t positions) {
  const Parts p = parts(tokens, batch, heads, kv_heads, positions);
  if (p.most < 2) return 0;
  const int64_t group = heads / kv_heads;
  const int rows = tile_rows(tokens, batch, group);
  return static_cast<size_t>(p.units * kv_heads * part_floats(rows, dim)) * sizeof(float);
}

// n / d for n < 2^31 as (mulhi(n, mul) + n) >> shift.
struct Divisor {
  uint32_t mul, shift;
};
inline Divisor divisor(uint32_t d) {
  uint32_t s = 0;
  while ((uint64_t{1} << s) < d) ++s;
  return {static_cast<uint32_t>(((uint64_t{1} << 32) * ((uint64_t{1} << s) - d)) / d + 1), s};
}

}  // namespace attention
}  // namespace credit
