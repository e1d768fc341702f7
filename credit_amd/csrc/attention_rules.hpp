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
constexpr int kMaxBatch = 1024;  // sequences that a wave counts through
constexpr int kResident = 512;   // workgroups: two a CU

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

// How a call's steps are dealt out: to `units` workgroups a key head, in runs of one
// length of at least least_steps, whose first and last tile may be parts of theirs.
// units 0: a workgroup a tile, none in parts.
struct Parts {
  int units, least_steps;
};
inline Parts parts(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads,
                   int64_t positions) {
  const int64_t group = heads / kv_heads;
  const int rows = tile_rows(tokens, batch, group);
  const int64_t all = tiles(tokens, batch, group, rows);
  const int keys = rows == kFew ? kFewKeys : kKeys;
  const int64_t least = rows == kFew ? 8 : 16;
  const int64_t longest = (positions + keys - 1) / keys;
  const int64_t units = std::max<int64_t>(1, kResident / kv_heads);
  // Many tiles of a few steps, and long prompts, are dealt by the dispatcher.
  if (longest <= least || batch > kMaxBatch || all * longest >= (int64_t{1} << 31) ||
      kv_heads > kResident ||  // places lie within 32-bit offsets
      (rows == kMany && all > units))
    return {0, 0};
  return {static_cast<int>(std::min(units, (all * longest + least - 1) / least)),
          static_cast<int>(least)};
}

// Columns that the products take.
inline int padded_dim(int dim) {
  return dim <= 64 ? 64 : dim <= 96 ? 96 : dim <= 128 ? 128 : dim <= 192 ? 192 : 256;
}

// Floats that a part of a tile leaves: its rows' outputs, maxima and sums.
inline int64_t part_floats(int rows, int dim) {
  return static_cast<int64_t>(rows) * (padded_dim(dim) + 2);
}

inline size_t workspace(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int dim,
                        int64_t positions) {
  const Parts p = parts(tokens, batch, heads, kv_heads, positions);
  const int rows = tile_rows(tokens, batch, heads / kv_heads);
  return static_cast<size_t>(2 * p.units * kv_heads * part_floats(rows, dim)) * sizeof(float);
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
