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

// Small tiles serve where a sequence has no more rows than one.  us, small / large,
// 32 heads over 8 key heads of 128, 8 sequences of 8192 positions: 8 new tokens each
// (32 rows) 60 / 68, 16 tokens 83 / 75, 32 tokens 128 / 80; 64 sequences, one token
// each 355 / 448.
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
//
// Meeting costs some 4 us, which a tile of up to 16 steps takes by itself: one sequence
// of 512 positions 11.6 us in parts, 9.5 whole; of 1024 11.7 / 14.0, of 8192 13.3 / 83.
// 64 ragged sequences of up to 16384 390 / 493, 512 tokens over 8192 positions 93 /
// 194.  A run of at least 8 small steps: 4 / 8 / 16 of them 15.1 / 13.3 / 14.2 us at
// 8192 positions (10.5 / 11.7 / 14.0 at 1024), and of at least 16 large ones: 8 / 16 /
// 32 of them 51 / 42 / 60 us, 256 tokens over 4096 positions.
// More large tiles than there are units go whole, a prompt's later ones, which see
// more, first: a prompt of 8192 549 us whole, 785 in parts, of 4096 160 / 222, 4 chunks
// of 1024 over 8192 505 / 521.
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
  if (longest <= 16 || batch > kMaxBatch || all * longest >= (int64_t{1} << 31) ||
      kv_heads > kResident ||  // places lie within 32-bit offsets
      (rows == kMany && all > units))
    return {0, 0};
  return {static_cast<int>(std::min(units, (all * longest + least - 1) / least)),
          static_cast<int>(least)};
}

// Columns that the products take: 80 of 96 instead of 128 were 90 us against 102 (six
// sequences of up to 500 new tokens), 192 instead of 256 169 against 406.
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
