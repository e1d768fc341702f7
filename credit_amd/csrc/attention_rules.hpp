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
constexpr int kManyDim = 192;  // of large tiles
constexpr int kFew = 32;     // query rows (tokens times heads of a group) of a small tile
constexpr int kMany = 128;   // of a large one
constexpr int kKeys = 64;    // positions of a step of large tiles
constexpr int kFewKeys = 32; // of small ones
constexpr int kMaxBatch = 1024;  // sequences that a wave counts through
constexpr int kResident = 512;   // workgroups: two a CU

// Columns that the products take: 80 of 96 instead of 128 were 90 us against 102 (six
// sequences of up to 500 new tokens), 192 instead of 256 169 against 406.
inline int padded_dim(int dim) {
  return dim <= 64 ? 64 : dim <= 96 ? 96 : dim <= 128 ? 128 : dim <= 192 ? 192 : 256;
}

// Small tiles serve where a sequence has no more rows than one; where they leave each
// a CU of its own and the positions are few, as there is not work enough to share; and
// for the widest heads, of which a large tile's wave has no registers for.  us, small /
// large, 32 heads over 8 key heads of 128: 8 sequences of 8192 positions with 8 new
// tokens each (32 rows) 61 / 68, with 16 84 / 75, with 32 124 / 85; 64 sequences with one
// 327 / 426; one sequence, 40 tokens over 500 positions 10.2 / 26, 64 over 2048 24 / 27,
// 128 over 8192 59 / 45; against the rule 10 tokens each of 9 sequences over 1024 31 / 26.
// 16 heads over 4 of 256: 13 tokens each of 9 sequences over 10818 171 / 292, 2048
// tokens over 4096 244 / 436.
//
// Lengths are on the device: `positions` is what a row of the table of pages holds, and
// the figures here and below are of tables as wide as the longest sequence (in a graph,
// three sets of inputs in turn).  A wider one is taken for longer sequences: 40 tokens
// over 500 positions 10.2 us with 512 in a row, 18.5 with 2048, 22 with 8192, 38 with
// 131072; 500 tokens over 500 26, 23, 38, 38; one over 500 9.2, then 11.1.
inline int tile_rows(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int dim,
                     int64_t positions) {
  const int64_t rows = tokens * (heads / kv_heads);
  if (rows <= kFew * batch || padded_dim(dim) > kManyDim) return kFew;
  return positions <= 2048 && (rows / kFew + batch) * kv_heads <= kResident / 2 ? kFew : kMany;
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
// of 512 positions 10.8 us in parts, 8.7 whole; of 1024 10.8 / 13.2, of 8192 14.7 / 102.
// 64 ragged sequences of up to 16384 357 / 459, 512 tokens over 8192 positions 90 /
// 197.  A run of at least 8 small steps: 4 / 8 / 16 of them 16.1 / 14.7 / 16.6 us at
// 8192 positions (9.7 / 10.8 / 13.2 at 1024).  Of large ones at least 16, which counts
// where a row of pages holds more than the sequences have: 8 / 16 / 32 of them 55 / 61 /
// 90 us, 100 tokens each of 3 over 3000 positions of 16384; 53 / 52 / 69, 300 each of 4
// over 1000 of 16384.
// Where even whole rows of pages would leave units idle with that, one a CU with as few
// as 4.  us, so / at least 16 / at least 8, one a CU: 40 tokens over 4096 37 / 46 / 32, 16
// each of 4 over 4096 36 / 49 / 35, 100 over 3000 43 / 45 / 40, 50 each of 3 over 2500
// with 16 heads over 2 34 / 46 / 33, 128 over 4096 with 32 heads of 64 27 / 31 / 26; where
// there is more to do it loses, 128 over 8192 48 / 46 / 45, 256 over 4096 42 / 41 / 40, 64
// over 8192 with 8 heads over 1 68 / 42 / 42.
// More tiles than there are units, of sequences with several, go whole, a prompt's
// later ones, which see more, first: a prompt of 8192 555 us whole, 795 in parts, of 4096
// 153 / 210, 4 chunks of 1024 over 8192 516 / 528.
struct Parts {
  int units, least_steps;
};
inline Parts parts(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int dim,
                   int64_t positions, int64_t window) {
  const int64_t group = heads / kv_heads;
  const int rows = tile_rows(tokens, batch, heads, kv_heads, dim, positions);
  const int64_t all = tiles(tokens, batch, group, rows);
  const int keys = rows == kFew ? kFewKeys : kKeys;
  // Whether there are parts does not depend on a window but where it makes them few.
  int64_t longest = (positions + keys - 1) / keys;
  const bool countable = all * longest < (int64_t{1} << 31);
  if (window > 0) longest = std::min(longest, (window + rows + keys - 1) / keys + 1);
  int64_t units = std::max<int64_t>(1, kResident / kv_heads);
  if (longest <= (rows == kFew ? 16 : 8) || batch > kMaxBatch || !countable ||
      kv_heads > kResident ||  // offsets within 32 bits
      (tokens * group > kFew * batch && all > units))
    return {0, 0};
  int64_t least = 8;
  if (rows == kMany) {
    least = 16;
    if (all * longest < least * units) {
      least = 4;
      units = std::max<int64_t>(1, units / 2);
    }
  }
  return {static_cast<int>(std::min(units, (all * longest + least - 1) / least)),
          static_cast<int>(least)};
}

// Floats that a part of a tile leaves: its rows' outputs, maxima and sums.
inline int64_t part_floats(int rows, int dim) {
  return static_cast<int64_t>(rows) * (padded_dim(dim) + 2);
}

inline size_t workspace(int64_t tokens, int64_t batch, int64_t heads, int64_t kv_heads, int dim,
                        int64_t positions, int64_t window) {
  const Parts p = parts(tokens, batch, heads, kv_heads, dim, positions, window);
  const int rows = tile_rows(tokens, batch, heads, kv_heads, dim, positions);
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
