// Where the tensors of the operators on heads (heads.hip, attention.hip) may lie
// and how a token's heads are dealt to lanes.  Host arithmetic alone, so that the
// CPU tests build it with g++ (tests/cpp/heads_rules_query.cpp).
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <algorithm>

namespace credit {
namespace heads {

constexpr int kMaxDim = 512;

// Vectors that are `step` bytes apart, `count` of them in each of `outer` runs
// that are `run` bytes apart, `width` bytes each.
struct Place {
  uintptr_t at = 0;
  int64_t run = 0, step = 0;
  int64_t outer = 0, count = 0, width = 0;

  bool empty() const { return outer == 0 || count == 0 || width == 0; }
  // Bytes from the first to behind the last.
  int64_t span() const { return empty() ? 0 : (outer - 1) * run + (count - 1) * step + width; }
  // Of one run.
  int64_t extent() const { return (count - 1) * step + width; }
};

// Whether no byte of a tensor belongs to two of its vectors.
inline bool apart_within(const Place& p) {
  if (p.empty()) return true;
  const int64_t step = p.count == 1 ? p.width : p.step, run = p.outer == 1 ? p.span() : p.run;
  if (step >= p.width && run >= (p.count - 1) * step + p.width) return true;
  return run >= p.width && step >= (p.outer - 1) * run + p.width;
}

// Whether two tensors share no byte, as far as can be told: spans apart, or
// vectors or whole runs of one distance that lie between each other's (heads or
// column ranges of one buffer).
inline bool between(uintptr_t a, int64_t wa, uintptr_t b, int64_t wb, int64_t distance) {
  if (distance <= 0 || wa > distance || wb > distance) return false;
  const int64_t d = b >= a ? static_cast<int64_t>(b - a) : -static_cast<int64_t>(a - b);
  const int64_t after = ((d % distance) + distance) % distance;
  return after >= wa && after + wb <= distance;
}
inline bool apart(const Place& a, const Place& b) {
  if (a.empty() || b.empty()) return true;
  if (a.at >= b.at + b.span() || b.at >= a.at + a.span()) return true;
  if (a.run == b.run && between(a.at, a.extent(), b.at, b.extent(), a.run)) return true;
  const auto whole = [](const Place& p) { return p.outer == 1 || p.run % p.step == 0; };
  return a.step == b.step && a.step > 0 && whole(a) && whole(b) &&
         between(a.at, a.width, b.at, b.width, a.step);
}

inline bool same(const Place& a, const Place& b) {
  return a.at == b.at && a.count == b.count && (a.outer <= 1 || a.run == b.run) &&
         (a.count <= 1 || a.step == b.step);
}

// Heads that a group of lanes takes of each tensor of a launch, a power of two up to
// `most`: one where that leaves the device short of waves (four a SIMD), more where a
// group's angles then serve them all.  `all`: heads of a token in all tensors,
// `widest`: of the one with the most.  us, a
// head a group -> `most` of them: 16384 tokens of 32 + 8 heads of 128 in bf16, norm and
// rotation 89 -> 66, their gradients 125 -> 106; 64 tokens, which stay at a head a
// group, 4.8.
inline int run_of(int64_t tokens, int64_t all, int widest, int group_lanes, int most) {
  constexpr double kLanes = 64.0 * 4096.0;
  int run = most;
  while (run > 1 && (run / 2 >= widest ||
                     static_cast<double>(tokens) * all * group_lanes < kLanes * run))
    run /= 2;
  return run;
}
// Groups (a power of two of them) that share a token's heads, group g taking heads g,
// g + groups, ...
inline int groups_of(int heads, int run) {
  int groups = 1;
  while (groups * run < heads) groups *= 2;
  return groups;
}

}  // namespace heads
}  // namespace credit
