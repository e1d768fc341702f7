// Where the tensors of the operators on heads (heads.hip, attention.hip) may lie
// and how a token's heads are dealt to lanes.  Host arithmetic alone, so that the
// CPU tests build it with g++ (tests/cpp/heads_rules_query.cpp).
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <algorithm>
#include <iterator>

namespace credit {
namespace heads {

constexpr int kMaxDim = 512;

// Vectors that are `step` bytes apart, `count` of them in each of `outer` runs
// that are `run` bytes apart, `width` bytes each; a cache's pages: `leads` of these,
// `lead` bytes apart.  Any of the distances may be the largest.
struct Place {
  uintptr_t at = 0;
  int64_t run = 0, step = 0;
  int64_t outer = 0, count = 0, width = 0;
  int64_t lead = 0, leads = 1;

  bool empty() const { return outer == 0 || count == 0 || width == 0 || leads == 0; }
  // Bytes from the first to behind the last.
  int64_t span() const {
    return empty() ? 0 : (leads - 1) * lead + (outer - 1) * run + (count - 1) * step + width;
  }
  // Bytes from the first vector's to behind the last one's, counted modulo `distance`,
  // of which the levels at its multiples take no part.
  int64_t extent(int64_t distance) const {
    const auto own = [&](int64_t stride, int64_t n) {
      return n == 1 || stride % distance == 0 ? 0 : (n - 1) * stride;
    };
    return own(lead, leads) + own(run, outer) + own(step, count) + width;
  }
};

// Whether no byte of a tensor belongs to two of its vectors: each level's distance
// holds all that lies within it.
inline bool apart_within(const Place& p) {
  if (p.empty()) return true;
  struct Level {
    int64_t stride, n;
  } levels[] = {{p.lead, p.leads}, {p.run, p.outer}, {p.step, p.count}};
  std::sort(std::begin(levels), std::end(levels),
            [](const Level& a, const Level& b) { return a.stride < b.stride; });
  int64_t within = p.width;
  for (const Level& l : levels) {
    if (l.n == 1) continue;
    if (l.stride < within) return false;
    within += (l.n - 1) * l.stride;
  }
  return true;
}

// Whether two tensors share no byte, as far as can be told: spans apart, or all of
// each one's bytes between the other's modulo one of their distances (heads, slots,
// pages or column ranges of one buffer).
inline bool between(const Place& a, const Place& b, int64_t distance) {
  if (distance <= 0) return false;
  const int64_t wa = a.extent(distance), wb = b.extent(distance);
  if (wa > distance || wb > distance) return false;
  const int64_t d = b.at >= a.at ? static_cast<int64_t>(b.at - a.at)
                                 : -static_cast<int64_t>(a.at - b.at);
  const int64_t after = ((d % distance) + distance) % distance;
  return after >= wa && after + wb <= distance;
}
inline bool apart(const Place& a, const Place& b) {
  if (a.empty() || b.empty()) return true;
  if (a.at >= b.at + b.span() || b.at >= a.at + a.span()) return true;
  for (const int64_t distance : {a.lead, a.run, a.step, b.lead, b.run, b.step})
    if (between(a, b, distance)) return true;
  return false;
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
