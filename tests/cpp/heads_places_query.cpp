// Places of three levels (heads_rules.hpp) behind a C ABI, for tests/test_heads_places.py.
#include "../../credit_amd/csrc/heads_rules.hpp"

using namespace credit;

namespace {
// at, run, step, outer, count, width, lead, leads
heads::Place place(const int64_t* p) {
  return {static_cast<uintptr_t>(p[0]), p[1], p[2], p[3], p[4], p[5], p[6], p[7]};
}
}  // namespace

extern "C" {
int places_apart(const int64_t* a, const int64_t* b) { return heads::apart(place(a), place(b)); }
int places_apart_within(const int64_t* a) { return heads::apart_within(place(a)); }
}
