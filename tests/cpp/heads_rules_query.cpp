// heads_rules.hpp and attention_rules.hpp behind a C ABI, for tests/test_heads_rules.py.
#include "../../credit_amd/csrc/attention_rules.hpp"
#include "../../credit_amd/csrc/heads_rules.hpp"

using namespace credit;

namespace {
// at, run, step, outer, count, width
heads::Place place(const int64_t* p) {
  return {static_cast<uintptr_t>(p[0]), p[1], p[2], p[3], p[4], p[5]};
}
}  // namespace

extern "C" {
int heads_apart(const int64_t* a, const int64_t* b) { return heads::apart(place(a), place(b)); }
int heads_apart_within(const int64_t* a) { return heads::apart_within(place(a)); }
int heads_same(const int64_t* a, const int64_t* b) { return heads::same(place(a), place(b)); }
int heads_run_of(int64_t tokens, int64_t all, int widest, int lanes, int most) {
  return heads::run_of(tokens, all, widest, lanes, most);
}
int heads_groups_of(int n, int run) { return heads::groups_of(n, run); }
int attention_tile_rows(int64_t tokens, int64_t batch, int64_t n, int64_t kv, int dim,
                        int64_t positions) {
  return attention::tile_rows(tokens, batch, n, kv, dim, positions);
}
int64_t attention_tiles(int64_t tokens, int64_t batch, int64_t group, int rows) {
  return attention::tiles(tokens, batch, group, rows);
}
int attention_units(int64_t tokens, int64_t batch, int64_t n, int64_t kv, int dim,
                    int64_t positions, int64_t window) {
  return attention::parts(tokens, batch, n, kv, dim, positions, window).units;
}
size_t attention_workspace(int64_t tokens, int64_t batch, int64_t n, int64_t kv, int dim,
                           int64_t positions, int64_t window) {
  return attention::workspace(tokens, batch, n, kv, dim, positions, window);
}
int attention_padded_dim(int dim) { return attention::padded_dim(dim); }
uint32_t attention_divide(uint32_t n, uint32_t d) {
  const attention::Divisor by = attention::divisor(d);
  const uint32_t high = static_cast<uint32_t>((uint64_t{n} * by.mul) >> 32);
  return (high + n) >> by.shift;
}
}
