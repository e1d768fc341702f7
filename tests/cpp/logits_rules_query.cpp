// logits_rules.hpp behind a C ABI, for tests/test_logits_rules.py.
#include "../../credit_amd/csrc/logits_rules.hpp"

using namespace credit::logits;

extern "C" {
int64_t logits_auto_parts(int64_t rows, int64_t batches, int alternatives) {
  return auto_parts(rows, batches, alternatives != 0);
}
size_t logits_workspace(int64_t rows, int64_t cols, int read, int64_t split, int alternatives) {
  return workspace(rows, cols, read, split, alternatives != 0);
}
size_t logits_parts_bytes(int64_t rows, int64_t parts, int64_t batches, int alternatives) {
  return parts_bytes(rows, parts, batches, alternatives != 0);
}
}
