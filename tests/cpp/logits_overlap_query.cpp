// The overlap rule of logits_rules.hpp behind a C ABI, for tests/test_logits_overlap.py.
#include "../../credit_amd/csrc/logits_rules.hpp"

extern "C" int logits_may_share(uintptr_t a, int64_t lda, uintptr_t b, int64_t ldb, int64_t rows,
                                int64_t cols, size_t elem) {
  return credit::logits::may_share(a, lda, b, ldb, rows, cols, elem) ? 1 : 0;
}
