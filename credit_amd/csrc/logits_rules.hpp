// How the forwards of the operators on logits (logits.hip) cut rows into parts,
// the workspace that takes, and where a gradient may lie beside its logits.  Host
// arithmetic alone, so that the CPU tests build it with g++
// (tests/cpp/logits_rules_query.cpp, logits_overlap_query.cpp).
#pragma once

#include <stddef.h>
#include <stdint.h>

#include <algorithm>

namespace credit {
namespace logits {

constexpr int kThreads = 256;
constexpr int kBatch = 8192;    // columns that a workgroup takes at once
constexpr int kMaxParts = 64;   // of a row
constexpr int kPartValues = 4;  // fp64 values a part leaves
constexpr int64_t kMaxSplitRows = 1024;

// Parts of a row of `batches` batches; 1: one workgroup a row.  As many as give
// every CU a workgroup, where that saves a part four batches or more: a batch is
// 0.5 us of a lone workgroup's time, the meeting of the parts 1.5 us.  us a call,
// one workgroup a row -> parts:
//   distillation with tail   1 x 131072 bf16 14.8 -> 7.4, 64 x 131072 16.0 -> 10.5,
//                            128 x 131072 16.3 -> 13.4, 16 x 262144 fp32 28.5 -> 9.8
//   but 64 x 32768 fp32 (4 batches) 9.0 -> 8.4 (log-probabilities alone 7.3 -> 7.5);
//   256 x 131072, two parts: 17.4 -> 18.5
// With alternatives the last part reads every lane's maxima back, which takes
// more (K = 20): 1 x 131072 15.2 -> 9.8, 64 x 131072 17.2 -> 14.3, 96 x 131072, two
// parts 17.2 -> 17.5, 128 x 131072 17.4 -> 18.1, 1 x 32768 fp32 9.2 -> 9.3.
// Not the best choice above its limits in bf16 rows of more than 16 batches, which
// keep whole rows: K = 20, 65 x 262144 27.8 -> 21.9 in four parts, 96 rows 27.9 ->
// 23.7, 128 rows 28.3 -> 26.2 (fp32 29.8 -> 27.8, 31.1 -> 30.9, 32.0 -> 35.8; 65 x
// 131072 bf16 17.2 -> 14.9, 200 x 262144 29.6 -> 37.0), and without alternatives
// 130 x 262144 23.1 -> 15.6 in three parts, 200 x 262144 24.7 -> 20.7 in two (fp32
// 27.0 -> 24.8, 31.9 -> 34.8).
inline int64_t auto_parts(int64_t rows, int64_t batches, bool alternatives) {
  if (alternatives && rows > 64) return 1;
  const int64_t a_cu_each = std::max<int64_t>(1, 256 / std::max<int64_t>(1, rows));
  const int64_t parts = std::min<int64_t>({kMaxParts, batches, a_cu_each});
  const int64_t saved = batches - (batches + parts - 1) / parts;
  return saved >= (alternatives ? 5 : 4) ? parts : 1;
}

inline size_t part_values_bytes(int64_t rows, int64_t parts) {
  return (static_cast<size_t>(rows * parts) * kPartValues * sizeof(double) + 255) / 256 * 256;
}
// Scratch of a call whose rows are in `parts` of `batches` batches each.
inline size_t parts_bytes(int64_t rows, int64_t parts, int64_t batches, bool alternatives) {
  return part_values_bytes(rows, parts) +
         (alternatives ? static_cast<size_t>(rows * parts * batches) * kThreads * sizeof(float)
                       : 0);
}

// Scratch that any call of this shape can take, whatever its type and alignment:
// a row's batches start at a 128-byte line, at most one more than its columns
// fill, its parts at most `split` (0: as AUTO takes them, with alternatives or
// without).
inline size_t workspace(int64_t rows, int64_t cols, int variant_read, int64_t split,
                        bool alternatives) {
  size_t most = 0;
  for (int64_t batches : {(cols + kBatch - 1) / kBatch, (cols + 63 + kBatch - 1) / kBatch})
    for (bool top : {false, alternatives}) {
      const int64_t want =
          variant_read ? 1 : split > 0 ? split : auto_parts(rows, batches, top);
      const int64_t each = (batches + want - 1) / want, n = (batches + each - 1) / each;
      if (n >= 2 && rows <= kMaxSplitRows)
        most = std::max(most, parts_bytes(rows, n, each, top));
    }
  return most;
}

// Whether a gradient of `rows` rows at b, ldb elements apart, may be written while
// logits at a, lda apart, are read: in place (a lane writes what it has read), or
// where no element is in both: memory apart, or rows of one distance that lie
// between each other's.  Rows of two distances whose spans meet are not looked at.
inline bool may_share(uintptr_t a, int64_t lda, uintptr_t b, int64_t ldb, int64_t rows,
                      int64_t cols, size_t elem) {
  if (a == b && (rows == 1 || lda == ldb)) return true;
  const uintptr_t width = cols * elem;
  const uintptr_t na = (rows - 1) * lda * elem + width, nb = (rows - 1) * ldb * elem + width;
  if (a >= b + nb || b >= a + na) return true;
  if (rows == 1 || lda != ldb) return false;
  const uintptr_t step = lda * elem, after = (a < b ? b - a : a - b) % step;
  return after >= width && step - after >= width;
}

}  // namespace logits
}  // namespace credit
