// Stable order of n ids by value, for the kernels that sum or multiply rows that share an id (embedding.hip, adapters.hip).
#pragma once
#include "sx_common.h"

namespace sx {

// ids outside [0, rows) fall into bucket `rows`.
//   perm [n]          position of the i-th entry in bucket order (equal ids keep their order)
//   key  [n]          its bucket
//   start[rows + 1], end[rows + 1]   first entry of each bucket and the one behind its last
// The buckets follow one another, `rows` last.  One launch, no scratch memory, the same result on every run.
int launch_sort_ids(const void* ids, int ids64, int64_t n, int64_t rows, int* perm, int* key, int* start, int* end,
                    hipStream_t st);

}  // namespace sx
