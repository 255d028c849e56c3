// Stable order of n ids by value, for the kernels that sum or multiply rows that share an id (embedding.hip, adapters.hip).
#pragma once
#include "sx_common.h"

namespace sx {

// ids outside [0, rows) fall into bucket `rows`, behind the others.
//   perm [n]          position of the i-th entry in sorted order (equal ids keep their order)
//   key  [n]          its bucket, or null
//   start[rows + 2]   first entry of each bucket; start[rows + 1] = n
// One launch, no scratch memory, the same result on every run.
int launch_sort_ids(const void* ids, int ids64, int64_t n, int64_t rows, int* perm, int* key, int* start, hipStream_t st);

}  // namespace sx
