// Launches of attention over a paged cache.
#pragma once
#include <cuda_runtime.h>

#include "handles.h"

namespace turq {
struct AttendArgs;
// Sequences of up to TOKEN_ROWS rows; others are left alone. a.part / part_ml: max_chunks pieces of part_rows rows for every key head
// of every sequence (unused where max_chunks is 1).
cudaError_t launch_attend_tokens(const turq_kv_cache* kc, const AttendArgs& a, cudaStream_t s, int* launches);
// Sequences of more rows, as `tiles` (or fewer) pairs of row tiles per key head, the keys of each in `splits` pieces (1: rows are finished).
cudaError_t launch_attend_tiles(const turq_kv_cache* kc, const AttendArgs& a, int64_t tiles, int splits, cudaStream_t s, int* launches);
}  // namespace turq
