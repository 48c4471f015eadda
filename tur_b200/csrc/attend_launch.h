// Launches of attention over a paged cache.
#pragma once
#include <cuda_runtime.h>

#include "handles.h"

namespace turq {
struct AttendArgs;
// Sequences of up to TOKEN_ROWS rows; others are left alone. a.part / part_ml: max_chunks pieces of part_rows rows for every key head
// of every sequence (unused where max_chunks is 1).
cudaError_t launch_attend_tokens(const turq_kv_cache* kc, const AttendArgs& a, cudaStream_t s, int* launches);
// Sequences of more rows. blocks: at least the pairs of row tiles x key heads, and a.tile_pieces.
cudaError_t launch_attend_tiles(const turq_kv_cache* kc, const AttendArgs& a, unsigned blocks, cudaStream_t s, int* launches);
// The second step where a.tile_pieces > 0: rows whose keys were cut.
cudaError_t launch_join_tiles(const turq_kv_cache* kc, const AttendArgs& a, cudaStream_t s, int* launches);
}  // namespace turq
