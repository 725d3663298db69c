// The paged cache as a 2-D byte tensor for the copy engine (defined in decode.cu).
#pragma once
#include <cuda.h>   // CUtensorMap (a type only: the encoder is looked up at run time)
#include <stdint.h>

namespace cda {
// Row = one slot position (all heads, H_kv * slot_bytes bytes), rows = slot positions.  A copy box is 16 rows x box_bytes
// starting at byte head * slot_bytes: one 16-token group of one head.
int make_cache_map(const char* who, const void* cache, int H_kv, int slot_bytes, int64_t num_slots, int box_bytes, CUtensorMap* out);
}  // namespace cda
