// Tensor maps for bulk-tensor copies, encoded on the host (project.cu).
#pragma once

#include <cuda.h>
#include <stdint.h>

namespace pa {
int tensor_map(CUtensorMap *map, CUtensorMapDataType type, const void *base, int rank,
               const uint64_t *dims, const uint64_t *strides, const uint32_t *box);
}  // namespace pa
