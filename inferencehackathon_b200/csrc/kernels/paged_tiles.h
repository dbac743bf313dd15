// Host side of paged_tiles.cu, called by the entry point in paged_attn.cu.
#pragma once
#include "api.h"

namespace ihb {
cudaError_t paged_tiles_launch(const IhbPagedAttn& a, cudaStream_t stream);
size_t paged_tiles_scratch(const IhbPagedAttn& a);
}  // namespace ihb
