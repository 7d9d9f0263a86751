// esda_prefix_tiles.h -- the launch of a shared prefix's query tiles, for esda_prefix.hip.
#pragma once

#include <hip/hip_runtime.h>

#include "esda_prefill_plan.h"

namespace esda_detail {
void prefix_tiles(const esda_prefill_plan::PrefixParams &p, int head_dim, hipStream_t st);
}  // namespace esda_detail
