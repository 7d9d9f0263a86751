// esda_tree_tiles.h -- the launch of a step of drafted tokens in query tiles, for esda_tree.hip.
#pragma once

#include <hip/hip_runtime.h>

#include "esda_prefill_plan.h"

namespace esda_detail {
void tree_tiles(const esda_prefill_plan::TreeParams &p, int head_dim, hipStream_t st);
}  // namespace esda_detail
