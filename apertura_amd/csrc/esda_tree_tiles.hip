// esda_tree_tiles.hip -- prefill_kernel (esda_prefill_kernel.h) with TreeParams: steps of many drafted
// tokens as query tiles.

#include "esda_tree_tiles.h"

#include "esda_prefill_kernel.h"

void esda_detail::tree_tiles(const esda_prefill_plan::TreeParams &p, int head_dim, hipStream_t st) {
    if (head_dim == 512) launch_tiles<512>(p, st);
    else if (head_dim == 256) launch_tiles<256>(p, st);
    else launch_tiles<128>(p, st);
}
