// esda_prefix_tiles.hip -- prefill_kernel (esda_prefill_kernel.h) with PrefixParams: the prefix of
// a decode batch as query tiles, and behind them the sequences' own rows.  A source of its own, as
// it is compiled with the default instruction scheduler.

#include "esda_prefix_tiles.h"

#include "esda_prefill_kernel.h"

void esda_detail::prefix_tiles(const esda_prefill_plan::PrefixParams &p, int head_dim, hipStream_t st) {
    if (head_dim == 512) launch_tiles<512>(p, st);
    else if (head_dim == 256) launch_tiles<256>(p, st);
    else launch_tiles<128>(p, st);
}
