// esda_prefix_tiles.hip -- the shared prefix of a decode batch as query tiles for MI355X (gfx950):
// prefill_kernel (esda_prefill_kernel.h) with PrefixParams.  The B * G query rows of a kv head
// are the rows of its tiles, so a tile reads each prefix key once for all of them; every key
// split leaves a partial for the merge with the sequences' own rows (esda_prefix.hip).

#include <hip/hip_runtime.h>

#include <cstdint>

#include "esda_internal.h"
#include "esda_prefill_kernel.h"
#include "esda_prefix.h"

namespace {

const char *plan(const esda_prefix_desc *d, PrefixParams *p) {
    const int D = d->own.head_dim;
    esda_prefill_desc t{};
    t.num_q_heads = d->own.num_q_heads;
    t.num_kv_heads = d->own.num_kv_heads;
    t.head_dim = D;
    t.seq_q = d->own.batch;
    t.seq_k = d->prefix_len;
    t.q_pos0 = d->prefix_len - 1;  // every row at or past the last key
    t.q_head_stride = D;
    t.q_row_stride = (int64_t) t.num_q_heads * D;
    t.kv_head_stride = d->prefix_head_stride;
    t.split_keys = d->split_keys;
    t.scale = d->own.scale;
    return last_plan(&t, 0, p);
}

}  // namespace

const char *esda_detail::prefix_tiles_plan(const esda_prefix_desc *d, int *splits) {
    PrefixParams p{};
    if (const char *why = plan(d, &p)) return why;
    *splits = p.splits;
    return nullptr;
}

int esda_detail::prefix_tiles(const esda_prefix_desc *d, const esda_prefix_args *a, float *part_acc, float *part_ml,
                              hipStream_t st) {
    PrefixParams p{};
    if (plan(d, &p)) return hipErrorInvalidValue;  // planned before
    p.q = static_cast<const uint16_t *>(a->own.q);
    p.k = static_cast<const uint16_t *>(a->prefix_k);
    p.v = static_cast<const uint16_t *>(a->prefix_v);
    p.part_acc = part_acc;
    p.part_ml = part_ml;
    if (d->own.head_dim == 512) launch_tiles<512>(p, st);
    else if (d->own.head_dim == 256) launch_tiles<256>(p, st);
    else launch_tiles<128>(p, st);
    return hipGetLastError();
}
