// esda_scored_decode.hip -- the decode step with capped or biased scores for MI355X (gfx950):
// attend_kernel (esda_attend.h) with ScoredAttendParams, and the plain step's split merge.  The C
// ABI is include/esda_scored.h.

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "esda.h"
#include "esda_attend.h"
#include "esda_internal.h"
#include "esda_scored.h"

extern "C" int esda_scored_decode(const esda_decode_desc *d, const esda_score *s, const esda_decode_args *a, void *stream) {
    Plan pl;
    int rc = make_plan(d, &pl);
    if (rc) return rc;
    if (!s) return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_scored_decode: null score");
    if (!(s->softcap >= 0.0f) || !std::isfinite(s->softcap))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_scored_decode: softcap must be 0 or positive and finite");
    if (s->prefix < 0) return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_scored_decode: prefix must not be negative");
    if (reinterpret_cast<uintptr_t>(s->slopes) & 3u)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_scored_decode: slopes must be 4-byte aligned");
    if (!(d->scale > 0.0f) || !std::isfinite(d->scale))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_scored_decode: scale must be positive and finite");
    rc = check_decode_args(d, a);
    if (rc) return rc;
    if (!a->workspace || a->workspace_bytes < pl.bytes || !aligned16(a->workspace))
        return fail(ESDA_ERR_WORKSPACE, "esda_scored_decode: workspace missing or smaller than esda_decode_workspace_size");
    ScoredAttendParams ap{};
    static_cast<AttendParams &>(ap) = decode_params(d, a);
    if (s->softcap > 0.0f) {
        ap.cap_in = (float) (2.0 * 1.4426950408889634 * d->scale / s->softcap);
        ap.cap_out = (float) (1.4426950408889634 * s->softcap);
        if (!std::isfinite(ap.cap_in) || !std::isfinite(ap.cap_out) || ap.cap_in == 0.0f)
            return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_scored_decode: softcap and scale are too far apart");
    }
    ap.slopes = s->slopes;
    rc = esda_detail::check_device();
    if (rc) return rc;
    const DecodeSpace sp = space_of(pl, a->workspace);
    uint16_t *out = static_cast<uint16_t *>(a->out);
    fill_attend(d, pl, sp, static_cast<int *>(a->workspace), out, ap);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const hipError_t e = dispatch_attend(d->head_dim, d->kv_shared != 0, ap, attend_grid(d, pl), st);
    if (e != hipSuccess) return hip_fail(e, "attend_kernel launch");
    return launch_merge(d, pl, sp, a->pos, a->row_base, 0, out, st);
}
