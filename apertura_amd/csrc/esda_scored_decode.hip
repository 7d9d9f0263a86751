// esda_scored_decode.hip -- the decode step with capped or biased scores for MI355X (gfx950):
// attend_kernel (esda_attend.h) with ScoredAttendParams, at head_dim 128 stream_kernel below, and
// the plain step's plan and split merge.  The C ABI is include/esda_scored.h.

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <type_traits>

#include "esda.h"
#include "esda_attend.h"
#include "esda_internal.h"
#include "esda_scored.h"
#include "esda_stream.h"

namespace {

// head_dim 128: a 16-row stage is 4 or 8 KB, too little for a barrier and a score exchange between
// the waves.  Here each of eight waves streams stages of its own: a step of 16 sequences of 2K .. 16K
// rows, 8 kv heads, 599 MB 101 us (5.9 TB/s; attend_kernel 144), one of 131,072 rows 83 us (6.5 TB/s;
// 115), of 16,384 16.1 (22.3), of 300 8.2 (9.0); K = V, 16 of 512 .. 4096 24.2 (40).  At 256 and 512 dims
// attend_kernel: 16 of 1024 .. 8192 rows of 512 dims, K = V, 318 MB 74 us from HBM (4.2 TB/s), one of
// 131,072 90 (6.0).
constexpr int kStreamWaves = 8;

template <bool SH, class P>
__global__ __launch_bounds__(64 * kStreamWaves, 1) void stream_kernel(P p) {
    constexpr int D = 128, SLOTS = 2;
    using L = esda_stream::Layout<D, SH, kStreamWaves, SLOTS>;
    __shared__ __attribute__((aligned(16))) unsigned char lds[L::BYTES];
    const int li = threadIdx.x & 15;
    auto segment = [&](const int b, const int kvh, const int j0, const int j1, const SeqView sv, const size_t slot,
                       const bool direct) __attribute__((always_inline)) {
        const size_t head = (size_t) b * p.seq_stride + (size_t) kvh * p.head_stride, at = ((size_t) b * p.Hkv + kvh) * D;
        const esda_stream::Run x{p.k_cache + head, p.v_cache + head, p.k_new + at, SH ? p.k_new + at : p.v_new + at,
                                 p.G, j0, j1, sv.nvis, sv.first, p.cap, sv.newrow};
        const uint16_t *const q = p.q + ((size_t) b * p.Hq + (size_t) kvh * p.G) * D;
        uint16_t *const out = p.out + ((size_t) b * p.Hq + (size_t) kvh * p.G) * D;
        const float slope = p.slopes && li < p.G ? p.slopes[kvh * p.G + li] * kLog2e : 0.0f;
        esda_stream::attend_run<D, SH, kStreamWaves, SLOTS, 1>(
            lds, x, [&](int h) { return q + (size_t) h * D; },
            [&](float s, int j) {
                float y = s * p.scale_log2e;
                if constexpr (std::is_same<P, WideScoredAttendParams>::value) y = capped_wide(s, y, p.soft);
                else if (p.soft.out != 0.0f) y = capped_narrow(s, p.soft);
                return __builtin_fmaf(-slope, (float) (sv.nvis - 1 - j), y);
            },
            [&](int h, int d, const f32x4 &o, float M, float T) {
                if (direct) {
                    const float inv = 1.0f / T;
                    bf16x4 r;
#pragma unroll
                    for (int e = 0; e < 4; ++e) r[e] = (__bf16) (o[e] * inv);
                    *reinterpret_cast<bf16x4 *>(out + (size_t) h * D + d) = r;
                } else {
                    const size_t at = slot * p.G + h;
                    *reinterpret_cast<f32x4 *>(p.part_acc + at * D + d) = o;
                    if (d == 0) *reinterpret_cast<f32x2 *>(p.part_ml + 2 * at) = f32x2{M, T};
                }
            });
    };
    walk_segments<kStreamWaves>(p, segment);
}

}  // namespace

extern "C" int esda_scored_decode(const esda_decode_desc *d, const esda_score *s, const esda_decode_args *a, void *stream) {
    Plan pl;
    int rc = make_plan(d, &pl);
    if (rc) return rc;
    // One kv head a workgroup (the same partials): a value that is not finite stays with its head's queries.
    pl.pk = 1;
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
    if (!set_softcap(s->softcap, d->scale, &ap.soft))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_scored_decode: softcap and scale are too far apart");
    ap.slopes = s->slopes;
    rc = esda_detail::check_device();
    if (rc) return rc;
    const DecodeSpace sp = space_of(pl, a->workspace);
    uint16_t *out = static_cast<uint16_t *>(a->out);
    fill_attend(d, pl, sp, static_cast<int *>(a->workspace), out, ap);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    auto launch = [&](const auto &x) {
        using P = std::decay_t<decltype(x)>;
        const dim3 grid = attend_grid(d, pl), block(64 * kStreamWaves);
        if (d->head_dim != 128) return dispatch_attend(d->head_dim, d->kv_shared != 0, x, grid, st);
        if (d->kv_shared) hipLaunchKernelGGL((stream_kernel<true, P>), grid, block, 0, st, x);
        else hipLaunchKernelGGL((stream_kernel<false, P>), grid, block, 0, st, x);
        return hipGetLastError();
    };
    hipError_t e;
    if (ap.soft.wide) {
        WideScoredAttendParams wp{};
        static_cast<ScoredAttendParams &>(wp) = ap;
        e = launch(wp);
    } else {
        e = launch(ap);
    }
    if (e != hipSuccess) return hip_fail(e, "attend_kernel launch");
    return launch_merge(d, pl, sp, a->pos, a->row_base, 0, out, st);
}
