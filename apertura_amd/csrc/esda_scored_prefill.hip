// esda_scored_prefill.hip -- prefill attention with capped or biased scores and document and
// prefix masks for MI355X (gfx950): prefill_kernel and prefill_merge_kernel (esda_prefill_kernel.h)
// with ScoredParams or, with documents, DocParams.  The C ABI is include/esda_scored.h.

#include <hip/hip_runtime.h>

#include <climits>
#include <cmath>
#include <cstdint>
#include <initializer_list>
#include <string>
#include <type_traits>

#include "esda.h"
#include "esda_internal.h"
#include "esda_prefill_kernel.h"
#include "esda_scored.h"
#include "esda_views.h"

namespace {

int fail(int code, const std::string &msg) {
    esda_detail::set_error(msg);
    return code;
}

bool aligned16(const void *ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0; }

// The plan of a call, or what is wrong with it.
const char *plan(const esda_prefill_desc *d, const esda_score *s, ScoredParams *p) {
    if (!d || !s) return "esda_scored_prefill: null description or score";
    if (!(s->softcap >= 0.0f) || !std::isfinite(s->softcap))
        return "esda_scored_prefill: softcap must be 0 or positive and finite";
    if (s->prefix < 0) return "esda_scored_prefill: prefix must not be negative";
    if ((long long) d->k_pos0 + d->seq_k > INT_MAX - 64) return "esda_scored_prefill: key positions must stay below 2^31 - 64";
    if (const char *why = last_plan(d, s->prefix, p)) return why;
    if (!set_softcap(s->softcap, d->scale, &p->soft)) return "esda_scored_prefill: softcap and scale are too far apart";
    p->slopes = s->slopes;
    return nullptr;
}

}  // namespace

extern "C" {

int esda_scored_prefill_workspace_size(const esda_prefill_desc *desc, const esda_score *score, size_t *bytes) {
    if (!bytes) return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_scored_prefill_workspace_size: null output");
    ScoredParams p;
    if (const char *why = plan(desc, score, &p)) return fail(ESDA_ERR_INVALID_ARGUMENT, why);
    *bytes = workspace_of(p, desc->head_dim);
    return ESDA_OK;
}

int esda_scored_prefill(const esda_prefill_desc *desc, const esda_score *score, const esda_scored_prefill_args *a,
                        void *stream) {
    ScoredParams p;
    if (const char *why = plan(desc, score, &p)) return fail(ESDA_ERR_INVALID_ARGUMENT, why);
    if (!a || !a->q || !a->k || !a->v || !a->out)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_scored_prefill: null pointer");
    if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->out))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_scored_prefill: tensors must be 16-byte aligned");
    const int D = desc->head_dim;
    // (a row of q is read again after rows of out are written, where a value is not finite)
    auto view = [](const void *ptr, long long rows, long long rs, long long heads, long long hs, long long width) {
        return esda_views::View{reinterpret_cast<uintptr_t>(ptr), {rows, heads}, {rs, hs}, width};
    };
    const long long keys = (long long) p.Sk * D;
    const esda_views::View out = view(a->out, p.Sq, p.o_rs, p.Hq, p.o_hs, D);
    for (const auto &in : {view(a->q, p.Sq, p.q_rs, p.Hq, p.q_hs, D), view(a->k, 1, 0, p.Hkv, p.kv_hs, keys),
                           view(a->v, 1, 0, p.Hkv, p.kv_hs, keys)}) {
        if (in.extent() > (__int128) 1 << 60 || out.extent() > (__int128) 1 << 60)
            return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_scored_prefill: strides are too large");
        if (!esda_views::disjoint(in, out))
            return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_scored_prefill: out must not overlap q, k or v");
    }
    if (!a->q_doc != !a->k_doc)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_scored_prefill: q_doc and k_doc go together");
    if ((reinterpret_cast<uintptr_t>(a->k_doc) | reinterpret_cast<uintptr_t>(a->q_doc) |
         reinterpret_cast<uintptr_t>(score->slopes)) & 3u)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_scored_prefill: document ids and slopes must be 4-byte aligned");
    const size_t need = workspace_of(p, D);
    if (need) {
        if (!a->workspace || a->workspace_bytes < need || !aligned16(a->workspace))
            return fail(ESDA_ERR_WORKSPACE, "esda_scored_prefill: workspace missing or smaller than "
                                            "esda_scored_prefill_workspace_size");
        const size_t rows = (size_t) p.Sq * p.Hq;
        p.part_acc = static_cast<float *>(a->workspace);
        p.part_ml = reinterpret_cast<float *>(static_cast<char *>(a->workspace) + (size_t) p.splits * rows * D * 4);
    }
    const int rc = esda_detail::check_device();
    if (rc != ESDA_OK) return rc;
    p.q = static_cast<const uint16_t *>(a->q);
    p.k = static_cast<const uint16_t *>(a->k);
    p.v = static_cast<const uint16_t *>(a->v);
    p.out = static_cast<uint16_t *>(a->out);
    hipStream_t st = static_cast<hipStream_t>(stream);
    auto launch = [&](const auto &x) {
        using P = std::decay_t<decltype(x)>;
        if (D == 512) launch_prefill<512, P>(x, 3, st);
        else if (D == 256) launch_prefill<256, P>(x, 3, st);
        else launch_prefill<128, P>(x, 3, st);
    };
    auto with_documents = [&](auto dp) {
        static_cast<ScoredParams &>(dp) = p;
        dp.q_doc = a->q_doc;
        dp.k_doc = a->k_doc;
        launch(dp);
    };
    if (a->k_doc) {
        if (p.soft.wide) with_documents(WideDocParams{});
        else with_documents(DocParams{});
    } else if (p.soft.wide) {
        WideScoredParams wp{};
        static_cast<ScoredParams &>(wp) = p;
        launch(wp);
    } else {
        launch(p);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(ESDA_ERR_HIP, std::string("esda_scored_prefill launch: ") + hipGetErrorString(e));
    return ESDA_OK;
}

}  // extern "C"
