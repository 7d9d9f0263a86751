// esda_prefix.hip -- the decode step of a batch that shares a prefix for MI355X (gfx950).
//
// Three launches: the prefix's query tiles (esda_prefix_tiles.hip), the sequences' own rows with
// the fused append (attend_kernel, esda_attend.h, with TailParams), and the merge below over the
// partials of both.  The C ABI is include/esda_prefix.h.

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <string>

#include "esda.h"
#include "esda_attend.h"
#include "esda_internal.h"
#include "esda_prefix.h"

namespace {

struct PrefixMergeParams : MergeParams {
    int base;
    int splits;                      // prefix splits
    const float *pre_acc, *pre_ml;   // [splits][B * Hq][D] and [..][2]
};
__device__ __forceinline__ int base_of(const PrefixMergeParams &p, int) { return p.base; }

// out = sum_s acc_s 2^(m_s - M) / sum_s l_s 2^(m_s - M) over the partials of the prefix and of the
// sequence's own rows.  One wave per (sequence, query head): lane j loads (m, l) of partial j, so
// the weights take one round trip and wave reductions; then the wave walks the partial rows,
// MB of them in flight.
template <int D>
__global__ __launch_bounds__(256) void prefix_merge_kernel(PrefixMergeParams p) {
    constexpr int VEC = D / 64;             // dims per lane
    constexpr int MB = 32 / VEC < 8 ? 32 / VEC : 8;
    typedef float vec __attribute__((ext_vector_type(VEC)));
    typedef __bf16 bvec __attribute__((ext_vector_type(VEC)));
    const int lane = threadIdx.x & 63;
    const int rows = p.B * p.Hq;
    const int row = blockIdx.x * 4 + uniform(threadIdx.x >> 6);
    if (row >= rows) return;
    const int b = row / p.Hq, h = row % p.Hq, kvh = h / p.G, g = h % p.G;
    size_t pbase = 0;
    const int own = pair_splits(p, b, kvh, pbase);
    if (own == 0) return;  // skipped: its position lies outside its cache
    const int n = p.splits + own;
    auto at = [&](int j) { return j < p.splits ? (size_t) j * rows + row : (pbase + (j - p.splits)) * p.G + g; };
    auto ml_of = [&](int j) {
        return j < n ? *reinterpret_cast<const f32x2 *>((j < p.splits ? p.pre_ml : p.part_ml) + 2 * at(j))
                     : f32x2{-INFINITY, 0.0f};
    };
    f32x2 ml = ml_of(lane);
    float M = ml[0];
    for (int j = lane + 64; j < n; j += 64) M = fmaxf(M, ml_of(j)[0]);
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) M = fmaxf(M, __shfl_xor(M, o));
    float den = 0.0f;
    vec num = 0.0f;
    for (int j0 = 0; j0 < n; j0 += 64) {
        if (j0) ml = ml_of(j0 + lane);
        const float w = j0 + lane < n ? __builtin_amdgcn_exp2f(ml[0] - M) : 0.0f;
        den += ml[1] * w;
        const int m = n - j0 < 64 ? n - j0 : 64;
        for (int i0 = 0; i0 < m; i0 += MB) {
            vec a[MB];
#pragma unroll
            for (int i = 0; i < MB; ++i)
                if (i0 + i < m)
                    a[i] = *reinterpret_cast<const vec *>((j0 + i0 + i < p.splits ? p.pre_acc : p.part_acc) + at(j0 + i0 + i) * D + lane * VEC);
#pragma unroll
            for (int i = 0; i < MB; ++i)
                if (i0 + i < m)
                    num += __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), i0 + i)) * a[i];
        }
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) den += __shfl_xor(den, o);
    bvec r;
#pragma unroll
    for (int e = 0; e < VEC; ++e) r[e] = (__bf16) (num[e] / den);
    *reinterpret_cast<bvec *>(p.out + (size_t) row * D + lane * VEC) = r;
}

// Workspace: the own rows' plan (its status word first), then the prefix partials.
struct PrefixPlan {
    Plan own;
    int splits;
    size_t off_ml, off_acc, bytes;
};

int make_prefix_plan(const esda_prefix_desc *d, PrefixPlan *pl) {
    if (!d) return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_prefix_decode: null description");
    const int rc = make_plan(&d->own, &pl->own);
    if (rc) return rc;
    if (d->own.ring || d->own.window)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_prefix_decode: own caches are linear and without a window");
    if (d->prefix_len <= 0) return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_prefix_decode: prefix_len must be positive");
    if (d->prefix_head_stride < (int64_t) d->prefix_len * d->own.head_dim || d->prefix_head_stride % 8)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_prefix_decode: prefix_head_stride must be >= prefix_len * head_dim "
                                               "and a multiple of 8");
    if (const char *why = esda_detail::prefix_tiles_plan(d, &pl->splits)) return fail(ESDA_ERR_INVALID_ARGUMENT, why);
    const size_t parts = (size_t) pl->splits * d->own.batch * d->own.num_q_heads;
    pl->off_ml = (pl->own.bytes + 255) / 256 * 256;
    pl->off_acc = pl->off_ml + (parts * 8 + 255) / 256 * 256;
    pl->bytes = pl->off_acc + parts * d->own.head_dim * sizeof(float);
    return ESDA_OK;
}

}  // namespace

extern "C" {

int esda_prefix_decode_workspace_size(const esda_prefix_desc *desc, size_t *bytes) {
    PrefixPlan pl;
    const int rc = make_prefix_plan(desc, &pl);
    if (rc) return rc;
    if (!bytes) return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_prefix_decode_workspace_size: null output");
    *bytes = pl.bytes;
    return ESDA_OK;
}

int esda_prefix_decode(const esda_prefix_desc *d, const esda_prefix_args *a, void *stream) {
    PrefixPlan pl;
    int rc = make_prefix_plan(d, &pl);
    if (rc) return rc;
    if (!a) return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_prefix_decode: null arguments");
    rc = check_decode_args(&d->own, &a->own);
    if (rc) return rc;
    if (a->own.row_base) return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_prefix_decode: row_base must be null");
    if (!a->prefix_k || !a->prefix_v || !aligned16(a->prefix_k) || !aligned16(a->prefix_v))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_prefix_decode: prefix_k and prefix_v must be 16-byte aligned device memory");
    if ((d->own.kv_shared != 0) != (a->prefix_k == a->prefix_v))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_prefix_decode: prefix_v equals prefix_k when kv_shared, and only then");
    if (!a->own.workspace || a->own.workspace_bytes < pl.bytes || !aligned16(a->own.workspace))
        return fail(ESDA_ERR_WORKSPACE, "esda_prefix_decode: workspace missing or smaller than "
                                        "esda_prefix_decode_workspace_size");
    rc = esda_detail::check_device();
    if (rc) return rc;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    unsigned char *ws = static_cast<unsigned char *>(a->own.workspace);
    float *pre_ml = reinterpret_cast<float *>(ws + pl.off_ml), *pre_acc = reinterpret_cast<float *>(ws + pl.off_acc);
    hipError_t e = static_cast<hipError_t>(esda_detail::prefix_tiles(d, a, pre_acc, pre_ml, st));
    if (e != hipSuccess) return hip_fail(e, "prefix tiles launch");
    TailParams tp{};
    static_cast<AttendParams &>(tp) = decode_params(&d->own, &a->own);
    tp.base = d->prefix_len;
    const DecodeSpace sp = space_of(pl.own, ws);
    uint16_t *out = static_cast<uint16_t *>(a->own.out);
    fill_attend(&d->own, pl.own, sp, reinterpret_cast<int *>(ws), out, tp);
    e = dispatch_attend(d->own.head_dim, d->own.kv_shared != 0, tp, attend_grid(&d->own, pl.own), st);
    if (e != hipSuccess) return hip_fail(e, "attend_kernel launch");
    PrefixMergeParams mp{};
    fill_merge(&d->own, pl.own, sp, a->own.pos, nullptr, 0, out, mp);
    mp.base = d->prefix_len;
    mp.splits = pl.splits;
    mp.pre_acc = pre_acc;
    mp.pre_ml = pre_ml;
    const dim3 grid((d->own.batch * d->own.num_q_heads + 3) / 4), block(256);
    if (d->own.head_dim == 512) hipLaunchKernelGGL(prefix_merge_kernel<512>, grid, block, 0, st, mp);
    else if (d->own.head_dim == 256) hipLaunchKernelGGL(prefix_merge_kernel<256>, grid, block, 0, st, mp);
    else hipLaunchKernelGGL(prefix_merge_kernel<128>, grid, block, 0, st, mp);
    e = hipGetLastError();
    return e == hipSuccess ? ESDA_OK : hip_fail(e, "prefix_merge_kernel launch");
}

}  // extern "C"
