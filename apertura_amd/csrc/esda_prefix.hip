// esda_prefix.hip -- the decode step of a batch that shares a prefix for MI355X (gfx950).
//
// Two launches.  The first leaves partials (m, l, O) of the prefix and of the sequences' own rows,
// whose workgroups stand side by side in one grid: the prefix as query tiles, each key read once
// for the B * G query rows of its kv head (prefill_kernel with PrefixParams), or, for at most 16 of
// them, in runs (prefix_run_kernel); the own rows in runs, with the fused append.  The second
// merges them.  The C ABI is include/esda_prefix.h.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>

#include "esda.h"
#include "esda_attend.h"
#include "esda_internal.h"
#include "esda_prefill_kernel.h"
#include "esda_prefix.h"

namespace {

struct PrefixMergeParams {
    const float *pre_acc, *pre_ml;  // [splits][B * Hq][D], [..][2]
    const float *own_acc, *own_ml;  // [B * Hkv][own_splits][G][D], [..][2]
    const int *pos;
    uint16_t *out;
    int B, Hq, Hkv, G, base, cap, splits, own_splits, own_chunk;
};

// out = sum_s acc_s 2^(m_s - M) / sum_s l_s 2^(m_s - M) over the n partials of a row: its prefix
// splits, then the own splits that hold rows.
struct MergeRow {
    const PrefixMergeParams &p;
    int row, b, h, n;
    __device__ MergeRow(const PrefixMergeParams &q, int r) : p(q), row(r), b(r / q.Hq), h(r % q.Hq) {
        const SeqView sv = seq_view(p.pos[b], p.base, p.cap, 0, 0);
        n = sv.ok ? p.splits + esda_plan::grid_splits(sv.nvis, p.own_chunk, p.own_splits) : 0;
    }
    // partial j's row among its kind's
    __device__ size_t at(int j) const {
        if (j < p.splits) return (size_t) j * ((size_t) p.B * p.Hq) + row;
        return (((size_t) b * p.Hkv + h / p.G) * p.own_splits + (j - p.splits)) * p.G + h % p.G;
    }
    __device__ f32x2 ml(int j) const { return *reinterpret_cast<const f32x2 *>((j < p.splits ? p.pre_ml : p.own_ml) + 2 * at(j)); }
    __device__ const float *acc(int j) const { return j < p.splits ? p.pre_acc : p.own_acc; }
};

// A thread per row and 4 dims: plans of at most NS partials a row.  Every partial is loaded at once,
// beside the position that says how many of the own ones count (the others are dropped by a select).
template <int D, int NS>
__global__ __launch_bounds__(256) void prefix_merge_few_kernel(PrefixMergeParams p) {
    const long long t = (long long) blockIdx.x * 256 + threadIdx.x;
    const int row = (int) (t / (D / 4)), d = (int) (t % (D / 4)) * 4;
    if (row >= p.B * p.Hq) return;
    const MergeRow r(p, row);
    f32x2 ml[NS];
    f32x4 a[NS];
#pragma unroll
    for (int j = 0; j < NS; ++j) {
        ml[j] = f32x2{-INFINITY, 0.0f};
        a[j] = 0.0f;
        if (j < p.splits + p.own_splits) {
            ml[j] = r.ml(j);
            a[j] = *reinterpret_cast<const f32x4 *>(r.acc(j) + r.at(j) * D + d);
        }
    }
    if (r.n == 0) return;  // skipped: its position lies outside its cache
    float M = -INFINITY;
#pragma unroll
    for (int j = 0; j < NS; ++j) M = j < r.n ? fmaxf(M, ml[j][0]) : M;
    float den = 0.0f;
    f32x4 num = 0.0f;
#pragma unroll
    for (int j = 0; j < NS; ++j)
        if (j < r.n) {
            const float w = __builtin_amdgcn_exp2f(ml[j][0] - M);
            den = __builtin_fmaf(ml[j][1], w, den);
            num += a[j] * w;
        }
    bf16x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = (__bf16) (num[e] / den);
    *reinterpret_cast<bf16x4 *>(p.out + (size_t) row * D + d) = o;
}

// A workgroup per row and 64 dims: 16 groups of 16 lanes x 4 dims take the partials in turn, U of
// them in flight, each against its own maximum; the groups meet in LDS.
template <int D>
__global__ __launch_bounds__(256) void prefix_merge_many_kernel(PrefixMergeParams p) {
    constexpr int U = 4;
    __shared__ f32x4 part[16][16];
    __shared__ f32x2 gml[16];
    const int row = blockIdx.x / (D / 64), lane = threadIdx.x & 15, g = threadIdx.x >> 4;
    const int d = (int) (blockIdx.x % (D / 64)) * 64 + lane * 4;
    const MergeRow r(p, row);
    if (r.n == 0) return;  // skipped
    float M = -INFINITY, den = 0.0f;
    f32x4 num = 0.0f;
    for (int j0 = g; j0 < r.n; j0 += 16 * U) {
        f32x2 ml[U];
        f32x4 a[U];
        float top = M;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = j0 + 16 * u;
            ml[u] = f32x2{-INFINITY, 0.0f};
            a[u] = 0.0f;
            if (j < r.n) {
                ml[u] = r.ml(j);
                a[u] = *reinterpret_cast<const f32x4 *>(r.acc(j) + r.at(j) * D + d);
            }
            top = fmaxf(top, ml[u][0]);
        }
        const float c = __builtin_amdgcn_exp2f(M - (top == -INFINITY ? 0.0f : top));
        num *= c;
        den *= c;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float w = __builtin_amdgcn_exp2f(ml[u][0] - (top == -INFINITY ? 0.0f : top));
            den = __builtin_fmaf(ml[u][1], w, den);
            num += a[u] * w;
        }
        M = top;
    }
    part[g][lane] = num;
    if (lane == 0) gml[g] = f32x2{M, den};
    __syncthreads();
    if (g == 0) {
        float top = gml[0][0], l = 0.0f;
#pragma unroll
        for (int u = 1; u < 16; ++u) top = fmaxf(top, gml[u][0]);
        f32x4 o = 0.0f;
#pragma unroll
        for (int u = 0; u < 16; ++u) {
            const float w = gml[u][0] == -INFINITY && gml[u][1] == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(gml[u][0] - top);
            l = __builtin_fmaf(gml[u][1], w, l);
            o += part[u][lane] * w;
        }
        bf16x4 b;
#pragma unroll
        for (int e = 0; e < 4; ++e) b[e] = (__bf16) (o[e] / l);
        *reinterpret_cast<bf16x4 *>(p.out + (size_t) row * D + d) = b;
    }
}

// ------------------------------------------------------------------------ host side

// A step's prefix and own splits, and its workspace behind the status word.
struct PrefixPlan {
    PrefixParams p;
    size_t off_pre_ml, off_own_ml, off_pre_acc, off_own_acc, bytes;
};

constexpr int kRunRows = 128;  // fewest rows of a run: two stages a wave of four

int make_prefix_plan(const esda_prefix_desc *d, PrefixPlan *pl) {
    if (!d) return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_prefix_decode: null description");
    Plan own;
    const int rc = make_plan(&d->own, &own);  // its checks, and the bound on own rows
    if (rc) return rc;
    if (d->own.ring || d->own.window)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_prefix_decode: own caches are linear and without a window");
    if (d->prefix_len <= 0) return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_prefix_decode: prefix_len must be positive");
    if ((long long) d->prefix_len + d->own.batch > INT_MAX || (long long) d->prefix_len + d->own.cap > INT_MAX)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_prefix_decode: positions must stay below 2^31");
    if (d->prefix_head_stride < (int64_t) d->prefix_len * d->own.head_dim || d->prefix_head_stride % 8)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_prefix_decode: prefix_head_stride must be >= prefix_len * head_dim "
                                               "and a multiple of 8");
    const int D = d->own.head_dim, B = d->own.batch, Hkv = d->own.num_kv_heads, P = d->prefix_len;
    const size_t rows = (size_t) B * d->own.num_q_heads;
    esda_prefill_desc t{};
    t.num_q_heads = d->own.num_q_heads;
    t.num_kv_heads = Hkv;
    t.head_dim = D;
    t.seq_q = B;
    t.seq_k = P;
    t.q_pos0 = P - 1;  // every row at or past the last key
    t.q_head_stride = D;
    t.q_row_stride = (int64_t) t.num_q_heads * D;
    t.kv_head_stride = d->prefix_head_stride;
    t.split_keys = d->split_keys;
    t.scale = d->own.scale;
    PrefixParams &p = pl->p;
    if (const char *why = last_plan(&t, 0, &p)) return fail(ESDA_ERR_INVALID_ARGUMENT, why);
    if (B * p.G <= 16) {
        // runs: a workgroup per CU (two at 8 KB a stage), no fewer than kRunRows keys each
        const int per_head = std::max(1, (2 * D * (d->own.kv_shared ? 1 : 2) <= 512 ? 512 : 256) / Hkv);
        int keys = d->split_keys;
        if (keys == 0) {
            keys = std::max(kRunRows, ((P + per_head - 1) / per_head + 15) / 16 * 16);
            keys = std::min(keys, (P + 15) / 16 * 16);
        }
        p.run_keys = keys;
        p.splits = (P + keys - 1) / keys;
        p.tile_groups = (unsigned) (p.splits * Hkv);
    } else {
        p.run_keys = 0;
        p.tile_groups = (unsigned) (p.tiles * Hkv * p.splits);
    }
    // Own rows: runs of 128 KB, so that a workgroup of the grid takes about as long as a tile's.
    const int row_bytes = 2 * D * (d->own.kv_shared ? 1 : 2);
    int chunk = d->own.split_rows > 0 ? d->own.split_rows : std::max(kRunRows, 128 * 1024 / row_bytes);
    if ((own.maxvis + chunk - 1) / chunk > 64) chunk = ((own.maxvis + 63) / 64 + 15) / 16 * 16;
    p.own_chunk = chunk;
    p.own_splits = (own.maxvis + chunk - 1) / chunk;
    if ((long long) p.tile_groups + (long long) B * Hkv * p.own_splits > INT_MAX / 512)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_prefix_decode: too many splits");
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    const size_t pre = rows * p.splits, mine = rows * p.own_splits;
    pl->off_pre_ml = 256;
    pl->off_own_ml = pl->off_pre_ml + up(pre * 8);
    pl->off_pre_acc = pl->off_own_ml + up(mine * 8);
    pl->off_own_acc = pl->off_pre_acc + pre * D * sizeof(float);
    pl->bytes = pl->off_own_acc + mine * D * sizeof(float);
    return ESDA_OK;
}

template <int D>
hipError_t launch_step(const PrefixParams &p, const PrefixMergeParams &m, bool shared, hipStream_t st) {
    if (p.run_keys > 0) {
        const dim3 grid(p.tile_groups + (unsigned) (p.Sq * p.Hkv * p.own_splits)), block(256);
        if (shared) hipLaunchKernelGGL((prefix_run_kernel<D, true>), grid, block, 0, st, p);
        else hipLaunchKernelGGL((prefix_run_kernel<D, false>), grid, block, 0, st, p);
    } else {
        launch_tiles<D>(p, st);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const int rows = m.B * m.Hq, n = m.splits + m.own_splits;
    const unsigned few = (unsigned) (((long long) rows * (D / 4) + 255) / 256);
    if (n <= 4) hipLaunchKernelGGL((prefix_merge_few_kernel<D, 4>), dim3(few), dim3(256), 0, st, m);
    else if (n <= 8) hipLaunchKernelGGL((prefix_merge_few_kernel<D, 8>), dim3(few), dim3(256), 0, st, m);
    else hipLaunchKernelGGL(prefix_merge_many_kernel<D>, dim3(rows * (D / 64)), dim3(256), 0, st, m);
    return hipGetLastError();
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
    unsigned char *ws = static_cast<unsigned char *>(a->own.workspace);
    PrefixParams &p = pl.p;
    p.q = static_cast<const uint16_t *>(a->own.q);
    p.k = static_cast<const uint16_t *>(a->prefix_k);
    p.v = static_cast<const uint16_t *>(a->prefix_v);
    p.part_ml = reinterpret_cast<float *>(ws + pl.off_pre_ml);
    p.part_acc = reinterpret_cast<float *>(ws + pl.off_pre_acc);
    p.own_ml = reinterpret_cast<float *>(ws + pl.off_own_ml);
    p.own_acc = reinterpret_cast<float *>(ws + pl.off_own_acc);
    p.own_k = static_cast<uint16_t *>(a->own.k_cache);
    p.own_v = static_cast<uint16_t *>(a->own.v_cache);
    p.k_new = static_cast<const uint16_t *>(a->own.k_new);
    p.v_new = static_cast<const uint16_t *>(d->own.kv_shared ? a->own.k_new : a->own.v_new);
    p.pos = a->own.pos;
    p.status = reinterpret_cast<int *>(ws);
    p.own_seq_stride = d->own.seq_stride;
    p.own_head_stride = d->own.head_stride;
    p.own_cap = d->own.cap;
    p.own_base = d->prefix_len;
    const PrefixMergeParams m{p.part_acc, p.part_ml, p.own_acc, p.own_ml, p.pos, static_cast<uint16_t *>(a->own.out),
                              d->own.batch, d->own.num_q_heads, d->own.num_kv_heads, p.G, p.own_base, p.own_cap, p.splits,
                              p.own_splits, p.own_chunk};
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const bool shared = d->own.kv_shared != 0;
    const hipError_t e = d->own.head_dim == 512   ? launch_step<512>(p, m, shared, st)
                         : d->own.head_dim == 256 ? launch_step<256>(p, m, shared, st)
                                                  : launch_step<128>(p, m, shared, st);
    return e == hipSuccess ? ESDA_OK : hip_fail(e, "esda_prefix_decode launch");
}

}  // extern "C"
