// esda_prefix.hip -- the decode step of a batch that shares a prefix for MI355X (gfx950).
//
// Two launches.  The first leaves partials (m, l, O) of the prefix and of the sequences' own rows,
// whose workgroups stand side by side in one grid: the prefix as query tiles, each key read once
// for the B * G query rows of its kv head (prefill_kernel with PrefixParams), or, for few of them,
// in runs (prefix_run_kernel); the own rows in runs, with the fused append.  The second merges them.
// A step of few rows is bound by the latency of the two (2 sequences behind 2049 tokens: 13.5 us), a
// long one by the runs' starts and the reads that a key's two row groups do not share (4 behind 32,768:
// 169 MB read for 140, the first launch 34.7 us, 4.9 TB/s, where a step of plain decode reads such rows at
// 7; 40 us in all), one of many sequences by both kinds of workgroups sharing the CUs (64 behind 16,384,
// 200 MB and 18 GFLOP: 61 us).  At 512 dims a batch is bound by its tiles' starts and partials: 32 behind
// 8191 write 46 MB of them and read them back for 70 MB of keys, 50 us.  With prefix, own rows and their
// merges in launches one after the other the first three took 48, 99 and 123 us.
// The C ABI is include/esda_prefix.h.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <string>
#include <type_traits>

#include "esda.h"
#include "esda_attend.h"
#include "esda_internal.h"
#include "esda_prefill_kernel.h"
#include "esda_prefix.h"
#include "esda_prefix_tiles.h"

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

constexpr int kRunRows = 64;    // fewest rows of a run: a stage for each of four waves
constexpr int kOwnSplits = 64;  // most own splits

// How the prefix's query rows can be laid out: as tiles (nw > 0: a prefill form), or in runs of 16 NG
// rows.  us of a workgroup: `start`, and per KB of K and V `per_kb`; slots: workgroups the GPU holds at
// once.  Runs against tiles at the best splits and own chunks of random steps (StepCosts), time of the
// one over that of the other: D = 128, up to 16 rows 0.76, 32 0.84, 64 1.08 (0.83 .. 1.35); D = 256, 16
// rows 0.93, 32 1.10 (not offered); D = 512, 16 rows 0.90 (0.58 .. 1.33), 32 0.93.
struct Form {
    int qb, kh, nw, ng;
    float start, per_kb;
    int slots;
    int rows() const { return ng ? 16 * ng : 16 * qb * (kh ? nw / 2 : nw); }
};

// What else a step's time goes by: us of an own workgroup and its KB per us; us and KB per us of the
// bytes of both kinds; the share by which the two bounds add up; us of a merge of at most 8 partials a
// row and of more; us per byte of partials.
// These and the forms' costs are fitted, per head dim, to 230 .. 500 random steps (1 .. 64 sequences,
// prefixes of 64 .. 40,000 keys, own caches of 64 .. 2048 rows, full, at random and nearly empty), each in
// every form, up to 7 own chunks and 9 prefix splits, graph-replayed, at D = 256 and 512 over 4 .. 24
// copies of the caches in turn (from HBM).  The cheapest by them takes 1.03 of the best forced plan's
// time on average, 1.15 at the 95th percentile.
struct StepCosts {
    float own_start, own_rate, start, rate, add, few, many, part;
};
constexpr StepCosts kCosts512 = {6.3f, 40.0f, 3.8f, 5600.0f, 0.13f, 4.3f, 3.5f, 2.6e-7f};
constexpr StepCosts kCosts256 = {5.4f, 79.0f, 11.4f, 16500.0f, 0.09f, 4.5f, 4.0f, 3.3e-7f};
constexpr StepCosts kCosts128 = {4.4f, 43.0f, 5.3f, 7900.0f, 0.25f, 5.8f, 2.9f, 2.9e-7f};

// The forms a step may take; returns their number.
int forms_of(int D, int rows, bool shared, Form *f) {
    int n = 0;
    const Tiling *t = D == 512 ? kTilings512 : D == 256 ? kTilings256 : kTilings128;
    const int nt = D == 512 ? 2 : D == 256 ? 3 : 1;
    // (a prefill workgroup's costs, and what a step's add to its start and to its stages)
    constexpr float kMore512[][2] = {{1.8f, 1.02f}, {0.0f, 0.96f}};
    constexpr float kMore256[][2] = {{4.6f, 1.37f}, {-0.7f, 1.47f}, {-1.0f, 1.63f}};
    constexpr float kMore128[][2] = {{0.0f, 1.6f}};
    const float(*more)[2] = D == 512 ? kMore512 : D == 256 ? kMore256 : kMore128;
    const float stage_kb = 32.0f * 2 * D * (shared ? 1 : 2) / 1024;
    for (int i = 0; i < nt; ++i)
        if (!(D == 512 && rows <= 64 && t[i].nw == (shared ? 8 : 4)))  // (launch_tiles' choice for one tile)
            f[n++] = {t[i].qb, t[i].kh, t[i].nw, 0, t[i].wg + t[i].row * std::min(rows, t[i].rows()) + more[i][0],
                      t[i].stage / stage_kb * more[i][1], 256};
    if (D == 512 && rows <= 32) f[n++] = {0, 0, 0, 1, 8.0f, rows <= 16 ? 1 / 54.0f : 1 / 49.0f, 256};
    if (D == 256 && rows <= 16) f[n++] = {0, 0, 0, 1, 4.6f, 1 / 65.0f, 256};
    if (D == 128 && rows <= 64) f[n++] = rows <= 16 ? Form{0, 0, 0, 1, 5.8f, 1 / 65.0f, 512}
                                         : rows <= 32 ? Form{0, 0, 0, 2, 13.2f, 1 / 56.0f, 512} : Form{0, 0, 0, 4, 13.1f, 1 / 32.0f, 256};
    return n;
}

// us of na workgroups of `a` us, then nb of `b` us, on `slots`.
float makespan(long long na, float a, long long nb, float b, int slots) {
    const long long rem = na % slots, idle = slots - rem;  // slots of the first kind's last round, and without it
    const float early = (float) (na / slots) * a, late = early + (rem ? a : 0.0f);
    if (nb <= idle) return std::max(late, early + (nb ? b : 0.0f));
    // whole rounds that both sorts of slots take (the first sort starts late - early behind), then the rest
    const long long rounds = std::max(0LL, nb / slots - 2);
    nb -= rounds * slots;
    for (int i = 1;; ++i) {
        const long long by_idle = i * idle, by_rem = (long long) (std::max(0.0f, early + i * b - late) / b) * rem;
        if (by_idle + by_rem >= nb) return std::max(late, early + (rounds + i) * b);
    }
}

int fresh_prefix_plan(const esda_prefix_desc *d, PrefixPlan *pl) {
    if (!d) return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_prefix_decode: null description");
    Plan own;
    const int rc = make_plan(&d->own, &own);  // its checks, and the bound on own rows
    if (rc) return rc;
    if (d->own.ring || d->own.window)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_prefix_decode: own caches are linear and without a window");
    if (d->prefix_len <= 0 || d->prefix_len > 1 << 30)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_prefix_decode: prefix_len must be 1 .. 2^30");
    if ((long long) d->prefix_len + d->own.batch > INT_MAX || (long long) d->prefix_len + d->own.cap > INT_MAX)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_prefix_decode: positions must stay below 2^31");
    if (d->prefix_head_stride < (int64_t) d->prefix_len * d->own.head_dim || d->prefix_head_stride % 8)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_prefix_decode: prefix_head_stride must be >= prefix_len * head_dim "
                                               "and a multiple of 8");
    if (d->split_keys < 0 || d->split_keys % kStageKeys)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_prefix_decode: split_keys must be a multiple of 32");
    if (!(d->own.scale > 0.0f) || !std::isfinite(d->own.scale))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_prefix_decode: scale must be positive and finite");
    const int D = d->own.head_dim, B = d->own.batch, Hkv = d->own.num_kv_heads, P = d->prefix_len;
    const bool shared = d->own.kv_shared != 0;
    const size_t rows = (size_t) B * d->own.num_q_heads;
    if (rows * (D / 64) >= 1u << 24)  // a launch holds fewer than 2^32 threads, the merge 256 for 64 dims
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_prefix_decode: too many query rows");
    PrefixParams &p = pl->p;
    p = PrefixParams{};
    p.Hq = d->own.num_q_heads;
    p.Hkv = Hkv;
    p.G = own.G;
    p.Sq = B;
    p.Sk = P;
    p.q_pos0 = P - 1;  // every row at or past the last key
    p.q_hs = D;
    p.q_rs = (long long) p.Hq * D;
    p.kv_hs = d->prefix_head_stride;
    p.scale_log2e = d->own.scale * kLog2e;
    // Own chunk, form and key splits of the prefix: the cheapest by the workgroups of both kinds on the
    // GPU, the bytes, and the merge of the partials.  (With the own rows in about two workgroups a CU
    // whatever the prefix takes, drawn steps were 17% longer on average, up to three times as long.)
    const StepCosts &c = D == 512 ? kCosts512 : D == 256 ? kCosts256 : kCosts128;
    const float row_kb = 2.0f * D * (shared ? 1 : 2) / 1024;
    const int group_rows = B * p.G;
    const float floor_us = c.start + ((float) P * Hkv + (float) own.maxvis * B * Hkv) * row_kb / c.rate;
    Form f[4];
    const int nf = forms_of(D, group_rows, shared, f);
    float best = INFINITY;
    auto consider = [&](const Form &form, int chunk, int keys) {
        const int splits = (int) (((long long) P + keys - 1) / keys), tiles = (group_rows + form.rows() - 1) / form.rows();
        const int own_splits = (int) (((long long) own.maxvis + chunk - 1) / chunk), n = splits + own_splits;
        const long long groups = (long long) tiles * Hkv * splits, own_groups = (long long) B * Hkv * own_splits;
        const float us = form.start + std::min(keys, P) * row_kb * form.per_kb;
        const float own_us = c.own_start + std::min(chunk, own.maxvis) * row_kb / c.own_rate;
        const float span = form.ng ? makespan(own_groups, own_us, groups, us, form.slots)
                                   : makespan(groups, us, own_groups, own_us, form.slots);
        const float cost = std::max(span, floor_us) + c.add * std::min(span, floor_us) + (n <= 8 ? c.few : c.many) +
                           c.part * 4 * D * rows * n;
        if (cost >= best) return;
        best = cost;
        p.qb = form.qb;
        p.kh = form.kh;
        p.nw = form.nw;
        p.tiles = tiles;
        p.splits = splits;
        p.kps = keys;
        p.run_keys = form.ng ? keys : 0;
        p.row_groups = form.ng ? tiles : 0;
        p.own_chunk = chunk;
        p.own_splits = own_splits;
    };
    // Forced splits longer than the rows are cut to them, in whole units (the kernels add one to a row).
    auto whole = [](long long n, int unit) { return (n + unit - 1) / unit * unit; };
    const int forced_keys = (int) std::min<long long>(d->split_keys, whole(P, kStageKeys));
    auto with_chunk = [&](int chunk) {
        for (int i = 0; i < nf; ++i) {
            if (forced_keys > 0) {
                consider(f[i], chunk, forced_keys);
                continue;
            }
            const int least = f[i].ng ? kRunRows : kStageKeys, unit = f[i].ng ? 16 : kStageKeys;
            int last = 0;
            for (int s = 1; s <= 512; s += std::max(1, s / 8)) {
                const int keys = std::max(least, ((P + s - 1) / s + unit - 1) / unit * unit);
                if (keys != last) consider(f[i], chunk, keys);
                if (keys == least) break;
                last = keys;
            }
        }
    };
    const int least_chunk = (own.maxvis / kOwnSplits + 16) / 16 * 16;  // (at most kOwnSplits of them)
    if (d->own.split_rows > 0) {
        const int forced = (int) std::min<long long>(d->own.split_rows, whole(d->own.cap, kTile));
        with_chunk(((long long) own.maxvis + forced - 1) / forced > kOwnSplits ? least_chunk : forced);
    } else {
        int last = 0;
        for (int s = 1; s <= kOwnSplits; s += std::max(1, s / 2)) {
            const int chunk = (int) std::max<long long>(kRunRows, std::min(((long long) own.maxvis + s - 1) / s + 15, (long long) INT_MAX) / 16 * 16);
            if (chunk != last) with_chunk(chunk);
            if (chunk == kRunRows) break;
            last = chunk;
        }
    }
    p.part_nt = 4.0f * D * rows * p.splits <= kPartNtBytes;
    if (p.splits > 65535 || (long long) p.tiles * Hkv * p.splits > INT_MAX / 1024)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_prefix_decode: too many key splits");
    p.tile_groups = (unsigned) (p.run_keys ? (p.splits * Hkv + 7) / 8 * 8 * p.row_groups : p.tiles * Hkv * p.splits);
    p.own_groups = (unsigned) (B * Hkv * p.own_splits);
    if ((long long) p.tile_groups + p.own_groups > INT_MAX / 512)
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

// The plan of the calling thread's last description, kept: it depends on that alone, and a step asks
// for it at every call.  (Descriptions compare by their bytes; other padding only plans anew.)
int make_prefix_plan(const esda_prefix_desc *d, PrefixPlan *pl) {
    struct Last {
        esda_prefix_desc desc;
        PrefixPlan plan;
        bool set = false;
    };
    thread_local Last last;
    if (!d || !last.set || std::memcmp(d, &last.desc, sizeof(*d)) != 0) {
        const int rc = fresh_prefix_plan(d, pl);
        if (rc) return rc;
        std::memcpy(&last.desc, d, sizeof(*d));
        last.plan = *pl;
        last.set = true;
        return ESDA_OK;
    }
    *pl = last.plan;
    return ESDA_OK;
}

template <int D>
hipError_t launch_step(const PrefixParams &p, const PrefixMergeParams &m, bool shared, hipStream_t st) {
    if (p.run_keys > 0) {
        const dim3 grid(p.tile_groups + p.own_groups), block(256);
        auto run = [&](auto ng) {
            constexpr int NG = decltype(ng)::value;
            if (shared) hipLaunchKernelGGL((prefix_run_kernel<D, true, NG>), grid, block, 0, st, p);
            else hipLaunchKernelGGL((prefix_run_kernel<D, false, NG>), grid, block, 0, st, p);
        };
        // (forms_of: 16 rows a workgroup at D = 256 and 512, up to 64 at D = 128)
        if constexpr (D >= 256) run(std::integral_constant<int, 1>{});
        if constexpr (D == 128) {
            if (p.Sq * p.G <= 16) run(std::integral_constant<int, 1>{});
            else if (p.Sq * p.G <= 32) run(std::integral_constant<int, 2>{});
            else run(std::integral_constant<int, 4>{});
        }
    } else {
        esda_detail::prefix_tiles(p, D, st);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    // The threads of the first form hold a row's partials side by side: up to 8 of them always, up to 40
    // where there are threads to cover the loads.  64 rows (2,048 .. 8,192 threads) in 21 partials, first
    // form / second: 10.5 / 8.9, 19.0 / 17.5, 15.4 / 14.1 us a step (D = 128, 256, 512); 32,768 threads, 11
    // 15.3 / 16.3 and 20.9 / 21.8, 21 20.7 / 20.5 and 22.2 / 22.3; 65,536 20.1 / 23.7 and 24.7 / 28.4, 31
    // 33.6 / 35.5 and 41.3 / 43.6; 262,144 in 11 37.6 / 48.5, in 31 77.4 / 79.6.
    const int rows = m.B * m.Hq, n = m.splits + m.own_splits;
    const long long threads = (long long) rows * (D / 4);
    const unsigned few = (unsigned) ((threads + 255) / 256);
    if (n <= 4) hipLaunchKernelGGL((prefix_merge_few_kernel<D, 4>), dim3(few), dim3(256), 0, st, m);
    else if (n <= 8) hipLaunchKernelGGL((prefix_merge_few_kernel<D, 8>), dim3(few), dim3(256), 0, st, m);
    else if (n <= 16 && threads >= 1 << 15) hipLaunchKernelGGL((prefix_merge_few_kernel<D, 16>), dim3(few), dim3(256), 0, st, m);
    else if (n <= 24 && threads >= 1 << 15) hipLaunchKernelGGL((prefix_merge_few_kernel<D, 24>), dim3(few), dim3(256), 0, st, m);
    else if (n <= 40 && threads >= 1 << 16) hipLaunchKernelGGL((prefix_merge_few_kernel<D, 40>), dim3(few), dim3(256), 0, st, m);
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
