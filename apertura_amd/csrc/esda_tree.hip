// esda_tree.hip -- the step of drafted tokens over a cache in pages, or a linear one, for MI355X
// (gfx950).  The C ABI is include/esda_tree.h.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <string>
#include <type_traits>

#include "esda.h"
#include "esda_internal.h"
#include "esda_page_view.h"
#include "esda_parts_merge.h"
#include "esda_prefill_kernel.h"
#include "esda_tree.h"
#include "esda_tree_rows.h"
#include "esda_tree_tiles.h"

namespace {

// Query rows r0 .. of a (sequence, kv head) over one split of its keys, in a run (esda_stream.h).
template <int D, bool SH, int NG>
__global__ __launch_bounds__(256, 1) void tree_run_kernel(TreeParams p) {
    using Own = OwnRows<D, SH, 4, NG>;
    __shared__ __attribute__((aligned(16))) unsigned char lds[Own::BYTES];
    __shared__ unsigned long long paths[64];
    __shared__ int odd[16 * NG], any_odd;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6), li = lane & 15, lg = lane >> 4;
    // The row groups of the same keys are 8 workgroups apart: on one XCD, whose L2 hands the second what
    // the first read.
    const unsigned i = blockIdx.x >> 3, unit = i / (unsigned) p.row_groups * 8 + (blockIdx.x & 7);
    const int r0 = (int) (i % (unsigned) p.row_groups) * 16 * NG;
    const int split = (int) (unit % (unsigned) p.splits), pair = (int) (unit / (unsigned) p.splits);
    if (pair >= p.B * p.Hkv) return;
    const int b = pair / p.Hkv, kvh = pair % p.Hkv;
    unsigned long long path;
    const TreeView w = tree_view(p, b, lane, path);
    if (kvh == 0 && split == 0 && r0 == 0 && threadIdx.x == 0) {
        p.views[b] = w.ok ? w.total : -1;
        if (!w.ok) __hip_atomic_fetch_add(p.status, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    if (!w.ok) return;
    const int rows = p.Sq * p.G;
    const size_t head = ((size_t) b * p.Sq * p.Hq + (size_t) kvh * p.G);  // of q and out, in rows
    auto at = [&](int r) { return head + (size_t) (r / p.G) * p.Hq + r % p.G; };
    TreeRows<D, SH> x(p, w, b, kvh);
    if (!esda_plan::grid_split(split, p.splits, p.kps, w.total, &x.j0, &x.j1)) {
        if (split == 0 && p.splits == 1)  // no node at all
            for (int t = threadIdx.x; t < min(16 * NG, rows - r0) * (D / 8); t += 256)
                *reinterpret_cast<u32x4 *>(p.out + at(r0 + t / (D / 8)) * D + t % (D / 8) * 8) = u32x4{0u, 0u, 0u, 0u};
        return;
    }
    x.G = min(rows - r0, 16 * NG);
    if (wave == 0) paths[lane] = path;
    for (int t = threadIdx.x; t < 16 * NG; t += 256) odd[t] = 0;
    if (threadIdx.x == 0) any_odd = 0;
    lds_barrier();
    unsigned long long sees[NG];
    int lowest[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        const int r = r0 + 16 * g + li;
        sees[g] = r < rows ? paths[r / p.G] : 0ull;
        lowest[g] = p.window > 0 ? w.len + __popcll(sees[g]) - p.window : 0;
    }
    const int all_see = p.window > 0 ? w.len + p.Sq - p.window : 0;  // committed rows from it on: every node
    auto score = [&](f32x4 &s, int jst, int end, int g) {
        s *= p.scale_log2e;
        const int row = x.first + jst;
        if (row >= all_see && row + 16 <= w.len && jst + 16 <= end) return;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int j = jst + 4 * lg + e, r = x.first + j;
            const bool seen = r < w.len ? r >= lowest[g] : ((sees[g] >> ((r - w.len) & 63)) & 1) != 0;
            if (j >= end || !seen) s[e] = -INFINITY;
        }
    };
    const size_t nrows = (size_t) p.B * p.Sq * p.Hq, part = (size_t) split * nrows;
    auto finish = [&](int r, int d, f32x4 o, float m, float l) {  // dims d .. d + 3 of query row r
        if (paths[r / p.G] == 0ull) {  // no node: nothing seen
            o = 0.0f;
            l = 0.0f;
        }
        if (p.splits == 1) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            bf16x4 y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = (__bf16) (o[e] * inv);
            *reinterpret_cast<bf16x4 *>(p.out + at(r) * D + d) = y;
        } else {
            Own::store(p.part_acc, p.part_ml, part + at(r), d, o, m, l);
        }
    };
    Own::attend(
        lds, x, [&](int h) { return p.q + at(r0 + h) * D; }, score,
        [&](int h, int d, const f32x4 &o, float m, float l) {
            finish(r0 + h, d, o, m, l);
            float c = 0.0f;  // NaN where a value is not finite
#pragma unroll
            for (int e = 0; e < 4; ++e) c = __builtin_fmaf(o[e], 0.0f, c);
            if (c != c && paths[(r0 + h) / p.G] != 0ull) {
                odd[h] = 1;
                any_odd = 1;
            }
        });
    if (r0 == 0) append_nodes<D, SH>(x, paths, x.j0, x.j1);
    ESDA_WAIT_VM(0);  // the rows as written above, before they are written again
    lds_barrier();
    if (__builtin_expect(any_odd != 0, 0)) {
        for (int h = wave; h < x.G; h += 4) {
            if (!odd[h]) continue;
            const unsigned long long mine = paths[(r0 + h) / p.G];
            tree_row_again<D, SH>(x, p.q + at(r0 + h) * D, mine, p.window > 0 ? w.len + __popcll(mine) - p.window : 0, x.j0, x.j1,
                                  p.scale_log2e, [&](float m, float l, const float(&o)[D / 64]) {
                                      tree_row_store<D>(p, split, at(r0 + h), lane, m, l, o);
                                  });
        }
    }
}

// A row's partials for esda_parts_merge.h: the splits that its sequence's keys reach.
struct TreeMergeRow {
    using Params = TreeParams;
    static constexpr bool EMPTY = true;
    const TreeParams &p;
    int row, view, n;
    __device__ TreeMergeRow(const TreeParams &q, int r) : p(q), row(r) {
        view = q.views[r / (q.Sq * q.Hq)];
        n = view > 0 ? esda_plan::grid_splits(view, q.kps, q.splits) : 0;
    }
    static __host__ __device__ int rows(const TreeParams &q) { return q.B * q.Sq * q.Hq; }
    __device__ int most() const { return p.splits; }
    __device__ bool write() const { return view >= 0; }
    __device__ size_t at(int j) const { return (size_t) j * rows(p) + row; }
    __device__ f32x2 ml(int j) const { return *reinterpret_cast<const f32x2 *>(p.part_ml + 2 * at(j)); }
    __device__ const float *acc(int) const { return p.part_acc; }
};

// ------------------------------------------------------------------------ host side

int fail(int code, const std::string &msg) {
    esda_detail::set_error(msg);
    return code;
}

int refuse(const char *why) { return fail(ESDA_ERR_INVALID_ARGUMENT, std::string("esda_tree_decode: ") + why); }

bool aligned(const void *p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

struct TreePlan {
    TreeParams p;
    size_t off_views, off_ml, off_acc, bytes;
};

const char *check_desc(const esda_tree_desc *d) {
    using namespace esda_page_view;
    if (!d) return "null description";
    if (d->batch < 1 || d->batch > 256) return "batch must be 1 .. 256";
    if (d->nodes < 1 || d->nodes > 64) return "nodes must be 1 .. 64";
    if (d->num_q_heads <= 0 || d->num_kv_heads <= 0 || d->num_q_heads % d->num_kv_heads)
        return "num_q_heads must be a multiple of num_kv_heads";
    if (d->num_q_heads / d->num_kv_heads > 16) return "at most 16 query heads per kv head";
    if (d->head_dim != 128 && d->head_dim != 256 && d->head_dim != 512) return "head_dim must be 128, 256 or 512";
    if (d->window != 0 && d->window < d->nodes) return "window must be 0 or at least nodes";
    if (d->max_pages == 0) {
        if (d->page_rows < 1 || d->page_rows > 1 << 30) return "linear caches have 1 .. 2^30 rows";
        if (d->num_pages != d->batch) return "linear caches: num_pages is the batch";
    } else if (const char *why = check_table(d->num_pages, d->page_rows, d->batch, d->max_pages, d->table_stride)) {
        return why;
    }
    if (!whole16(d->page_stride) || !whole16(d->head_stride)) return "strides must be non-negative multiples of 8";
    if (!blocks_apart({1, d->num_pages, d->num_kv_heads}, {0, d->page_stride, d->head_stride}, (long long) d->page_rows * d->head_dim))
        return "the pages overlap";
    if (d->max_visible < 0) return "max_visible must not be negative";
    if (d->split_rows < 0 || d->split_rows % kStageKeys) return "split_rows must be a multiple of 32";
    if (!(d->scale > 0.0f) || !std::isfinite(d->scale)) return "scale must be positive and finite";
    if ((long long) d->batch * d->nodes * d->num_q_heads * (d->head_dim / 64) >= 1 << 24) return "too many query rows";
    return nullptr;
}

// How the query rows of a kv head can be laid out: as tiles (nw > 0: a prefill form), or in runs of 16 ng
// rows.  us of a workgroup: `start`, and `per_kb` per KB of K and V; slots: workgroups the GPU holds at once.
struct Form {
    int qb, kh, nw, ng;
    float start, per_kb;
    int slots;
    int rows() const { return ng ? 16 * ng : 16 * qb * (kh ? nw / 2 : nw); }
};

// The forms a step of `rows` query rows a kv head may take; returns their number.
int forms_of(int D, int rows, bool shared, Form *f) {
    int n = 0;
    const float stage_kb = 32.0f * 2 * D * (shared ? 1 : 2) / 1024;
    auto tile = [&](const Tiling &t, float more, float times) {
        f[n++] = {t.qb, t.kh, t.nw, 0, t.wg + t.row * std::min(rows, t.rows()) + more, t.stage / stage_kb * times, 256 * t.occ};
    };
    if (D == 512) {
        if (rows > 64 || shared == false) tile(kTilings512[0], 1.8f, 1.02f);
        if (rows > 64 || shared) tile(kTilings512[1], 0.0f, 0.96f);  // (launch_tiles' choice for one tile)
        f[n++] = {0, 0, 0, 1, 8.0f, 1 / 54.0f, 256};
    } else if (D == 256) {
        tile(kTilings256[1], -0.7f, 1.47f);
        tile(kTilings256[2], -1.0f, 1.63f);
        f[n++] = {0, 0, 0, 1, 4.6f, 1 / 65.0f, 256};
    } else {
        tile(kTilings128Scored[0], 0.0f, 1.6f);
        f[n++] = {0, 0, 0, 1, 5.8f, 1 / 65.0f, 512};
        if (rows > 16) f[n++] = {0, 0, 0, 2, 13.2f, 1 / 56.0f, 512};
        if (rows > 32) f[n++] = {0, 0, 0, 4, 13.1f, 1 / 32.0f, 256};
    }
    return n;
}

// Form and splits of a step over at most `most` keys a sequence: the cheapest by the workgroups' time on
// the GPU, the bytes, and the merge of the partials.
void choose(const esda_tree_desc *d, long long most, TreeParams *p) {
    const int D = d->head_dim, rows = p->Sq * p->G;
    const bool shared = d->kv_shared != 0;
    const float row_kb = 2.0f * D * (shared ? 1 : 2) / 1024;
    const long long pairs = (long long) p->B * p->Hkv, out_rows = (long long) p->B * p->Sq * p->Hq;
    const float floor_us = 4.0f + (float) (most * pairs) * row_kb / 5600.0f;
    Form f[4];
    const int nf = forms_of(D, rows, shared, f);
    float best = INFINITY;
    auto consider = [&](const Form &form, long long keys) {
        const long long splits = (most + keys - 1) / keys, tiles = (rows + form.rows() - 1) / form.rows();
        const long long groups = pairs * tiles * splits;
        const float us = form.start + (float) std::min(keys, most) * row_kb * form.per_kb;
        float span = std::max(us, (float) groups / form.slots * us);
        if (groups > form.slots) span += 0.5f * us;
        const float cost = std::max(span, floor_us) + 0.13f * std::min(span, floor_us) +
                           (splits == 1 ? 0.0f : splits <= 8 ? 4.3f : 4.8f) + (splits > 1 ? 2.6e-7f * 4 * D * out_rows * splits : 0.0f);
        if (cost >= best) return;
        best = cost;
        p->qb = form.qb;
        p->kh = form.kh;
        p->nw = form.nw;
        p->run_groups = form.ng;
        p->tiles = p->row_groups = (int) tiles;
        p->splits = (int) std::max(1LL, splits);
        p->kps = (int) keys;
    };
    for (int i = 0; i < nf; ++i) {
        if (d->split_rows > 0) {  // (one longer than the keys is cut to them)
            consider(f[i], std::min<long long>(d->split_rows, (most + kStageKeys - 1) / kStageKeys * kStageKeys));
            continue;
        }
        long long last = 0;
        for (int s = 1; s <= 512; s += std::max(1, s / 8)) {
            const long long keys = std::max(64LL, ((most + s - 1) / s + kStageKeys - 1) / kStageKeys * kStageKeys);
            if (keys != last) consider(f[i], keys);
            if (keys == 64) break;
            last = keys;
        }
    }
    p->part_nt = 4.0f * D * out_rows * p->splits <= kPartNtBytes;
}

int fresh_plan(const esda_tree_desc *d, TreePlan *pl) {
    if (const char *why = check_desc(d)) return refuse(why);
    const int D = d->head_dim;
    TreeParams &p = pl->p;
    p = TreeParams{};
    p.Hq = d->num_q_heads;
    p.Hkv = d->num_kv_heads;
    p.G = p.Hq / p.Hkv;
    p.Sq = d->nodes;
    p.B = d->batch;
    p.window = d->window;
    p.kv_hs = d->head_stride;
    p.page_stride = d->page_stride;
    p.table_stride = d->table_stride;
    p.linear = d->max_pages == 0;
    p.N = d->num_pages;
    p.P = p.linear ? 1 : d->max_pages;
    p.shift = p.linear ? 30 : __builtin_ctz((unsigned) d->page_rows);
    p.cap = d->page_rows;
    p.scale_log2e = d->scale * kLog2e;
    p.q_hs = p.o_hs = D;
    p.q_rs = p.o_rs = (long long) p.Hq * D;
    // most keys of a sequence: what its pages hold, the bound that is given, its window (from a multiple
    // of 32 on); longer ones only lengthen the last split
    long long most = p.linear ? p.cap : (long long) d->max_pages * d->page_rows;
    if (d->max_visible > 0) most = std::min(most, (long long) d->max_visible + p.Sq);
    if (p.window > 0) most = std::min(most, (long long) p.window + p.Sq + kStageKeys);
    choose(d, most, &p);
    const long long groups = (long long) p.B * p.Hkv * p.row_groups;
    if (p.splits > 4096 || groups * p.splits >= INT_MAX / 512) return refuse("too many splits");
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    const size_t parts = p.splits > 1 ? (size_t) p.B * p.Sq * p.Hq * p.splits : 0;
    pl->off_views = 256;
    pl->off_ml = pl->off_views + up((size_t) p.B * 4);
    pl->off_acc = pl->off_ml + up(parts * 8);
    pl->bytes = pl->off_acc + parts * D * sizeof(float);
    return ESDA_OK;
}

// The plan of the calling thread's last description, kept: it depends on that alone, and a step asks
// for it at every call.
int make_tree_plan(const esda_tree_desc *d, TreePlan *pl) {
    struct Last {
        esda_tree_desc desc;
        TreePlan plan;
        bool set = false;
    };
    thread_local Last last;
    if (!d || !last.set || std::memcmp(d, &last.desc, sizeof(*d)) != 0) {
        const int rc = fresh_plan(d, pl);
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
hipError_t launch_step(const TreeParams &p, bool shared, hipStream_t st) {
    if (!p.run_groups) {
        esda_detail::tree_tiles(p, D, st);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess || p.splits == 1) return e;
        launch_parts_merge<D, TreeMergeRow>(p, p.splits, st);
        return hipGetLastError();
    }
    const unsigned units = (unsigned) (p.B * p.Hkv * p.splits);
    const dim3 grid((units + 7) / 8 * 8 * p.row_groups), block(256);
    auto run = [&](auto ng) {
        constexpr int NG = decltype(ng)::value;
        if (shared) hipLaunchKernelGGL((tree_run_kernel<D, true, NG>), grid, block, 0, st, p);
        else hipLaunchKernelGGL((tree_run_kernel<D, false, NG>), grid, block, 0, st, p);
    };
    if (p.run_groups == 1) run(std::integral_constant<int, 1>{});
    if constexpr (D == 128) {
        if (p.run_groups == 2) run(std::integral_constant<int, 2>{});
        if (p.run_groups == 4) run(std::integral_constant<int, 4>{});
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits == 1) return e;
    launch_parts_merge<D, TreeMergeRow>(p, p.splits, st);
    return hipGetLastError();
}

}  // namespace

extern "C" {

int esda_tree_workspace_size(const esda_tree_desc *desc, size_t *bytes) {
    TreePlan pl;
    const int rc = make_tree_plan(desc, &pl);
    if (rc) return rc;
    if (!bytes) return refuse("null output");
    *bytes = pl.bytes;
    return ESDA_OK;
}

int esda_tree_decode(const esda_tree_desc *d, const esda_tree_args *a, void *stream) {
    TreePlan pl;
    int rc = make_tree_plan(d, &pl);
    if (rc) return rc;
    if (!a) return refuse("null arguments");
    const bool shared = d->kv_shared != 0;
    if (!a->q || !a->k_new || !a->k_pages || !a->v_pages || !a->out || (!shared && !a->v_new)) return refuse("null pointer");
    for (const void *t : {a->q, a->k_new, shared ? a->k_new : a->v_new, (const void *) a->k_pages, (const void *) a->v_pages, (const void *) a->out})
        if (!aligned(t, 16)) return refuse("tensors must be 16-byte aligned");
    if (shared != (a->k_pages == a->v_pages)) return refuse("v_pages equals k_pages when kv_shared, and only then");
    if ((d->max_pages == 0) != (a->table == nullptr)) return refuse("a table goes with pages, and only with them");
    if (!a->length || !aligned(a->length, 4) || !aligned(a->table, 4) || !aligned(a->parent, 4))
        return refuse("table, length and parent must be 4-byte aligned device memory");
    if (!a->workspace || a->workspace_bytes < pl.bytes || !aligned(a->workspace, 16))
        return fail(ESDA_ERR_WORKSPACE, "esda_tree_decode: workspace missing or smaller than esda_tree_workspace_size");
    rc = esda_detail::check_device();
    if (rc) return rc;
    unsigned char *const ws = static_cast<unsigned char *>(a->workspace);
    TreeParams &p = pl.p;
    p.q = static_cast<const uint16_t *>(a->q);
    p.k = static_cast<const uint16_t *>(a->k_pages);
    p.v = static_cast<const uint16_t *>(a->v_pages);
    p.out = static_cast<uint16_t *>(a->out);
    p.k_new = static_cast<const uint16_t *>(a->k_new);
    p.v_new = static_cast<const uint16_t *>(shared ? a->k_new : a->v_new);
    p.table = a->table;
    p.length = a->length;
    p.parent = a->parent;
    p.status = reinterpret_cast<int *>(ws);
    p.views = reinterpret_cast<int *>(ws + pl.off_views);
    p.part_ml = reinterpret_cast<float *>(ws + pl.off_ml);
    p.part_acc = reinterpret_cast<float *>(ws + pl.off_acc);
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const hipError_t e = d->head_dim == 512   ? launch_step<512>(p, shared, st)
                         : d->head_dim == 256 ? launch_step<256>(p, shared, st)
                                              : launch_step<128>(p, shared, st);
    return e == hipSuccess ? ESDA_OK : fail(ESDA_ERR_HIP, std::string("esda_tree_decode launch: ") + hipGetErrorString(e));
}

}  // extern "C"
