// esda_tree.hip -- the step of drafted tokens over a cache in pages, or a linear one, for MI355X
// (gfx950).  The C ABI is include/esda_tree.h.
//
//   out_i = sum_j 2^(s_ij - m_i) v_j / sum_j 2^(s_ij - m_i),  s_ij = scale log2 e q_i.k_j,
// over the committed rows within node i's window and the nodes on its path.  A path is 64 bits, bit j for
// node j; a wave works them out with a node to a lane, doubling the paths' length in each of six rounds,
// and a node's depth is the number of its bits.  Only stages that hold nodes, the window's edge or a page
// that is none look at them; the others are plain attention.  Rows that no node sees (of nodes that are none,
// before the window, of such a page) may hold anything: they are zeros in LDS.
//
// A launch of pieces (one kv head, one sequence, a share of its keys) and one that merges them.  Few query
// rows a kv head take runs (tree_run_kernel), bound by memory: 32 sequences of 1,024 .. 8,192 rows of 128
// dims, K and V of 8 heads in 16-row pages, 608 MB read in 102 us (6.0 TB/s; a read of a large buffer
// reaches 7.2), 8 of 5 nodes each over 16 heads of 256 dims, 831 MB, 132 (6.3).  More take query tiles
// (prefill_kernel with TreeParams), bound by the matrix instructions and the softmax in turn: 2 x 63 nodes
// over 16,384 and 15,347 rows of 4 heads of 512 dims, K = V, 131 GFLOP in 146 us with the merge, called over
// and over (0.90 PFLOP/s; esda_prefill's tiles over the same rows, linear, take 1 .. 5% less), the matrix pipes
// busy for 0.46 of the tiles' cycles.  One token over 1,000 rows is two dependent launches, 8.2 and 3.5 us
// each by itself, 11.0 together: the length and the table's first entries, the rows, the waves' sum.

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
#include "esda_prefill_kernel.h"
#include "esda_tree.h"
#include "esda_tree_forms.h"
#include "esda_tree_rows.h"
#include "esda_tree_tiles.h"

namespace {

// A run's rows (esda_tree_rows.h) with what is to be done once its first loads are under way, which says
// which nodes are none.
template <int D, bool SH, class Begin>
struct BegunRows : TreeRows<D, SH> {
    Begin &begin;
    __device__ __forceinline__ BegunRows(const TreeParams &p, const TreeUnit &t, int ids, Begin &f) : TreeRows<D, SH>(p, t, ids), begin(f) {}
    __device__ __forceinline__ void begun() { this->none = begin(); }
};

// 16 NG query rows of a (sequence, kv head) over one piece of its keys, in a run (esda_stream.h): four waves
// that stream 16-row stages of their own, each row read once for all 16 NG query rows.  The page of a stage
// comes from a register that holds the next 64 entries of the table, a lane each.  Tried and not kept: two
// stages of a wave under way at once and the entries by DMA (token of 32 sequences 104.0 -> 105.5 us), shares
// that go on from one sequence to the next (104.0 -> 102.9, but 8 sequences of 5 nodes 135 -> 138 and one
// token 11.0 -> 12.3), q's loads before the nodes' paths (no difference).
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
    const int ids = tree_ids(p, lane);
    const TreeUnit t = tree_unit(p, unit, lane);
    if (!t.there) return;
    const bool reports = t.piece == 0 && t.kvh == 0 && r0 == 0 && threadIdx.x == 0;
    if (t.keys == 0) {  // no length: skipped
        if (reports) tree_report(p, t, false);
        return;
    }
    const int rows = p.Sq * p.G;
    const size_t head = ((size_t) t.b * p.Sq * p.Hq + (size_t) t.kvh * p.G);  // of q and out, in rows
    auto at = [&](int r) { return head + (size_t) (r / p.G) * p.Hq + r % p.G; };
    unsigned long long sees[NG];
    int lowest[NG];
    bool ok = false;
    auto begin = [&]() {  // beside the first stage's loads; the workgroup meets again before its rows are written
        unsigned long long path;
        ok = tree_paths(p, t.b, t.len, lane, path);
        if (wave == 0) paths[lane] = path;
        for (int e = threadIdx.x; e < 16 * NG; e += 256) odd[e] = 0;
        if (threadIdx.x == 0) any_odd = 0;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const int r = min(r0 + 16 * g + li, rows - 1);
            sees[g] = __shfl(path, r / p.G);
            lowest[g] = p.window > 0 ? t.len + __popcll(sees[g]) - p.window : 0;
        }
        if (reports) tree_report(p, t, ok);
        return __builtin_amdgcn_ballot_w64(path == 0ull);  // the nodes that are none
    };
    BegunRows<D, SH, decltype(begin)> x(p, t, ids, begin);
    x.G = min(rows - r0, 16 * NG);
    const int all_see = p.window > 0 ? t.len + p.Sq - p.window : 0;  // committed rows from it on: every node
    auto score = [&](f32x4 &s, int jst, int end, int g) {
        s *= p.scale_log2e;
        const int row = t.first + jst;
        if (row >= all_see && row + 16 <= t.len && jst + 16 <= end) return;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int j = jst + 4 * lg + e, r = t.first + j;
            const bool seen = r < t.len ? r >= lowest[g] : ((sees[g] >> ((r - t.len) & 63)) & 1) != 0;
            if (j >= end || !seen) s[e] = -INFINITY;
        }
    };
    const size_t part = (size_t) tree_part(p, t);
    auto finish = [&](int r, int d, f32x4 o, float m, float l) {  // dims d .. d + 3 of query row r
        if (paths[r / p.G] == 0ull) {  // no node: nothing seen (its q may be anything, and m infinite)
            o = 0.0f;
            m = -INFINITY;
            l = 0.0f;
        }
        if (p.splits == 1) {
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            bf16x4 y;
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = (__bf16) (o[e] * inv);
            if (ok) *reinterpret_cast<bf16x4 *>(p.out + at(r) * D + d) = y;
        } else {
            Own::store(p.part_acc, p.part_ml, part + r, d, o, m, l);
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
    if (!ok) return;
    if (r0 == 0) append_nodes<D, SH>(x, paths, x.j0, x.j1);
    ESDA_WAIT_VM(0);  // the rows as written above, before they are written again
    lds_barrier();
    if (__builtin_expect(any_odd != 0, 0)) {
        for (int h = wave; h < x.G; h += 4) {
            if (!odd[h]) continue;
            const unsigned long long mine = paths[(r0 + h) / p.G];
            tree_row_again<D, SH>(x, p.q + at(r0 + h) * D, mine, p.window > 0 ? t.len + __popcll(mine) - p.window : 0, x.j0, x.j1,
                                  p.scale_log2e, [&](float m, float l, const float(&o)[D / 64]) {
                                      tree_row_store<D>(p, at(r0 + h), part + r0 + h, lane, m, l, o);
                                  });
        }
    }
}

// out = sum_s acc_s 2^(m_s - M) / sum_s l_s 2^(m_s - M) over the pieces of a row's sequence; 0 where it
// saw no key.  A workgroup takes 256 / GR lanes of 4 dims, and its GR groups of threads the pieces in
// turn, U of them in flight, each against its own maximum; the groups meet in LDS.  Few rows take many
// groups (launch_step), which cover the loads' latency; many rows are bound by the partials' bytes (4,032
// rows of 512 dims, 67 MB in 12.4 us, 5.4 TB/s; eight of a lane in flight were no faster).
template <int D, int GR>
__global__ __launch_bounds__(256) void tree_merge_kernel(TreeParams p) {
    constexpr int U = 4, LANES = 256 / GR;
    __shared__ f32x4 part[GR > 1 ? GR : 1][LANES];
    __shared__ f32x2 gml[GR > 1 ? GR : 1][LANES];
    const int lane = threadIdx.x % LANES, g = threadIdx.x / LANES;
    const long long x = (long long) blockIdx.x * LANES + lane;
    const int row = (int) (x / (D / 4)), d = (int) (x % (D / 4)) * 4;
    const bool there = row < p.B * p.Sq * p.Hq;
    const int i = (there ? row : 0) / p.Hq, h = (there ? row : 0) % p.Hq, b = i / p.Sq;
    const int base = p.views[2 * b], n = there ? p.views[2 * b + 1] : 0;  // 0: skipped, and left as it is
    const size_t first = ((size_t) base * p.Hkv + h / p.G) * (p.Sq * p.G) + (i - b * p.Sq) * p.G + h % p.G;
    const size_t step = (size_t) p.Hkv * p.Sq * p.G;
    float M = -INFINITY, den = 0.0f;
    f32x4 num = 0.0f;
    for (int j0 = g; j0 < n; j0 += GR * U) {
        f32x2 ml[U];
        f32x4 a[U];
        float top = M;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = j0 + GR * u;
            ml[u] = f32x2{-INFINITY, 0.0f};
            a[u] = 0.0f;
            if (j < n) {
                ml[u] = *reinterpret_cast<const f32x2 *>(p.part_ml + 2 * (first + j * step));
                a[u] = *reinterpret_cast<const f32x4 *>(p.part_acc + (first + j * step) * D + d);
            }
            top = fmaxf(top, ml[u][0]);
        }
        const float at = top == -INFINITY ? 0.0f : top;
        const float c = __builtin_amdgcn_exp2f(M - at);
        num *= c;
        den *= c;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float w = __builtin_amdgcn_exp2f(ml[u][0] - at);
            den = __builtin_fmaf(ml[u][1], w, den);
            num += a[u] * w;
        }
        M = top;
    }
    if constexpr (GR > 1) {
        part[g][lane] = num;
        gml[g][lane] = f32x2{M, den};
        __syncthreads();
        if (g != 0) return;
        float top = M;
#pragma unroll
        for (int u = 1; u < GR; ++u) top = fmaxf(top, gml[u][lane][0]);
        if (top == -INFINITY) top = 0.0f;
        num = 0.0f;
        den = 0.0f;
#pragma unroll
        for (int u = 0; u < GR; ++u) {
            const f32x2 ml = gml[u][lane];
            const float w = __builtin_amdgcn_exp2f(ml[0] - top);
            den = __builtin_fmaf(ml[1], w, den);
            num += part[u][lane] * w;
        }
    }
    if (n == 0) return;
    if (den == 0.0f) den = 1.0f;
    bf16x4 o;
#pragma unroll
    for (int e = 0; e < 4; ++e) o[e] = (__bf16) (num[e] / den);
    *reinterpret_cast<bf16x4 *>(p.out + (size_t) row * D + d) = o;
}

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
    if (d->max_pages != 0 && (long long) d->max_pages * d->page_rows > (1LL << 31) - 256) return "a table holds fewer than 2^31 - 256 rows";
    if (d->split_rows < 0 || d->split_rows % kStageKeys) return "split_rows must be a multiple of 32";
    if (!(d->scale > 0.0f) || !std::isfinite(d->scale)) return "scale must be positive and finite";
    if ((long long) d->batch * d->nodes * d->num_q_heads * (d->head_dim / 64) >= 1 << 24) return "too many query rows";
    return nullptr;
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
    const long long most = (p.linear ? p.cap : (long long) d->max_pages * d->page_rows) + p.Sq;  // keys of a sequence
    esda_tree_forms::choose(d, p.window > 0 ? std::min(most, (long long) p.window + p.Sq + kStageKeys) : most, &p);
    if (p.splits > 4096 || (long long) p.units * p.tiles >= INT_MAX / 512) return refuse("too many splits");
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    const size_t parts = p.splits > 1 ? (size_t) p.units * p.Sq * p.G : 0;
    p.part_nt = 4.0f * D * parts <= kPartNtBytes;
    pl->off_views = 256;
    pl->off_ml = pl->off_views + up((size_t) p.B * 8);
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
    if (p.run_groups) {
        const dim3 grid(p.units * p.row_groups), block(256);
        auto run = [&](auto ng) {
            constexpr int NG = decltype(ng)::value;
            if (shared) hipLaunchKernelGGL((tree_run_kernel<D, true, NG>), grid, block, 0, st, p);
            else hipLaunchKernelGGL((tree_run_kernel<D, false, NG>), grid, block, 0, st, p);
        };
        if (p.run_groups == 1) run(std::integral_constant<int, 1>{});
        if constexpr (D == 128) {
            if (p.run_groups == 2) run(std::integral_constant<int, 2>{});
        }
    } else {
        esda_detail::tree_tiles(p, D, st);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits == 1) return e;
    const long long lanes = (long long) p.B * p.Sq * p.Hq * (D / 4);
    auto merge = [&](auto gr) {
        constexpr int GR = decltype(gr)::value;
        hipLaunchKernelGGL((tree_merge_kernel<D, GR>), dim3((unsigned) ((lanes + 256 / GR - 1) / (256 / GR))), dim3(256), 0, st, p);
    };
    if (lanes <= 1 << 14) merge(std::integral_constant<int, 16>{});
    else if (lanes <= 1 << 16) merge(std::integral_constant<int, 4>{});
    else merge(std::integral_constant<int, 1>{});
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
    // What is written must not be what is read: rows of q are read again after rows of out are written, and
    // the new rows while they are written to the pages.
    struct Range {
        const void *at;
        long long n;
        bool meets(const Range &o) const { return esda_page_view::meet(at, n, o.at, o.n); }
    };
    const long long token = (long long) d->batch * d->nodes * d->head_dim;
    const long long extent = (d->num_pages - 1) * d->page_stride + (d->num_kv_heads - 1) * d->head_stride + (long long) d->page_rows * d->head_dim;
    const Range out{a->out, token * d->num_q_heads}, k_new{a->k_new, token * d->num_kv_heads},
        v_new{shared ? a->k_new : a->v_new, token * d->num_kv_heads}, k_pages{a->k_pages, extent}, v_pages{a->v_pages, extent};
    for (const Range &x : {Range{a->q, out.n}, k_new, v_new, k_pages, v_pages})
        if (out.meets(x)) return refuse("out must not overlap q, the new rows or the pages");
    for (const Range &x : {k_new, v_new})
        if (x.meets(k_pages) || x.meets(v_pages)) return refuse("the new rows must not overlap the pages");
    if (!shared) {
        auto plane = [&](const void *at) {
            return esda_page_view::Blocks{at, {1, d->num_pages, d->num_kv_heads}, {0, d->page_stride, d->head_stride}, (long long) d->page_rows * d->head_dim};
        };
        if (!esda_page_view::apart(plane(a->k_pages), plane(a->v_pages))) return refuse("k_pages and v_pages must not overlap");
    }
    if (!a->workspace || a->workspace_bytes < pl.bytes || !aligned(a->workspace, 16))
        return fail(ESDA_ERR_WORKSPACE, "esda_tree_decode: workspace missing or smaller than esda_tree_workspace_size");
    const Range workspace{a->workspace, (long long) pl.bytes / 2}, lists[] = {
        {a->length, 2LL * d->batch}, {a->parent, 2LL * d->batch * d->nodes}, {a->table, a->table ? 2 * ((d->batch - 1) * d->table_stride + d->max_pages) : 0}};
    for (const Range &x : {Range{a->q, out.n}, out, k_new, v_new, k_pages, v_pages, lists[0], lists[1], lists[2]})
        if (x.at && workspace.meets(x)) return refuse("the workspace must not overlap the tensors");
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
