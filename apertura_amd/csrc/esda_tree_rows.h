// esda_tree_rows.h -- the rows that a step of drafted tokens attends (gfx950): the nodes' paths, the
// place of a row in its page, and a query row done again where a value is not finite.  For esda_tree.hip
// and the tiles of esda_prefill_kernel.h.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "esda_device.h"
#include "esda_prefill_plan.h"

namespace {

using esda_prefill_plan::TreeParams;

// A sequence's keys: `total` of them from row `first` on (0: it has no node; then it is done).
struct TreeView {
    int ok, len, nodes, first, total;
};

__device__ __forceinline__ bool tree_page(const TreeParams &p, int id) { return (unsigned) id < (unsigned) p.N; }

// Sequence b as a wave: lane i < 64 gets node i's path (bit j: node j is above it, or is it; 0: no node).
// A node's path doubles in length each round: what is above the node that is above it.
__device__ __forceinline__ TreeView tree_view(const TreeParams &p, int b, int lane, unsigned long long &path) {
    TreeView v;
    v.len = uniform(p.length[b]);
    bool node = lane < p.Sq;
    path = node ? (2ull << lane) - 1 : 0ull;
    if (p.parent) {
        int above = node ? p.parent[(size_t) b * p.Sq + lane] : -2;
        if (above < -1 || above >= lane) above = -2;  // on no node
        path = 1ull << lane;
#pragma unroll
        for (int i = 0; i < 6; ++i) {
            const int from = max(above, 0);
            const unsigned long long more = __shfl(path, from);
            const int next = __shfl(above, from);
            if (above >= 0) {
                path |= more;
                above = next;
            }
        }
        node = above == -1;
        if (!node) path = 0ull;
    }
    const unsigned long long there = __builtin_amdgcn_ballot_w64(node);
    v.nodes = there ? 64 - __builtin_clzll(there) : 0;
    bool ok = v.len >= 0 && (long long) v.len + v.nodes <= (p.linear ? (long long) p.cap : (long long) p.P << p.shift);
    if (ok && node && !p.linear) ok = tree_page(p, p.table[b * p.table_stride + ((v.len + lane) >> p.shift)]);
    v.ok = __builtin_amdgcn_ballot_w64(!ok) == 0ull;
    v.first = p.window > 0 ? max(0, v.len - p.window + 1) & ~31 : 0;
    v.total = v.nodes ? v.len + v.nodes - v.first : 0;
    return v;
}

// The rows of one (sequence, kv head) as esda_stream.h's runs take them.
template <int D, bool SH>
struct TreeRows {
    uint16_t *k, *v;                // the kv head in page 0
    const uint16_t *k_new, *v_new;  // its rows of the nodes
    const int *table;               // of the sequence; null: page `page0` alone
    long long page_stride;
    int G, j0, j1;                  // query rows; keys (esda_stream.h)
    int len, first, new_stride, N, P, shift, page0;
    int ids, of;                    // lane i: page 64 of + i of the table
    int page;                       // of the last stage

    __device__ __forceinline__ TreeRows(const TreeParams &p, const TreeView &w, int b, int kvh) {
        k = const_cast<uint16_t *>(p.k) + kvh * p.kv_hs;
        v = const_cast<uint16_t *>(p.v) + kvh * p.kv_hs;
        const size_t at = ((size_t) b * p.Sq * p.Hkv + kvh) * D;
        k_new = p.k_new + at;
        v_new = SH ? k_new : p.v_new + at;
        table = p.linear ? nullptr : p.table + b * p.table_stride;
        page_stride = p.page_stride;
        len = w.len;
        first = w.first;
        new_stride = p.Hkv * D;
        N = p.N;
        P = p.P;
        shift = p.shift;
        page0 = p.linear ? b : 0;
        G = j0 = j1 = page = 0;
        ids = page0;  // (linear: every row in entry 0)
        of = p.linear ? 0 : -1;
    }

    struct Stage {
        const uint16_t *k, *v;
        int end;
    };
    // The page of entry n (the same in every lane), 64 entries a load; -1 where it is none.
    __device__ __forceinline__ int page_of(int n) {
        const int block = uniform(n >> 6);
        if (__builtin_expect(block != of, 0)) {
            of = block;
            const int i = (block << 6) + (int) (threadIdx.x & 63);
            ids = table[min(i, P - 1)];  // (entries past the last are not asked for)
            if ((unsigned) ids >= (unsigned) N) ids = -1;
        }
        return __builtin_amdgcn_readlane(ids, n & 63);
    }
    // A stage's 16 rows lie in one page.  Of a page that is none no row has weight: page 0 is read for it.
    __device__ __forceinline__ bool dense(int jst, Stage &st) {
        const int row = first + jst;
        st.end = j1;
        page = 0;
        if (row < len) {
            page = page_of(row >> shift);
            if (page < 0) {
                page = 0;
                st.end = jst;
            }
        }
        const long long at = page * page_stride + (long long) (row & ((1 << shift) - 1)) * D;
        st.k = k + at;
        st.v = v + at;
        return row + 16 <= len && jst + 16 <= j1;
    }
    __device__ __forceinline__ void row(int j, const uint16_t *&kr, const uint16_t *&vr) const {
        const int r = first + j;
        const long long at = r < len ? page * page_stride + (long long) (r & ((1 << shift) - 1)) * D : (long long) (r - len) * new_stride;
        kr = (r < len ? k : k_new) + at;
        if constexpr (!SH) vr = (r < len ? v : v_new) + at;
    }
    __device__ __forceinline__ void appended(int, int) const {}
};

// The rows of the nodes among keys [j0, j1) into the cache, by the threads of a workgroup.
template <int D, bool SH>
__device__ __forceinline__ void append_nodes(const TreeRows<D, SH> &x, const unsigned long long *paths, int j0, int j1) {
    const int i0 = max(0, x.first + j0 - x.len), i1 = x.first + j1 - x.len;
    for (int t = threadIdx.x + i0 * (D / 8); t < i1 * (D / 8); t += blockDim.x) {
        const int i = t / (D / 8), c = t % (D / 8), row = x.len + i;
        if (paths[i] == 0ull) continue;
        const int page = x.table ? x.table[row >> x.shift] : x.page0;
        const long long to = page * x.page_stride + (long long) (row & ((1 << x.shift) - 1)) * D + 8 * c, from = (long long) i * x.new_stride + 8 * c;
        *reinterpret_cast<u32x4 *>(x.k + to) = *reinterpret_cast<const u32x4 *>(x.k_new + from);
        if constexpr (!SH) *reinterpret_cast<u32x4 *>(x.v + to) = *reinterpret_cast<const u32x4 *>(x.v_new + from);
    }
}

// One query row over the keys [j0, j1) that it sees and no others, as a wave: for rows whose O was not
// finite, since a value that is not meets a weight of 0 in the products (0 x inf is NaN).  The lanes take
// 64 keys for the scores, then the row's dims: store(m, l, o) with dims DPL lane on.  Rare.
template <int D, bool SH, class Store>
__device__ __forceinline__ void tree_row_again(const TreeRows<D, SH> &x, const uint16_t *qr, unsigned long long path, int lowest,
                                            int j0, int j1, float scale_log2e, Store &&store) {
    constexpr int DPL = D / 64;
    typedef uint16_t piece __attribute__((ext_vector_type(DPL)));
    const int lane = threadIdx.x & 63;
    float m = -INFINITY, l = 0.0f, o[DPL];
#pragma unroll
    for (int e = 0; e < DPL; ++e) o[e] = 0.0f;
    for (int jb = j0; jb < j1; jb += 64) {
        const int j = jb + lane, row = x.first + j;
        const uint16_t *kr = x.k, *vr = x.v;
        bool seen = false;
        if (j < j1) {
            long long at;
            if (row < x.len) {
                const int id = x.table ? x.table[row >> x.shift] : x.page0;
                seen = row >= lowest && (unsigned) id < (unsigned) x.N;
                at = (seen ? id : 0) * x.page_stride + (long long) (row & ((1 << x.shift) - 1)) * D;
            } else {
                seen = (path >> (row - x.len)) & 1;
                at = (long long) (row - x.len) * x.new_stride;
                kr = x.k_new;
                vr = x.v_new;
            }
            kr += at;
            vr += at;
        }
        unsigned long long todo = __builtin_amdgcn_ballot_w64(seen);
        if (todo == 0ull) continue;
        float s = 0.0f;
        if (seen) {
#pragma unroll 1
            for (int d = 0; d < D; d += 8) {
                const u32x4 kv = *reinterpret_cast<const u32x4 *>(kr + d), qv = *reinterpret_cast<const u32x4 *>(qr + d);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s = __builtin_fmaf(bf16_lo(qv[e]), bf16_lo(kv[e]), s);
                    s = __builtin_fmaf(bf16_hi(qv[e]), bf16_hi(kv[e]), s);
                }
            }
            s *= scale_log2e;
        }
        float top = seen ? s : -INFINITY;
#pragma unroll
        for (int i = 32; i >= 1; i >>= 1) top = fmaxf(top, __shfl_xor(top, i));
        const float mn = fmaxf(m, top), corr = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - mn);
        const float w = seen ? (float) (__bf16) __builtin_amdgcn_exp2f(s - (mn == -INFINITY ? 0.0f : mn)) : 0.0f;
        float sum = w;
#pragma unroll
        for (int i = 32; i >= 1; i >>= 1) sum += __shfl_xor(sum, i);
        m = mn;
        l = l * corr + sum;
#pragma unroll
        for (int e = 0; e < DPL; ++e) o[e] *= corr;
        const uint64_t at = (uint64_t) (uintptr_t) (SH ? kr : vr);
        while (todo) {
            const int b = __builtin_ctzll(todo);
            todo &= todo - 1;
            const float wb = __shfl(w, b);
            const uint16_t *const of = (const uint16_t *) (uintptr_t) __shfl((unsigned long long) at, b);
            const piece pv = *reinterpret_cast<const piece *>(of + lane * DPL);
#pragma unroll
            for (int e = 0; e < DPL; ++e) o[e] = __builtin_fmaf(wb, __builtin_bit_cast(float, (unsigned) pv[e] << 16), o[e]);
        }
    }
    store(m, l, o);
}

// .. and its place in out or among the partials.
template <int D>
__device__ __forceinline__ void tree_row_store(const TreeParams &p, int split, long long row, int lane, float m, float l,
                                               const float (&o)[D / 64]) {
    constexpr int DPL = D / 64;
    if (p.splits == 1) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int e = 0; e < DPL; ++e) p.out[row * D + lane * DPL + e] = __builtin_bit_cast(uint16_t, (__bf16) (o[e] * inv));
        return;
    }
    const long long at = (long long) split * p.B * p.Sq * p.Hq + row;
#pragma unroll
    for (int e = 0; e < DPL; ++e) p.part_acc[at * D + lane * DPL + e] = o[e];
    if (lane == 0) *reinterpret_cast<f32x2 *>(p.part_ml + 2 * at) = f32x2{m, l};
}

}  // namespace
