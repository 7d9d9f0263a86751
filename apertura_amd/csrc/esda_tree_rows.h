// esda_tree_rows.h -- the rows that a step of drafted tokens attends (gfx950): the nodes' paths, the
// place of a row in its page, and a query row done again where a value is not finite.  For esda_tree.hip
// and the tiles of esda_prefill_kernel.h.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "esda_device.h"
#include "esda_prefill_plan.h"
#include "esda_tree_plan.h"

namespace {

using esda_prefill_plan::TreeParams;

__device__ __forceinline__ bool tree_page(const TreeParams &p, int id) { return (unsigned) id < (unsigned) p.N; }

// A workgroup's piece: keys [j0, j1) of sequence b and kv head kvh, counted from row `first` on; the
// sequence's pieces are base .. base + pieces - 1 of the batch's.
struct TreeUnit {
    int there, b, kvh, len, first, keys, piece, pieces, base, j0, j1;
};

// Keys of a sequence of len rows, and the first row that any node sees (a multiple of 32); 0 keys where
// the length is none (every node's row is counted, whether it is one or not).
__device__ __forceinline__ int tree_keys(const TreeParams &p, int len, int &first) {
    const long long most = p.linear ? (long long) p.cap : (long long) p.P << p.shift;
    first = p.window > 0 ? max(0, len - p.window + 1) & ~31 : 0;
    return len >= 0 && len <= most ? len - first + p.Sq : 0;
}

// tree_unit where sequences are several: piece g of the batch's, sequences 64 k + lane for k < K by each
// lane.  (Every workgroup does this before its first load: up to 64 sequences by themselves.)
template <int K>
__device__ __forceinline__ TreeUnit tree_unit_of(const TreeParams &p, int g, int lane, TreeUnit t) {
    using namespace esda_tree_plan;
    int len[K], n[K], first, sum = 0;
#pragma unroll
    for (int k = 0; k < K; ++k) {
        const int s = 64 * k + lane, n = p.length[min(s, p.B - 1)];
        len[k] = s < p.B ? n : -1;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
        n[k] = blocks_of(tree_keys(p, len[k], first));
        sum += n[k];
    }
    int chunk = p.forced;
    if (!p.forced) {
        auto total = [](int x) { return __builtin_amdgcn_readlane(wave_sums(x), 63); };
        sum = total(sum);
#pragma unroll 1
        for (int i = 0; i <= kTries; ++i) {
            chunk = chunk_of(sum, p.share, p.B, p.least, i);
            int count = 0;
#pragma unroll
            for (int k = 0; k < K; ++k)
                if (64 * k + lane < p.B) count += pieces_of(n[k], chunk, p.splits);
            if (total(count) <= p.share) break;
        }
    }
    int before = 0;  // pieces of the sequences of the rounds before
#pragma unroll
    for (int k = 0; k < K; ++k) {
        if (64 * k >= p.B) break;
        const bool mine = 64 * k + lane < p.B;
        const int count = mine ? pieces_of(n[k], chunk, p.splits) : 0;
        const int upto = before + wave_sums(count), from = upto - count;
        const unsigned long long who = __builtin_amdgcn_ballot_w64(from <= g && g < upto);
        if (who) {
            const int l = __builtin_ctzll(who);
            t.there = 1;
            t.b = 64 * k + l;
            t.base = __builtin_amdgcn_readlane(from, l);
            t.len = __builtin_amdgcn_readlane(len[k], l);
            t.pieces = __builtin_amdgcn_readlane(count, l);
            t.keys = tree_keys(p, t.len, t.first);
            t.piece = g - t.base;
            piece_keys(t.piece, t.pieces, chunk, t.keys, &t.j0, &t.j1);
            return t;
        }
        before = __builtin_amdgcn_readlane(upto, 63);
    }
    return t;
}

// Unit u as a wave: the pieces that the batch's lengths make, and which of them it is.
__device__ __forceinline__ TreeUnit tree_unit(const TreeParams &p, unsigned u, int lane) {
    using namespace esda_tree_plan;
    TreeUnit t;
    t.kvh = (int) (u % (unsigned) p.Hkv);
    const int g = (int) (u / (unsigned) p.Hkv);  // piece of the batch
    t.there = 0;
    if (p.B == 1) {
        t.b = t.base = 0;
        t.len = uniform(p.length[0]);
        t.keys = tree_keys(p, t.len, t.first);
        const int n = blocks_of(t.keys);
        const int chunk = p.forced ? p.forced : chunk_of(n, p.share, 1, p.least, 0);
        t.pieces = pieces_of(n, chunk, p.splits);
        t.piece = g;
        t.there = g < t.pieces;
        piece_keys(g, t.pieces, chunk, t.keys, &t.j0, &t.j1);
        return t;
    }
    return p.B <= 64 ? tree_unit_of<1>(p, g, lane, t) : tree_unit_of<4>(p, g, lane, t);
}

// Sequence b's nodes as a wave: lane i < 64 gets node i's path (bit j: node j is above it, or is it; 0: no
// node), and whether the sequence is one: its length and its nodes' rows lie in its cache.  A node's path
// doubles in length each round: what is above the node that is above it.
__device__ __forceinline__ bool tree_paths(const TreeParams &p, int b, int len, int lane, unsigned long long &path) {
    bool node = lane < p.Sq;
    path = node ? (2ull << lane) - 1 : 0ull;
    const long long most = p.linear ? (long long) p.cap : (long long) p.P << p.shift;
    const long long row = (long long) len + lane;
    const bool within = len >= 0 && row < most;
    int id = 0;
    if (!p.linear) id = p.table[b * p.table_stride + (node && within ? row >> p.shift : 0)];
    if (p.parent) {
        int above = p.parent[(size_t) b * p.Sq + min(lane, p.Sq - 1)];
        if (!node || above < -1 || above >= lane) above = -2;  // on no node
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
    const bool ok = len >= 0 && len <= most && (!node || (within && (p.linear || tree_page(p, id))));
    return __builtin_amdgcn_ballot_w64(!ok) == 0ull;
}

// The first partial of a unit, and what the merge is told of its sequence (by one thread of them all).
__device__ __forceinline__ long long tree_part(const TreeParams &p, const TreeUnit &t) {
    return ((long long) (t.base + t.piece) * p.Hkv + t.kvh) * (p.Sq * p.G);
}
__device__ __forceinline__ void tree_report(const TreeParams &p, const TreeUnit &t, bool ok) {
    p.views[2 * t.b] = t.base;
    p.views[2 * t.b + 1] = ok ? t.pieces : 0;
    if (!ok) __hip_atomic_fetch_add(p.status, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The first entries of a single sequence's table, read beside its length (0.5 us of a step's 11).
__device__ __forceinline__ int tree_ids(const TreeParams &p, int lane) {
    return p.B == 1 && !p.linear ? p.table[min(lane, p.P - 1)] : -1;
}

// The rows of one (sequence, kv head) as esda_stream.h's runs take them.
template <int D, bool SH>
struct TreeRows {
    static constexpr bool kUnseen = true;
    uint16_t *k, *v;                // the kv head in page 0
    const uint16_t *k_new, *v_new;  // its rows of the nodes
    const int *table;               // of the sequence; null: page `page0` alone
    long long page_stride;
    int G, j0, j1;                  // query rows; keys (esda_stream.h)
    int len, first, new_stride, N, P, shift, page0;
    int ids, of;                    // lane i: page 64 of + i of the table
    int page;                       // of the last stage
    int low;                        // committed rows before it are seen by no node
    unsigned long long none;        // bit i: node i is none, or past the last (said after the first loads)

    // ids0: the first 64 entries of the table (tree_ids), or anything
    __device__ __forceinline__ TreeRows(const TreeParams &p, const TreeUnit &w, int ids0) {
        const int b = w.b, kvh = w.kvh;
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
        G = page = 0;
        low = p.window > 0 ? max(0, w.len + 1 - p.window) : 0;
        none = 0ull;
        j0 = w.j0;
        j1 = w.j1;
        ids = p.linear ? page0 : (unsigned) ids0 < (unsigned) N ? ids0 : -1;  // (linear: every row in entry 0)
        of = p.linear || p.B == 1 ? 0 : -1;
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
    // Those of rows jst .. jst + 15 that no node sees, but for the rows of a page that is none.
    __device__ __forceinline__ unsigned unseen(int jst) const {
        const int row = first + jst, i = row - len;  // (i > -16: some row is a node's)
        unsigned rows = row < low ? (1u << min(low - row, 16)) - 1u : 0u;
        if (i > -16) rows |= i >= 64 ? 0xffffu : i >= 0 ? (unsigned) ~(~none >> i) : (unsigned) (none << -i);
        return rows & 0xffffu;
    }
    __device__ __forceinline__ void begun() const {}
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
        // (rounded to bf16, as the weights of the products are)
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

// .. and into out, row `row`, or its partial, number `at`.
template <int D>
__device__ __forceinline__ void tree_row_store(const TreeParams &p, long long row, long long at, int lane, float m, float l,
                                               const float (&o)[D / 64]) {
    constexpr int DPL = D / 64;
    if (p.splits == 1) {
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int e = 0; e < DPL; ++e) p.out[row * D + lane * DPL + e] = __builtin_bit_cast(uint16_t, (__bf16) (o[e] * inv));
        return;
    }
#pragma unroll
    for (int e = 0; e < DPL; ++e) p.part_acc[at * D + lane * DPL + e] = o[e];
    if (lane == 0) *reinterpret_cast<f32x2 *>(p.part_ml + 2 * at) = f32x2{m, l};
}

}  // namespace
