// esda_page_view.h -- where the rows of a cache in pages lie, and what a description of one must
// satisfy: for esda_pages.hip, esda_tree.hip and their kernels.  The checks are host code.
#pragma once

#include <algorithm>
#include <cstdint>

#include "esda_pages.h"

namespace esda_page_view {

constexpr int kMaxPages = 1 << 22, kMaxPageRows = 4096, kMaxSlots = 1 << 20, kMaxTable = 1 << 20;
constexpr int kMaxPlanes = 4096;

// Blocks of `block` elements at i st[0] + j st[1] + k st[2], i < n[0] .., that do not overlap, and end
// below 2^60.  (Ordered by stride, each step is at least as wide as what lies within it.)
inline bool blocks_apart(const long long (&count)[3], const long long (&stride)[3], long long block) {
    int order[3] = {0, 1, 2};
    std::sort(order, order + 3, [&](int a, int b) { return stride[a] < stride[b]; });
    __int128 width = block;
    for (int i : order) {
        if (count[i] <= 1) continue;
        if (stride[i] < width) return false;
        width += (__int128) (count[i] - 1) * stride[i];
    }
    return width < (__int128) 1 << 60;
}

// Blocks of `block` elements at i stride[0] + j stride[1] + k stride[2] from `at` on, i < count[0] ..
struct Blocks {
    const void *at;
    long long count[3], stride[3], block;
    // Elements from the first to the last of all, along the dims of `dims` (bits) alone.
    __int128 extent(unsigned dims) const {
        __int128 n = block;
        for (int i = 0; i < 3; ++i)
            if (dims >> i & 1) n += (__int128) (count[i] - 1) * stride[i];
        return n;
    }
};

// Whether the blocks of a and those of b, which start d elements behind a's, can be shown to have no element in
// common.  By the widest stride: of its steps only those matter that bring the rest of the two together, a
// few at most where each lies within a step; then the rest in the same way.
inline bool blocks_apart_from(const Blocks &a, unsigned of_a, const Blocks &b, unsigned of_b, __int128 d) {
    if (d >= a.extent(of_a) || -d >= b.extent(of_b)) return true;
    long long S = 0;
    auto widest = [&](const Blocks &x, unsigned of) {
        for (int i = 0; i < 3; ++i)
            if (of >> i & 1 && x.count[i] > 1) S = std::max(S, x.stride[i]);
    };
    widest(a, of_a);
    widest(b, of_b);
    if (S == 0) return false;
    auto without = [&](const Blocks &x, unsigned of, long long &steps) {  // .. the dim of stride S
        steps = 0;
        for (int i = 0; i < 3; ++i)
            if (of >> i & 1 && x.count[i] > 1 && x.stride[i] == S) {
                steps = x.count[i] - 1;
                return of & ~(1u << i);
            }
        return of;
    };
    long long back, on;
    of_a = without(a, of_a, back);
    of_b = without(b, of_b, on);
    auto floor_div = [](__int128 x, long long y) { return x / y - (x % y < 0); };
    // d + k S between -extent(b) and extent(a)
    const __int128 first = std::max<__int128>(-back, floor_div(-b.extent(of_b) - d, S) + 1);
    const __int128 last = std::min<__int128>(on, floor_div(a.extent(of_a) - 1 - d, S));
    if (last - first > 4) return false;
    for (__int128 k = first; k <= last; ++k)
        if (!blocks_apart_from(a, of_a, b, of_b, d + k * S)) return false;
    return true;
}
inline bool apart(const Blocks &a, const Blocks &b) {  // (both 16-byte aligned)
    return blocks_apart_from(a, 7, b, 7, ((__int128) reinterpret_cast<uintptr_t>(b.at) - (__int128) reinterpret_cast<uintptr_t>(a.at)) / 2);
}

inline bool power_of_two(int x) { return x > 0 && (x & (x - 1)) == 0; }
inline bool whole16(long long a) { return a >= 0 && a % 8 == 0; }

// Whether the na elements from a on meet the nb from b on.
inline bool meet(const void *a, long long na, const void *b, long long nb) {
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + 2 * (uintptr_t) nb && y < x + 2 * (uintptr_t) na;
}

inline Blocks blocks_of(const esda_pool &p, int num_pages, int page_rows) {
    return {p.data, {p.planes, num_pages, p.num_kv_heads}, {p.plane_stride, p.page_stride, p.head_stride}, (long long) page_rows * p.head_dim};
}
inline Blocks bytes_at(const void *at, size_t bytes) { return {at, {1, 1, 1}, {0, 0, 0}, (long long) (bytes + 1) / 2}; }

// What is wrong with a pool of pages of page_rows rows, or null.
inline const char *check_pool(const esda_pool &p, int num_pages, int page_rows) {
    if (!p.data || (reinterpret_cast<uintptr_t>(p.data) & 15u)) return "a pool must be 16-byte aligned device memory";
    if (p.planes <= 0 || p.planes > kMaxPlanes || p.num_kv_heads <= 0 || p.num_kv_heads > kMaxPlanes)
        return "a pool has 1 .. 4096 planes and kv heads";
    if (p.head_dim != 128 && p.head_dim != 256 && p.head_dim != 512) return "head_dim must be 128, 256 or 512";
    if (!whole16(p.plane_stride) || !whole16(p.page_stride) || !whole16(p.head_stride))
        return "strides must be non-negative multiples of 8";
    if (!blocks_apart({p.planes, num_pages, p.num_kv_heads}, {p.plane_stride, p.page_stride, p.head_stride},
                      (long long) page_rows * p.head_dim))
        return "the pages of a pool overlap";
    return nullptr;
}

// What is wrong with the pages of a table, or null.
inline const char *check_table(int num_pages, int page_rows, int slots, int max_pages, long long table_stride) {
    if (num_pages <= 0 || num_pages > kMaxPages) return "num_pages must be 1 .. 2^22";
    if (!power_of_two(page_rows) || page_rows < 16 || page_rows > kMaxPageRows)
        return "page_rows must be a power of two, 16 .. 4096";
    if (slots <= 0 || slots > kMaxSlots) return "slots must be 1 .. 2^20";
    if (max_pages <= 0 || max_pages > kMaxTable || (long long) max_pages * page_rows >= 1LL << 31)
        return "max_pages must be 1 .. 2^20 and hold fewer than 2^31 rows";
    if (table_stride < max_pages || table_stride > 1LL << 40) return "table_stride must be at least max_pages";
    return nullptr;
}

}  // namespace esda_page_view
