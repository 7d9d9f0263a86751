// esda_views.h -- whether the tensors of a call share memory, for the entry points whose outputs may
// not overlap their inputs.  Host code; tests/views_check.cpp compiles it with g++ and compares it with
// the elements themselves.
#pragma once

#include <cstdint>
#include <utility>

namespace esda_views {

// Rows of `width` 2-byte elements at ptr + i st[0] + j st[1], i < n[0], j < n[1] (strides >= 0).
struct View {
    uintptr_t ptr;
    long long n[2], st[2], width;
    // elements from the first to the last
    __int128 extent() const { return (__int128) (n[0] - 1) * st[0] + (__int128) (n[1] - 1) * st[1] + width; }
};

// Apart in memory as a whole.
inline bool apart(const View &a, const View &b) {
    return a.ptr >= b.ptr + 2 * b.extent() || b.ptr >= a.ptr + 2 * a.extent();
}

// Side by side in each period of a common stride: the q and the k part of a packed row, or of a packed
// head.
inline bool side_by_side(const View &a, const View &b) {
    for (int i = 0; i < 2; ++i)
        for (int j = 0; j < 2; ++j) {
            const long long s = a.st[i];
            if (s <= 0 || s != b.st[j]) continue;
            const __int128 wa = (__int128) (a.n[1 - i] - 1) * a.st[1 - i] + a.width;
            const __int128 wb = (__int128) (b.n[1 - j] - 1) * b.st[1 - j] + b.width;
            const long long bytes = (long long) ((__int128) b.ptr - (__int128) a.ptr);
            if (bytes % 2) continue;
            long long delta = bytes / 2 % s;
            if (delta < 0) delta += s;
            if (delta >= wa && delta + wb <= s) return true;
        }
    return false;
}

// Whether two views share no element.  Views that interleave in another way count as sharing, except
// where one is a few blocks (kv heads) that each keep clear of the other.
inline bool disjoint(const View &a, const View &b, int depth = 2) {
    if (apart(a, b) || side_by_side(a, b)) return true;
    constexpr int kBlocks = 64;
    for (int turn = 0; turn < 2 && depth > 0; ++turn) {
        const View &x = turn ? b : a, &y = turn ? a : b;
        const int o = x.n[0] > 1 && (x.n[1] <= 1 || x.st[0] >= x.st[1]) ? 0 : 1;  // the wider stride
        if (x.n[o] <= 1 || x.n[o] > kBlocks) continue;
        bool clear = true;
        for (long long i = 0; i < x.n[o] && clear; ++i) {
            View block = x;
            block.n[o] = 1;
            block.ptr += 2 * (uintptr_t) (i * x.st[o]);
            clear = disjoint(block, y, depth - 1);
        }
        if (clear) return true;
    }
    return false;
}

// Rows of one view that overlap one another.
inline bool overlaps_itself(const View &v) {
    long long n[2] = {v.n[0], v.n[1]}, st[2] = {v.st[0], v.st[1]};
    if (st[0] > st[1]) {
        std::swap(n[0], n[1]);
        std::swap(st[0], st[1]);
    }
    if (n[0] > 1 && st[0] < v.width) return true;
    return n[1] > 1 && (__int128) st[1] < (__int128) (n[0] - 1) * st[0] + v.width;
}

}  // namespace esda_views
