// views_check.cpp -- esda_views.h's disjoint() and overlaps_itself() beside the elements themselves, for
// random small views.  disjoint() may call views that interleave oddly shared, never shared ones
// disjoint; packed rows, packed heads and separate buffers it has to tell apart.
#include "esda_views.h"

#include <cstdio>
#include <random>
#include <set>

using esda_views::View;

static std::multiset<long long> elements(const View &v) {
    std::multiset<long long> s;
    for (long long i = 0; i < v.n[0]; ++i)
        for (long long j = 0; j < v.n[1]; ++j)
            for (long long d = 0; d < v.width; ++d) s.insert((long long) v.ptr / 2 + i * v.st[0] + j * v.st[1] + d);
    return s;
}

int main() {
    std::mt19937 rng(7);
    auto pick = [&](int lo, int hi) { return (long long) std::uniform_int_distribution<int>(lo, hi)(rng); };
    int apart = 0, shared = 0, odd = 0;
    for (int t = 0; t < 200000; ++t) {
        View v[2];
        for (auto &x : v) x = View{(uintptr_t) (1000 + 2 * pick(0, 60)), {pick(1, 4), pick(1, 4)}, {pick(0, 24), pick(0, 24)}, pick(1, 4)};
        if (pick(0, 1)) v[1].st[0] = v[0].st[pick(0, 1)];
        const auto a = elements(v[0]), b = elements(v[1]);
        bool meet = false;
        for (long long e : a) meet = meet || b.count(e);
        const bool says = esda_views::disjoint(v[0], v[1]);
        if (says != esda_views::disjoint(v[1], v[0])) return std::printf("case %d: not symmetric\n", t), 1;
        if (says && meet) return std::printf("case %d: shared views called disjoint\n", t), 1;
        ++(meet ? shared : says ? apart : odd);
        const std::set<long long> once(a.begin(), a.end());
        if (once.size() != a.size() && !esda_views::overlaps_itself(v[0])) return std::printf("case %d: overlaps itself\n", t), 1;
    }
    // q, k, v and out of packed rows; heads side by side; kv heads of an arena with out between them
    const long long T = 100, D = 8, row = 10 * D;
    const View q{4096, {T, 4}, {row, D}, D}, k{4096 + 2 * 4 * D, {T, 2}, {row, D}, D}, out{4096 + 2 * 6 * D, {T, 4}, {row, D}, D};
    const View hq{4096, {4, T}, {2 * T * D, D}, D}, ho{4096 + 2 * T * D, {4, T}, {2 * T * D, D}, D};
    const View kv{4096, {3, 1}, {5000, 0}, T * D}, between{4096 + 2 * 1000, {T, 4}, {4 * D, D}, D};
    for (auto *p : {&k, &out})
        if (!esda_views::disjoint(q, *p)) return std::puts("packed rows"), 1;
    if (!esda_views::disjoint(hq, ho)) return std::puts("packed heads"), 1;
    if (!esda_views::disjoint(kv, between) || !esda_views::disjoint(between, kv)) return std::puts("between heads"), 1;
    // the far ends of the address range
    const View far{4096, {1LL << 30, 65536}, {1LL << 40, 1LL << 23}, 512};
    if (esda_views::disjoint(far, q)) return std::puts("far"), 1;
    std::printf("%d apart, %d shared, %d undecided\n", apart, shared, odd);
    return apart < 1000 || shared < 1000;
}
