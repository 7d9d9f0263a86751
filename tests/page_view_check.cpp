// Checks apart() of esda_page_view.h on the host against the elements themselves: random blocks, one set
// beside, between or over the other.  What is apart has no element in common; what has none is found
// apart where both sets have the same strides, or one's are whole steps of the other's.  Prints "ok" or what failed.
#include <algorithm>
#include <cstdio>
#include <random>
#include <vector>

#include "esda_page_view.h"

using namespace esda_page_view;

static std::vector<long long> elements(const Blocks &b, long long at) {
    std::vector<long long> all;
    for (int i = 0; i < b.count[0]; ++i)
        for (int j = 0; j < b.count[1]; ++j)
            for (int k = 0; k < b.count[2]; ++k)
                for (int e = 0; e < b.block; ++e) all.push_back(at + i * b.stride[0] + j * b.stride[1] + k * b.stride[2] + e);
    std::sort(all.begin(), all.end());
    return all;
}

int main() {
    std::mt19937 rng(3);
    auto below = [&](int n) { return (int) (rng() % (unsigned) n); };
    long long found = 0, lost = 0, met = 0;
    static char memory[1 << 22];
    for (int turn = 0; turn < 200000; ++turn) {
        Blocks x[2];
        int order[3] = {0, 1, 2};
        std::shuffle(order, order + 3, rng);
        const bool alike = turn % 3 != 0;  // the same strides, with room for both sets
        for (int s = 0; s < 2; ++s) {
            if (s == 1 && alike) {
                x[1] = x[0];
                for (long long &c : x[1].count) c = turn % 2 ? c : 1 + below((int) c);
                x[1].block = 1 + below((int) x[0].block);
                break;
            }
            x[s].block = 1 + below(4);
            long long width = x[s].block + below(6);
            if (s == 0 || below(2)) std::shuffle(order, order + 3, rng);
            for (int i : order) {
                x[s].count[i] = 1 + below(4);
                x[s].stride[i] = width;
                width = width * x[s].count[i] + below(3) * (1 + below((int) width));
            }
        }
        const long long base = 1 << 20, size = (long long) x[0].extent(7), d = below((int) (2 * size + 4)) - size - 2;
        x[0].at = memory + 2 * base;
        x[1].at = memory + 2 * (base + d);
        const std::vector<long long> a = elements(x[0], 0), b = elements(x[1], d);
        std::vector<long long> both;
        std::set_intersection(a.begin(), a.end(), b.begin(), b.end(), std::back_inserter(both));
        const bool says = apart(x[0], x[1]);
        if (says != apart(x[1], x[0])) return std::printf("apart() goes by the order\n"), 1;
        if (says && !both.empty()) return std::printf("turn %d: %zu elements in common\n", turn, both.size()), 1;
        if (!says && both.empty()) {
            if (alike) return std::printf("turn %d: not found apart\n", turn), 1;
            ++lost;
        }
        found += says;
        met += !both.empty();
    }
    if (found < 20000 || met < 20000) return std::printf("%lld apart, %lld met\n", found, met), 1;
    std::printf("ok\n");
    std::fprintf(stderr, "%lld apart, %lld met, %lld not shown\n", found, met, lost);
}
