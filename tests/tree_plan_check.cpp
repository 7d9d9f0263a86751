// Checks esda_tree_plan.h on the host: over random batches, the pieces of every sequence cover its keys
// once and in order, none is empty, they start at whole blocks, and there are no more of them than the
// host's bound.  Prints "ok" or what failed.
#include <cstdio>
#include <cstdlib>
#include <random>

#include "esda_tree_plan.h"

using namespace esda_tree_plan;

int main() {
    std::mt19937 rng(1);
    auto below = [&](long long n) { return (int) (((unsigned long long) rng() << 31 | rng()) % (unsigned long long) n); };
    for (int turn = 0; turn < 200000; ++turn) {
        const int B = 1 + below(turn % 3 ? 40 : 256), share = B + below(turn % 2 ? 600 : 8), least = 1 + below(9);
        const bool even = turn % 5 != 0;
        const int most = turn % 7 ? share : 1 + below(5);
        static int keys[256];
        int sum = 0;
        for (int b = 0; b < B; ++b) {
            const int kind = below(10);
            keys[b] = kind == 0 ? 0 : kind == 1 ? 2147483391 : kind < 5 ? below(2000) : below(200000);
            sum += blocks_of(keys[b]);
        }
        if (sum < 0) return std::printf("the batch's blocks pass 2^31\n"), 1;
        int chunk = 1 + below(300);
        for (int t = 0; even && t <= kTries; ++t) {
            chunk = chunk_of(sum, share, B, least, t);
            long long n = 0;
            for (int b = 0; b < B; ++b) n += pieces_of(blocks_of(keys[b]), chunk, most);
            if (n <= share) break;
            if (t == kTries) return std::printf("%lld pieces in the last try, share %d, batch %d\n", n, share, B), 1;
        }
        long long all = 0;
        for (int b = 0; b < B; ++b) {
            const int count = pieces_of(blocks_of(keys[b]), chunk, most);
            if (count < 1 || count > most) return std::printf("count %d of %d\n", count, most), 1;
            all += count;
            int at = 0;
            for (int i = 0; i < count; ++i) {
                int j0, j1;
                piece_keys(i, count, chunk, keys[b], &j0, &j1);
                if (j0 != at || j1 < j0 || j0 % kBlock || (keys[b] > 0 && j1 == j0))
                    return std::printf("keys %d chunk %d: piece %d of %d is %d .. %d behind %d\n", keys[b], chunk, i, count, j0, j1, at), 1;
                at = j1;
            }
            if (at != keys[b]) return std::printf("keys %d: %d covered\n", keys[b], at), 1;
        }
        if (even && all > share) return std::printf("%lld pieces, share %d, batch %d\n", all, share, B), 1;
    }
    std::printf("ok\n");
}
