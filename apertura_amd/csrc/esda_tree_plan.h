// esda_tree_plan.h -- how the keys of a step of drafted tokens are split over workgroups.  The lengths
// are known on the device only, so every workgroup works its share out from them; the host fixes how
// many pieces a kv head's keys make at most.  Lengths count in blocks of 32 rows.  Host and device;
// tests/tree_plan_check.cpp compiles it with g++.
#pragma once

#include "esda_plan.h"

namespace esda_tree_plan {

constexpr int kBlock = 32;
constexpr int kMaxBlocks = 1 << 22;  // a sequence counts as at most this many: the batch's sum stays below 2^31

ESDA_HD int blocks_of(int keys) {
    const int n = (int) (((long long) keys + kBlock - 1) / kBlock);
    return n < kMaxBlocks ? n : kMaxBlocks;
}

// Blocks of a piece, none shorter than `least`, when the batch's `sum` blocks are to make at most `share`
// pieces a kv head (share >= B sequences, each of which rounds up).  Tries 0 .. kTries, the first of which
// whose pieces are that few is taken; the last one's always are.
constexpr int kTries = 4;
ESDA_HD int chunk_of(int sum, int share, int B, int least, int t) {
    const unsigned n = (unsigned) (share - (int) ((long long) (B == 1 ? 0 : B) * t / kTries));
    const int even = n ? (int) (((unsigned) sum + n - 1u) / n) : kMaxBlocks;
    return even > least ? even : least;
}

// Pieces of `chunk` blocks that a sequence of n makes; at most `most`.
ESDA_HD int pieces_of(int n, int chunk, int most) {
    const int count = (int) (((unsigned) n + (unsigned) chunk - 1u) / (unsigned) chunk);
    return count < 1 ? 1 : count > most ? most : count;
}

// Keys [j0, j1) of piece i of `count` of a sequence of `keys` (the last takes what is left).
ESDA_HD void piece_keys(int i, int count, int chunk, int keys, int *j0, int *j1) {
    const long long a = (long long) i * chunk * kBlock, b = a + (long long) chunk * kBlock;
    *j0 = a < keys ? (int) a : keys;
    *j1 = i == count - 1 || b > keys ? keys : (int) b;
}

}  // namespace esda_tree_plan
