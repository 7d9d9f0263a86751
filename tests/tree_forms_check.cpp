// tree_forms_check.cpp -- the form of esda_tree_decode (apertura_amd/csrc/esda_tree_forms.h) for descriptions read
// from standard input, one per line: "batch nodes Hq Hkv D shared window room split_rows" (room: rows of
// a sequence's table or linear cache).  Prints, per line, "run" or "tile", the query rows of a workgroup, its waves
// and "one" piece or "split".  Built and run by tests/test_tree_forms.py with g++.
#include "esda_tree_forms.h"

#include <cstdio>

int main() {
    esda_tree_desc d{};
    long long room = 0;
    int n = 0;
    while (std::scanf("%d %d %d %d %d %d %d %lld %d", &d.batch, &d.nodes, &d.num_q_heads, &d.num_kv_heads, &d.head_dim, &d.kv_shared,
                      &d.window, &room, &d.split_rows) == 9) {
        esda_prefill_plan::TreeParams p{};
        p.B = d.batch;
        p.Hkv = d.num_kv_heads;
        p.G = d.num_q_heads / d.num_kv_heads;
        p.Sq = d.nodes;
        p.window = d.window;
        const long long most = room + p.Sq;
        esda_tree_forms::choose(&d, p.window > 0 ? std::min(most, (long long) p.window + p.Sq + esda_tree_forms::kStageKeys) : most, &p);
        const bool run = p.run_groups > 0;
        std::printf("%s %d %d %s\n", run ? "run" : "tile", run ? 16 * p.run_groups : 16 * p.qb * (p.kh ? p.nw / 2 : p.nw), run ? 4 : p.nw,
                    p.splits == 1 ? "one" : "split");
        ++n;
    }
    return n == 0;
}
