// esda_tree_forms.h -- which kernel a step of drafted tokens takes, and into how many pieces its keys are
// split at most.  Host code; tests/tree_forms_check.cpp compiles it with g++.
#pragma once

#include <algorithm>
#include <climits>
#include <cmath>

#include "esda_prefill_plan.h"
#include "esda_tree.h"

namespace esda_tree_forms {

using esda_prefill_plan::kStageKeys;
using esda_prefill_plan::TreeParams;

// How the query rows of a kv head can be laid out: as tiles (nw > 0: a prefill form), or in runs of 16 ng
// rows.  slots: workgroups the GPU holds at once; stage: us of one for 32 keys.
struct Form {
    int qb, kh, nw, ng, slots;
    float stage;
    int rows() const { return ng ? 16 * ng : 16 * qb * (kh ? nw / 2 : nw); }
};
constexpr Form kRun128 = {0, 0, 0, 1, 512, 0.25f}, kRun128x2 = {0, 0, 0, 2, 512, 0.3f}, kTile128 = {2, 0, 4, 0, 512, 1.2f};
constexpr Form kRun256 = {0, 0, 0, 1, 256, 0.5f}, kTile256 = {1, 0, 8, 0, 256, 1.0f}, kTile256Half = {1, 1, 8, 0, 256, 0.8f};
constexpr Form kRun512 = {0, 0, 0, 1, 256, 0.8f}, kTile512 = {1, 0, 8, 0, 256, 1.6f}, kTile512Half = {1, 0, 4, 0, 256, 1.6f};

// The form of a step of `rows` query rows a kv head over caches with room for `room` bytes of keys and
// values (the host does not know how many are there).  Up to 16 rows a run reads every key once; more
// take a run's rows again for each 16, or fill a tile, which starts later.  Of 2,170 random steps (1 .. 64
// sequences and nodes, 32 .. 49,152 rows, a quarter to all of the room filled), times over the fastest
// form's, below 10 MB / below 100 / above:
//   D = 128  17 .. 32 rows   run 1.00 / 1.06 / 1.21   two blocks a run 1.15 / 1.03 / 1.00   tile 1.15 / 1.12 / 1.13
//            33 .. 64            1.00 / 1.07 / 1.40                    1.16 / 1.04 / 1.06        1.22 / 1.09 / 1.01
//            65 .. 256           1.05 / 1.27 / 1.8                     1.16 / 1.09 / 1.2         1.33 / 1.03 / 1.00
//            more                1.14 / 1.47                           1.10 / 1.21               1.21 / 1.00
//   D = 256  up to 16        run 1.01 / 1.00 / 1.00   tile of 64 rows 1.06 / 1.09 / 1.14    of 128 1.03 / 1.10 / 1.26
//            17 .. 64            1.05 / 1.07 / 1.30                   1.09 / 1.02 / 1.00           1.06 / 1.03 / 1.10
//            more                1.26 / 1.65 / 2.0                    1.06 / 1.03 / 1.09           1.18 / 1.07 / 1.00
//   D = 512  up to 16        run 1.00 / 1.00 / 1.00   tile of 64 rows 1.11 / 1.16 / 1.32
//            17 .. 32            1.03 / 1.00 / 1.02                   1.18 / 1.10 / 1.05   (K and V apart, tile of 128: 1.00, run 1.2)
//            33 .. 64            1.05 / 1.18 / 1.50                   1.23 / 1.03 / 1.00
//            65 .. 128           1.08 / 1.3  / 1.8                    1.17 / 1.02 / 1.25    of 128 1.31 / 1.05 / 1.00
//            more                1.1  / 1.7  / 2.3                    1.15 / 1.2  / 1.5            1.3  / 1.00 / 1.00;
// and a form whose workgroups do not fit the GPU at once, for `pairs` sequences and kv heads, gives way to
// one of more rows (12 sequences of 59 rows, 64 nodes, D = 128: 31.4 us in runs, 19.1 in tiles).
inline Form pick(int D, int rows, bool shared, float room, long long pairs) {
    const bool small = room <= 1e7f, large = room > 1e8f;
    auto fits = [&](const Form &f) { return pairs * ((rows + f.rows() - 1) / f.rows()) <= f.slots; };
    if (D == 128) {
        if (rows <= 16) return kRun128;
        if (small && rows <= 256 && fits(kRun128)) return kRun128;
        if (small && fits(kRun128x2)) return kRun128x2;
        return rows <= (large ? 32 : 64) ? kRun128x2 : kTile128;
    }
    if (D == 256) {
        if (rows <= 16) return kRun256;
        return rows <= 64 || (!large && fits(kTile256Half)) ? kTile256Half : kTile256;
    }
    if (rows <= 16 || (rows <= 32 && shared) || (small && rows <= 256 && fits(kRun512))) return kRun512;
    if (rows <= 64) return shared ? kTile512Half : kTile512;  // (launch_tiles' choice for one tile)
    return (small || (rows <= 128 && !large)) && fits(kTile512Half) ? kTile512Half : kTile512;
}

// The form of a step, and how many pieces its keys are to make (esda_tree_plan.h shares them out): at most
// as many workgroups as the GPU holds at once.  Fewer where the room for keys is little: k pieces of a full
// sequence take t / k, but a second launch (4 us) and k partials of every row, written and read back (at 4
// TB/s); then k = sqrt(t / what one partial of all rows takes), or a single piece.  (As many pieces as
// fit, whatever the room: 12 sequences of 39 rows, 64 nodes, D = 128, 32.8 us, with one each 19.7.)
inline void choose(const esda_tree_desc *d, long long most, TreeParams *p) {
    const int D = d->head_dim, rows = p->Sq * p->G;
    const bool shared = d->kv_shared != 0;
    const long long pairs = (long long) p->B * p->Hkv;
    const float room = (float) (most * pairs) * 2.0f * D * (shared ? 1 : 2);
    const Form x = pick(D, rows, shared, room, pairs);
    p->qb = x.qb;
    p->kh = x.kh;
    p->nw = x.nw;
    p->run_groups = x.ng;
    p->tiles = p->row_groups = (rows + x.rows() - 1) / x.rows();
    long long units;
    if (d->split_rows > 0) {
        p->forced = (int) std::min<long long>(d->split_rows / kStageKeys, (most + kStageKeys - 1) / kStageKeys);
        p->splits = (int) std::min<long long>((most + d->split_rows - 1) / d->split_rows, INT_MAX);
        p->share = 1;
        units = pairs * p->splits;
    } else {
        p->least = rows <= 64 ? 2 : rows <= 256 ? 4 : 8;
        const float t = (float) most / kStageKeys * x.stage, part = 5.0e-7f * 4 * D * (float) (pairs * rows);
        const float k = std::min((float) x.slots / (float) (pairs * p->tiles), std::sqrt(t / part));
        const bool split = k > 1.0f && t / k + 4.0f + part * k < t;
        p->share = split ? std::max(p->B + 1, (int) (k * p->B)) : p->B;
        p->splits = split ? p->share : 1;
        units = (long long) p->share * p->Hkv;
    }
    p->units = (int) std::min<long long>((units + 7) / 8 * 8, INT_MAX);
}

}  // namespace esda_tree_forms
