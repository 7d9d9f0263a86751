// esda_prefill_kernel.h -- the prefill attention kernel, its split merge and their launch
// (gfx950), for the sources that build entry points on them: esda_prefill.hip (causal and sliding
// masks), esda_scored_prefill.hip (capped and biased scores, document and prefix masks) and
// esda_prefix_tiles.hip (the rows of a decode batch over its shared prefix), esda_tree_tiles.hip (steps of
// many drafted tokens).  What the kernel does
// is described at the head of esda_prefill.hip.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>
#include <type_traits>

#include "esda_device.h"
#include "esda_plan.h"
#include "esda_prefill_plan.h"
#include "esda_stream.h"
#include "esda_tree_rows.h"

namespace {

using namespace esda_prefill_plan;

constexpr int kBlk = 1056;                 // LDS bytes per DMA block: 1 KB + 32 B pad
constexpr int kRingBudget = 136 * 1024;    // LDS bytes for the K / V ring
// K / V stream loads without the non-temporal hint: the tiles of one kv head read the
// same keys, and the L2 keeping them for the next tile was measured 2-12% faster.
constexpr bool kStreamNT = false;
typedef int i32x4 __attribute__((ext_vector_type(4)));

// LDS ring geometry for head dim D: a 16-key half stage is NI DMA blocks of kBlk bytes,
// block b holding keys b + NI*q (q < 512/D) at +2D*q; a stage is the K halves then the V
// halves.  Both the 128-bit row reads (QK A operand) and the transpose reads (PV A
// operand) are bank-conflict-free in this layout (the decode kernel's measured layout).
// Eight waves per workgroup (two per SIMD) and QB 16-query blocks per wave.  O^T takes
// QB * D / 16 accumulator registers per lane beside Q^T's QB * D / 8 and 8 QB of scores,
// within the 256 registers of two waves per SIMD: QB = 1 at D = 512 (two blocks do not
// fit without spills), 1 or 2 at D = 256 (kTilings256), 2 at D = 128.  (Measured: at D = 256,
// four waves of two blocks -- one wave per SIMD -- ran 6% slower than eight waves of one
// block, and forming the next stage's scores during this stage's softmax -- a second set
// of score registers, forcing one block per wave at D = 256 -- was 5-20% slower.)
//
// KH (stage halves, D = 256 with one block per wave): waves w and w + 4 own the same query
// block and take the even and the odd stages of the tile's keys, over a ring of four
// stages per tensor (132 KB), and fold their (m, l, O^T) together through LDS at the end.
// A tile is then 64 query rows, so a chunk whose 128-row tiles would leave CUs idle gets
// twice the tiles before any key split -- no fp32 partials and no merge launch -- while
// each wave's work per stage and the barriers per stage stay those of the plain kernel.
constexpr int kWaves = 8;
#ifndef PV_DEPTH
#define PV_DEPTH 4
#endif
constexpr int kPairSpin = 1 << 20;  // PS: polls of the partner's flag before a wave gives up

// A run of the prefix step (esda_prefix.h) on a workgroup of NW waves, for up to 16 NG query rows: by
// waves that stream stages of their own, as many in flight as the prefill kernel's LDS holds; short
// runs of 512 dims, whose waves' O^T would take longer to sum than the run, in groups of stages.  A
// step of 128 such runs over one K = V buffer, streamed / in groups, us: 64 rows 15.5 / 12.4, 128 16.5 /
// 13.7, 256 19.8 / 18.5, 384 22.5 / 22.3, 512 25.4 / 26.6, 1024 35.1 / 41.5.  (256 dims: 64 rows 9.1 /
// 9.0, 256 14.4 / 15.0, 1024 30.7 / 35.3.)
template <int D, bool SH, int NW, int NG = 1>
struct OwnRows {
    static constexpr int kStage = (SH ? 1 : 2) * 2 * D * 16;  // bytes of a 16-row stage
    static constexpr int SLOTS = 2 * kStage * NW > 128 * 1024 ? 1 : 2;
    static constexpr bool GROUPS = D == 512, ONLY = GROUPS && NW > 4;  // (eight waves' registers do not hold the streaming form)
    static constexpr int kGroupRows = 384;  // longest run in groups
    static constexpr int kGroupBytes = esda_stream::GroupLayout<D, SH>::BYTES;
    static constexpr int kStreamBytes = esda_stream::Layout<D, SH, NW, SLOTS, NG>::BYTES;
    static constexpr int BYTES = ONLY || (GROUPS && kGroupBytes > kStreamBytes) ? kGroupBytes : kStreamBytes;
    using Run = esda_stream::RunOf<D, SH>;
    template <class Rows, class Query, class Score, class Put>
    static __device__ __forceinline__ void attend(unsigned char *lds, Rows &x, Query &&query, Score &&score, Put &&put) {
        if constexpr (GROUPS) {
            static_assert(NG == 1, "16 query rows a group");
            if (ONLY || x.j1 - x.j0 <= kGroupRows) {
                esda_stream::attend_groups<D, SH, NW>(lds, x, query, score, put);
                return;
            }
        }
        if constexpr (!ONLY) esda_stream::attend_run<D, SH, NW, SLOTS, NG>(lds, x, query, score, put);
    }

    static __device__ __forceinline__ void store(float *acc, float *ml, size_t at, int d, const f32x4 &o, float M, float T) {
        __builtin_nontemporal_store(o, reinterpret_cast<f32x4 *>(acc + at * D + d));
        if (d == 0) *reinterpret_cast<f32x2 *>(ml + 2 * at) = f32x2{M, T};
    }
    // own workgroup w: split w % own_splits of pair w / own_splits
    static __device__ __forceinline__ void run(const PrefixParams &p, unsigned w, unsigned char *lds) {
        const int split = (int) (w % (unsigned) p.own_splits), pair = (int) (w / (unsigned) p.own_splits);
        const int b = pair / p.Hkv, kvh = pair % p.Hkv;
        const esda_plan::SeqView sv = esda_plan::seq_view(p.pos[b], p.own_base, p.own_cap, 0, 0);
        if (!sv.ok) {
            if (split == 0 && kvh == 0 && threadIdx.x == 0) atomicAdd(p.status, 1);
            return;
        }
        Run x;
        if (!esda_plan::grid_split(split, p.own_splits, p.own_chunk, sv.nvis, &x.j0, &x.j1)) return;
        const size_t head = (size_t) b * p.own_seq_stride + (size_t) kvh * p.own_head_stride;
        x.k = p.own_k + head;
        x.v = p.own_v + head;
        x.k_new = p.k_new + (size_t) pair * D;
        x.v_new = SH ? x.k_new : p.v_new + (size_t) pair * D;
        x.G = p.G;
        x.nvis = sv.nvis;
        x.first = sv.first;
        x.cap = p.own_cap;
        x.newrow = sv.newrow;
        const uint16_t *const q = p.q + (size_t) b * p.q_rs + (size_t) kvh * p.G * D;
        const size_t slot = ((size_t) pair * p.own_splits + split) * p.G;
        attend(
            lds, x, [&](int h) { return q + (size_t) h * D; }, [&](float s, int) { return s * p.scale_log2e; },
            [&](int h, int d, const f32x4 &o, float M, float T) { store(p.own_acc, p.own_ml, slot + h, d, o, M, T); });
    }
    // Prefix workgroup w: 16 NG of the B * G query rows of a kv head over run_keys keys.  The row groups
    // of the same keys are 8 workgroups apart: on one XCD, whose L2 hands the second what the first read.
    static __device__ __forceinline__ void run_prefix(const PrefixParams &p, unsigned w, unsigned char *lds) {
        const unsigned i = w >> 3, pair = i / (unsigned) p.row_groups * 8 + (w & 7);
        const int r0 = (int) (i % (unsigned) p.row_groups) * 16 * NG;
        const int kvh = (int) (pair % (unsigned) p.Hkv), split = (int) (pair / (unsigned) p.Hkv);
        if (split >= p.splits) return;
        Run x{};
        x.j0 = split * p.run_keys;
        x.j1 = min(p.Sk, x.j0 + p.run_keys);
        x.k = const_cast<uint16_t *>(p.k) + (size_t) kvh * p.kv_hs;
        x.v = const_cast<uint16_t *>(p.v) + (size_t) kvh * p.kv_hs;
        x.G = min(p.Sq * p.G - r0, 16 * NG);
        x.nvis = p.Sk + 1;  // (no appended row)
        x.cap = p.Sk;
        const size_t rows = (size_t) p.Sq * p.Hq, slot = (size_t) split * rows;
        auto row = [&](int h) { return (size_t) ((r0 + h) / p.G) * p.Hq + kvh * p.G + (r0 + h) % p.G; };
        attend(
            lds, x, [&](int h) { return p.q + row(h) * D; }, [&](float s, int) { return s * p.scale_log2e; },
            [&](int h, int d, const f32x4 &o, float M, float T) { store(p.part_acc, p.part_ml, slot + row(h), d, o, M, T); });
    }
};

// Prefix and own rows in runs, for batches of few query rows a kv head (esda_prefix.hip's forms):
// bound by memory where the prefix is long (2 sequences behind 32,768 tokens, 4 kv heads of one
// 512-dim stream, 135 MB in 32 us), else by the latency of a few stages.  Every wave holds 16 NG query
// rows and its own keys, so that a K or V value is read from LDS once for those, where the tiles'
// waves each hold 16 rows and read every key.  The registers bound NG (O^T and Q^T take 6 D NG / 16
// of 512 a lane: NG D = 1024 spills, and 32 rows of 512 dims in groups of stages took 42 us where two
// workgroups of 16 take 40); more rows are row_groups workgroups of the same keys.
template <int D, bool SH, int NG>
__global__ __launch_bounds__(256, 1) void prefix_run_kernel(PrefixParams p) {
    __shared__ __attribute__((aligned(16))) unsigned char lds[OwnRows<D, SH, 4, NG>::BYTES];
    if (blockIdx.x >= p.own_groups) OwnRows<D, SH, 4, NG>::run_prefix(p, blockIdx.x - p.own_groups, lds);
    else OwnRows<D, SH, 4>::run(p, blockIdx.x, lds);
}

template <int D, int NSL, int NT = 2>
struct PRing {
    static constexpr int NI = D / 32;                 // DMA blocks per 16-key half
    static constexpr int HB = NI * kBlk;              // one half stage of one tensor
    static constexpr int BYTES = 2 * NT * NSL * HB;   // NSL K stages, then NSL V stages (NT = 2)
    static constexpr int CPR = D / 8;                 // 16-byte chunks per row
    static_assert(BYTES <= kRingBudget, "the K / V slots must fit the LDS budget");
    __host__ __device__ static constexpr int off(int r) { return (r % NI) * kBlk + (r / NI) * 2 * D; }
};

// SH: V is the K buffer (attention_k_eq_v): one tensor streams, and PV reads V^T from the
// stage's K slot.  S2 (with SH, in the LDS the second tensor leaves free): every wave computes
// two stages per iteration, so the workgroup meets at one barrier per 64 keys.
//
// PS (pair split, one block per wave): waves w and w^1 (on different SIMDs) each score and
// softmax their own query block over the whole head dim, as above, but accumulate O^T for
// both blocks of the pair over half of the head dim each (wave w: dims D/2 (w & 1) on).
// Each V^T tile read from LDS then feeds two MFMAs, which halves the kernel's transpose
// reads for an exchange of P^T (1 KB per wave and stage) through LDS: the wave writes its
// P^T (and, after a rescale, its factors), then a flag, and reads its partner's once the
// partner's flag shows the stage.  The buffers alternate by stage parity: a wave rewrites a
// parity only after reading its partner's next flag, which the partner writes after reading
// this stage's P^T.  Used by the K = V kernel at D = 512 (p512gs 436 -> 422 us on one box);
// with separate K and V -- one stage per barrier -- it measured 1-3% slower and is not used.
//
// P = ScoredParams (esda_scored.h): scores are capped and lose slope * distance, a prefix opens
// keys ahead of a query, a row that sees nothing gives 0, and a value that is not finite reaches
// only the rows that see its key.  Bound as the plain form, by the MFMAs and the softmax in turn: a
// cap adds 6 .. 9% at D = 256 and 512 (2048 queries 92 -> 100 us, 143 -> 151) and 25% at D = 128,
// whose stages have half or a quarter of the products to a score (4096 queries 150 -> 187).  Wide caps
// have kernels of their own (P = WideScoredParams, WideDocParams): as a branch in these, their form cost
// the others up to 8% (4096 local queries at D = 256, 153 -> 166, no cap).  Beside a narrow cap it takes
// 201 -> 240 us (4096 queries, D = 128), 93 -> 116 (2048 local, 256), 476 -> 535 (512 over 16K, 512).
// P = DocParams: document ids (equal, not negative) close the other keys, too.  The waves first
// read the range of ids of every 32-key stage: stages that hold no id of the tile's range are never
// loaded, those that hold nothing but the tile's one id need no mask, and the ids of the others
// come with their keys by DMA.
// P = TreeParams (esda_tree.h): a unit of workgroups is one piece of the keys of one sequence and kv head
// (tree_unit), its query rows the nodes' heads; a wave's DMAs fill one half of a stage, 16 rows of one page.
// Stages that hold nodes, the window's edge or a page that is none are masked by the nodes' paths.
template <int D, int QB, bool KH = false, bool SH = false, bool S2 = false, bool PS = false, int NW = kWaves,
          class P = PrefillParams>
// (D == 128 on four waves: two workgroups per CU)
__global__ __launch_bounds__(64 * NW, D == 128 && NW == 4 ? 2 : 1) void prefill_kernel(P p) {
    constexpr bool DOCS = std::is_base_of<DocParams, P>::value;
    constexpr bool SCORED = std::is_base_of<ScoredParams, P>::value;
    constexpr bool WIDE = std::is_same<P, WideScoredParams>::value || std::is_same<P, WideDocParams>::value;
    constexpr bool PARTS = std::is_same<P, PrefixParams>::value;  // a partial from every split, also one
    constexpr bool TREE = std::is_same<P, TreeParams>::value;
    constexpr bool ODD = SCORED || TREE;  // rows whose O^T is not finite are done again
    static_assert(!S2 || !KH, "two stages per iteration: all waves on both");
    static_assert(!PS || (QB == 1 && !KH), "pair split: one block per wave, every wave on every stage");
    constexpr int NQW = KH ? NW / 2 : NW;  // waves with distinct query blocks
    constexpr int NSL = KH || S2 ? 4 : 2;          // ring stages per tensor
    constexpr int SPI = KH || S2 ? 2 : 1;          // stages per iteration (KH: one per wave group)
    using R = PRing<D, NSL, SH ? 1 : 2>;
    constexpr int QT = 16 * QB * NQW;   // query rows per tile
    constexpr int KS = D / 32;          // QK k-steps
    constexpr int DT = D / 16;          // PV dim tiles
    constexpr int NB = PS ? 2 : QB;     // O^T blocks per wave
    constexpr int DW = PS ? DT / 2 : DT;  // O^T dim tiles per wave
    constexpr int kLds = PARTS && OwnRows<D, SH, NW>::BYTES > R::BYTES ? OwnRows<D, SH, NW>::BYTES : R::BYTES;
    __shared__ __attribute__((aligned(16))) unsigned char ring[kLds];
    if constexpr (PARTS) {
        if (blockIdx.x >= p.tile_groups) {
            OwnRows<D, SH, NW>::run(p, blockIdx.x - p.tile_groups, ring);
            return;
        }
    }
    // PS exchange, per stage parity: each wave's P^T (16 B per lane) and rescale factors
    // (4 B per lane), then one flag per wave; after both parities, each wave's row sums.
    constexpr int XP = 64 * 16 + 64 * 4;
    constexpr int XPAR = NW * XP + NW * 4;
    __shared__ __attribute__((aligned(16))) unsigned char xch[PS ? 2 * XPAR + NW * 16 * 4 : 16];
    __shared__ __attribute__((aligned(16))) int dids[DOCS ? NSL : 1][kStageKeys];  // the slots' document ids
    // of each 64 stages, which to compute and which of them without a mask; those past the last
    // of kDocWindows (131,072 keys of a split) are computed with one
    constexpr int kDocWindows = 64;
    __shared__ unsigned long long paths[TREE ? 64 : 1];  // the nodes'
    __shared__ unsigned char odd_row[ODD ? QT : 1];  // tile rows whose O^T is not finite
    __shared__ int any_odd;
    // the tile rows' positions, slopes (log2 units) and documents, read where a stage needs them:
    // held in registers they cost the stages reloads of spilled ones, whose waits wait for the DMAs
    __shared__ int row_pos[SCORED ? QT : 1], row_doc[DOCS ? QT : 1];
    __shared__ float row_slope[SCORED ? QT : 1];
    __shared__ unsigned long long live_of[DOCS ? kDocWindows : 1], pure_of[DOCS ? kDocWindows : 1];

    // (scored: said to be scalar, which frees the registers that the score's form needs)
    const int lane = threadIdx.x & 63, wave = ODD ? uniform(threadIdx.x >> 6) : threadIdx.x >> 6;
    const int li = lane & 15, lg = lane >> 4;
    // Query-block wave and stage parity (both constant for the plain kernel, whose code
    // does not change: a wave-dependent parity there measured 3% slower).
    const int wq = KH ? wave % NQW : wave, kh = KH ? wave / NQW : 0;
    const int hd = PS ? (wave & 1) : 0;  // PS: this wave's half of the head dim
    // Workgroup -> (tile, kv head, split): consecutive workgroups go to consecutive XCDs
    // (dispatch is round-robin over the 8), so the (kv head, split) pair is the fastest
    // index and the workgroups on one XCD share one K / V stream in its L2; tiles run
    // heaviest (latest) first.
    // (TREE: units of one piece of keys and one kv head.)
    int combos = p.Hkv * p.splits;
    if constexpr (TREE) combos = p.units;
    const int wg = (int) blockIdx.x;
    const int tile = p.tiles - 1 - wg / combos;
    TreeUnit tu{};
    int tree_first = -1;
    if constexpr (TREE) {
        tree_first = tree_ids(p, lane);
        tu = tree_unit(p, (unsigned) (wg % combos), lane);
        if (!tu.there) return;
    }
    const int kvh = TREE ? tu.kvh : (wg % combos) % p.Hkv, split = TREE ? tu.piece : (wg % combos) / p.Hkv;
    const long long nrows = (long long) p.Sq * p.Hq;
    const long long row0 = TREE ? tu.b * nrows : 0;  // the sequence's first row of q and out
    const uint16_t *const qb0 = TREE ? p.q + row0 * D : p.q;
    uint16_t *const out0 = TREE ? p.out + row0 * D : p.out;

    int j0, j1;
    if constexpr (TREE) {
        j0 = tu.j0;
        j1 = tu.j1;
        if (tu.keys == 0) {  // no length: skipped
            if (kvh == 0 && tile == 0 && threadIdx.x == 0) tree_report(p, tu, false);
            return;
        }
    } else {
        int tj0, tj1;
        tile_keys(p, tile, QT, tj0, tj1);
        j0 = min(tj1, tj0 + split * p.kps);
        j1 = min(tj1, j0 + p.kps);
    }

    // This lane's query row in block qb: tile row wq*16*QB + 16qb + li, global row gr
    // (position gr / G, head kvh*G + gr % G); rows past the end repeat the last row and
    // are not written.
    const long long nq = (long long) p.Sq * p.G;
    auto qrow = [&](int qb) -> long long {
        const long long gr = (long long) tile * QT + wq * 16 * QB + qb * 16 + li;
        return gr < nq ? gr : nq - 1;
    };
    auto qvalid = [&](int qb) { return (long long) tile * QT + wq * 16 * QB + qb * 16 + li < nq; };

    if (!TREE && j0 >= j1) {  // an empty split: no keys for this tile; the merge skips it
        if (p.splits > 1 && lg == 0 && kh == 0) {
#pragma unroll
            for (int qb = 0; qb < QB; ++qb)
                if (qvalid(qb)) {
                    const long long gr = qrow(qb);
                    const unsigned qi = position_of(gr, p.G);
                    const long long row = (long long) qi * p.Hq + kvh * p.G + (int) ((unsigned) gr - qi * p.G);
                    *reinterpret_cast<f32x2 *>(p.part_ml + 2 * ((long long) split * nrows + row)) =
                        f32x2{-INFINITY, 0.0f};
                }
        }
        if constexpr (SCORED) {  // unsplit: a tile whose rows see nothing is 0
            if (p.splits == 1) {
                for (int r = wave; r < QT; r += NW) {
                    const long long gr = (long long) tile * QT + r;
                    if (gr >= nq) break;
                    const unsigned qi = position_of(gr, p.G);
                    uint16_t *o = p.out + (size_t) qi * p.o_rs + (size_t) (kvh * p.G + (int) ((unsigned) gr - qi * p.G)) * p.o_hs;
                    for (int d = 4 * lane; d < D; d += 256) *reinterpret_cast<u32x2 *>(o + d) = u32x2{0u, 0u};
                }
            }
        }
        return;
    }

    // Q^T B operands: lane (li, lg) holds dims 32ks + 8lg .. +8 of its query row.
    bf16x8 qreg[QB][KS];
    int qabs[QB];  // absolute position of this lane's query in block qb
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        const long long gr = qrow(qb);
        const unsigned qi = position_of(gr, p.G);
        const uint16_t *qr = qb0 + (size_t) (kvh * p.G + (int) ((unsigned) gr - qi * p.G)) * p.q_hs +
                             (size_t) qi * p.q_rs + lg * 8;
        if constexpr (!ODD) qabs[qb] = p.q_pos0 + (int) qi;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            u32x4 w = qvalid(qb) ? *reinterpret_cast<const u32x4 *>(qr + ks * 32) : u32x4{0u, 0u, 0u, 0u};
            qreg[qb][ks] = __builtin_bit_cast(bf16x8, w);
        }
    }

    // LDS: NSL K slots then NSL V slots, each a 32-key stage (two 16-key halves).  Stage
    // s's K sits in K slot s % NSL and its V in V slot s % NSL.  Iteration i computes the
    // SPI stages SPI*i .. (one per wave group); after its barrier the stages of iteration
    // i+1 replace those of iteration i-1 (every wave is done with them) and land while
    // iteration i computes.
    //
    // DMA: K instruction t of this wave (ii = wave*KPW + t of the stage's 2 NI) fills block
    // b = ii % NI of half hh = ii / NI; lane l reads chunk l % CPR of stage row
    // r = 16hh + b + NI*(l / CPR).  V likewise.  Interior stages add the lane's byte offset
    // to a wave-uniform base; the last, partial stage clamps each row to the range.
    constexpr int KPW = 2 * R::NI / NW;  // DMA instructions per wave per tensor per stage
    static_assert(KPW * NW == 2 * R::NI, "whole DMA blocks per wave");
    const uint16_t *kvb = p.k + (size_t) kvh * p.kv_hs;
    const uint16_t *vvb = p.v + (size_t) kvh * p.kv_hs;
    const int nst = (j1 - j0 + kStageKeys - 1) / kStageKeys;
    unsigned voff[KPW];
    int vrow[KPW], ldso[KPW];
#pragma unroll
    for (int t = 0; t < KPW; ++t) {
        const int ii = wave * KPW + t, hh = ii / R::NI, b = ii % R::NI;
        vrow[t] = 16 * hh + b + R::NI * (lane / R::CPR);
        voff[t] = (unsigned) ((vrow[t] * D + (lane % R::CPR) * 8) * 2);
        ldso[t] = hh * R::HB + b * kBlk;
    }
    static_assert((NSL & (NSL - 1)) == 0, "stage slots: a power of two");
    auto kslot = [&](int s) { return ring + (s & (NSL - 1)) * 2 * R::HB; };
    auto vslot = [&](int s) { return SH ? kslot(s) : ring + 2 * NSL * R::HB + (s & (NSL - 1)) * 2 * R::HB; };
    // TREE: this wave's DMAs fill one half of a stage, 16 rows of one page
    struct None {};
    std::conditional_t<TREE, TreeRows<D, SH>, None> tr = [&] {
        if constexpr (TREE) {
            return TreeRows<D, SH>(p, tu, tree_first);
        } else {
            return None{};
        }
    }();
    auto issue = [&](const uint16_t *head, int s, unsigned char *slot) {
        const int jb = j0 + s * kStageKeys;
        if constexpr (TREE) {
            const int half = 16 * (wave / (NW / 2));
            typename TreeRows<D, SH>::Stage rows;
            if (tr.dense(jb + half, rows)) {
                const uint16_t *base = (head == vvb && !SH ? rows.v : rows.k) - half * D;
#pragma unroll
                for (int t = 0; t < KPW; ++t) lds_dma16_s<kStreamNT>(base, voff[t], lds_addr(slot) + ldso[t]);
            } else {
#pragma unroll
                for (int t = 0; t < KPW; ++t) {
                    const uint16_t *kr, *vr;
                    tr.row(min(jb + vrow[t], j1 - 1), kr, vr);  // rows past the range repeat the last node's
                    if constexpr (!SH) kr = head == vvb ? vr : kr;
                    lds_dma16<kStreamNT>(kr + (lane % R::CPR) * 8, lds_addr(slot) + ldso[t]);
                }
            }
            return;
        }
        if (jb + kStageKeys <= j1) {
            const uint16_t *base = head + (size_t) jb * D;
#pragma unroll
            for (int t = 0; t < KPW; ++t) lds_dma16_s<kStreamNT>(base, voff[t], lds_addr(slot) + ldso[t]);
        } else {
#pragma unroll
            for (int t = 0; t < KPW; ++t) {
                const int j = min(jb + vrow[t], j1 - 1);  // rows past the range repeat the last key
                lds_dma16<kStreamNT>(head + (size_t) j * D + (lane % R::CPR) * 8, lds_addr(slot) + ldso[t]);
            }
        }
    };

    if constexpr (SCORED) {
        for (int r = threadIdx.x; r < QT; r += 64 * NW) {
            const long long gr = min((long long) tile * QT + r, nq - 1);
            const unsigned qi = position_of(gr, p.G);
            odd_row[r] = 0;
            row_pos[r] = p.q_pos0 + (int) qi;
            row_slope[r] = p.slopes ? p.slopes[kvh * p.G + (int) ((unsigned) gr - qi * p.G)] * kLog2e : 0.0f;
            if constexpr (DOCS) row_doc[r] = p.q_doc[qi];
        }
        if (threadIdx.x == 0) any_odd = 0;
        lds_barrier();
    }
    const int qk_off = R::off(li) + lg * 16;                    // + 64 ks (+ HB: keys 16..31)
    const int tr_off = R::off(4 * lg + li / 4) + (li % 4) * 8;  // + 32 dt (+ HB)
    // V^T of dims 16 dt .. of a stage's slot (PS: from its half), the PV A operand
    auto vtile_of = [&](const unsigned char *vbh, int dt) {
        const short4v a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) short4v *) (vbh + tr_off + 32 * dt));
        const short4v a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
            (__attribute__((address_space(3))) short4v *) (vbh + R::HB + tr_off + 32 * dt));
        const short8v a8 = {a0[0], a0[1], a0[2], a0[3], a1[0], a1[1], a1[2], a1[3]};
        return __builtin_bit_cast(bf16x8, a8);
    };

    float m[QB], l[QB];
    f32x4 acc[NB][DW];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        m[qb] = -INFINITY;
        l[qb] = 0.0f;
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb)
#pragma unroll
        for (int dt = 0; dt < DW; ++dt) acc[nb][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    // PS flags start at 0 (stage s shows as 2 (s + 1), plus 1 after a rescale); the loop's
    // first barrier orders these stores before any wave reads them.
    // (Flags are read and written through LDS pointers: a generic volatile access would be
    // a flat one, whose wait also drains the ring's DMAs.)
    using lds_flag = __attribute__((address_space(3))) volatile unsigned;
    if constexpr (PS) {
        if (lane < 2) *(lds_flag *) (xch + lane * XPAR + NW * XP + wave * 4) = 0u;
    }
    // Positions of the tile's first and last rows (the host keeps positions below 2^31).
    const int qa_min = TREE ? 0 : p.q_pos0 + (int) position_of((long long) tile * QT, p.G);
    const int qa_max = TREE ? 0 : p.q_pos0 +
                       (int) position_of(((long long) tile * QT + QT < nq ? (long long) tile * QT + QT : nq) - 1, p.G);

    // S^T[keys x queries] of a stage: s[h][qb] covers keys 16h + 4lg + r of query column li.
    struct Scores {
        f32x4 s[2][QB];
    };
    auto qk = [&](const unsigned char *kb) {
        Scores sc;
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) sc.s[h][qb] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const bf16x8 ka0 = *reinterpret_cast<const bf16x8 *>(kb + qk_off + 64 * ks);
            const bf16x8 ka1 = *reinterpret_cast<const bf16x8 *>(kb + R::HB + qk_off + 64 * ks);
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) {
                sc.s[0][qb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ka0, qreg[qb][ks], sc.s[0][qb], 0, 0, 0);
                sc.s[1][qb] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ka1, qreg[qb][ks], sc.s[1][qb], 0, 0, 0);
            }
        }
        return sc;
    };

    // Scored: stages from the last to the first, so that a bias by distance meets its largest scores
    // first (from the first on, steep slopes raised the maximum and rescaled O^T in every stage: 512
    // queries over 16K keys, 32 slopes 2^-0.25 .. 2^-8, 541 us against 442).
    // Documents: only those to compute.  cur[i] / ahead[i] are the key stages of this and of the next
    // iteration (-1 past the last), and whether they need no mask for their documents; live and pure
    // describe the 64 stages of `window`.  The i-th stage computed takes ring slot i % NSL.
    struct Stage {
        int st;
        bool pure;
    };
    Stage cur[SPI], ahead[SPI];
    int window = -1;
    unsigned long long live = 0ull, pure = 0ull;
    // to[0 .. SPI-1]: the first SPI stages to compute from stage s down
    auto next_stages = [&](int s, auto &to) {
        if constexpr (DOCS) {
#pragma unroll
            for (int i = 0; i < SPI; ++i) {
                to[i] = {-1, true};
                while (s >= 0) {
                    if ((s >> 6) != window) {
                        window = s >> 6;
                        const bool known = window < kDocWindows;
                        auto word = [&](const unsigned long long *x) {
                            const unsigned long long v = known ? x[window] : 0ull;
                            return (unsigned long long) (unsigned) uniform((int) (unsigned) (v >> 32)) << 32 |
                                   (unsigned) uniform((int) (unsigned) v);
                        };
                        live = known ? word(live_of) : ~0ull;
                        pure = word(pure_of);
                    }
                    const unsigned long long m = live << (63 - (s & 63));
                    if (m == 0ull) {
                        s = (s & ~63) - 1;
                        continue;
                    }
                    s -= __builtin_clzll(m);
                    to[i] = {s, ((pure >> (s & 63)) & 1) != 0};
                    --s;
                    break;
                }
            }
        }
    };
    if constexpr (DOCS) {
        // lowest and highest document of the tile's positions; negative ids are nobody's
        int qlo = INT_MAX, qhi = -1;
        bool one_doc = true;  // all of its rows in one
        for (int i = qa_min - p.q_pos0 + lane; i <= qa_max - p.q_pos0; i += 64) {
            const int d = p.q_doc[i];
            if (d < 0) one_doc = false;
            else {
                qlo = min(qlo, d);
                qhi = max(qhi, d);
            }
        }
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            qlo = min(qlo, __shfl_xor(qlo, o));
            qhi = max(qhi, __shfl_xor(qhi, o));
        }
        one_doc = __builtin_amdgcn_ballot_w64(!one_doc) == 0ull && qlo == qhi;
        // Eight stages a wave and step: one load, 8 lanes of 4 keys to a stage (past the last key: its id
        // again), lowest and highest id over those lanes, and a byte of each set.
        typedef int i32x4_a4 __attribute__((ext_vector_type(4), aligned(4)));
        for (int c = wave; c < 8 * kDocWindows && 8 * c < nst; c += NW) {
            const long long j = (long long) j0 + 256LL * c + 4 * lane, last = p.Sk - 1;
            i32x4 d;
            if (j + 3 <= last) d = *reinterpret_cast<const i32x4_a4 *>(p.k_doc + j);
            else
#pragma unroll
                for (int e = 0; e < 4; ++e) d[e] = p.k_doc[min(j + e, last)];
            int lo = min(min(d[0], d[1]), min(d[2], d[3])), hi = max(max(d[0], d[1]), max(d[2], d[3]));
            // lanes ^1, ^2, then the other four of the eight
            lo = min(lo, __builtin_amdgcn_mov_dpp(lo, 0xb1, 0xf, 0xf, true));
            hi = max(hi, __builtin_amdgcn_mov_dpp(hi, 0xb1, 0xf, 0xf, true));
            lo = min(lo, __builtin_amdgcn_mov_dpp(lo, 0x4e, 0xf, 0xf, true));
            hi = max(hi, __builtin_amdgcn_mov_dpp(hi, 0x4e, 0xf, 0xf, true));
            lo = min(lo, __builtin_amdgcn_mov_dpp(lo, 0x141, 0xf, 0xf, true));
            hi = max(hi, __builtin_amdgcn_mov_dpp(hi, 0x141, 0xf, 0xf, true));
            auto eight = [](bool x) {  // bit 8i of the ballot (lane 8i: stage i of the eight) -> bit i
                return (unsigned char) (((__builtin_amdgcn_ballot_w64(x) & 0x0101010101010101ull) * 0x0102040810204080ull) >> 56);
            };
            const unsigned char a = eight(hi >= qlo && lo <= qhi), b = eight(one_doc && lo == qlo && hi == qhi);
            if (lane == 0) {
                reinterpret_cast<unsigned char *>(live_of)[c] = a;
                reinterpret_cast<unsigned char *>(pure_of)[c] = b;
            }
        }
        lds_barrier();
        next_stages(nst - 1, cur);
    }
    auto issue_docs = [&](int st, int s) {
        if constexpr (DOCS) {
            if (wave == 0 && lane < kStageKeys)
                lds_dma4(p.k_doc + min(j0 + st * kStageKeys + lane, j1 - 1), lds_addr(dids[s & (NSL - 1)]));
        }
    };

    if constexpr (!SCORED) {
        issue(kvb, 0, kslot(0));  // nst >= 1 here
        if (!SH) issue(vvb, 0, vslot(0));
        if ((KH || S2) && nst > 1) {
            issue(kvb, 1, kslot(1));
            if (!SH) issue(vvb, 1, vslot(1));
        }
    } else {
#pragma unroll
        for (int i = 0; i < SPI; ++i) {
            const int st = DOCS ? cur[i].st : nst - 1 - i;
            if (st >= 0) {
                issue(kvb, st, kslot(i));
                if (!SH) issue(vvb, st, vslot(i));
                issue_docs(st, i);
            }
        }
    }

    bool holes = false;  // TREE: some committed row among the keys lies in no page
    int all_see = 0;     // .. and committed rows from it on are seen by every node
    bool is_seq = true;
    if constexpr (TREE) {  // beside the first stage's loads
        unsigned long long path;
        is_seq = tree_paths(p, tu.b, tu.len, lane, path);
        if (wave == 0) paths[lane] = path;
        for (int r = threadIdx.x; r < QT; r += 64 * NW) odd_row[r] = 0;
        if (threadIdx.x == 0) any_odd = 0;
        if (!p.linear) {
            const int k0 = (tu.first + j0) >> p.shift, k1 = (min(tu.len, tu.first + j1) - 1) >> p.shift;  // (k1 < k0: none)
            for (int k = k0 + lane; k <= k1; k += 64) holes = holes || !tree_page(p, tr.table[k]);
            holes = __builtin_amdgcn_ballot_w64(holes) != 0ull;
        }
        if (p.window > 0) all_see = tu.len + p.Sq - p.window;
        if (kvh == 0 && split == 0 && tile == 0 && threadIdx.x == 0) tree_report(p, tu, is_seq);
        if (!is_seq) {  // (its DMAs end before the workgroup's LDS is another's)
            ESDA_WAIT_VM(0);
            return;
        }
        tr.none = __builtin_amdgcn_ballot_w64(path == 0ull);
    }
    // TREE: rows of stage s that no node sees may hold anything, with a weight of 0: zeros instead (0 x inf is
    // NaN).  By the wave whose DMAs they are, once these have landed.
    auto clear_unseen = [&](int s) {
        if constexpr (TREE) {
            const int jst = j0 + s * kStageKeys + 16 * (wave / (NW / 2)), row = tu.first + jst;
            unsigned rows = tr.unseen(jst);
            if (holes && row < tu.len && tr.page_of(row >> p.shift) < 0) rows = 0xffffu;
#pragma unroll
            for (int t = 0; t < KPW; ++t)
                if ((rows >> (vrow[t] & 15)) & 1) *reinterpret_cast<u32x4 *>(vslot(s) + ldso[t] + 16 * lane) = u32x4{0u, 0u, 0u, 0u};
        }
    };
    auto shift = [&]() {
        if constexpr (DOCS) {
#pragma unroll
            for (int i = 0; i < SPI; ++i) cur[i] = ahead[i];
        }
    };
    auto scored_full = [&](int jb, int ka_first, int ka_last, bool pure) {
        if constexpr (SCORED)
            return jb + kStageKeys <= j1 && (ka_last <= qa_min || ka_last < p.prefix) &&
                   (p.window == 0 || ka_first > qa_max - p.window) && pure;
        else return false;
    };
    for (int s0 = 0; DOCS ? cur[0].st >= 0 : s0 < nst; s0 += SPI, shift()) {
        // the key stage of the i-th stage from s0 on
        auto at = [&](int i) -> int {
            if constexpr (!SCORED) return s0 + i;
            else if constexpr (!DOCS) return nst - 1 - (s0 + i);
            else if (i < SPI) return i == 0 ? cur[0].st : cur[SPI - 1].st;
            else return i == SPI ? ahead[0].st : ahead[SPI - 1].st;
        };
        auto there = [&](int st) { return SCORED ? st >= 0 : st < nst; };
        // The iteration's stages s0 .. s0+SPI-1 landed (this wave's loads; the barrier covers
        // the other waves') and every wave is done with the previous iteration
        ESDA_WAIT_VM(0);
        if constexpr (TREE) {
            const int row = tu.first + j0 + s0 * kStageKeys;
            if (__builtin_expect(holes || row < tr.low || row + SPI * kStageKeys > tu.len, 0))
                for (int s = s0; s < min(s0 + SPI, nst); ++s) clear_unseen(s);
        }
        lds_barrier();
        if constexpr (PARTS) {
            // rows past the prefix repeat its last key: with a weight of 0, but 0 x inf is NaN
            const int past = j1 - (j0 + s0 * kStageKeys);  // keys from this iteration's first on
            if (s0 + SPI >= nst && past % kStageKeys != 0) {
                for (int r = past % kStageKeys + wave; r < kStageKeys; r += NW) {
                    unsigned char *const row = vslot(nst - 1) + (r >> 4) * R::HB + R::off(r & 15);
                    for (int c = lane; c < D / 8; c += 64) *reinterpret_cast<u32x4 *>(row + 16 * c) = u32x4{0u, 0u, 0u, 0u};
                }
                lds_barrier();
            }
        }
        if constexpr (DOCS) next_stages(cur[SPI - 1].st - 1, ahead);
        // The next iteration's DMAs, spread over this iteration so that the workgroup's loads
        // do not all queue at the barrier (each slot is free once the barrier has passed):
        //  - separate K and V (plain, S2): K of the next stage at the barrier, its V after
        //    this iteration's first QK;
        //  - one K = V stream (S2): the next stage after the first QK;
        //  - S2: the stage after that once this iteration's first stage is done;
        //  - KH: all at the barrier (spreading measured slower there).
        constexpr bool kVLate = !SH && !KH;
        auto issue_k = [&]() {
            if (there(at(SPI))) {
                issue(kvb, at(SPI), kslot(s0 + SPI));
                issue_docs(at(SPI), s0 + SPI);
            }
        };
        auto issue_v = [&]() {
            if (!SH && there(at(SPI))) issue(vvb, at(SPI), vslot(s0 + SPI));
        };
        auto issue_second = [&]() {
            if (there(at(SPI + 1))) {
                issue(kvb, at(SPI + 1), kslot(s0 + SPI + 1));
                if (!SH) issue(vvb, at(SPI + 1), vslot(s0 + SPI + 1));
                issue_docs(at(SPI + 1), s0 + SPI + 1);
            }
        };
        auto after_first_qk = [&]() {
            if constexpr (SH) issue_k();
            if constexpr (kVLate) issue_v();
        };
        if constexpr (!SH) issue_k();
        if constexpr (!kVLate && !SH) issue_v();
        if constexpr (KH) issue_second();
        // stage s in the order computed (its ring slot), key stage st
        auto stage = [&](const int s, const int st, const bool pure, auto after_qk) {
        const Scores cur = qk(kslot(s));
        after_qk();
        const unsigned char *vb = vslot(s);
        const int jb = j0 + st * kStageKeys;

        // Stage s's raw scores q.k; positions a boundary stage does not show to a row are
        // -inf.  A stage is fully visible to every row of the tile when its last key is at
        // or before the tile's first position, its first key is inside the window of the
        // tile's last position, and it lies inside the split.  The softmax scale (times
        // log2 e, > 0) is applied to the row maxima and inside the exponent's fma.
        // (Scored: the cap and the bias first, the mask last -- a masked score may be NaN.)
        float c2 = p.scale_log2e;
        float sv[QB][8];
#pragma unroll
        for (int qb = 0; qb < QB; ++qb)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int r = 0; r < 4; ++r) sv[qb][4 * h + r] = cur.s[h][qb][r];
        const int ka_first = p.k_pos0 + jb, ka_last = ka_first + kStageKeys - 1;
        const int krow = tu.first + jb;  // TREE: the stage's first row
        const bool full = TREE     ? jb + kStageKeys <= j1 && krow + kStageKeys <= tu.len && krow >= all_see && !holes
                          : SCORED ? scored_full(jb, ka_first, ka_last, pure)
                                 : jb + kStageKeys <= j1 && ka_last <= qa_min &&
                                       (p.window == 0 || ka_first > qa_max - p.window);
        if constexpr (SCORED) {
            if constexpr (WIDE) {
                c2 = 1.0f;
#pragma unroll
                for (int qb = 0; qb < QB; ++qb)
#pragma unroll
                    for (int e = 0; e < 8; ++e) sv[qb][e] = capped_wide(sv[qb][e], sv[qb][e] * p.scale_log2e, p.soft);
            } else if (p.soft.out != 0.0f) {
                // the softmax drops the 1 of 1 - 2 / (1 + e^2x): -1 / (1 + e^2x) in units of 2 cap log2 e
                c2 = 2.0f * p.soft.out;
#pragma unroll
                for (int qb = 0; qb < QB; ++qb)
#pragma unroll
                    for (int e = 0; e < 8; ++e)
                        sv[qb][e] = __builtin_amdgcn_rcpf(-1.0f - __builtin_amdgcn_exp2f(sv[qb][e] * p.soft.in));
            }
            if (p.slopes) {
                // Keys at or before their queries: the bias is linear, base + slope (key's place in the
                // stage).  (Keys ahead of a query are masked unless they lie in the prefix.)
                if (ka_last <= qa_min || p.prefix <= ka_first) {
#pragma unroll
                    for (int qb = 0; qb < QB; ++qb) {
                        const int r = wq * 16 * QB + qb * 16 + li;
                        const float slope = row_slope[r], base = -slope * (float) (row_pos[r] - ka_first - 4 * lg);
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            sv[qb][e] = __builtin_fmaf(sv[qb][e], c2, __builtin_fmaf(slope, (float) (16 * (e / 4) + e % 4), base));
                    }
                } else {
#pragma unroll
                    for (int qb = 0; qb < QB; ++qb) {
                        const int r = wq * 16 * QB + qb * 16 + li, d0 = row_pos[r] - ka_first - 4 * lg;
                        const float slope = row_slope[r];
#pragma unroll
                        for (int e = 0; e < 8; ++e) {
                            const float dist = (float) (d0 - (16 * (e / 4) + e % 4));
                            sv[qb][e] = __builtin_fmaf(sv[qb][e], c2, -slope * __builtin_fabsf(dist));
                        }
                    }
                }
                c2 = 1.0f;
            }
        }
        if constexpr (TREE) {
            if (!full) {
                bool held[2] = {true, true};  // the halves' pages
                if (holes)
#pragma unroll
                    for (int h = 0; h < 2; ++h)
                        if (krow + 16 * h < tu.len) held[h] = tr.page_of((krow + 16 * h) >> p.shift) >= 0;
#pragma unroll
                for (int qb = 0; qb < QB; ++qb) {
                    const unsigned long long sees = paths[position_of(qrow(qb), p.G)];
                    const int lowest = p.window > 0 ? tu.len + __popcll(sees) - p.window : 0;
#pragma unroll
                    for (int h = 0; h < 2; ++h)
#pragma unroll
                        for (int r = 0; r < 4; ++r) {
                            const int j = jb + 16 * h + 4 * lg + r, row = tu.first + j;
                            const bool seen = row < tu.len ? row >= lowest && held[h] : ((sees >> ((row - tu.len) & 63)) & 1) != 0;
                            if (!(j < j1 && seen)) sv[qb][4 * h + r] = -INFINITY;
                        }
                }
            }
        } else if (!full) {
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) {
                const int qa = SCORED ? row_pos[SCORED ? wq * 16 * QB + qb * 16 + li : 0] : qabs[qb];
                const int lo = p.window > 0 ? qa - p.window : INT_MIN;  // visible: lo < ka <= qa
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const int j = jb + 16 * h + 4 * lg + r;
                        const int ka = p.k_pos0 + j;
                        if constexpr (SCORED) {
                            if (!((j < j1) & (ka <= max(qa, p.prefix - 1)) & (ka > lo))) sv[qb][4 * h + r] = -INFINITY;
                        } else {
                            if (!(j < j1 && ka <= qa && ka > lo)) sv[qb][4 * h + r] = -INFINITY;
                        }
                    }
            }
        }

        if constexpr (DOCS) {
            if (!pure) {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const i32x4 d = *reinterpret_cast<const i32x4 *>(&dids[s & (NSL - 1)][16 * h + 4 * lg]);
#pragma unroll
                    for (int qb = 0; qb < QB; ++qb)
#pragma unroll
                        for (int r = 0; r < 4; ++r)
                            if ((d[r] != row_doc[wq * 16 * QB + qb * 16 + li]) | (d[r] < 0)) sv[qb][4 * h + r] = -INFINITY;
                }
            }
        }

        // Row maxima of the stage in log2 units (scaling by c2 > 0 keeps the order).
        float mt[QB];
        bool need = false;
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
            float x = sv[qb][0];
#pragma unroll
            for (int e = 1; e < 8; ++e) x = fmaxf(x, sv[qb][e]);
            mt[qb] = wave_max_across_groups(x) * c2;
            need = need || mt[qb] > m[qb] + kRescaleSlack;
        }

        // Raise the running max where a score exceeds it by the slack (rare): one
        // wave-uniform branch; lanes that do not need it scale by 1.
        unsigned char *const xs = xch + (PS ? (s & 1) * XPAR : 0);  // PS: this stage's exchange
        bool resc = false;
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(need) != 0, 0)) {
            asm volatile("" ::: "memory");  // keeps the rare rescale a branch (no if-conversion)
            resc = true;
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) {
                const bool up = mt[qb] > m[qb] + kRescaleSlack;
                const float corr = up ? __builtin_amdgcn_exp2f(m[qb] - mt[qb]) : 1.0f;  // 0 while m is -inf
                l[qb] *= corr;
#pragma unroll
                for (int dt = 0; dt < DW; ++dt) acc[qb][dt] *= corr;
                m[qb] = up ? mt[qb] : m[qb];
                if constexpr (PS) *reinterpret_cast<float *>(xs + wave * XP + 1024 + lane * 4) = corr;
            }
        }

        bf16x8 pb[QB];
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
            const float mu = m[qb] == -INFINITY ? 0.0f : m[qb];  // all keys so far masked
            // The weights are bf16, as the product's operands are; the sum takes them rounded, too, so that
            // a row of equal values comes out exact.  (At most 2^-8 of a weight: outputs are 0.0016 .. 0.0023
            // off in relative norm, 0.0016 of it by their own rounding to bf16.)
            bf16x8 pv;
#pragma unroll
            for (int e = 0; e < 8; ++e) pv[e] = (__bf16) __builtin_amdgcn_exp2f(__builtin_fmaf(sv[qb][e], c2, -mu));
            // l += the eight bf16 weights, two per v_dot2_f32_bf16 against (1, 1)
            const bf16x2 one2 = {(__bf16) 1.0f, (__bf16) 1.0f};
#pragma unroll
            for (int e = 0; e < 8; e += 2) l[qb] = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{pv[e], pv[e + 1]}, one2, l[qb], false);
            pb[qb] = pv;
        }
        if constexpr (PS) {  // P^T (and factors) to the partner, then the flag
            *reinterpret_cast<bf16x8 *>(xs + wave * XP + lane * 16) = pb[0];
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            if (lane == 0)
                *(lds_flag *) (xs + NW * XP + wave * 4) = 2u * (unsigned) (s + 1) + (resc ? 1u : 0u);
        }

        // O^T += V^T . P^T: lane (li, lg) gets dim 16dt + li of keys 4lg .. 4lg+3 (first
        // half) and 16 + 4lg .. (second half): the k order of the P^T registers.
        // The V^T tiles are read PD ahead of their MFMAs (the scheduler alone kept one in flight).
        const unsigned char *const vbh = vb + 32 * DW * hd;  // PS: this wave's dims
        auto vtile = [&](int dt) { return vtile_of(vbh, dt); };
        constexpr int PD = PV_DEPTH;
        bf16x8 vf[PD];
#pragma unroll
        for (int i = 0; i < PD && i < DW; ++i) vf[i] = vtile(i);
        bf16x8 pq[NB];  // B operands: the wave's blocks (PS: its own, then its partner's)
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) pq[qb] = pb[qb];
        if constexpr (PS) {
            // The partner's flag for this stage (bounded: a wave that gave up would compute
            // garbage, not hang), then its P^T and, after its rescale, its factors.
            const unsigned want = 2u * (unsigned) (s + 1);
            lds_flag *fl = (lds_flag *) (xs + NW * XP + (wave ^ 1) * 4);
            unsigned f = __builtin_amdgcn_readfirstlane(*fl);
            for (int it = 0; (f & ~1u) != want && it < kPairSpin; ++it) {
                __builtin_amdgcn_s_sleep(1);
                f = __builtin_amdgcn_readfirstlane(*fl);
            }
            asm volatile("" ::: "memory");
            const unsigned char *const xp = xs + (wave ^ 1) * XP;
            pq[1] = *reinterpret_cast<const bf16x8 *>(xp + lane * 16);
            if (f & 1u) {
                const float pc = *reinterpret_cast<const float *>(xp + 1024 + lane * 4);
#pragma unroll
                for (int dt = 0; dt < DW; ++dt) acc[1][dt] *= pc;
            }
        }
#pragma unroll
        for (int dt = 0; dt < DW; ++dt) {
            const bf16x8 a = vf[dt % PD];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
                acc[nb][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, pq[nb], acc[nb][dt], 0, 0, 0);
            if (dt + PD < DW) vf[dt % PD] = vtile(dt + PD);
            __builtin_amdgcn_sched_barrier(0);
        }
        };
        if constexpr (S2) {
            stage(s0, at(0), !DOCS || cur[0].pure, after_first_qk);
            issue_second();
            if (there(at(1))) stage(s0 + 1, at(1), !DOCS || cur[SPI - 1].pure, [] {});
        } else {
            const int s = s0 + kh, st = at(kh);  // this wave group's stage
            if (KH && !there(st)) continue;  // an odd stage count: the odd group's last iteration is empty
            stage(s, st, !DOCS || (kh ? cur[SPI - 1].pure : cur[0].pure), after_first_qk);
        }
    }

    if constexpr (KH) {
        // The odd-stage wave of each query block hands its (m, l, O^T) to the even-stage
        // wave through the ring's LDS (no DMA is outstanding and, after the barrier, no wave
        // reads the ring): lane-major, so each store and load of a wave is one contiguous
        // 1 KB.  A group that saw no key of a row holds m = -inf, l = 0 and adds nothing.
        constexpr int XA = QB * DT * 64 * 16;  // O^T bytes per wave
        constexpr int XW = XA + QB * 64 * 8;   // + (m, l)
        static_assert(NQW * XW <= R::BYTES, "the hand-over must fit the ring");
        unsigned char *xb = ring + wq * XW;
        lds_barrier();
        if (kh) {
#pragma unroll
            for (int qb = 0; qb < QB; ++qb) {
#pragma unroll
                for (int dt = 0; dt < DT; ++dt)
                    *reinterpret_cast<f32x4 *>(xb + ((qb * DT + dt) * 64 + lane) * 16) = acc[qb][dt];
                *reinterpret_cast<f32x2 *>(xb + XA + (qb * 64 + lane) * 8) = f32x2{m[qb], l[qb]};
            }
        }
        lds_barrier();
        if (!ODD && kh) return;
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
            if (ODD && kh) break;
            const f32x2 mlb = *reinterpret_cast<const f32x2 *>(xb + XA + (qb * 64 + lane) * 8);
            const float M = fmaxf(m[qb], mlb[0]);
            const float wa = m[qb] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m[qb] - M);
            const float wb = mlb[0] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mlb[0] - M);
            l[qb] = l[qb] * wa + mlb[1] * wb;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
                acc[qb][dt] = acc[qb][dt] * wa +
                              *reinterpret_cast<const f32x4 *>(xb + ((qb * DT + dt) * 64 + lane) * 16) * wb;
            m[qb] = M;
        }
    }

    // Row totals over the four lane groups; then the output (one split) or the partial.
    float lb[NB];  // row sums of the wave's O^T blocks
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
        l[qb] += __shfl_xor(l[qb], 16);
        l[qb] += __shfl_xor(l[qb], 32);
        lb[qb] = l[qb];
    }
    if constexpr (PS) {  // the partner's row sums, through LDS past every wave's last stage
        float *xl = reinterpret_cast<float *>(xch + 2 * XPAR);
        if (lg == 0) xl[wave * 16 + li] = l[0];
        lds_barrier();
        lb[1] = xl[(wave ^ 1) * 16 + li];
    }
#pragma unroll
    for (int nb = 0; nb < NB; ++nb) {
        // the block's first tile row (PS: the wave's own block, then its partner's)
        const int br = PS ? (nb == 0 ? wave : wave ^ 1) * 16 : wq * 16 * QB + nb * 16;
        const long long gr0 = (long long) tile * QT + br + li;
        if (gr0 >= nq || (ODD && KH && kh)) continue;
        if constexpr (TREE) {
            if (paths[position_of(gr0, p.G)] == 0ull) {  // no node: nothing seen (its q may be anything, and m infinite)
                lb[nb] = 0.0f;
                if (nb < QB) {
                    m[nb < QB ? nb : 0] = -INFINITY;
                    l[nb < QB ? nb : 0] = 0.0f;
                }
#pragma unroll
                for (int dt = 0; dt < DW; ++dt) acc[nb][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            }
        }
        if constexpr (ODD) {
            float c = 0.0f;  // NaN where a value is not finite
#pragma unroll
            for (int dt = 0; dt < DW; ++dt)
#pragma unroll
                for (int r = 0; r < 4; ++r) c = __builtin_fmaf(acc[nb][dt][r], 0.0f, c);
            if (c != c) {
                odd_row[br + li] = 1;
                any_odd = 1;
            }
        }
        const long long gr = gr0;
        const int qi = (int) position_of(gr, p.G), qh = kvh * p.G + (int) ((unsigned) gr - (unsigned) qi * p.G);
        const long long row = (long long) qi * p.Hq + qh;
        long long part = (long long) split * nrows + row;  // its partial
        if constexpr (TREE) part = tree_part(p, tu) + gr;
        const int d0 = 16 * DW * hd;  // the wave's first O^T dim
        if (!PARTS && p.splits == 1) {
            float inv = 1.0f / lb[nb];
            if constexpr (ODD) inv = lb[nb] == 0.0f ? 0.0f : inv;  // a row that sees nothing
            uint16_t *o = out0 + (size_t) qi * p.o_rs + (size_t) qh * p.o_hs + d0 + 4 * lg;
#pragma unroll
            for (int dt = 0; dt < DW; ++dt) {
                const f32x4 v4 = acc[nb][dt] * inv;
                bf16x4 b4 = {(__bf16) v4[0], (__bf16) v4[1], (__bf16) v4[2], (__bf16) v4[3]};
                *reinterpret_cast<bf16x4 *>(o + 16 * dt) = b4;
            }
        } else {
            float *pa = p.part_acc + part * D + d0 + 4 * lg;
            if (p.part_nt) {
                // (the barriers keep the two branches' stores from being merged into plain ones)
                asm volatile("" ::: "memory");
#pragma unroll
                for (int dt = 0; dt < DW; ++dt) __builtin_nontemporal_store(acc[nb][dt], reinterpret_cast<f32x4 *>(pa + 16 * dt));
                asm volatile("" ::: "memory");
            } else {
#pragma unroll
                for (int dt = 0; dt < DW; ++dt) *reinterpret_cast<f32x4 *>(pa + 16 * dt) = acc[nb][dt];
            }
            if (lg == 0 && nb < QB)  // (m, l) from the block's owner
                *reinterpret_cast<f32x2 *>(p.part_ml + 2 * part) = f32x2{m[nb < QB ? nb : 0], l[nb < QB ? nb : 0]};
        }
    }
    if constexpr (TREE) {
        if (tile == 0) append_nodes<D, SH>(tr, paths, j0, j1);
        ESDA_WAIT_VM(0);  // the rows as written above, before they are written again
        lds_barrier();
        if (__builtin_expect(any_odd != 0, 0)) {
            for (int r = wave; r < QT; r += NW) {
                if (!odd_row[r]) continue;
                const long long gr = (long long) tile * QT + r;
                const int qi = (int) position_of(gr, p.G), qh = kvh * p.G + (int) ((unsigned) gr - (unsigned) qi * p.G);
                const long long row = row0 + (long long) qi * p.Hq + qh;
                tree_row_again<D, SH>(tr, p.q + row * D, paths[qi], p.window > 0 ? tu.len + __popcll(paths[qi]) - p.window : 0, j0, j1,
                                      p.scale_log2e, [&](float mr, float lr, const float(&o)[D / 64]) {
                                          tree_row_store<D>(p, row, tree_part(p, tu) + gr, lane, mr, lr, o);
                                      });
            }
        }
    }
    if constexpr (SCORED) {
        // Rare: rows whose O^T is not finite.  A value that is not was seen, or met a weight of 0 (0 x inf
        // is NaN): those rows again, over the keys they see only.  The lanes take 64 keys for the scores,
        // then the row's dims for the product.  (Testing the values of every masked stage took 5% to 70%
        // of a chunk's time, a second form of the product in the stage O^T's registers.)
        ESDA_WAIT_VM(0);  // the rows as written above, before they are written again
        lds_barrier();
        if (__builtin_expect(any_odd != 0, 0)) {
            constexpr int DPL = D / 64;
            typedef uint16_t piece __attribute__((ext_vector_type(DPL)));
            for (int r = wave; r < QT; r += NW) {
                if (!odd_row[r]) continue;
                const long long gr = (long long) tile * QT + r;
                const int qi = (int) position_of(gr, p.G), qh = kvh * p.G + (int) ((unsigned) gr - (unsigned) qi * p.G);
                const uint16_t *const qr = p.q + (size_t) qh * p.q_hs + (size_t) qi * p.q_rs;
                const int qa = p.q_pos0 + qi, lo = p.window > 0 ? qa - p.window : INT_MIN;
                const float sl = p.slopes ? p.slopes[qh] * kLog2e : 0.0f;
                int doc = 0;
                if constexpr (DOCS) doc = p.q_doc[qi];
                float mr = -INFINITY, lr = 0.0f, o[DPL];
#pragma unroll
                for (int e = 0; e < DPL; ++e) o[e] = 0.0f;
                for (int jb = j0; jb < j1; jb += 64) {
                    const int j = jb + lane, ka = p.k_pos0 + j;
                    bool seen = j < j1 && ka <= max(qa, p.prefix - 1) && ka > lo;
                    if constexpr (DOCS) {
                        if (seen) seen = doc >= 0 && p.k_doc[j] == doc;
                    }
                    unsigned long long todo = __builtin_amdgcn_ballot_w64(seen);
                    if (todo == 0ull) continue;
                    float x = 0.0f;
                    if (seen) {
                        const uint16_t *const kr = kvb + (size_t) j * D;
#pragma unroll 1
                        for (int d = 0; d < D; d += 8) {
                            const u32x4 kv = *reinterpret_cast<const u32x4 *>(kr + d);
                            const u32x4 qv = *reinterpret_cast<const u32x4 *>(qr + d);
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                x = __builtin_fmaf(bf16_lo(qv[e]), bf16_lo(kv[e]), x);
                                x = __builtin_fmaf(bf16_hi(qv[e]), bf16_hi(kv[e]), x);
                            }
                        }
                        const float raw = x;
                        x *= p.scale_log2e;
                        if constexpr (WIDE) x = capped_wide(raw, x, p.soft);
                        else if (p.soft.out != 0.0f)
                            x = 2.0f * p.soft.out * __builtin_amdgcn_rcpf(-1.0f - __builtin_amdgcn_exp2f(raw * p.soft.in));
                        x = __builtin_fmaf(-sl, __builtin_fabsf((float) (qa - ka)), x);
                    }
                    float top = seen ? x : -INFINITY;
#pragma unroll
                    for (int i = 32; i >= 1; i >>= 1) top = fmaxf(top, __shfl_xor(top, i));
                    const float mn = fmaxf(mr, top), corr = mr == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mr - mn);
                    const float w = seen ? (float) (__bf16) __builtin_amdgcn_exp2f(x - (mn == -INFINITY ? 0.0f : mn)) : 0.0f;
                    float sum = w;
#pragma unroll
                    for (int i = 32; i >= 1; i >>= 1) sum += __shfl_xor(sum, i);
                    mr = mn;
                    lr = lr * corr + sum;
#pragma unroll
                    for (int e = 0; e < DPL; ++e) o[e] *= corr;
                    while (todo) {
                        const int b = __builtin_ctzll(todo);
                        todo &= todo - 1;
                        const float wb = __shfl(w, b);
                        const piece v = *reinterpret_cast<const piece *>(vvb + (size_t) (jb + b) * D + lane * DPL);
#pragma unroll
                        for (int e = 0; e < DPL; ++e)
                            o[e] = __builtin_fmaf(wb, __builtin_bit_cast(float, (unsigned) v[e] << 16), o[e]);
                    }
                }
                const long long row = (long long) qi * p.Hq + qh;
                if (p.splits == 1) {
                    const float inv = lr == 0.0f ? 0.0f : 1.0f / lr;
                    piece b;
#pragma unroll
                    for (int e = 0; e < DPL; ++e) b[e] = __builtin_bit_cast(uint16_t, (__bf16) (o[e] * inv));
                    *reinterpret_cast<piece *>(p.out + (size_t) qi * p.o_rs + (size_t) qh * p.o_hs + lane * DPL) = b;
                } else {
                    float *pa = p.part_acc + ((long long) split * nrows + row) * D + lane * DPL;
#pragma unroll
                    for (int e = 0; e < DPL; ++e) pa[e] = o[e];
                    if (lane == 0)
                        *reinterpret_cast<f32x2 *>(p.part_ml + 2 * ((long long) split * nrows + row)) = f32x2{mr, lr};
                }
            }
        }
    }
}

// out(i, h, :) = sum_s acc_s 2^(m_s - M) / sum_s l_s 2^(m_s - M) over the splits with
// l_s > 0.  One wave per (row, 64 * VEC dims), or per two rows of 128 dims (in up to 8 splits; a
// block is then two waves, since four rows a block keep a GQA group of four on the XCD that
// wrote it: 143 queries of 32 heads over 8 in 8 splits, 4.1 us and 5.9 with eight rows a block).
// Memory-bound: splits * D * 4 bytes per row, read once, so the two forms differ in how they
// cover the latency:
//  - NS > 0, for plans of at most NS splits: every (m, l) and partial row is loaded at once
//    (one round trip; a row that an empty split never wrote is dropped by a select), or with
//    GAPS, where the plan leaves many tiles' last splits empty, the (m, l) and then the live
//    splits' rows: a fresh prompt's rows see the splits up to their own, a little over half of
//    them (2048 queries of 32 heads in 4 splits, D = 512, 0.54 GB: 116 us reading all, 75 the
//    live ones; 805 MB in 6, 174 and 114);
//  - NS = 0: lane j loads (m, l) of split j (and j + 64, ..), so the max, the weights and the
//    denominator take one round trip and wave reductions, and the wave then walks the live
//    splits (a ballot: wave-uniform) with MB of their rows in flight.
// A thread per 4 dims walking the splits one after another was bound by their latency:
// 512 rows of D = 512 with 18 splits 8.2 us against 4.3 here, with 32 splits 19.9 against
// 6.3; 16384 rows with 2 splits 17.2 against 14.4 (67 MB at 4.7 TB/s).  A wave per row of 128
// dims, 2 a lane, had too few bytes in flight for many rows: 16,384 rows with 2 splits 6.9 us
// against 5.4 here, 32,768 10.9 against 9.3.
// P = ScoredParams: a row without a live split gives 0 (and a NaN sum is live: its row is NaN).
template <int D, int NS, bool GAPS = false, class P = PrefillParams>
__global__ __launch_bounds__(256) void prefill_merge_kernel(P p) {
    constexpr bool SCORED = std::is_same<P, ScoredParams>::value;
    auto alive = [](float l) { return SCORED ? l != 0.0f : l > 0.0f; };
    auto inverse = [](float den) { return SCORED && den == 0.0f ? 0.0f : 1.0f / den; };
    constexpr int VEC = D >= 256 || NS > 0 ? 4 : D / 64;              // dims per lane
    constexpr int LPR = D / VEC < 64 ? D / VEC : 64, RPW = 64 / LPR;  // lanes per row and wave, rows per wave
    constexpr int PARTS = D / (LPR * VEC);                            // waves per row
    constexpr int MB = 8;                       // partial rows in flight
    typedef float vec __attribute__((ext_vector_type(VEC)));
    typedef __bf16 bvec __attribute__((ext_vector_type(VEC)));
    const int lane = threadIdx.x & 63;
    const long long nrows = (long long) p.Sq * p.Hq;
    const long long wv = p.merge_wave0 + (long long) blockIdx.x * (4 / RPW) + uniform(threadIdx.x >> 6);
    const long long row = RPW * (wv / PARTS) + (RPW > 1 ? lane / LPR : 0);
    if (row >= nrows) return;
    const int d0 = (int) (wv % PARTS) * 64 * VEC + lane % LPR * VEC;
    const float *acc = p.part_acc + row * D + d0;
    const long long ss = nrows * D;
    auto write = [&](const vec &v) {
        bvec b;
#pragma unroll
        for (int e = 0; e < VEC; ++e) b[e] = (__bf16) v[e];
        const int i = (int) (row / p.Hq), h = (int) (row % p.Hq);
        *reinterpret_cast<bvec *>(p.out + (size_t) i * p.o_rs + (size_t) h * p.o_hs + d0) = b;
    };
    if constexpr (NS > 0) {
        f32x2 mls[NS];
        vec a[NS];
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            mls[s] = f32x2{-INFINITY, 0.0f};
            a[s] = 0.0f;
            if (s < p.splits) {
                mls[s] = *reinterpret_cast<const f32x2 *>(p.part_ml + 2 * ((long long) s * nrows + row));
                if (!GAPS) a[s] = *reinterpret_cast<const vec *>(acc + s * ss);
            }
        }
        if (GAPS) {
#pragma unroll
            for (int s = 0; s < NS; ++s)
                if (alive(mls[s][1])) a[s] = *reinterpret_cast<const vec *>(acc + s * ss);
        }
        float M = -INFINITY, den = 0.0f;
#pragma unroll
        for (int s = 0; s < NS; ++s) M = alive(mls[s][1]) ? fmaxf(M, mls[s][0]) : M;
        vec num = 0.0f;
#pragma unroll
        for (int s = 0; s < NS; ++s) {
            // (the operands selected, not the products: those stay fused into the sums)
            const bool live = alive(mls[s][1]);
            const float w = live ? __builtin_amdgcn_exp2f(mls[s][0] - M) : 0.0f;
            den = __builtin_fmaf(live ? mls[s][1] : 0.0f, w, den);
#pragma unroll
            for (int e = 0; e < VEC; ++e) num[e] = __builtin_fmaf(live ? a[s][e] : 0.0f, w, num[e]);
        }
        write(num * inverse(den));
        return;
    }
    auto ml_of = [&](int s) {
        return s < p.splits ? *reinterpret_cast<const f32x2 *>(p.part_ml + 2 * ((long long) s * nrows + row))
                            : f32x2{-INFINITY, 0.0f};
    };
    f32x2 ml = ml_of(lane);
    float M = alive(ml[1]) ? ml[0] : -INFINITY;
    for (int s = lane + 64; s < p.splits; s += 64) {
        const f32x2 x = ml_of(s);
        if (alive(x[1])) M = fmaxf(M, x[0]);
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) M = fmaxf(M, __shfl_xor(M, o));
    float den = 0.0f;
    vec num = 0.0f;
    for (int s0 = 0; s0 < p.splits; s0 += 64) {
        if (s0) ml = ml_of(s0 + lane);
        const float w = alive(ml[1]) ? __builtin_amdgcn_exp2f(ml[0] - M) : 0.0f;
        den += alive(ml[1]) ? ml[1] * w : 0.0f;
        unsigned long long live = __builtin_amdgcn_ballot_w64(alive(ml[1]));
        while (live) {
            vec a[MB];
            float wj[MB];
            int n = 0;
#pragma unroll
            for (int j = 0; j < MB; ++j)
                if (live) {
                    const int b = __builtin_ctzll(live);
                    live &= live - 1;
                    wj[j] = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), b));
                    a[j] = *reinterpret_cast<const vec *>(acc + (s0 + b) * ss);
                    n = j + 1;
                }
#pragma unroll
            for (int j = 0; j < MB; ++j)
                if (j < n) num += wj[j] * a[j];
        }
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) den += __shfl_xor(den, o);
    write(num * inverse(den));
}

template <int D, class P = PrefillParams>
void launch_tiles(const P &p, hipStream_t st) {
    // Up to 64 rows of D = 512 are one tile, and a plan, of either height; the kernel then goes by
    // the streams, which the plan does not know.  Of 499 such (chunk, split) pairs of K = V four
    // waves took 0.95 of eight's time on average (0.92 .. 0.99 from the 10th to the 90th
    // percentile); of 117 of separate K and V 1.05 (1.03 .. 1.12).
    const bool shared = p.k == p.v, one = D == 512 && (long long) p.Sq * p.G <= 64;
    const int nw = one ? (shared ? 4 : 8) : p.nw;
    unsigned groups = p.tiles * p.Hkv * p.splits;
    if constexpr (std::is_same<P, PrefixParams>::value) groups += p.own_groups;
    if constexpr (std::is_same<P, TreeParams>::value) groups = p.tiles * p.units;
    const dim3 grid(groups), block(64 * nw);
    if constexpr (D == 512) {
        if (nw == 4 && shared) hipLaunchKernelGGL((prefill_kernel<512, 1, false, true, true, true, 4, P>), grid, block, 0, st, p);
        else if (nw == 4) hipLaunchKernelGGL((prefill_kernel<512, 1, false, false, false, false, 4, P>), grid, block, 0, st, p);
        else if (shared) hipLaunchKernelGGL((prefill_kernel<512, 1, false, true, true, true, kWaves, P>), grid, block, 0, st, p);
        else hipLaunchKernelGGL((prefill_kernel<512, 1, false, false, false, false, kWaves, P>), grid, block, 0, st, p);
    }
    else if constexpr (D == 128 && (std::is_base_of<ScoredParams, P>::value || std::is_same<P, TreeParams>::value))
        hipLaunchKernelGGL((prefill_kernel<128, 2, false, false, false, false, 4, P>), grid, block, 0, st, p);
    else if constexpr (D == 128)
        hipLaunchKernelGGL((prefill_kernel<128, 2, false, false, false, false, kWaves, P>), grid, block, 0, st, p);
    else {
        // (a tree's rows of a kv head fill few tiles of 256, whose kernel would spill registers there)
        if constexpr (!std::is_same<P, TreeParams>::value) {
            if (p.qb == 2) {
                hipLaunchKernelGGL((prefill_kernel<256, 2, false, false, true, false, kWaves, P>), grid, block, 0, st, p);
                return;
            }
        }
        if (p.kh)
            hipLaunchKernelGGL((prefill_kernel<256, 1, true, false, false, false, kWaves, P>), grid, block, 0, st, p);
        else
            hipLaunchKernelGGL((prefill_kernel<256, 1, false, false, false, false, kWaves, P>), grid, block, 0, st, p);
    }
}

template <int D, class P = PrefillParams>
void launch_prefill(const P &p, int stages, hipStream_t st) {
    if (stages & 1) launch_tiles<D, P>(p, st);
    if ((stages & 2) && p.splits > 1) {
        const long long waves = merge_waves(p, D);
        using M = std::conditional_t<std::is_base_of<ScoredParams, P>::value, ScoredParams, P>;
        M mp = p;
        for (mp.merge_wave0 = 0; mp.merge_wave0 < waves; mp.merge_wave0 += kMergeLaunchWaves) {
            const long long n = std::min(kMergeLaunchWaves, waves - mp.merge_wave0);
            const int wpb = D == 128 && p.splits <= 8 ? 2 : 4;  // waves per block: the kernel's 4 / RPW
            const dim3 grid((unsigned) ((n + wpb - 1) / wpb)), block(64 * wpb);
            if (p.part_gaps && p.splits <= 4) hipLaunchKernelGGL((prefill_merge_kernel<D, 4, true, M>), grid, block, 0, st, mp);
            else if (p.part_gaps && p.splits <= 8) hipLaunchKernelGGL((prefill_merge_kernel<D, 8, true, M>), grid, block, 0, st, mp);
            else if (p.splits <= 4) hipLaunchKernelGGL((prefill_merge_kernel<D, 4, false, M>), grid, block, 0, st, mp);
            else if (p.splits <= 8) hipLaunchKernelGGL((prefill_merge_kernel<D, 8, false, M>), grid, block, 0, st, mp);
            else hipLaunchKernelGGL((prefill_merge_kernel<D, 0, false, M>), grid, block, 0, st, mp);
        }
    }
}

}  // namespace
