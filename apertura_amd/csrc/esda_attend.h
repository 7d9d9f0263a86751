// esda_attend.h -- the decode attention kernel over a bf16 cache, the split merges and the host
// side that plans and launches them (gfx950), for the sources that build entry points on them:
// esda_decode.hip, and esda_scored_decode.hip (ScoredAttendParams); esda_prefix.hip takes its plan
// and checks.  What the kernels do is described at the head of esda_decode.hip.
#pragma once

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>
#include <type_traits>
#include <utility>

#include "esda.h"
#include "esda_device.h"
#include "esda_internal.h"
#include "esda_plan.h"
#include "esda_softcap.h"

namespace {

constexpr int kTile = 16;          // MFMA row block; split sizes are multiples of it
constexpr int kMaxGroup = 16;
constexpr int kTargetGroups = 256;  // one workgroup per MI355X CU; plans of two per CU aim at twice that
constexpr int kWaves256 = 4;        // waves per workgroup of the plain kernels at D = 256
constexpr int kOcc256 = 2;          // and their workgroups per CU
// The 512-dim shared stream's kernel is built with its ring in half the LDS (4 stages) although
// its plans place one workgroup per CU: see dispatch_attend.
constexpr int kOcc512Shared = 2;
constexpr int kMinRows = 64;        // fewest rows per workgroup the automatic plan gives
constexpr int kMinRowsOcc2 = 32;    // the same for grids of two workgroups per CU (C1: step
                                    // 8.3 -> 7.8 us with 32-row splits; 16 rows: 8.0)
constexpr int kMaxGroups = 16384;   // workgroups per launch
constexpr int kMaxBatch = 256;      // sequences per call (one per thread of the prefix scan)

// Per-sequence views, the prefix table, shares, segments and merge owners: the integer
// arithmetic of esda_plan.h (shared with the host tests).
using esda_plan::SeqView;
using esda_plan::seq_view;

struct AttendParams {
    const uint16_t *q, *k_new, *v_new;
    uint16_t *k_cache, *v_cache;
    const int *pos, *row_base;
    float *part_acc, *part_ml;
    int *status;
    long long seq_stride, head_stride;
    // Hkv and G count packed kv heads: a workgroup serves pk consecutive kv heads of one
    // sequence (gk query heads each) as one group of G = pk * gk query heads.
    int B, Hq, Hkv, G, cap, window, ring;
    int pk, gk;
    int balanced;      // 1: W balanced shares of all rows; 0: grid (S, Hkv, B) of chunk-row splits
    int W, S, chunk;
    float scale_log2e;
    long long *table;  // balanced: prefix sums of visible rows per sequence, for the merge
    uint16_t *out;     // written directly for (sequence, kv head) pairs of one segment
    // raw-K mode only
    const uint16_t *kw;
    const float *inv_freq;
    const unsigned *rope_tab;  // optional [rows][64] cos/sin pairs (esda_rope_table), row = cache row
    float eps;
    // q8 raw-K mode: u8 rows at q8 (strides as for k_cache, in bytes) and per-row scale /
    // bias at qsc / qbs[b * sb_seq_stride + kv head * sb_head_stride + row]
    unsigned char *q8;
    float *qsc, *qbs;
    long long sb_seq_stride, sb_head_stride;
};



// A step with modified scores (esda_scored.h): capped by `soft`, less slopes[head] log2 e per position
// of distance.
struct ScoredAttendParams : AttendParams {
    SoftCap soft;
    const float *slopes;
};
// .. with a wide cap (esda_softcap.h), in kernels of their own
struct WideScoredAttendParams : ScoredAttendParams {};

// ---------------------------------------------------------------- LDS ring layout
//
// A workgroup streams its rows through a ring of NS stages of 16 rows in LDS.  Rows
// arrive by LDS DMA (global_load_lds_dwordx4: 64 lanes x 16 B land contiguously at
// M0 + 16*lane), non-temporal, so in-flight data costs no registers and each
// instruction reads 1 KB of contiguous HBM.  One instruction carries RPI = 512/D rows:
// instruction i of a stage holds rows i + q*NI (q < RPI) in a 1056-byte block (1 KB +
// 32 B pad), sub-row q at +2D*q bytes.  The 32-byte pad (a measured choice: 16 B leaves
// both the 128-bit row reads and the transpose reads 2-way bank-conflicted on gfx950)
// makes both read patterns conflict-free with every address a base plus an immediate.
// LDSB: the LDS bytes of one workgroup.
template <int D, bool SHARED, int NW, int LDSB>
struct Ring {
    static constexpr int RPI = 512 / D;                     // rows per DMA instruction
    static constexpr int NI = 16 / RPI;                     // DMA instructions per stage
    static constexpr int CPR = D / 8;                       // 16-byte chunks per row
    static constexpr int BLK = 1056;                        // LDS bytes per DMA block
    static constexpr int TB = NI * BLK;                     // one tensor's stage
    static constexpr int SB = (SHARED ? 1 : 2) * TB;        // stage bytes (K [+ V])
    static constexpr int DW = D / NW;                       // dims per wave
    static constexpr int SL = DW / 8;                       // chunks per wave slice
    static constexpr int KKW = DW / 32;                     // QK k-steps per wave
    static constexpr int DTW = DW / 16;                     // PV dim tiles per wave
    static constexpr int DPT = NI / NW;                     // DMA per wave per tensor
    static constexpr int DPW = DPT * (SHARED ? 1 : 2);      // DMA per wave per stage
    static constexpr int XB = 2 * NW * 64 * 16;             // score-exchange bytes
    // reserve: kernel arguments' spill room (256 B) and the batch prefix scan (int64 per
    // sequence + one per wave)
    static constexpr int NS_ = (LDSB - XB - 256 - ((kMaxBatch + 1) + NW) * 8) / SB;
    static constexpr int NS = NS_ > 16 ? 16 : NS_;          // stages in the ring
    static_assert(DW % 32 == 0 && NI % NW == 0, "wave slices must cover whole MFMA steps");
    static_assert(NS >= 4, "the ring needs at least 4 stages");
    static_assert((NS - 3) * DPW <= 60, "vmcnt holds at most 63 outstanding loads");
    // Byte offset of (row r, chunk cin of wave slice ws) inside a tensor stage.
    __device__ static __forceinline__ int off(int r, int ws, int cin) {
        return (r % NI) * BLK + (r / NI) * 2 * D + (ws * SL + cin) * 16;
    }
};


// The segments of one launch's workgroup: grid plans give workgroup (split, kv head,
// sequence) rows [split * chunk, ...) of its pair; balanced plans give workgroup w its share
// of all visible rows of the batch, walked pair by pair (esda_plan.h).  segment(b, kvh, j0,
// j1, view, slot, direct) runs each; the ring is free again when it returns (the walk puts
// a barrier between segments).  NW: waves per workgroup; PAD: rows a pair counts beside its
// own in a balanced plan's shares.
template <int NW, int PAD = 0, class Seg>
__device__ __forceinline__ void walk_segments(const AttendParams &p, Seg &&segment) {
    const int wg = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    if (!p.balanced) {
        // Fixed splits (uniform lengths: one sequence, or windowed local layers): workgroup
        // (split, kvh, b) takes rows [split * chunk, (split + 1) * chunk) of its pair.
        const int split = blockIdx.x, kvh = blockIdx.y, b = blockIdx.z;
        const SeqView sv = seq_view(p.pos[b], p.row_base ? p.row_base[b] : 0, p.cap, p.window, p.ring);
        if (!sv.ok) {
            if (split == 0 && kvh == 0 && tid == 0) atomicAdd(p.status, 1);
            return;
        }
        int j0, j1;
        if (!esda_plan::grid_split(split, p.S, p.chunk, sv.nvis, &j0, &j1)) return;
        segment(b, kvh, j0, j1, sv, ((size_t) b * p.Hkv + kvh) * p.S + split, j0 == 0 && j1 == sv.nvis);
        return;
    }

    // Balanced shares (ragged batches).
    // Visible rows of every sequence and their exclusive prefix sums (the rows that
    // precede sequence b in the linearised order).  Up to 64 sequences every wave scans
    // the batch in its own lanes (no LDS, no barrier); larger batches (up to 256, one per
    // thread) go through LDS.
    __shared__ long long s_pref[kMaxBatch + 1];
    __shared__ long long s_wtot[NW];
    const bool single = p.B == 1;
    const bool wave_scan = p.B <= 64;
    long long w_incl = 0, w_nv = 0;  // wave scan: lane t's inclusive sum and rows of sequence t
    SeqView w_view{0, 0, 0, 0};
    long long rows_seq = 0;          // sum of visible rows over the batch
    if (single) {
        // one sequence: its view straight from the (wave-uniform) position word
        w_view = seq_view(p.pos[0], p.row_base ? p.row_base[0] : 0, p.cap, p.window, p.ring);
        rows_seq = w_view.ok ? w_view.nvis + PAD : 0;
        if (wg == 0 && tid == 0) {
            if (!w_view.ok) atomicAdd(p.status, 1);
            esda_plan::write_prefix_entry(p.table, 0, 1, 0, rows_seq);
        }
    } else {
        const int t = wave_scan ? lane : tid;
        SeqView v{0, 0, 0, 0};
        if (t < p.B) v = seq_view(p.pos[t], p.row_base ? p.row_base[t] : 0, p.cap, p.window, p.ring);
        const long long nv = v.ok ? v.nvis + PAD : 0;
        long long x = nv;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const long long y = __shfl_up(x, o);
            if (lane >= o) x += y;
        }
        if (wave_scan) {
            w_incl = x;
            w_nv = nv;
            w_view = v;
            rows_seq = __shfl(x, 63);
            if (wg == 0 && wave == 0) {
                if (t < p.B && !v.ok) atomicAdd(p.status, 1);
                esda_plan::write_prefix_entry(p.table, t, p.B, x - nv, rows_seq);
            }
        } else {
            if (lane == 63) s_wtot[wave] = x;
            __syncthreads();  // no DMA is in flight yet
            long long off = 0;
            for (int i = 0; i < wave; ++i) off += s_wtot[i];
            if (tid < p.B) s_pref[tid + 1] = off + x;
            if (tid == 0) s_pref[0] = 0;
            if (wg == 0 && tid < p.B && !v.ok) atomicAdd(p.status, 1);
            __syncthreads();
            // B + 1 entries (B may be 256 = one per thread): the total goes in separately
            if (wg == 0) esda_plan::write_prefix_entry(p.table, tid, p.B, tid < p.B ? s_pref[tid] : 0, s_pref[p.B]);
            rows_seq = s_pref[p.B];
        }
    }
    const long long rows_total = rows_seq * p.Hkv;
    // Rows before sequence b (b <= B) and its view; the same in every lane.
    auto lane64 = [](long long v, int l) {
        const unsigned lo = __builtin_amdgcn_readlane((unsigned) v, l);
        const unsigned hi = __builtin_amdgcn_readlane((unsigned) ((unsigned long long) v >> 32), l);
        return (long long) (((unsigned long long) hi << 32) | lo);
    };
    auto pref_at = [&](int b) -> long long {
        if (single) return b == 0 ? 0 : rows_seq;
        if (!wave_scan) return s_pref[b];
        return b >= p.B ? rows_seq : lane64(w_incl - w_nv, b);
    };
    auto view_at = [&](int b) -> SeqView {
        if (single) return w_view;
        if (!wave_scan) return seq_view(p.pos[b], p.row_base ? p.row_base[b] : 0, p.cap, p.window, p.ring);
        return SeqView{__builtin_amdgcn_readlane(w_view.nvis, b), __builtin_amdgcn_readlane(w_view.first, b),
                       __builtin_amdgcn_readlane(w_view.newrow, b), __builtin_amdgcn_readlane(w_view.ok, b)};
    };

    // This workgroup's share of all visible rows, linearised as (sequence, kv head, row):
    // [rows_total * wg / Wr, rows_total * (wg + 1) / Wr) with Wr = min(W, rows_total), so
    // that every share holds at least one row (W is sized from the bound on rows; early in
    // a long cache fewer rows are visible) and workgroups wg >= Wr have nothing to do.  A
    // share covers one or more segments; the partial of workgroup wg for pair
    // u = b * Hkv + kvh goes to slot u + wg, so the slots of one pair are consecutive and
    // distinct pairs never share a slot.
    const int Wr = esda_plan::active_shares(rows_total, p.W);
    if (wg >= Wr) return;
    const long long lo = esda_plan::share_begin(rows_total, Wr, wg), hi = esda_plan::share_begin(rows_total, Wr, wg + 1);
    long long x = lo;
    int b = 0;
    while (x < hi) {
        // the sequence holding row x (x < rows_total): the count of sequences that end at
        // or before it
        if (single) {
            b = 0;
        } else if (wave_scan) {
            b = __popcll(__ballot(lane < p.B && w_incl * p.Hkv <= x));
        } else {
            while (pref_at(b + 1) * p.Hkv <= x) ++b;
        }
        const long long pb = pref_at(b);
        const int n = (int) (pref_at(b + 1) - pb);
        const esda_plan::Segment sg = esda_plan::segment_at(x, hi, pb * p.Hkv, n);
        const int kvh = sg.kvh, j0 = sg.j0, j1 = sg.j1;
        const long long seg_end = sg.end;
        const SeqView v = view_at(b);
        // Every value of the segment is the same in all lanes (computed from LDS and kernel
        // arguments); saying so keeps the ring's control flow and addresses scalar.
        const SeqView sv{uniform(v.nvis), uniform(v.first), uniform(v.newrow), uniform(v.ok)};
        const int ub = uniform(b), ukvh = uniform(kvh), uj0 = uniform(j0);
        const int uj1 = PAD ? min(uniform(j1), sv.nvis) : uniform(j1), un = PAD ? sv.nvis : n;
        if (PAD == 0 || uj0 < un) {
            segment(ub, ukvh, uj0, uj1, sv, (size_t) esda_plan::share_slot((long long) ub * p.Hkv + ukvh, wg),
                    uj0 == 0 && uj1 == un);
            lds_barrier();  // every wave is done with the ring before the next segment refills it
        }
        x = seg_end;
    }
}

// --------------------------------------------------------------------- attend kernel
//
// grid (splits, kv heads, sequences), NW waves per workgroup, the ring in 1/OCC of
// the LDS (so that OCC workgroups fit per CU).  A workgroup owns `chunk` consecutive visible rows
// of one (sequence, kv head) and streams them through the LDS ring in 16-row stages.
// When each pair needs one split and pairs are plentiful, pk = 2 or 4 kv heads of a
// sequence share a workgroup:
// a stage then holds 16 / pk rows of each, their query heads fill the MFMA N dimension
// side by side, and scores of a head against another kv head's rows are masked.
// Ragged batches use balanced shares instead: workgroup w takes rows
// [total * w / W, total * (w + 1) / W) of all visible rows linearised by (sequence, kv
// head, row), one segment per pair it touches.  The head dim is split
// across the waves: per stage, each wave forms partial scores S^T[16 rows x 16 heads]
// over its dims with v_mfma_f32_16x16x32_bf16 (the GQA group is the MFMA N dimension,
// zero-padded to 16, so each K/V byte is read from HBM once per group), the partials
// are summed through LDS, every wave runs the same online softmax, and each wave
// accumulates O^T for its own dims with v_mfma_f32_16x16x16_bf16 (V^T from LDS by
// transpose reads).  One barrier per stage: the scores of stage s+1 are formed while
// stage s is accumulated.  With attention_k_eq_v the V rows are the K rows in LDS.
//
// The new token's row is copied from k_new/v_new into the cache by the workgroup whose
// split ends at it (bit-exact copy); that workgroup's own loads read the row from
// k_new/v_new and no other workgroup reads it, so the copy needs no ordering.
//
// P = ScoredAttendParams: the four scores a lane holds of a stage are capped and biased before
// the softmax; row j of the visible ones lies nvis - 1 - j positions behind the token.  (Wide caps
// as a branch here: 16 sequences of 1024 .. 8192 rows of 512 dims 64 us -> 68, capped 72.)
template <int D, bool SHARED, int NW, int OCC = 1, class P = AttendParams>
// The LDS ring allows OCC workgroups per CU, i.e. OCC * NW/4 waves per SIMD: telling the
// compiler so lifts the register limit it would otherwise keep for higher occupancy,
// which it meets by serialising LDS reads behind their uses.  (Plans may still place one
// workgroup per CU on a kernel built with OCC = 2: its shallower ring is what they want.)
__global__ __attribute__((amdgpu_flat_work_group_size(64 * NW, 64 * NW), amdgpu_waves_per_eu(OCC * NW / 4, OCC * NW / 4)))
void attend_kernel(P p) {
    constexpr bool SCORED = std::is_base_of<ScoredAttendParams, P>::value;
    constexpr bool WIDE = std::is_same<P, WideScoredAttendParams>::value;
    using R = Ring<D, SHARED, NW, 160 * 1024 / OCC>;
    // D = 512 exchanges only the live heads' partial scores (the padding columns are zero)
    constexpr bool kLiveX = D == 512;
    constexpr int NS = R::NS, DW = R::DW, KKW = R::KKW, DTW = R::DTW;
    constexpr int DPW = R::DPW;  // DMA instructions per wave per stage
    static_assert(NS >= 4, "the ring must hold the look-ahead stage and one in flight");
    // Distinct arrays per stage: the compiler tracks DMA completion per LDS object, so a
    // read of stage u only waits for stage u's DMA, never for the stages behind it.
    __shared__ __attribute__((aligned(16))) unsigned char r0[R::SB], r1[R::SB], r2[R::SB], r3[R::SB],
        r4[R::SB], r5[R::SB], r6[R::SB], r7[R::SB], r8[R::SB], r9[R::SB], r10[R::SB], r11[R::SB],
        r12[R::SB], r13[R::SB], r14[R::SB], r15[R::SB];
    // Stage buffer u (a compile-time index).
    auto ring = [&](auto uc) -> unsigned char * {
        constexpr int u = decltype(uc)::value % NS;
        if constexpr (u == 0) return r0;
        else if constexpr (u == 1) return r1;
        else if constexpr (u == 2) return r2;
        else if constexpr (u == 3) return r3;
        else if constexpr (u == 4) return r4;
        else if constexpr (u == 5) return r5;
        else if constexpr (u == 6) return r6;
        else if constexpr (u == 7) return r7;
        else if constexpr (u == 8) return r8;
        else if constexpr (u == 9) return r9;
        else if constexpr (u == 10) return r10;
        else if constexpr (u == 11) return r11;
        else if constexpr (u == 12) return r12;
        else if constexpr (u == 13) return r13;
        else if constexpr (u == 14) return r14;
        else return r15;
    };
    __shared__ f32x4 xch[2][NW][64];  // partial scores, double-buffered by stage parity
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 15, lg = lane >> 4;

    // Packed kv heads: a stage holds RPP = 16 / pk rows of each of the pk kv heads (stage
    // row r belongs to kv head r / RPP, row r % RPP of the stage's row range).  pk is 1, 2
    // or 4 and the same in every lane (scored steps: 1).
    const int pk = SCORED ? 1 : uniform(p.pk);
    const int lrpp = 4 - __builtin_ctz(pk), RPP = 1 << lrpp;
    // Query head li belongs to kv head li / gk of the group (padding heads li >= G take
    // the last); the C rows 4lg .. 4lg+3 of this lane come from one kv head (RPP >= 4).
    const bool hmatch = ((4 * lg) >> lrpp) == min(li / p.gk, pk - 1);
    const int jl = (4 * lg) & (RPP - 1);

    // One segment: rows [j0, j1) of (sequence b, packed kv head kvh).  `slot` indexes its
    // partial; `direct` means the segment is the whole pair and writes the output itself.
    auto segment = [&](const int b, const int kvh, const int j0, const int j1, const SeqView sv,
                       const size_t slot, const bool direct) {
    const bool append = p.k_new != nullptr;

    // kv head kvh * pk + i of sequence b sits at head_off + i * head_stride
    const size_t head_off = (size_t) b * p.seq_stride + (size_t) kvh * pk * p.head_stride;
    uint16_t *kbase = p.k_cache + head_off;
    uint16_t *vbase = p.v_cache + head_off;
    const uint16_t *knew = append ? p.k_new + ((size_t) b * p.Hkv + kvh) * pk * D : nullptr;
    const uint16_t *vnew = SHARED ? knew : p.v_new + ((size_t) b * p.Hkv + kvh) * pk * D;
    auto qk_chunk = [&](int kk) { return wave * KKW + kk; };  // 32-dim chunk of QK k-step kk of this wave

    // Q^T operand for this wave's dims: lane (li, lg) = head li, dims 32*chunk + 8lg .. +8
    // (zero for heads >= G).
    bf16x8 qv[KKW];
    {
        const bool qok = li < p.G;
        const uint16_t *qrow = p.q + ((size_t) b * p.Hq + (size_t) kvh * p.G + (qok ? li : 0)) * D + lg * 8;
#pragma unroll
        for (int kk = 0; kk < KKW; ++kk) {
            const u32x4 t = qok ? *reinterpret_cast<const u32x4 *>(qrow + 32 * qk_chunk(kk)) : u32x4{0u, 0u, 0u, 0u};
            qv[kk] = __builtin_bit_cast(bf16x8, t);
        }
    }
    float slope = 0.0f;  // of this lane's head, log2 units
    if constexpr (SCORED) {
        if (p.slopes && li < p.G) slope = p.slopes[kvh * p.G + li] * kLog2e;
    }
    ESDA_WAIT_VM(0);  // operands are in registers before the ring starts counting its own loads

    // DMA source slot of this lane: sub-row dq, chunk dchunk of the row.
    const int dq = lane / R::CPR, dchunk = lane % R::CPR;
    const int nst = (j1 - j0 + RPP - 1) >> lrpp;
    // Per-lane byte offsets of this wave's DMA slots inside a stage's row range (stage row
    // r: kv head r / RPP of the group, row r % RPP; below 2^31 bytes, checked by the host).
    unsigned dvoff[R::DPT];
#pragma unroll
    for (int t = 0; t < R::DPT; ++t) {
        const int r = wave * R::DPT + t + dq * R::NI;
        dvoff[t] = (unsigned) ((size_t) (r >> lrpp) * p.head_stride * 2 + (size_t) (r & (RPP - 1)) * D * 2 + dchunk * 16);
    }
    // DMA of stage st into ring buffer `buf`.
    auto dma = [&](int st, unsigned char *buf) {
        const int jst = j0 + st * RPP;
        if (jst + RPP < j1 && sv.first + jst + RPP <= p.cap) {
            // Interior stage: RPP consecutive cache rows per kv head, none clamped or new.
            const uint16_t *kb = kbase + (size_t) (sv.first + jst) * D;
            const uint16_t *vb = vbase + (size_t) (sv.first + jst) * D;
#pragma unroll
            for (int t = 0; t < R::DPT; ++t) {
                const int i = wave * R::DPT + t;
                lds_dma16_s(kb, dvoff[t], lds_addr(buf) + i * R::BLK);
                if constexpr (!SHARED) lds_dma16_s(vb, dvoff[t], lds_addr(buf) + R::TB + i * R::BLK);
            }
            return;
        }
#pragma unroll
        for (int t = 0; t < R::DPT; ++t) {
            const int i = wave * R::DPT + t;           // DMA block of this stage
            const int sr = i + dq * R::NI;             // stage row this lane feeds
            const int pr = sr >> lrpp;                  // its kv head within the group
            const int j = jst + (sr & (RPP - 1));       // its logical row
            const int jj = j < j1 ? j : j1 - 1;          // clamp: masked rows read a visible row
            int r = sv.first + jj;
            if (r >= p.cap) r -= p.cap;
            const bool from_new = append && (jj == sv.nvis - 1);
            const size_t hoff = (size_t) pr * p.head_stride + (size_t) r * D;
            const uint16_t *ks = (from_new ? knew + pr * D : kbase + hoff) + dchunk * 8;
            lds_dma16(ks, lds_addr(buf) + i * R::BLK);
            if constexpr (!SHARED) {
                const uint16_t *vs = (from_new ? vnew + pr * D : vbase + hoff) + dchunk * 8;
                lds_dma16(vs, lds_addr(buf) + R::TB + i * R::BLK);
            }
        }
    };
    // Per-lane LDS offsets: the QK A operand (row li, chunk qk_chunk(kk), 16 bytes at
    // 8lg dims) and the V^T transpose read (lane (li, lg) supplies row 4lg + li/4, dims
    // wave*DW + 16dt + 4(li%4) .. +4; ds_read_b64_tr_b16 hands lane li of the group dim
    // 16dt + li of rows 4lg .. 4lg+3, the PV A operand).
    const int qk_off = R::off(li, 0, 0) + lg * 16;                     // + 64*qk_chunk(kk)
    const int tr_off = R::off(4 * lg + li / 4, wave, 0) + (li % 4) * 8;  // + 32*dt
    constexpr int VOFF = SHARED ? 0 : R::TB;

    float m = kNoScore, l = 0.0f;
    f32x4 acc[DTW];
#pragma unroll
    for (int dt = 0; dt < DTW; ++dt) acc[dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    // Partial scores of a stage over this wave's dims, published for the other waves.
    auto qk_partial = [&](const unsigned char *kb, int par) {
        f32x4 sp = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int kk = 0; kk < KKW; ++kk) {
            const bf16x8 a = *reinterpret_cast<const bf16x8 *>(kb + qk_off + 64 * qk_chunk(kk));
            sp = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, qv[kk], sp, 0, 0, 0);
        }
        // D = 512: only the live heads' columns (lanes li < G) are exchanged; the padding
        // heads' partials are zero (their Q^T operand is)
        if (!kLiveX || li < p.G) xch[par][wave][lane] = sp;
    };

    // Prologue: fill NS-1 stages; the first stage's scores.
    unroll<NS - 1>([&](auto uc) {
        constexpr int u = decltype(uc)::value;
        if (u < nst) dma(u, ring(uc));
    });
    if (nst - 1 >= NS - 2) {
        ESDA_WAIT_VM((NS - 2) * DPW);
    } else {
        ESDA_WAIT_VM(0);
    }
    lds_barrier();
    qk_partial(ring(std::integral_constant<int, 0>{}), 0);

    // Iteration st: one barrier, after which (a) every wave's stage-st partial scores
    // are in xch, (b) stage st+1 has landed from every wave's DMA, and (c) every wave
    // is done with stage st-1's buffer, which is refilled at once.  The scores of stage
    // st+1 are computed alongside stage st's PV, so the two dependency chains overlap.
    auto stage = [&](int s0, auto uc) {
        constexpr int u = decltype(uc)::value;
        const int st = s0 + u;
        if (st >= nst) return;
        if (st + 1 < nst) {
            // own DMA for stage st+1 done; the stages behind it may stay in flight --
            // except at D = 256, whose two workgroups per CU then keep twice the 512-dim
            // kernel's bytes in flight (16.8 MB over the GPU, past the 6-15 MB at which the
            // read probe peaks): waiting for every issued stage there took C5 7.50 -> 7.44 ms
            if (D != 256 && nst - st - 2 >= NS - 3) {
                ESDA_WAIT_VM((NS - 3) * DPW);
            } else {
                ESDA_WAIT_VM(0);
            }
        }
        lds_barrier();
        if (st + NS - 1 < nst) dma(st + NS - 1, ring(std::integral_constant<int, (u + NS - 1) % NS>{}));
        f32x4 sc = {0.0f, 0.0f, 0.0f, 0.0f};
        if (!kLiveX || li < p.G) {
            sc = xch[st & 1][0][lane];
#pragma unroll
            for (int w = 1; w < NW; ++w) sc += xch[st & 1][w][lane];
        }
        // V^T operands of this stage, read behind the exchange so that
        // their latency hides under the softmax instead of following it
        const unsigned char *vb = ring(uc) + VOFF;
        short4v va[DTW];
#pragma unroll
        for (int dt = 0; dt < DTW; ++dt)
            va[dt] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) short4v *) (vb + tr_off + 32 * dt));
        // The look-ahead work runs unconditionally (one basic block with the softmax, so
        // the two interleave): past the last stage it reads stale but in-bounds LDS and
        // writes exchange slots that are never read again.
        qk_partial(ring(std::integral_constant<int, (u + 1) % NS>{}), (st + 1) & 1);
        // Online softmax (log2 domain), identical in every wave; rows past the split
        // end (last stage only) and rows of another kv head of the group are masked.
        const int jt = j0 + st * RPP + jl;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float x = sc[r] * p.scale_log2e;
            if constexpr (SCORED) {
                if constexpr (WIDE) x = capped_wide(sc[r], x, p.soft);
                else if (p.soft.out != 0.0f) x = capped_narrow(sc[r], p.soft);
                x = __builtin_fmaf(-slope, (float) (sv.nvis - 1 - jt - r), x);
            }
            sc[r] = hmatch && (jt + r) < j1 ? x : -INFINITY;
        }
        if constexpr (SCORED) {
            // rows past the end repeat the last one: with a weight of 0, but 0 x inf is NaN
            if (st + 1 == nst) {
#pragma unroll
                for (int dt = 0; dt < DTW; ++dt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) va[dt][r] = jt + r < j1 ? va[dt][r] : (short) 0;
            }
        }
        const float tmax = wave_max_across_groups(fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3])));
        if (__any(tmax > m + kRescaleSlack)) {
            const float mnew = fmaxf(m, tmax);
            const float corr = __builtin_amdgcn_exp2f(m - mnew);
            l *= corr;
#pragma unroll
            for (int dt = 0; dt < DTW; ++dt) acc[dt] *= corr;
            m = mnew;
        }
        short4v pbs;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const __bf16 pr = (__bf16) __builtin_amdgcn_exp2f(sc[r] - m);
            l += (float) pr;
            pbs[r] = __builtin_bit_cast(short, pr);
        }
        // O^T (this wave's dims) += V^T . P^T
#pragma unroll
        for (int dt = 0; dt < DTW; ++dt)
            acc[dt] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(va[dt], pbs, acc[dt], 0, 0, 0);
    };
    for (int s0 = 0; s0 < nst; s0 += NS) unroll<NS>([&](auto uc) { stage(s0, uc); });

    // Fused append: the workgroup whose rows end at the new token copies k_new / v_new
    // into its cache row (bit-exact).  Its own DMA reads that row from k_new / v_new and
    // no other workgroup reads it; the copy runs after this workgroup's ring has
    // drained, so no outstanding load is counted against the ring's waits.
    if (append && j1 == sv.nvis) {
        for (int pr = wave; pr < pk; pr += NW) {  // wave pr copies kv head pr of the group
            const size_t row = (size_t) pr * p.head_stride + (size_t) sv.newrow * D;
            for (int c = lane; c < D / 8; c += 64) {
                *reinterpret_cast<u32x4 *>(kbase + row + c * 8) =
                    *reinterpret_cast<const u32x4 *>(knew + pr * D + c * 8);
                if constexpr (!SHARED)
                    *reinterpret_cast<u32x4 *>(vbase + row + c * 8) =
                        *reinterpret_cast<const u32x4 *>(vnew + pr * D + c * 8);
            }
        }
    }

    // Partial of this split: every wave holds the same (m, l) and its own dim slice.
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (direct) {
        // The only segment of this (sequence, kv head): normalise here, with the merge's
        // arithmetic (acc * (1 / l), then bf16); the merge skips this pair.
        if (li < p.G) {
            const float inv = 1.0f / l;
            uint16_t *dst = p.out + ((size_t) b * p.Hq + (size_t) kvh * p.G + li) * D + wave * DW;
#pragma unroll
            for (int dt = 0; dt < DTW; ++dt) {
                bf16x4 r;
#pragma unroll
                for (int e = 0; e < 4; ++e) r[e] = (__bf16) (acc[dt][e] * inv);
                *reinterpret_cast<uint2 *>(dst + 16 * dt + 4 * lg) = __builtin_bit_cast(uint2, r);
            }
        }
        return;
    }
    if (li < p.G) {
        const size_t pidx = slot * p.G + li;
        float *dst = p.part_acc + pidx * D + wave * DW;
        // D = 512: the partials are stored non-temporal (the merge reads them from another
        // XCD; C4 step 82.2 -> 81.2 us, C2 14.7 -> 14.2).  The short D = 256 launches finish
        // sooner with write-back stores (C1 attend 5.4 against 5.8 us).
        if constexpr (D == 512) {
#pragma unroll
            for (int dt = 0; dt < DTW; ++dt) __builtin_nontemporal_store(acc[dt], reinterpret_cast<f32x4 *>(dst + 16 * dt + 4 * lg));
            if (wave == 0 && lg == 0) __builtin_nontemporal_store(f32x2{m, l}, reinterpret_cast<f32x2 *>(p.part_ml + pidx * 2));
        } else {
#pragma unroll
            for (int dt = 0; dt < DTW; ++dt) *reinterpret_cast<f32x4 *>(dst + 16 * dt + 4 * lg) = acc[dt];
            if (wave == 0 && lg == 0) *reinterpret_cast<f32x2 *>(p.part_ml + pidx * 2) = f32x2{m, l};
        }
    }
    };

    walk_segments<NW>(p, segment);
}

struct MergeParams {
    const float *part_acc, *part_ml;
    const long long *table;
    const int *pos, *row_base;
    uint16_t *out;
    int B, Hq, Hkv, G, D, cap, window, ring;
    int balanced, W, S, chunk;
    int pad;  // balanced: rows a pair counted beside its own (walk_segments' PAD)
};

constexpr int kMergeThreads = 256;
constexpr int kMergeDims = 64;      // output dims per merge workgroup (16 lanes x float4)
constexpr int kMergeGroups = kMergeThreads / (kMergeDims / 4);  // split groups reduced in parallel (16)

// Cross-split merge (ESDecodeAttn.mm:253-273 restated in the log2 domain):
// M = max_s m_s; O = sum_s acc_s 2^(m_s - M) / sum_s l_s 2^(m_s - M).
// One workgroup per (sequence, query head, 64 output dims); 16 split groups x 16 float4
// lanes.  Each thread issues its partial loads together with the (m, l) loads, so the
// whole merge is one memory round trip; each split group weighs its splits against its
// own max, and the final sum over the groups rescales them to the largest (no block-wide
// reduction before the weights).  (Against 128 dims x 8 groups, the narrower workgroups and one 8-byte
// (m, l) load per split took 1.8 us off the C4 step and 1.2 us off C2's.)
// REGS: splits per thread held in registers (S <= 16 * REGS in one pass): 4, or 16 for
// more splits (the raw-K C4 shape packs two kv heads into 128 splits).

// The splits that hold partials of pair (b, kvh): their count ns (0 when the sequence
// is skipped) and the slot of the first, as the attend kernel laid them out.
__device__ __forceinline__ int pair_splits(const MergeParams &p, int b, int kvh, size_t &pbase) {
    int ns;
    if (p.balanced) {
        // The attend workgroups w0 .. w1 that covered pair (b, kvh) (every one of them holds
        // rows of the pair and wrote its slot); an inconsistent table reads nothing.
        int w0 = 0;
        ns = esda_plan::pair_owners(p.table[b], p.table[b + 1], p.table[p.B], p.Hkv, kvh, p.W, &w0, p.pad);
        if (ns == 0) return 0;
        pbase = (size_t) esda_plan::share_slot((long long) b * p.Hkv + kvh, w0);
    } else {
        const SeqView sv = seq_view(p.pos[b], p.row_base ? p.row_base[b] : 0, p.cap, p.window, p.ring);
        if (!sv.ok) return 0;
        ns = esda_plan::grid_splits(sv.nvis, p.chunk, p.S);
        pbase = ((size_t) b * p.Hkv + kvh) * p.S;
    }
    return ns;
}

template <int REGS>
__global__ __launch_bounds__(kMergeThreads) void merge_kernel(MergeParams p) {
    __shared__ f32x4 part[kMergeGroups][kMergeDims / 4];
    __shared__ float lsum[kMergeGroups], gmax[kMergeGroups];
    const int h = blockIdx.y, b = blockIdx.z;
    const int kvh = h / p.G, g = h % p.G;
    const int tid = threadIdx.x;
    size_t pbase;
    const int ns = pair_splits(p, b, kvh, pbase);
    if (ns <= 1) return;  // one workgroup covered the pair and wrote the output itself
    const int dq = tid % (kMergeDims / 4), sg = tid / (kMergeDims / 4);
    const int d0 = blockIdx.x * kMergeDims + dq * 4;

    float mloc = -INFINITY;
    float ms[REGS], ls[REGS];
    f32x4 av[REGS];
    // Fast path: every split this thread owns fits in registers.
    const bool in_regs = ns <= kMergeGroups * REGS;
    if (in_regs) {
#pragma unroll
        for (int u = 0; u < REGS; ++u) {
            const int s = sg + u * kMergeGroups;
            if (s < ns) {
                const size_t ix = (pbase + s) * p.G + g;
                av[u] = *reinterpret_cast<const f32x4 *>(p.part_acc + ix * p.D + d0);
                const f32x2 ml = *reinterpret_cast<const f32x2 *>(p.part_ml + ix * 2);
                ms[u] = ml[0];
                ls[u] = ml[1];
            } else {
                av[u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                ms[u] = -INFINITY;
                ls[u] = 0.0f;
            }
            mloc = fmaxf(mloc, ms[u]);
        }
    } else {
        for (int s = sg; s < ns; s += kMergeGroups) mloc = fmaxf(mloc, p.part_ml[((pbase + s) * p.G + g) * 2]);
    }
    // Each split group combines its splits against its own max (the same in the group's 16
    // lanes: m is per split); the groups are rescaled to their common max in the final sum.
    const float mx = mloc == -INFINITY ? 0.0f : mloc;  // a group without splits: weights 0

    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    float lt = 0.0f;
    if (in_regs) {
#pragma unroll
        for (int u = 0; u < REGS; ++u) {
            const float w = __builtin_amdgcn_exp2f(ms[u] - mx);  // 0 for absent splits
            o += av[u] * w;
            lt += ls[u] * w;
        }
    } else {
        for (int s = sg; s < ns; s += kMergeGroups) {
            const size_t ix = (pbase + s) * p.G + g;
            const float w = __builtin_amdgcn_exp2f(p.part_ml[ix * 2] - mx);
            o += *reinterpret_cast<const f32x4 *>(p.part_acc + ix * p.D + d0) * w;
            lt += p.part_ml[ix * 2 + 1] * w;
        }
    }
    part[sg][dq] = o;
    if (dq == 0) {
        lsum[sg] = lt;
        gmax[sg] = mloc;
    }
    __syncthreads();
    if (tid < kMergeDims / 4) {
        float M = gmax[0];
#pragma unroll
        for (int u = 1; u < kMergeGroups; ++u) M = fmaxf(M, gmax[u]);
        f32x4 t = {0.0f, 0.0f, 0.0f, 0.0f};
        float l = 0.0f;
#pragma unroll
        for (int u = 0; u < kMergeGroups; ++u) {
            // a group with no split (its max -inf) adds nothing
            const float c = gmax[u] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(gmax[u] - M);
            t += part[u][tid] * c;
            l += lsum[u] * c;
        }
        const float inv = 1.0f / l;
        uint16_t *dst = p.out + ((size_t) b * p.Hq + h) * p.D + blockIdx.x * kMergeDims + tid * 4;
        bf16x4 r;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = (__bf16) (t[e] * inv);
        *reinterpret_cast<uint2 *>(dst) = __builtin_bit_cast(uint2, r);
    }
}

// Merge for pairs of few splits: one thread per (sequence,
// query head, 4 output dims), no barriers.  Splits are read 8 at a time -- the loads of
// a chunk issue together, so up to 8 splits cost one memory round trip -- with the
// running max raised per chunk (same result as merge_kernel up to summation order).
constexpr int kMergeRowsThreads = 256;
constexpr int kMergeShares = 6;  // balanced shares per pair from which merge_kernel is the faster merge
constexpr int kMergeRowsChunk = 8;

__global__ __launch_bounds__(kMergeRowsThreads) void merge_rows_kernel(MergeParams p) {
    const int D4 = p.D / 4;
    const int t = blockIdx.x * kMergeRowsThreads + threadIdx.x;
    const int b = blockIdx.y;
    if (t >= p.Hq * D4) return;
    const int h = t / D4, d4 = t - (t / D4) * D4;
    const int kvh = h / p.G, g = h % p.G;
    size_t pbase;
    const int ns = pair_splits(p, b, kvh, pbase);
    if (ns <= 1) return;  // written by the attend kernel, or skipped
    float mx = -INFINITY, lt = 0.0f;
    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
    for (int s0 = 0; s0 < ns; s0 += kMergeRowsChunk) {
        float mv[kMergeRowsChunk], lv[kMergeRowsChunk];
        f32x4 av[kMergeRowsChunk];
#pragma unroll
        for (int u = 0; u < kMergeRowsChunk; ++u) {
            mv[u] = -INFINITY;
            lv[u] = 0.0f;
            av[u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if (s0 + u < ns) {
                const size_t ix = (pbase + s0 + u) * p.G + g;
                mv[u] = p.part_ml[ix * 2];
                lv[u] = p.part_ml[ix * 2 + 1];
                av[u] = *reinterpret_cast<const f32x4 *>(p.part_acc + ix * p.D + d4 * 4);
            }
        }
        float cm = mv[0];
#pragma unroll
        for (int u = 1; u < kMergeRowsChunk; ++u) cm = fmaxf(cm, mv[u]);
        const float mn = fmaxf(mx, cm);
        const float c = __builtin_amdgcn_exp2f(mx - mn);  // 0 on the first chunk
        o *= c;
        lt *= c;
#pragma unroll
        for (int u = 0; u < kMergeRowsChunk; ++u) {
            const float w = __builtin_amdgcn_exp2f(mv[u] - mn);  // 0 for absent splits
            o += av[u] * w;
            lt += lv[u] * w;
        }
        mx = mn;
    }
    const float inv = 1.0f / lt;
    bf16x4 r;
#pragma unroll
    for (int e = 0; e < 4; ++e) r[e] = (__bf16) (o[e] * inv);
    *reinterpret_cast<uint2 *>(p.out + ((size_t) b * p.Hq + h) * p.D + d4 * 4) = __builtin_bit_cast(uint2, r);
}


// ------------------------------------------------------------------------ host side

int fail(int code, const std::string &msg) {
    esda_detail::set_error(msg);
    return code;
}


int hip_fail(hipError_t e, const char *what) {
    return fail(ESDA_ERR_HIP, std::string(what) + ": " + hipGetErrorString(e));
}

bool aligned16(const void *ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0; }

struct Plan {
    int G, maxvis, balanced, W, S, chunk;
    int pk;   // kv heads packed per workgroup (the kernels see Hkv / pk heads of G * pk)
    int per_cu;  // attend workgroups per CU the plan is sized for (1 or 2)
    size_t off_table, off_ml, off_acc, bytes;
};

// Kv heads per workgroup for a grid of one split per (sequence, kv head): with several
// workgroups' worth of pairs per CU, packing pk kv heads (pk * G <= 16 query heads, the
// MFMA's N dimension) gives each workgroup one pk-times longer stream instead of pk short
// ones, each of which would pay the ring's fill and drain.  Local layers (G = 2) at C5's
// batch: 512 pairs -> 256 workgroups of two kv heads.
int choose_pack(const esda_decode_desc *d, int G, long long S, int target) {
    const long long pairs = (long long) d->batch * d->num_kv_heads;
    int pk = 1;
    while (pk < 4 && S == 1 && G * pk * 2 <= kMaxGroup && d->num_kv_heads % (pk * 2) == 0 &&
           pairs / (pk * 2) >= target &&
           (long long) d->head_stride * 2 * (pk * 2) + 16LL * d->head_dim * 2 < (1LL << 31))
        pk *= 2;
    return pk;
}

// raw: the raw-K kernels take one kv head per workgroup.
int make_plan(const esda_decode_desc *d, Plan *pl, bool raw = false) {
    if (!d) return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode: null description");
    if (d->batch <= 0 || d->num_q_heads <= 0 || d->num_kv_heads <= 0)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode: batch and head counts must be positive");
    if (d->batch > kMaxBatch)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode: at most 256 sequences per call");
    if (d->head_dim != 128 && d->head_dim != 256 && d->head_dim != 512)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode: head_dim must be 128, 256 or 512");
    if (d->num_q_heads % d->num_kv_heads)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode: num_q_heads must be a multiple of num_kv_heads");
    const int G = d->num_q_heads / d->num_kv_heads;
    if (G > kMaxGroup)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode: at most 16 query heads per kv head");
    if (d->cap <= 0) return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode: cap must be positive");
    if (d->window < 0) return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode: window must be >= 0");
    if (d->ring && (d->window <= 0 || d->window > d->cap))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode: ring mode needs 0 < window <= cap");
    if (d->head_stride < (int64_t) d->cap * d->head_dim || (d->head_stride % 8) != 0)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode: head_stride must be >= cap*head_dim and a multiple of 8");
    if (d->seq_stride < (int64_t) d->num_kv_heads * d->head_stride || (d->seq_stride % 8) != 0)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode: seq_stride must be >= num_kv_heads*head_stride and a multiple of 8");
    if (d->split_rows < 0 || (d->split_rows % kTile) != 0)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode: split_rows must be a multiple of 16");
    int bound = d->ring ? d->window : (d->window > 0 ? std::min(d->window, d->cap) : d->cap);
    int maxvis = d->max_visible > 0 ? std::min(d->max_visible, bound) : bound;
    // Several full-causal sequences have ragged lengths: workgroups then take balanced
    // shares of all rows (the kernel scans the lengths).  Otherwise (one sequence, or
    // windowed local layers whose lengths are nearly equal) a plain grid of fixed splits
    // per (sequence, kv head) starts faster.
    pl->balanced = d->batch > 1 && !d->ring;
    // Workgroups per CU: two at D = 256 (C5 step 7.47 ms against 7.58 with plans of one per
    // CU), else one.  At D = 512 two per CU measured slower on grid plans (twice the splits
    // cost more in the merge than they gain: C4 step 82.7 -> 85.1 us) and on balanced shares
    // (C5 7.64 against 7.52 ms with 256 shares).
    pl->per_cu = (!raw && d->head_dim == 256) ? kOcc256 : 1;
    const int target = pl->per_cu * kTargetGroups;  // workgroups that fill the GPU
    pl->pk = 1;
    // Work split.  Sizing uses the upper bound on rows (the kernels see the real ones),
    // counted per packed kv head (a row of a pk-packed head is pk cache rows).
    // Automatic: about one workgroup per CU, no fewer than 64 rows each; split_rows > 0
    // asks for that many rows per workgroup.
    const long long rows_max = (long long) maxvis * d->batch * (d->num_kv_heads / pl->pk);
    const long long per = d->split_rows > 0 ? d->split_rows : kMinRows;
    pl->G = G;
    pl->maxvis = maxvis;
    size_t slots;
    if (pl->balanced) {
        long long W = (rows_max + per - 1) / per;
        if (d->split_rows == 0 && W > target) W = target;
        if (W > kMaxGroups) W = kMaxGroups;
        if (W < 1) W = 1;
        pl->W = (int) W;
        pl->S = pl->chunk = 0;
        slots = (size_t) d->batch * (d->num_kv_heads / pl->pk) + (size_t) W;  // pair u's partial from workgroup w at u + w
    } else {
        long long chunk = d->split_rows;
        if (chunk == 0) {
            // The fewest rows per split that keep the grid within one workgroup per CU, in
            // whole 16-row tiles (C2, 4 pairs of 8193 rows: 64-row rounding gave 192-row
            // splits and 176 workgroups, 11.4 us; 16-row rounding gives 144 and 228, 10.3).
            const long long pairs = (long long) d->batch * (d->num_kv_heads / pl->pk);
            const long long per_pair = std::max(1LL, target / pairs);
            chunk = (maxvis + per_pair - 1) / per_pair;
            chunk = (chunk + kTile - 1) / kTile * kTile;
            const int min_rows = pl->per_cu == 2 ? kMinRowsOcc2 : kMinRows;
            if (chunk < min_rows) chunk = min_rows;
            if (chunk > 8192) chunk = 8192;
        }
        long long S = (maxvis + chunk - 1) / chunk;
        if (S > kMaxGroups) {
            chunk = (maxvis + kMaxGroups - 1) / kMaxGroups;
            chunk = (chunk + kTile - 1) / kTile * kTile;
            S = (maxvis + chunk - 1) / chunk;
        }
        pl->W = 0;
        pl->S = (int) S;
        pl->chunk = (int) chunk;
        if (!raw && d->split_rows == 0) pl->pk = choose_pack(d, G, S, target);
        slots = (size_t) d->batch * (d->num_kv_heads / pl->pk) * S;
    }
    const size_t parts = slots * G * pl->pk;
    pl->off_table = 256;
    pl->off_ml = pl->off_table + (((size_t) (d->batch + 1) * sizeof(long long) + 255) / 256) * 256;
    pl->off_acc = pl->off_ml + ((parts * 2 * sizeof(float) + 255) / 256) * 256;
    pl->bytes = pl->off_acc + parts * d->head_dim * sizeof(float);
    return ESDA_OK;
}

// Waves per workgroup (the head dim is split across them); workgroups per CU: Plan::per_cu.  D = 256:
// two workgroups of 4 waves per CU, each with half the LDS for its ring (4 stages of 16
// rows), so each SIMD runs two waves of independent workgroups that never wait on each
// other's barriers.  Against one workgroup of 8 waves (two per SIMD in barrier lockstep,
// the softmax repeated by all 8): C3 attend 23.9 -> 22.3 us, C5 step 7.80 -> 7.61 ms, C1
// 5.7 -> 5.3 us.  D = 512 keeps 4 waves (its 8-wave form loses a ring stage to the larger
// score exchange and runs C4 ~6% slower).  D = 128 has too few dims for 8 waves of 32-dim MFMA
// steps.
template <int D>
constexpr int ring_waves() { return D == 256 ? kWaves256 : 4; }

template <int D, bool SHARED, int OCC, class P>
hipError_t launch_attend(const P &ap, dim3 grid, hipStream_t st) {
    constexpr int NW = ring_waves<D>();
    hipLaunchKernelGGL((attend_kernel<D, SHARED, NW, OCC, P>), grid, dim3(64 * NW), 0, st, ap);
    return hipGetLastError();
}

// The 512-dim shared stream (C2, C4, C5's global layers) runs the kernel whose ring takes half
// the LDS -- 4 stages of 16 rows, two of them in flight (32 KB) -- at one workgroup per CU.
// Shallower rings measured faster there, the register budget of two waves per SIMD making no
// difference: C4 step 78.8-79.1 us at 4 stages (80 KB budget), 79.9-80.1 at 5, 80.4-80.6 at 6,
// 81.5-81.9 at 9 (the full LDS), 108.6 at 3; C2 13.4 against 14.2 us at 9.  Over 256
// workgroups two stages each keep ~8.4 MB in flight, enough to saturate HBM (a read probe reads
// 7.1-7.3 TB/s with 6-15 MB in flight, less with ~30 MB), where 9 stages keep ~29 MB.  A
// separate 512-dim V needs the whole LDS for 4 stages; D = 128 stages are 4 KB.
template <class P>
hipError_t dispatch_attend(int D, bool shared, const P &ap, dim3 grid, hipStream_t st) {
    constexpr int O256 = kOcc256, O512 = kOcc512Shared;
    switch (D) {
        case 128:
            // (scored steps of 128 dims run stream_kernel)
            if constexpr (std::is_base_of<ScoredAttendParams, P>::value) return hipErrorInvalidValue;
            else return shared ? launch_attend<128, true, 1>(ap, grid, st) : launch_attend<128, false, 1>(ap, grid, st);
        case 256:
            return shared ? launch_attend<256, true, O256>(ap, grid, st)
                          : launch_attend<256, false, O256>(ap, grid, st);
        default:
            return shared ? launch_attend<512, true, O512>(ap, grid, st)
                          : launch_attend<512, false, 1>(ap, grid, st);
    }
}

// The step's shape, plan and workspace in a kernel's parameters.
struct DecodeSpace {
    long long *table;
    float *part_ml, *part_acc;
};
DecodeSpace space_of(const Plan &pl, void *workspace) {
    unsigned char *ws = static_cast<unsigned char *>(workspace);
    return {reinterpret_cast<long long *>(ws + pl.off_table), reinterpret_cast<float *>(ws + pl.off_ml),
            reinterpret_cast<float *>(ws + pl.off_acc)};
}
void fill_attend(const esda_decode_desc *d, const Plan &pl, const DecodeSpace &sp, int *status, uint16_t *out,
                 AttendParams &ap) {
    ap.part_acc = sp.part_acc;
    ap.part_ml = sp.part_ml;
    ap.status = status;
    ap.table = sp.table;
    ap.out = out;
    ap.seq_stride = d->seq_stride;
    ap.head_stride = d->head_stride;
    ap.B = d->batch;
    ap.Hq = d->num_q_heads;
    ap.Hkv = d->num_kv_heads / pl.pk;
    ap.G = pl.G * pl.pk;
    ap.pk = pl.pk;
    ap.gk = pl.G;
    ap.cap = d->cap;
    ap.window = d->window;
    ap.ring = d->ring;
    ap.balanced = pl.balanced;
    ap.W = pl.W;
    ap.S = pl.S;
    ap.chunk = pl.chunk;
    ap.scale_log2e = d->scale * kLog2e;
}
dim3 attend_grid(const esda_decode_desc *d, const Plan &pl) {
    return pl.balanced ? dim3(pl.W) : dim3(pl.S, d->num_kv_heads / pl.pk, d->batch);
}

// The split merge of a step.  pad: rows a pair counted beside its own (walk_segments' PAD).
int launch_merge(const esda_decode_desc *d, const Plan &pl, const DecodeSpace &sp, const int *pos, const int *row_base,
                 int pad, uint16_t *out, hipStream_t st) {
    // One split per pair: the attend workgroups wrote every output themselves.
    if (!pl.balanced && pl.S == 1) return ESDA_OK;
    MergeParams mp;
    mp.part_acc = sp.part_acc;
    mp.part_ml = sp.part_ml;
    mp.table = sp.table;
    mp.pos = pos;
    mp.row_base = row_base;
    mp.out = out;
    mp.B = d->batch;
    mp.Hq = d->num_q_heads;
    mp.Hkv = d->num_kv_heads / pl.pk;
    mp.G = pl.G * pl.pk;
    mp.D = d->head_dim;
    mp.cap = d->cap;
    mp.window = d->window;
    mp.ring = d->ring;
    mp.balanced = pl.balanced;
    mp.W = pl.W;
    mp.S = pl.S;
    mp.chunk = pl.chunk;
    mp.pad = pad;
    // Partials per pair: a grid's S, or about W / pairs + 1 of the balanced shares.
    const long long pairs = (long long) d->batch * d->num_kv_heads / pl.pk;
    if (pl.balanced ? pl.W < kMergeShares * pairs : pl.S <= kMergeRowsChunk) {
        // A few splits per pair: the thread-per-output merge, one memory round trip per
        // kMergeRowsChunk of them (C5's global layers, 128 pairs of 3 partials: 11 -> 4.4
        // us).  With more, merge_kernel's workgroups reduce 16 split groups side by side:
        // at C1's 16 splits over 8 pairs the rows kernel takes two round trips (9.0 ->
        // 11.8 us a step), and on balanced shares (step us, rows / merge_kernel): 8 pairs of
        // 32 partials 46.1 / 30.0, 16 of 16 47.7 / 38.4, 32 of 8 41.6 / 38.7, 40 of 6.4
        // 50.4 / 49.6, 48 of 5.3 51.0 / 50.8, 64 of 4 39.5 / 42.5.
        const int threads = d->num_q_heads * (d->head_dim / 4);
        dim3 grid((threads + kMergeRowsThreads - 1) / kMergeRowsThreads, d->batch);
        hipLaunchKernelGGL(merge_rows_kernel, grid, dim3(kMergeRowsThreads), 0, st, mp);
    } else {
        dim3 grid(d->head_dim / kMergeDims, d->num_q_heads, d->batch);
        // (balanced: room for a pair of twice the average partials; longer ones are looped over)
        if (pl.balanced ? 2LL * pl.W <= kMergeGroups * 4 * pairs : pl.S <= kMergeGroups * 4)
            hipLaunchKernelGGL(merge_kernel<4>, grid, dim3(kMergeThreads), 0, st, mp);
        else
            hipLaunchKernelGGL(merge_kernel<16>, grid, dim3(kMergeThreads), 0, st, mp);
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return hip_fail(e, "merge_kernel launch");
    return ESDA_OK;
}

// Argument checks shared by the decode entry points over a bf16 cache (everything but the
// workspace).
int check_decode_args(const esda_decode_desc *d, const esda_decode_args *a) {
    if (!a) return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode: null arguments");
    if (!a->q || !a->k_new || !a->k_cache || !a->v_cache || !a->pos || !a->out)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode: null device pointer");
    if (!d->kv_shared && !a->v_new)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode: v_new is required unless kv_shared");
    if (d->kv_shared && a->v_cache != a->k_cache)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode: kv_shared needs v_cache == k_cache");
    if (!d->kv_shared && a->v_cache == a->k_cache)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode: separate K/V need distinct caches");
    if (!aligned16(a->q) || !aligned16(a->k_new) || (a->v_new && !aligned16(a->v_new)) ||
        !aligned16(a->k_cache) || !aligned16(a->v_cache) || !aligned16(a->out))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode: tensors must be 16-byte aligned");
    return ESDA_OK;
}

AttendParams decode_params(const esda_decode_desc *d, const esda_decode_args *a) {
    AttendParams ap{};
    ap.q = static_cast<const uint16_t *>(a->q);
    ap.k_new = static_cast<const uint16_t *>(a->k_new);
    ap.v_new = static_cast<const uint16_t *>(d->kv_shared ? a->k_new : a->v_new);
    ap.k_cache = static_cast<uint16_t *>(a->k_cache);
    ap.v_cache = static_cast<uint16_t *>(a->v_cache);
    ap.pos = a->pos;
    ap.row_base = a->row_base;
    return ap;
}

}  // namespace
