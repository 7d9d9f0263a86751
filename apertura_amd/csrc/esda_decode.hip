// esda_decode.hip -- Gemma-4 decode attention for MI355X (gfx950, CDNA4).
//
// One decode step = fused KV append + split-K single-query attention + fp32 merge.
// Reference behaviour (Apertura tree): ESKVCache::update prealloc append
// (ESKVCache.mm:64-109) followed by mx::fast::scaled_dot_product_attention at
// ESAttention.mm:188, with the visibility rule of ESGemma4TextModel.mm:68-83 and the
// split merge of ESDecodeAttn.mm:253-273; in raw-K mode, ESKVCache::updateRaw
// (ESKVCache.mm:458-504) followed by esDecodeAttnGlobal (ESDecodeAttn.mm:17-117, 415-453).
//
// Kernels
//   attend_kernel  grid (splits, kv heads, sequences) or balanced shares of a ragged
//                  batch; 4 waves, one workgroup per CU (two at D = 256), the
//                  ring in the whole LDS or in half of it.  A workgroup streams
//                  visible rows of one (sequence, kv head) -- or of 2 or 4 kv heads
//                  packed together -- through an LDS ring filled by LDS DMA, splits the head dim across its
//                  waves for the QK and PV MFMAs (the GQA group is the MFMA N dimension),
//                  runs an fp32 online softmax and writes (m, l, acc) partials.  The
//                  workgroup whose split ends at the new token also copies its row into
//                  the cache.  Details at the kernel.
//   raw_attend_kernel  the same over a raw-K or q8 raw-K stream, K and V rebuilt per row.
//   merge_kernel   reduces the partials of all splits per (sequence, query head).
//   append_kernel  multi-row append (slice_update) for prefill-style callers.
// attend_kernel, the merges and their launch are in esda_attend.h, which other entry points use too.
// The C ABI (include/esda.h) is at the end of the file.

#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>
#include <cstring>
#include <mutex>
#include <string>
#include <type_traits>
#include <utility>

#include "esda.h"
#include "esda_attend.h"
#include "esda_device.h"
#include "esda_internal.h"
#include "esda_plan.h"

namespace {

// ------------------------------------------------------------ raw-K reconstruction
//
// Raw mode (ESDecodeAttn.mm:51-106): the cache holds pre-norm k_proj rows.  Per row,
// rinv = rsqrt(mean(kraw^2) + eps); K = bf16(rope(kraw * rinv * kw)) with rotary pairs
// (d, d + 256) for d < 64, whose cos / sin are those of the fp32 angle t * inv_freq[d]
// rounded to bf16; V = kraw * rinv, with rinv folded into the softmax weight.

constexpr int kRawDim = 512;
constexpr int kRopePairs = 64;

// ------------------------------------------------- raw-K attend with wave-private rings
//
// Raw-K decode (ESDecodeAttn.mm:17-117).  A workgroup serves one kv head (a contiguous run of its rows, as
// the composite kernel's) with four waves, one per SIMD.  Each wave owns whole 16-row stages
// (16 consecutive positions) over the full 512-dim head, in turn: wave w takes stages w,
// w + 4, w + 8, ... of a segment.  It streams their rows through two LDS slots of its own and
// their cos / sin table rows through a table buffer of its own, filled by its own LDS DMA and
// waited on with its own vmcnt, so the main loop has no barrier and no exchange between
// waves.  Per stage a wave:
//   - reads the 16 raw rows as MFMA A operands (lane (li, lg): row li, dims kdim(kk, lg)
//     of k-step kk);
//   - forms their 16x16 Gram matrix with 16 MFMAs: the diagonal is each row's sum of
//     squares (exact bf16 products, fp32 sums), hence rinv = rsqrt(mean + eps);
//   - rebuilds K = bf16(rope(kraw * rinv * kw)), rounded where the reference rounds it:
//     kraw * kw comes exactly (a product of two bf16 values fits fp32) from MFMAs of the
//     lane's own rows against diag(kw) operands built once per kernel, whose C layout
//     hands every lane the dims it supplied; one multiply by rinv, the rotation and the
//     bf16 rounding remain per element.  The rotary partners (d, d + 256), d < 64, sit in
//     one lane (k-steps 0, 1 and 8, 9); their bf16 cos / sin come from the table rows,
//     whose buffer takes the next stage's table rows once the rotary k-steps have read it,
//     or, when the caller passes no table, are computed by the lane that uses them (16 per
//     lane and stage, about 500 VALU instructions: 131072 rows x 4 heads raw 104 us a step
//     against 95 with the table and 164 by an 8-wave kernel that shared a computed table
//     through LDS; q8 118, 96 and 207);
//   - scores the kv head's query heads (up to 16: the MFMA's N dimension, zero-padded) with
//     16 MFMAs, runs its own online softmax, and accumulates O^T[512 x 16 heads] with 32
//     MFMAs over V = kraw read back by transpose reads, rinv folded into the weight:
//     P = bf16(e * rinv), l += P / rinv.
// Q8 (esDecodeAttnGlobalQ8, ESDecodeAttn.mm:275-369): rows are u8 with a per-row scale and
// bias (x = q * scale + bias).  sum(q^2) and sum(q) of each row are exact integer dot products
// of the u8 bytes (v_dot4_u32_u8, summed over the four lane groups), hence mean(x^2), and every
// lane computes its own row's factors;
// K = bf16(rope(fma(q, scale * rinv, bias * rinv) * kw)); q is also written to a bf16 tile
// of the wave's that the transpose reads use as V, with P = bf16(e * scale * rinv) and the
// bias entering as sum(P * bias / scale) per head.
// At the end of a segment the four waves' (m, l, O) merge through LDS into one partial.

constexpr int kWaves = 4;                  // waves of the wave-private-ring kernels
constexpr int kBlk = 1056;                 // LDS bytes per 1 KiB DMA block (1 KiB + 32 B pad)

// Dims of k-step kk held by lane group lg: 8 consecutive dims, the four lane groups side by
// side (32 kk + 8 lg), so that a row's lane groups read (and the q8 V tile's writes write)
// adjacent 16-byte pieces, without LDS bank conflicts; the rotary partners of k-steps 0, 1 are
// k-steps 8, 9 of the same lane.
__device__ __forceinline__ int kdim(int kk, int lg) { return 32 * kk + 8 * lg; }
// The rotary k-steps: dims 0 .. 63 (k-steps 0, 1) and their partners 256 .. 319 (8, 9).
__device__ __forceinline__ constexpr bool rot_step(int kk) { return (kk & 7) < 2; }

// Lazy-rescale threshold of the raw kernels (log2 units).  Their V rows are RMS-normalised
// (|v_d| <= sqrt(512)), so with probabilities up to 2^64 before normalisation the partial
// sums stay below rows * 2^64 * 2^6 < 2^101 for any row count under 2^31, far from fp32's
// limit.  The in-model scale of these layers is 1.0, which spreads the scores widely:
// with the generic threshold of 8 about half of all stages would rescale.
constexpr float kRawRescaleSlack = 64.0f;

// Balanced shares without a table: a pair counts this many rows beside its own, about what
// starting its segment costs (~6 us: q, the first rows, the waves' merge, each a round trip;
// a row of a long segment takes 0.05), so that no share collects many short pairs.  8 heads x
// 61, 4 and 101 rows 59.2 us a step with 0 and 18.1 with 128 (the tiny sequence's 8 segments
// were one share), 15.4 with 64, 17.6 with 256; 3 x 129 rows 21.5, 18.2, 21.2, 21.0; 16
// sequences of 6 .. 156 rows 54.4, 20.3, 22.9, 22.0; 7 x 1030 x 4 heads 28.2, 22.2, 24.8, 24.1.
constexpr int kOwnTablePad = 128;

template <bool Q8, bool TABLE>
struct WRing {
    static constexpr int ROWS = Q8 ? 8 * kBlk : 16 * kBlk;  // a stage's 16 rows (q8: two per block)
    static constexpr int SB = Q8 ? 128 : 0;                  // q8: 16 scales, 16 biases
    static constexpr int SLOT = ROWS + SB;
    static constexpr int STG = Q8 ? 16 * kBlk : 0;           // q8: the bf16 V tile
    static constexpr int TAB = TABLE ? 4 * kBlk : 0;         // the stage's 16 cos/sin table rows (swizzled)
    static constexpr int WAVE = 2 * SLOT + STG + TAB;        // one wave's LDS: two slots, the V tile, the table
    static constexpr int MERGE = kWaves * 16 * 516 * 4;      // end-of-segment merge area (aliases the rings)
    static constexpr int LDS = kWaves * WAVE > MERGE ? kWaves * WAVE : MERGE;
};

// DMA of LDS blocks I .. N-1 of an interior stage: block i is 1 KiB of memory at
// base[i / 4] + (i % 4) KiB and lands at LDS block i (lds + i * kBlk), so four blocks share
// one scalar base (immediate offsets) and each costs one scalar instruction beside its DMA.
template <int I, int N>
__device__ __forceinline__ void ring_blocks(const uint64_t *base, unsigned voff, unsigned lds) {
    if constexpr (I < N) {
        constexpr int k = I & 3;
        lds_dma16_o<k * 1024, 4 * (I >> 2) * kBlk + k * (kBlk - 1024)>(base[I >> 2], voff, lds);
        ring_blocks<I + 1, N>(base, voff, lds);
    }
}

template <bool Q8, bool TABLE>
__global__ __attribute__((amdgpu_flat_work_group_size(64 * kWaves, 64 * kWaves), amdgpu_waves_per_eu(1, 1)))
void raw_attend_kernel(AttendParams p) {
    using W = WRing<Q8, TABLE>;
    __shared__ __attribute__((aligned(16))) unsigned char wlds[W::LDS];
    // per-wave row factors of the stage being computed (the softmax's rows 4lg .. 4lg + 3):
    // [0] rinv (q8: scale * rinv), [1] its inverse, [2] (q8) bias / scale
    __shared__ __attribute__((aligned(16))) float xf[kWaves][3][16];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int li = lane & 15, lg = lane >> 4;
    unsigned char *const wl = wlds + wave * W::WAVE;

    // q8: the k-norm weights in fp32, read per k-step (the lanes of a lane group read the
    // same 32 bytes); 128 of them per lane would not fit in registers beside O^T and Q^T.
    __shared__ __attribute__((aligned(16))) float kwl[Q8 ? kRawDim : 1];
    // no table: the rotary frequencies, a copy per wave (no barrier), read back per stage.  A call
    // of a few stages is latency from end to end: with the copy ahead of every DMA, the first
    // rows requested before q and the cos / sin computed while they are in flight, 31 rows x 4
    // heads take 9.0 us against 9.7 (q8 10.4 against 11.7).
    __shared__ __attribute__((aligned(16))) float invl[TABLE ? 1 : kWaves][kRopePairs];
    float freq = 0.0f;
    if constexpr (!TABLE) freq = p.inv_freq[lane];
    if constexpr (Q8) {
        const unsigned t = reinterpret_cast<const unsigned *>(p.kw)[tid];
        kwl[2 * tid] = bf16_lo(t);
        kwl[2 * tid + 1] = bf16_hi(t);
    }
    if constexpr (Q8) __syncthreads();
    // Raw: the A operands of the x * kw products, diag(kw) over 16 dims.  For k-step kk and half
    // hh the B operand is the lane's own dims kdim(kk, lg) + 4hh .. + 3 of row li; lane
    // (li, lg) then holds kw of dim kdim(kk, lg) + 4hh + (li & 3) at slot li & 3 when
    // lg == li / 4 and zeros elsewhere, and the product's C layout hands every lane x * kw
    // of the same dims it supplied.
    short4v dg[Q8 ? 1 : 16][2];
    if constexpr (!Q8) {
        // The lane's 8 weights of a k-step come in one load and are masked: 32 two-byte loads and
        // their selects took 0.7 us more of every workgroup (802 rows x 4 heads 12.0 -> 11.4 us a step).
        const int s = li & 3;
        const unsigned on = (li >> 2) == lg ? (s & 1 ? 0xffff0000u : 0xffffu) : 0u;
        const unsigned m0 = s < 2 ? on : 0u, m1 = s < 2 ? 0u : on;
#pragma unroll
        for (int kk = 0; kk < 16; ++kk) {
            const u32x4 w = *reinterpret_cast<const u32x4_a2 *>(p.kw + kdim(kk, lg));
            dg[kk][0] = __builtin_bit_cast(short4v, u32x2{w[0] & m0, w[1] & m1});
            dg[kk][1] = __builtin_bit_cast(short4v, u32x2{w[2] & m0, w[3] & m1});
        }
    }

    // (ahead of any DMA: a wait for this load must not wait for rows behind it)
    if constexpr (!TABLE) invl[wave][lane] = freq;

    auto segment = [&](const int b, const int kvh, const int j0, const int j1, const SeqView sv, const size_t slot,
                       const bool direct) {
        const bool append = p.k_new != nullptr;
        const size_t head_off = (size_t) b * p.seq_stride + (size_t) kvh * p.head_stride;
        uint16_t *const kbase = p.k_cache + head_off;
        const uint16_t *const knew = append ? p.k_new + ((size_t) b * p.Hkv + kvh) * kRawDim : nullptr;
        unsigned char *const q8base = Q8 ? p.q8 + head_off : nullptr;
        const size_t sb_off = Q8 ? (size_t) b * p.sb_seq_stride + (size_t) kvh * p.sb_head_stride : 0;

        // Q^T operand: head li of the packed pair (zero for padding heads li >= G)
        bf16x8 qv[16];
        auto load_q = [&]() {
            const bool qok = li < p.G;
            const uint16_t *qrow = p.q + ((size_t) b * p.Hq + (size_t) kvh * p.G + (qok ? li : 0)) * kRawDim;
#pragma unroll
            for (int kk = 0; kk < 16; ++kk) {
                const u32x4 t = qok ? *reinterpret_cast<const u32x4 *>(qrow + kdim(kk, lg)) : u32x4{0u, 0u, 0u, 0u};
                qv[kk] = __builtin_bit_cast(bf16x8, t);
            }
        };
        if constexpr (TABLE) load_q();
        if constexpr (Q8) {
            // The new row is quantized into the cache before any DMA (wave 0),
            // esQuantizeRawRows' arithmetic (ESDecodeAttn.mm:491-509).
            if (append && j1 == sv.nvis && wave == 0) {
                const u32x4 t = *reinterpret_cast<const u32x4 *>(knew + lane * 8);
                float x[8];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    x[2 * e] = bf16_lo(t[e]);
                    x[2 * e + 1] = bf16_hi(t[e]);
                }
                float mn = x[0], mx = x[0];
#pragma unroll
                for (int e = 1; e < 8; ++e) {
                    mn = fminf(mn, x[e]);
                    mx = fmaxf(mx, x[e]);
                }
#pragma unroll
                for (int o = 32; o > 0; o >>= 1) {
                    mn = fminf(mn, __shfl_xor(mn, o));
                    mx = fmaxf(mx, __shfl_xor(mx, o));
                }
                float scl = (mx - mn) / 255.0f;
                if (!(scl > 1e-8f)) scl = 1e-8f;
                unsigned lo = 0u, hi = 0u;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const unsigned qi = (unsigned) fminf(roundf((x[e] - mn) / scl), 255.0f);
                    if (e < 4) lo |= qi << (8 * e);
                    else hi |= qi << (8 * (e - 4));
                }
                unsigned char *row = q8base + (size_t) sv.newrow * kRawDim;
                *reinterpret_cast<uint2 *>(row + lane * 8) = uint2{lo, hi};
                if (lane == 0) {
                    const size_t at = sb_off + (size_t) sv.newrow;
                    p.qsc[at] = scl;
                    p.qbs[at] = mn;
                }
            }
        }
        if constexpr (TABLE) ESDA_WAIT_VM(0);  // operands in registers (and the q8 row stored) before the ring counts its loads
        if constexpr (Q8) {
            if (append && j1 == sv.nvis) {
                if constexpr (!TABLE) ESDA_WAIT_VM(0);
                lds_barrier();  // the quantized row is in memory before any DMA
            }
        }

        const int nst = (j1 - j0 + 15) >> 4;  // 16-row stages: 16 positions
        // DMA of stage st's rows into slot sl.  Rows past the segment end repeat its last row
        // (their scores are masked); the new token's raw row comes from k_new.
        auto dma_rows = [&](int st, unsigned char *sl) {
            const int jst = j0 + 16 * st;
            const unsigned lb = lds_addr(sl);
            // q8 block i: rows 2i, 2i + 1; lane l loads row 2i + (l & 1), 16-byte piece l >> 1
            const int h = lane & 1, pc = lane >> 1;
            if (jst + 16 < j1) {
                // Interior stage: all sixteen positions exist (the segment's last row is in the
                // last stage).  Four consecutive 1 KiB blocks of memory (raw rows; pairs of q8
                // rows) share one scalar base through the DMA's immediate offset (ring_blocks).
                if constexpr (Q8) {
                    const unsigned char *r0 = q8base + (size_t) (sv.first + jst) * kRawDim;
                    const uint64_t base[2] = {sbase64(r0), sbase64(r0 + 4096)};
                    const unsigned v = (unsigned) (h * kRawDim + pc * 16);
                    ring_blocks<0, 8>(base, v, lb);
                } else {
                    const unsigned char *r0 = reinterpret_cast<const unsigned char *>(kbase + (size_t) (sv.first + jst) * kRawDim);
                    const uint64_t base[4] = {sbase64(r0), sbase64(r0 + 4096), sbase64(r0 + 8192), sbase64(r0 + 12288)};
                    ring_blocks<0, 16>(base, (unsigned) (lane * 16), lb);
                }
            } else {
                if constexpr (Q8) {
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        const int j = min(jst + 2 * i + h, j1 - 1);
                        lds_dma16(q8base + (size_t) (sv.first + j) * kRawDim + pc * 16, lb + i * kBlk);
                    }
                } else {
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int j = min(jst + r, j1 - 1);
                        const uint16_t *src = (append && j == sv.nvis - 1) ? knew : kbase + (size_t) (sv.first + j) * kRawDim;
                        lds_dma16(src + lane * 8, lb + r * kBlk);
                    }
                }
            }
            if constexpr (Q8) {
                // scales (lanes 0..15) and biases (16..31) of the stage's rows
                if (lane < 32) {
                    const int j = min(jst + (lane & 15), j1 - 1);
                    lds_dma4((lane < 16 ? p.qsc : p.qbs) + sb_off + (size_t) (sv.first + j), lb + W::ROWS);
                }
            }
        };
        // raw: chunk c (of 4) of stage st's row DMAs, rows 4c .. 4c + 3.  The next stage's rows
        // go out in four chunks over the iteration (at the top, after the Gram pass, beside the
        // table rows, after the scores) rather than sixteen DMAs at once, which stalled their
        // issue behind the other waves' loads (c4raw attend 91.3 -> 90.8 us).
        auto dma_rows_part = [&](int st, unsigned char *sl, auto cc) {
            constexpr int c = decltype(cc)::value;
            const int jst = j0 + 16 * st;
            const unsigned lb = lds_addr(sl);
            if (jst + 16 < j1) {
                const unsigned char *r0 = reinterpret_cast<const unsigned char *>(kbase + (size_t) (sv.first + jst) * kRawDim);
                const uint64_t base[4] = {sbase64(r0), sbase64(r0 + 4096), sbase64(r0 + 8192), sbase64(r0 + 12288)};
                ring_blocks<4 * c, 4 * c + 4>(base, (unsigned) (lane * 16), lb);
            } else {
#pragma unroll
                for (int r = 4 * c; r < 4 * c + 4; ++r) {
                    const int j = min(jst + r, j1 - 1);
                    const uint16_t *src = (append && j == sv.nvis - 1) ? knew : kbase + (size_t) (sv.first + j) * kRawDim;
                    lds_dma16(src + lane * 8, lb + r * kBlk);
                }
            }
        };
        // DMA of stage st's 16 table rows into the wave's table buffer: block bt holds positions
        // 4bt .. 4bt + 3, piece c of position rib at 16 * (16 rib + (c + 4 rib) mod 16).  Loaded
        // temporal (the rows non-temporal): the workgroups of the other kv heads at the same
        // positions run on the same XCD and read them from the L2.
        auto dma_tab = [&](int st) {
            const int jst = j0 + 16 * st;
            const int rib = lane >> 4, c = (lane - 4 * rib) & 15;
            const unsigned tdst = lds_addr(wl + 2 * W::SLOT + W::STG);
            if (jst + 16 <= j1) {
                const uint64_t tb = sbase64(p.rope_tab + (size_t) (sv.first + jst) * kRopePairs);
                const unsigned tvoff = (unsigned) (rib * 256 + c * 16);
                lds_dma16_o<0, 0, false>(tb, tvoff, tdst);
                lds_dma16_o<1024, kBlk - 1024, false>(tb, tvoff, tdst);
                lds_dma16_o<2048, 2 * kBlk - 2048, false>(tb, tvoff, tdst);
                lds_dma16_o<3072, 3 * kBlk - 3072, false>(tb, tvoff, tdst);
            } else {
#pragma unroll
                for (int bt = 0; bt < 4; ++bt) {
                    const int j = min(jst + 4 * bt + rib, j1 - 1);
                    lds_dma16<false>(p.rope_tab + (size_t) (sv.first + j) * kRopePairs + c * 4, tdst + bt * kBlk);
                }
            }
        };

        // This wave's stages: w, w + 4, ...; local index i uses slot i & 1.  One stage is in
        // flight at a time: the next one's DMA is issued as soon as the current one has
        // landed (the other slot was consumed by the previous iteration).  Two in flight
        // while waiting measured slower (c4raw attend 96.4 against 94.5 us, c4q8 110.1
        // against 108.5): the loads of all waves together then oversubscribe the memory system.
        const int st0 = wave;
        if (st0 < nst) {
            dma_rows(st0, wl);
            if constexpr (TABLE) dma_tab(st0);
        }
        if constexpr (!TABLE) load_q();  // behind the first rows: one round trip for both

        float m = -INFINITY, l = 0.0f;
        float bt = 0.0f;  // q8: sum of P * bias / scale of this lane's head
        f32x4 acc[32];
#pragma unroll
        for (int dt = 0; dt < 32; ++dt) acc[dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        float *const xfw = &xf[wave][0][0];

        for (int st = st0, it = 0; st < nst; st += kWaves, ++it) {
            unsigned char *const sl = wl + (it & 1) * W::SLOT;
            u32x4 tab[4];
            if constexpr (!TABLE) {
                // Computed (rope_table_kernel's arithmetic; the lanes of a stage need 16 x 64 pairs, so
                // each computes the 16 it uses) while the stage's rows are in flight
                const float t = (float) (sv.first + min(j0 + 16 * st + li, j1 - 1));
#pragma unroll
                for (int c4 = 0; c4 < 4; ++c4) {
                    const f32x4 f = *reinterpret_cast<const f32x4 *>(&invl[wave][32 * (c4 >> 1) + 8 * lg + 4 * (c4 & 1)]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float sn, cs;
                        sincos_f32(t * f[e], sn, cs);
                        tab[c4][e] = __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{cs, sn}, bf16x2));
                    }
                }
            }
            ESDA_WAIT_VM(0);  // this stage's rows and table rows landed
            unsigned char *const nsl = wl + ((it + 1) & 1) * W::SLOT;
            const bool more = st + kWaves < nst;
            if (more) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the other slot's reads are done
                if constexpr (Q8) dma_rows(st + kWaves, nsl);
                else dma_rows_part(st + kWaves, nsl, std::integral_constant<int, 0>{});
            }
            // Scores S^T[16 rows x 16 heads] of K = bf16(rope(x * rinv * kw)) (q8: x = q * scale
            // + bias), rounded where ESDecodeAttn.mm:51-93 rounds it.
            f32x4 sp0 = {0.0f, 0.0f, 0.0f, 0.0f}, sp1 = {0.0f, 0.0f, 0.0f, 0.0f};
            // cos / sin of row li's position for the rotary pairs this lane holds, from the table
            auto load_tab = [&](u32x4 (&tab)[4]) {
                const int bt2 = li >> 2, rib = li & 3;  // row li: position li of the stage
#pragma unroll
                for (int c4 = 0; c4 < 4; ++c4) {
                    // the pieces (4 frequencies each) of the lane's rotary dims kdim(kr, lg) .. + 7
                    const int c = 8 * (c4 >> 1) + 2 * lg + (c4 & 1);
                    tab[c4] = *reinterpret_cast<const u32x4 *>(wl + 2 * W::SLOT + W::STG + bt2 * kBlk +
                                                               16 * (16 * rib + ((c + 4 * rib) & 15)));
                }
            };
            auto pack = [](const float (&v)[8]) -> bf16x8 {
                bf16x8 r;
#pragma unroll
                for (int e = 0; e < 8; ++e) r[e] = (__bf16) v[e];
                return r;
            };
            // rope over rotary k-steps kr, kr + 8 (dims kdim(kr, lg) + e and their partners + 256)
            auto rotate = [](const u32x4 (&tab)[4], int kr, float (&lo)[8], float (&hi)[8]) {
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const unsigned w = tab[2 * kr + e / 4][e & 3];
                    const float c = bf16_lo(w), s = bf16_hi(w);
                    const float x0 = lo[e], x1 = hi[e];
                    lo[e] = x0 * c - x1 * s;
                    hi[e] = x1 * c + x0 * s;
                }
            };
            // Pass 1: the row norms.  Raw: from Gram products of the rows as stored.  q8: from
            // integer sums of the u8 bytes (the rebuild below widens them to bf16 for the V tile).
            uint2 w8[Q8 ? 16 : 1];  // q8: the lane's 8 u8 values of row li for k-step kk
            u32x4 xr[Q8 ? 1 : 16];  // raw: the lane's row pieces, k-step kk (pass 1, kept for the rebuild)
            float rq = 0.0f, fq = 0.0f;  // q8: scale * rinv and bias * rinv of row li
            {
                if constexpr (Q8) {
                    // All sixteen u8 reads go out before the first V-tile write: LDS accesses
                    // complete in order, so a read issued after a write would wait for it.
                    // Row r's 16-byte piece pc (dims 16 pc ..) sits at (r / 2) * kBlk + 32 pc +
                    // 16 (r % 2) (two rows interleaved per DMA block); the lane's dims kdim(kk, lg)
                    // are half of piece 2kk + lg / 2.
#pragma unroll
                    for (int kk = 0; kk < 16; ++kk)
                        w8[kk] = *reinterpret_cast<const uint2 *>(sl + (li >> 1) * kBlk + 32 * (2 * kk + (lg >> 1)) +
                                                                  16 * (li & 1) + 8 * (lg & 1));
                    const float scl = reinterpret_cast<const float *>(sl + W::ROWS)[li];
                    const float bias = reinterpret_cast<const float *>(sl + W::ROWS)[16 + li];
                    __builtin_amdgcn_sched_barrier(0);
                    // sum(q^2) and sum(q) of the lane's quarter of row li, exact in integers
                    unsigned s2 = 0u, s1 = 0u;
#pragma unroll
                    for (int kk = 0; kk < 16; ++kk)
#pragma unroll
                        for (int w = 0; w < 2; ++w) {
                            const unsigned x = w ? w8[kk].y : w8[kk].x;
                            s2 = __builtin_amdgcn_udot4(x, x, s2, false);
                            s1 = __builtin_amdgcn_udot4(x, 0x01010101u, s1, false);
                        }
                    // whole-row sums in every lane of row li's column (lanes li + 16 lg)
                    s2 = wave_sum_across_groups(s2);
                    s1 = wave_sum_across_groups(s1);
                    // mean(x^2) = scale^2 var(q) + mean(x)^2 with 512^2 var(q) = 512 sum(q^2) - sum(q)^2,
                    // formed exactly in fp64 (below 2^35) and rounded once
                    const float var = (float) (512.0 * (double) s2 - (double) s1 * (double) s1);
                    const float mean = __builtin_fmaf(scl, (float) s1 * (1.0f / kRawDim), bias);
                    const float ms = scl * scl * var * (1.0f / (kRawDim * kRawDim)) + __builtin_fmaf(mean, mean, p.eps);
                    const float rinv = __builtin_amdgcn_rsqf(ms);
                    rq = scl * rinv;
                    fq = bias * rinv;
                    // Without a table both quotients are IEEE divisions: within half an ulp each, where
                    // the reciprocal instruction is within one (~25 more VALU instructions a stage
                    // beside the ~500 of the cos / sin).
                    if (lg == 0) {
                        xfw[0 * 16 + li] = rq;
                        xfw[1 * 16 + li] = TABLE ? __builtin_amdgcn_rcpf(rq) : 1.0f / rq;
                        xfw[2 * 16 + li] = TABLE ? bias * __builtin_amdgcn_rcpf(scl) : bias / scl;
                    }
                } else {
                    // C layout: lane (li, lg) holds C[4lg + i][li]; row li's diagonal is register
                    // li - 4lg of the lanes with lg == li / 4, which publish the row factors.
                    const int i = li - 4 * lg;
                    auto diagonal = [&](const f32x4 &g) { return i == 0 ? g[0] : i == 1 ? g[1] : i == 2 ? g[2] : g[3]; };
                    f32x4 g = {0.0f, 0.0f, 0.0f, 0.0f};
                    float sq[8];
                    if constexpr (TABLE) {
#pragma unroll
                        for (int kk = 0; kk < 16; ++kk) {
                            xr[kk] = *reinterpret_cast<const u32x4 *>(sl + li * kBlk + 2 * kdim(kk, lg));
                            const bf16x8 x = __builtin_bit_cast(bf16x8, xr[kk]);
                            g = __builtin_amdgcn_mfma_f32_16x16x32_bf16(x, x, g, 0, 0, 0);
                        }
                    } else {
                        // Eight chains of two k-steps, added by pairs: a chain of sixteen drops every
                        // 32-dim sum below half an ulp of the running one (and each diagonal is taken
                        // at once: eight live accumulators do not fit beside O^T and Q^T).
#pragma unroll
                        for (int kk = 0; kk < 16; ++kk) xr[kk] = *reinterpret_cast<const u32x4 *>(sl + li * kBlk + 2 * kdim(kk, lg));
#pragma unroll
                        for (int c = 0; c < 8; ++c) {
                            const bf16x8 x0 = __builtin_bit_cast(bf16x8, xr[c]), x1 = __builtin_bit_cast(bf16x8, xr[c + 8]);
                            const f32x4 z = {0.0f, 0.0f, 0.0f, 0.0f};
                            sq[c] = diagonal(__builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                x1, x1, __builtin_amdgcn_mfma_f32_16x16x32_bf16(x0, x0, z, 0, 0, 0), 0, 0, 0));
                        }
#pragma unroll
                        for (int o = 4; o >= 1; o >>= 1)
#pragma unroll
                            for (int c = 0; c < o; ++c) sq[c] += sq[c + o];
                    }
                    if (i >= 0 && i < 4) {
                        const float s2 = TABLE ? diagonal(g) : sq[0];
                        const float ms = s2 * (1.0f / kRawDim) + p.eps;
                        const float rinv = __builtin_amdgcn_rsqf(ms);
                        xfw[0 * 16 + li] = rinv;
                        xfw[1 * 16 + li] = ms * rinv;
                    }
                }
            }
            // q8: the u8 values are converted once, in pass 2; this keeps the compiler from
            // hoisting the conversions above the row-factor exchange, which would hold 128 floats
            // live across it (it parks such values in accumulation registers)
            if constexpr (Q8) {
#pragma unroll
                for (int kk = 0; kk < 16; ++kk) asm volatile("" : "+v"(w8[kk]));
            }
            if constexpr (!Q8) {
                if (more) dma_rows_part(st + kWaves, nsl, std::integral_constant<int, 1>{});
            }
            // Other lanes read the factors back: a compiler memory barrier keeps those loads
            // after the stores above (the lanes' LDS accesses then run in order).
            asm volatile("" ::: "memory");
            if constexpr (TABLE) load_tab(tab);
            const float rk = Q8 ? rq : xfw[0 * 16 + li];  // rinv of row li (q8: scale * rinv)
            // Pass 2: x * rinv * kw of k-step kk, dims kdim(kk, lg) .. + 7 of row li.
            auto xkw = [&](int kk, float (&v)[8]) {
                if constexpr (Q8) {
                    // fma(q, scale * rinv, bias * rinv) * kw, per element; the same floats of q,
                    // packed to bf16 (exact), are the k-step's part of the V tile
                    float q[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) q[e] = (float) ((((e >> 2) ? w8[kk].y : w8[kk].x) >> (8 * (e & 3))) & 255u);
                    unsigned o[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        o[e] = __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, q[2 * e + 1]), __builtin_bit_cast(unsigned, q[2 * e]),
                                                     0x07060302u);
                    *reinterpret_cast<u32x4 *>(wl + 2 * W::SLOT + li * kBlk + 2 * kdim(kk, lg)) = u32x4{o[0], o[1], o[2], o[3]};
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = __builtin_fmaf(q[e], rk, fq) * kwl[kdim(kk, lg) + e];
                } else {
                    // x * kw exactly (a product of two bf16 values fits fp32) by MFMAs against
                    // the diagonal kw operands, then times rinv
                    const u32x4 t = xr[kk];
                    const f32x4 z = {0.0f, 0.0f, 0.0f, 0.0f};
                    const f32x4 d0 = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(
                        dg[kk][0], __builtin_bit_cast(short4v, uint2{t[0], t[1]}), z, 0, 0, 0);
                    const f32x4 d1 = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(
                        dg[kk][1], __builtin_bit_cast(short4v, uint2{t[2], t[3]}), z, 0, 0, 0);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        v[e] = d0[e] * rk;
                        v[4 + e] = d1[e] * rk;
                    }
                }
            };
#pragma unroll
            for (int kr = 0; kr < 2; ++kr) {
                float lo[8], hi[8];
                xkw(kr, lo);
                xkw(kr + 8, hi);
                rotate(tab, kr, lo, hi);
                sp0 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pack(lo), qv[kr], sp0, 0, 0, 0);
                sp1 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pack(hi), qv[kr + 8], sp1, 0, 0, 0);
            }
            // the table buffer is read (the rotary k-steps above): the next stage's rows may land
            if (st + kWaves < nst) {
                if constexpr (TABLE) {
                    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                    dma_tab(st + kWaves);
                }
                if constexpr (!Q8) dma_rows_part(st + kWaves, nsl, std::integral_constant<int, 2>{});
            }
#pragma unroll
            for (int kk = 2; kk < 16; ++kk) {
                if (rot_step(kk)) continue;
                float v[8];
                xkw(kk, v);
                if (kk & 1) sp1 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pack(v), qv[kk], sp1, 0, 0, 0);
                else sp0 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pack(v), qv[kk], sp0, 0, 0, 0);
            }
            f32x4 sc = sp0 + sp1;
            if constexpr (!Q8) {
                if (more) dma_rows_part(st + kWaves, nsl, std::integral_constant<int, 3>{});
            }
            // Online softmax (log2 domain) over stage rows 4lg .. 4lg + 3: rows past the
            // segment end are masked.
            const int jt = j0 + 16 * st + 4 * lg;
#pragma unroll
            for (int r = 0; r < 4; ++r) sc[r] = (jt + r) < j1 ? sc[r] * p.scale_log2e : -INFINITY;
            const float tmax = wave_max_across_groups(fmaxf(fmaxf(sc[0], sc[1]), fmaxf(sc[2], sc[3])));
            m = m == -INFINITY ? tmax : m;  // first stage: nothing accumulated to rescale
            if (__builtin_expect(__any(tmax > m + kRawRescaleSlack), 0)) {
                const float mnew = fmaxf(m, tmax);
                const float corr = __builtin_amdgcn_exp2f(m - mnew);
                l *= corr;
                if constexpr (Q8) bt *= corr;
#pragma unroll
                for (int dt = 0; dt < 32; ++dt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        float x = acc[dt][e];
                        acc_scale(x, corr);
                        acc[dt][e] = x;
                    }
                m = mnew;
            }
            short4v pbs;
            {
                const f32x4 ri = *reinterpret_cast<const f32x4 *>(xfw + 0 * 16 + 4 * lg);
                const f32x4 rn = *reinterpret_cast<const f32x4 *>(xfw + 1 * 16 + 4 * lg);
                f32x4 gm = {0.0f, 0.0f, 0.0f, 0.0f};
                if constexpr (Q8) gm = *reinterpret_cast<const f32x4 *>(xfw + 2 * 16 + 4 * lg);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float e = __builtin_amdgcn_exp2f(sc[r] - m);
                    const __bf16 pw = (__bf16) (e * ri[r]);
                    l += (float) pw * rn[r];
                    if constexpr (Q8) bt += (float) pw * gm[r];
                    pbs[r] = __builtin_bit_cast(short, pw);
                }
            }
            // O^T += V^T . P^T over all 512 dims (V^T by transpose reads: lane (li, lg)
            // supplies row 4lg + li/4, dims 16dt + 4(li % 4) .. + 4)
            const unsigned char *vb = Q8 ? wl + 2 * W::SLOT : sl;
            const int tr_off = (4 * lg + li / 4) * kBlk + (li % 4) * 8;
#pragma unroll
            for (int dt = 0; dt < 32; ++dt) {
                const short4v av = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) short4v *) (vb + tr_off + 32 * dt));
                acc[dt] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(av, pbs, acc[dt], 0, 0, 0);
                if ((dt & 7) == 7) __builtin_amdgcn_sched_barrier(0);  // at most 8 reads in flight
            }
        }

        // Fused append (raw): the workgroup whose rows end at the new token copies k_new
        // into its cache row (its DMA read the row from k_new; no other workgroup reads it).
        if (!Q8 && append && j1 == sv.nvis && wave == 0) {
            const size_t row = (size_t) sv.newrow * kRawDim;
            *reinterpret_cast<u32x4 *>(kbase + row + lane * 8) = *reinterpret_cast<const u32x4 *>(knew + lane * 8);
        }

        // This wave's (m, l, O): l and (q8) the bias term summed over the lane groups.
        l += __shfl_xor(l, 16);
        l += __shfl_xor(l, 32);
        if constexpr (Q8) {
            bt += __shfl_xor(bt, 16);
            bt += __shfl_xor(bt, 32);
#pragma unroll
            for (int dt = 0; dt < 32; ++dt) acc[dt] += bt;
        }
        // Merge the four waves through LDS (aliasing the rings, which are all consumed).
        ESDA_WAIT_VM(0);
        lds_barrier();
        float *const accb = reinterpret_cast<float *>(wlds);          // [wave][head][516]
        float *const mlb = &xf[0][0][0];                               // [wave][2][16] (m, l)
        // Live heads only: at most 8 of them take 32 threads each, more take 16.
        if (li < p.G) {
#pragma unroll
            for (int dt = 0; dt < 32; ++dt)
                *reinterpret_cast<f32x4 *>(accb + (wave * 16 + li) * 516 + 16 * dt + 4 * lg) = acc[dt];
        }
        if (lg == 0) {
            mlb[wave * 32 + li] = m;
            mlb[wave * 32 + 16 + li] = l;
        }
        lds_barrier();
        {
            const int lt = p.G <= 8 ? 5 : 4;  // log2 of the threads per head
            const int h = tid >> lt, d4 = tid & ((1 << lt) - 1);  // head h, dims 4 d4 + (4 << lt) k
            float mw[kWaves], M = -INFINITY;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                mw[w] = mlb[w * 32 + h];
                M = fmaxf(M, mw[w]);
            }
            float cw[kWaves], L = 0.0f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                cw[w] = mw[w] == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(mw[w] - M);
                L += cw[w] * mlb[w * 32 + 16 + h];
            }
            if (h < p.G) {
                const size_t hq = (size_t) b * p.Hq + (size_t) kvh * p.G + h;
                const size_t pidx = slot * p.G + h;
                const float inv = 1.0f / L;
#pragma unroll 4
                for (int d = 4 * d4; d < kRawDim; d += 4 << lt) {
                    f32x4 o = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int w = 0; w < kWaves; ++w) o += *reinterpret_cast<const f32x4 *>(accb + (w * 16 + h) * 516 + d) * cw[w];
                    if (direct) {
                        bf16x4 r;
#pragma unroll
                        for (int e = 0; e < 4; ++e) r[e] = (__bf16) (o[e] * inv);
                        *reinterpret_cast<uint2 *>(p.out + hq * kRawDim + d) = __builtin_bit_cast(uint2, r);
                    } else {
                        // non-temporal, as the 512-dim attend kernel's partials
                        __builtin_nontemporal_store(o, reinterpret_cast<f32x4 *>(p.part_acc + pidx * kRawDim + d));
                    }
                }
                if (!direct && d4 == 0) {
                    __builtin_nontemporal_store(f32x2{M, L}, reinterpret_cast<f32x2 *>(p.part_ml + pidx * 2));
                }
            }
        }
        lds_barrier();  // the merge area is read before the next segment's DMA overwrites it
    };
    walk_segments<kWaves, TABLE ? 0 : kOwnTablePad>(p, segment);
}

// Per-row affine u8 of raw rows (esQuantizeRawRows, ESDecodeAttn.mm:491-539): one wave
// per row of src [kv heads, n, 512] bf16; row (h, i) -> q8[h * q_head_stride + (row0 + i)
// * 512 ..], scale / bias at [h * sb_head_stride + row0 + i].  raw_attend_kernel's q8 form
// quantizes the decode step's new row with the same arithmetic.
__global__ __launch_bounds__(256) void quantize_rows_kernel(const uint16_t *src, int n, long long rows,
                                                            unsigned char *q8, long long q_head_stride,
                                                            float *scale, float *bias, long long sb_head_stride,
                                                            int row0) {
    const long long r = (long long) blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= rows) return;
    const int lane = threadIdx.x & 63;
    const long long h = r / n, i = r - (r / n) * n;
    const u32x4 t = *reinterpret_cast<const u32x4 *>(src + r * kRawDim + lane * 8);
    float x[8];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        x[2 * e] = bf16_lo(t[e]);
        x[2 * e + 1] = bf16_hi(t[e]);
    }
    float mn = x[0], mx = x[0];
#pragma unroll
    for (int e = 1; e < 8; ++e) {
        mn = fminf(mn, x[e]);
        mx = fmaxf(mx, x[e]);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) {
        mn = fminf(mn, __shfl_xor(mn, o));
        mx = fmaxf(mx, __shfl_xor(mx, o));
    }
    float scl = (mx - mn) / 255.0f;
    if (!(scl > 1e-8f)) scl = 1e-8f;
    unsigned lo = 0u, hi = 0u;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const unsigned qi = (unsigned) fminf(roundf((x[e] - mn) / scl), 255.0f);
        if (e < 4) lo |= qi << (8 * e);
        else hi |= qi << (8 * (e - 4));
    }
    *reinterpret_cast<uint2 *>(q8 + h * q_head_stride + (row0 + i) * kRawDim + lane * 8) = uint2{lo, hi};
    if (lane == 0) {
        scale[h * sb_head_stride + row0 + i] = scl;
        bias[h * sb_head_stride + row0 + i] = mn;
    }
}

// Rotary cos/sin table for raw-K decode: entry (t, f) = bf16 cos | bf16 sin << 16 of the
// fp32 angle t * inv_freq[f], t < rows, f < 64 -- what raw_attend_kernel computes without a table.
__global__ __launch_bounds__(256) void rope_table_kernel(const float *inv_freq, long long n, unsigned *tab) {
    const long long i = (long long) blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const int t = (int) (i / kRopePairs), f = (int) (i % kRopePairs);
    float s, c;
    sincos_f32((float) t * inv_freq[f], s, c);
    tab[i] = __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{c, s}, bf16x2));
}

__global__ void fill_i32_kernel(int *dst, int value, int n) {
    const int i = blockIdx.x * blockDim.x + threadIdx.x;
    if (i < n) dst[i] = value;
}

// Plain row copy for multi-row appends (slice_update at rows row0 .. row0 + n - 1).
__global__ __launch_bounds__(256) void append_kernel(uint16_t *cache, long long seq_stride,
                                                      long long head_stride, int Hkv, int D,
                                                      int cap, const uint16_t *src, int n_new,
                                                      const int *row0, int *status) {
    const int b = blockIdx.z, h = blockIdx.y;
    const int r0 = row0[b];
    if (r0 < 0 || r0 + n_new > cap) {
        if (h == 0 && blockIdx.x == 0 && threadIdx.x == 0 && status) atomicAdd(status, 1);
        return;
    }
    const int chunks = D / 8;
    const size_t total = (size_t) n_new * chunks;
    for (size_t i = (size_t) blockIdx.x * blockDim.x + threadIdx.x; i < total;
         i += (size_t) gridDim.x * blockDim.x) {
        const int r = (int) (i / chunks), c = (int) (i % chunks);
        const uint4 v = *reinterpret_cast<const uint4 *>(src + (((size_t) b * Hkv + h) * n_new + r) * D + c * 8);
        *reinterpret_cast<uint4 *>(cache + (size_t) b * seq_stride + (size_t) h * head_stride +
                                   (size_t) (r0 + r) * D + c * 8) = v;
    }
}

// Read-only stream over `blocks` 1 KiB blocks through the attend kernel's load path
// (global_load_lds_dwordx4 ... nt into LDS, 64 lanes x 16 B = 1 KiB per instruction,
// up to 15 in flight per wave): the memory system's ceiling for that path, and the
// reference point of the HBM counters for it.  Workgroup w reads blocks [blocks * w / G,
// blocks * (w + 1) / G) round-robin over its 4 waves; each wave keeps one word of what it
// read, so the loads feed an output (sink[4 * w + wave]).
__global__ __launch_bounds__(256) void stream_read_kernel(const unsigned char *src, long long blocks, unsigned *sink) {
    __shared__ __attribute__((aligned(16))) unsigned char buf[4][16][1024];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const long long b0 = blocks * blockIdx.x / gridDim.x, b1 = blocks * (blockIdx.x + 1) / gridDim.x;
    int i = 0;
    for (long long b = b0 + wave; b < b1; b += 4, ++i) {
        // at most 14 outstanding before this one: the load that last filled slot i % 16
        // (16 loads ago) has landed
        ESDA_WAIT_VM(14);
        lds_dma16(src + b * 1024 + lane * 16, lds_addr(&buf[wave][i & 15][0]));
    }
    ESDA_WAIT_VM(0);
    lds_barrier();
    const unsigned x = reinterpret_cast<const unsigned *>(&buf[wave][lane & 15][0])[lane];
    unsigned s = x;
    for (int o = 32; o > 0; o >>= 1) s ^= __shfl_xor(s, o);
    if (lane == 0) sink[4 * blockIdx.x + wave] = s;
}

// ------------------------------------------------------------------------ host side

thread_local std::string g_err;

}  // namespace

void esda_detail::set_error(const std::string &msg) { g_err = msg; }

namespace {

// The library is built for gfx950 only: refuse other devices loudly.
int check_device() {
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return hip_fail(e, "hipGetDevice");
    static std::mutex mu;
    static int checked[64] = {0};
    std::lock_guard<std::mutex> lk(mu);
    if (dev < 0 || dev >= 64) return fail(ESDA_ERR_DEVICE, "device index out of range");
    if (checked[dev] == 0) {
        hipDeviceProp_t prop;
        e = hipGetDeviceProperties(&prop, dev);
        if (e != hipSuccess) return hip_fail(e, "hipGetDeviceProperties");
        checked[dev] = std::strncmp(prop.gcnArchName, "gfx950", 6) == 0 ? 1 : -1;
    }
    if (checked[dev] < 0) return fail(ESDA_ERR_DEVICE, "libesda.so is built for gfx950 only");
    return ESDA_OK;
}


}  // namespace

int esda_detail::check_device() { return ::check_device(); }

namespace {

// The raw-mode step as a plain decode description: linear rows, full causal span, one
// shared stream of 512-dim rows.
int raw_as_decode(const esda_raw_desc *r, esda_decode_desc *d) {
    if (!r) return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode_raw: null description");
    if (r->head_dim != kRawDim) return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode_raw: head_dim must be 512");
    if (!(r->eps >= 0.0f)) return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode_raw: eps must be >= 0");
    std::memset(d, 0, sizeof(*d));
    d->batch = r->batch;
    d->num_q_heads = r->num_q_heads;
    d->num_kv_heads = r->num_kv_heads;
    d->head_dim = r->head_dim;
    d->cap = r->cap;
    d->window = 0;
    d->ring = 0;
    d->kv_shared = 1;
    d->seq_stride = r->seq_stride;
    d->head_stride = r->head_stride;
    d->max_visible = r->max_visible;
    d->split_rows = r->split_rows;
    d->scale = r->scale;
    return ESDA_OK;
}

// Launches the requested stages of one decode step (raw: the raw-K attend kernel).
// mode: 0 composite, 1 raw-K, 2 q8 raw-K.  status: the skipped-sequence counter (null =
// the workspace's first word).
int run_stages(const esda_decode_desc *d, const Plan &pl, const AttendParams &ap_in, uint16_t *out,
               void *workspace, int stages, int mode, hipStream_t st, int *status = nullptr) {
    const DecodeSpace sp = space_of(pl, workspace);
    if (stages & ESDA_STAGE_ATTEND) {
        AttendParams ap = ap_in;
        fill_attend(d, pl, sp, status ? status : static_cast<int *>(workspace), out, ap);
        const dim3 grid = attend_grid(d, pl);
        hipError_t e;
        if (mode == 0) {
            e = dispatch_attend(d->head_dim, d->kv_shared != 0, ap, grid, st);
        } else {
            const dim3 block(64 * kWaves);
            if (mode == 1 && ap.rope_tab) hipLaunchKernelGGL((raw_attend_kernel<false, true>), grid, block, 0, st, ap);
            else if (mode == 1) hipLaunchKernelGGL((raw_attend_kernel<false, false>), grid, block, 0, st, ap);
            else if (ap.rope_tab) hipLaunchKernelGGL((raw_attend_kernel<true, true>), grid, block, 0, st, ap);
            else hipLaunchKernelGGL((raw_attend_kernel<true, false>), grid, block, 0, st, ap);
            e = hipGetLastError();
        }
        if (e != hipSuccess) return hip_fail(e, "attend_kernel launch");
    }
    if (stages & ESDA_STAGE_MERGE)
        return launch_merge(d, pl, sp, ap_in.pos, ap_in.row_base, mode != 0 && !ap_in.rope_tab ? kOwnTablePad : 0, out, st);
    return ESDA_OK;
}

}  // namespace

// ------------------------------------------------ static scratch of esda_decode_noalloc
//
// The split partials, the batch prefix table and (when the caller passes no status word)
// the skipped-sequence counter of esda_decode_noalloc live here instead of in a caller
// workspace.  Every GPU the library runs on holds its own copy for the life of the
// process.  In host code `scratch` names a host-side stand-in, never the device memory:
// kernels get the address hipGetSymbolAddress returns for the current device.
constexpr size_t kScratchBytes = size_t(32) << 20;
static __device__ __align__(256) unsigned char scratch[kScratchBytes];

namespace {

// Device address of `scratch` on the current device, looked up once per device.
int scratch_address(void **out) {
    int dev = 0;
    hipError_t e = hipGetDevice(&dev);
    if (e != hipSuccess) return hip_fail(e, "hipGetDevice");
    if (dev < 0 || dev >= 64) return fail(ESDA_ERR_DEVICE, "device index out of range");
    static std::mutex mu;
    static void *addr[64] = {nullptr};
    std::lock_guard<std::mutex> lk(mu);
    if (!addr[dev]) {
        void *p = nullptr;
        e = hipGetSymbolAddress(&p, HIP_SYMBOL(scratch));
        if (e != hipSuccess) return hip_fail(e, "hipGetSymbolAddress(scratch)");
        if (!p) return fail(ESDA_ERR_RUNTIME, "hipGetSymbolAddress(scratch) returned null");
        addr[dev] = p;
    }
    *out = addr[dev];
    return ESDA_OK;
}

}  // namespace

extern "C" {

const char *esda_last_error(void) { return g_err.c_str(); }

int esda_version(void) { return 100; }

int esda_decode_workspace_size(const esda_decode_desc *desc, size_t *bytes) {
    Plan pl;
    int rc = make_plan(desc, &pl);
    if (rc) return rc;
    if (!bytes) return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode_workspace_size: null output");
    *bytes = pl.bytes;
    return ESDA_OK;
}

int esda_decode_stages(const esda_decode_desc *d, const esda_decode_args *a, int stages,
                       void *stream) {
    Plan pl;
    int rc = make_plan(d, &pl);
    if (rc) return rc;
    rc = check_decode_args(d, a);
    if (rc) return rc;
    if (!a->workspace || a->workspace_bytes < pl.bytes || !aligned16(a->workspace))
        return fail(ESDA_ERR_WORKSPACE, "esda_decode: workspace missing or smaller than esda_decode_workspace_size");
    if ((stages & (ESDA_STAGE_ATTEND | ESDA_STAGE_MERGE)) == 0 || (stages & ~3))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode_stages: bad stage mask");
    rc = check_device();
    if (rc) return rc;
    return run_stages(d, pl, decode_params(d, a), static_cast<uint16_t *>(a->out), a->workspace, stages, 0,
                      reinterpret_cast<hipStream_t>(stream));
}

int esda_decode_noalloc(const esda_decode_desc *d, const esda_decode_args *a, void *stream) {
    Plan pl;
    int rc = make_plan(d, &pl);
    if (rc) return rc;
    rc = check_decode_args(d, a);
    if (rc) return rc;
    // The workspace argument is optional here and only ever the status word.
    if (a->workspace && (a->workspace_bytes < sizeof(int32_t) || (reinterpret_cast<uintptr_t>(a->workspace) & 3u)))
        return fail(ESDA_ERR_WORKSPACE, "esda_decode_noalloc: a status word needs >= 4 bytes, 4-byte aligned");
    if (pl.bytes > kScratchBytes)
        return fail(ESDA_ERR_WORKSPACE, "esda_decode_noalloc: this step needs " + std::to_string(pl.bytes) +
                                            " bytes of scratch; the library's static scratch holds " +
                                            std::to_string(kScratchBytes) + " (use esda_decode with a workspace)");
    rc = check_device();
    if (rc) return rc;
    void *ws = nullptr;
    rc = scratch_address(&ws);
    if (rc) return rc;
    int *status = a->workspace ? static_cast<int *>(a->workspace) : static_cast<int *>(ws);
    return run_stages(d, pl, decode_params(d, a), static_cast<uint16_t *>(a->out), ws,
                      ESDA_STAGE_ATTEND | ESDA_STAGE_MERGE, 0, reinterpret_cast<hipStream_t>(stream), status);
}

int esda_decode(const esda_decode_desc *desc, const esda_decode_args *args, void *stream) {
    return esda_decode_stages(desc, args, ESDA_STAGE_ATTEND | ESDA_STAGE_MERGE, stream);
}

int esda_decode_raw_workspace_size(const esda_raw_desc *desc, size_t *bytes) {
    esda_decode_desc d;
    int rc = raw_as_decode(desc, &d);
    if (rc) return rc;
    Plan pl;
    rc = make_plan(&d, &pl, /*raw=*/true);
    if (rc) return rc;
    if (!bytes) return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode_raw_workspace_size: null output");
    *bytes = pl.bytes;
    return ESDA_OK;
}

int esda_decode_raw_stages(const esda_raw_desc *desc, const esda_raw_args *a, int stages, void *stream) {
    esda_decode_desc d;
    int rc = raw_as_decode(desc, &d);
    if (rc) return rc;
    Plan pl;
    rc = make_plan(&d, &pl, /*raw=*/true);
    if (rc) return rc;
    if (!a) return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode_raw: null arguments");
    if (!a->q || !a->raw_cache || !a->pos || !a->kw || !a->inv_freq || !a->out)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode_raw: null device pointer");
    if (!aligned16(a->q) || (a->k_new && !aligned16(a->k_new)) || !aligned16(a->raw_cache) ||
        !aligned16(a->kw) || !aligned16(a->inv_freq) || !aligned16(a->out))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode_raw: tensors must be 16-byte aligned");
    if (a->rope_table && (a->rope_table_rows < d.cap || !aligned16(a->rope_table)))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode_raw: rope_table needs >= cap rows, 16-byte aligned");
    if (!a->workspace || a->workspace_bytes < pl.bytes || !aligned16(a->workspace))
        return fail(ESDA_ERR_WORKSPACE, "esda_decode_raw: workspace missing or smaller than esda_decode_raw_workspace_size");
    if ((stages & (ESDA_STAGE_ATTEND | ESDA_STAGE_MERGE)) == 0 || (stages & ~3))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode_raw_stages: bad stage mask");
    rc = check_device();
    if (rc) return rc;
    AttendParams ap{};
    ap.q = static_cast<const uint16_t *>(a->q);
    ap.k_new = static_cast<const uint16_t *>(a->k_new);
    ap.v_new = ap.k_new;
    ap.k_cache = static_cast<uint16_t *>(a->raw_cache);
    ap.v_cache = ap.k_cache;
    ap.pos = a->pos;
    ap.row_base = nullptr;
    ap.kw = static_cast<const uint16_t *>(a->kw);
    ap.inv_freq = a->inv_freq;
    ap.rope_tab = static_cast<const unsigned *>(a->rope_table);
    ap.eps = desc->eps;
    return run_stages(&d, pl, ap, static_cast<uint16_t *>(a->out), a->workspace, stages, 1,
                      reinterpret_cast<hipStream_t>(stream));
}

int esda_decode_raw(const esda_raw_desc *desc, const esda_raw_args *args, void *stream) {
    return esda_decode_raw_stages(desc, args, ESDA_STAGE_ATTEND | ESDA_STAGE_MERGE, stream);
}

int esda_decode_raw_q8_stages(const esda_raw_desc *desc, const esda_raw_q8_args *a, int stages, void *stream) {
    esda_decode_desc d;
    int rc = raw_as_decode(desc, &d);
    if (rc) return rc;
    if ((d.head_stride % 16) || (d.seq_stride % 16))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode_raw_q8: u8 strides must be multiples of 16 bytes");
    Plan pl;
    rc = make_plan(&d, &pl, /*raw=*/true);
    if (rc) return rc;
    if (!a) return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode_raw_q8: null arguments");
    if (!a->q || !a->q8_cache || !a->scale || !a->bias || !a->pos || !a->kw || !a->inv_freq || !a->out)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode_raw_q8: null device pointer");
    if (!aligned16(a->q) || (a->k_new && !aligned16(a->k_new)) || !aligned16(a->q8_cache) ||
        !aligned16(a->kw) || !aligned16(a->inv_freq) || !aligned16(a->out) ||
        (reinterpret_cast<uintptr_t>(a->scale) & 3u) || (reinterpret_cast<uintptr_t>(a->bias) & 3u))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode_raw_q8: tensors must be 16-byte aligned (scale / bias 4)");
    if (a->rope_table && (a->rope_table_rows < d.cap || !aligned16(a->rope_table)))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode_raw_q8: rope_table needs >= cap rows, 16-byte aligned");
    if (a->sb_head_stride < d.cap || a->sb_seq_stride < (int64_t) d.num_kv_heads * a->sb_head_stride)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode_raw_q8: scale / bias strides smaller than the cache");
    if (!a->workspace || a->workspace_bytes < pl.bytes || !aligned16(a->workspace))
        return fail(ESDA_ERR_WORKSPACE, "esda_decode_raw_q8: workspace missing or smaller than esda_decode_raw_workspace_size");
    if ((stages & (ESDA_STAGE_ATTEND | ESDA_STAGE_MERGE)) == 0 || (stages & ~3))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode_raw_q8_stages: bad stage mask");
    rc = check_device();
    if (rc) return rc;
    AttendParams ap{};
    ap.q = static_cast<const uint16_t *>(a->q);
    ap.k_new = static_cast<const uint16_t *>(a->k_new);
    ap.v_new = ap.k_new;
    ap.k_cache = static_cast<uint16_t *>(a->q8_cache);  // not read in q8 mode
    ap.v_cache = ap.k_cache;
    ap.q8 = static_cast<unsigned char *>(a->q8_cache);
    ap.qsc = a->scale;
    ap.qbs = a->bias;
    ap.sb_seq_stride = a->sb_seq_stride;
    ap.sb_head_stride = a->sb_head_stride;
    ap.pos = a->pos;
    ap.row_base = nullptr;
    ap.kw = static_cast<const uint16_t *>(a->kw);
    ap.inv_freq = a->inv_freq;
    ap.rope_tab = static_cast<const unsigned *>(a->rope_table);
    ap.eps = desc->eps;
    return run_stages(&d, pl, ap, static_cast<uint16_t *>(a->out), a->workspace, stages, 2,
                      reinterpret_cast<hipStream_t>(stream));
}

int esda_decode_raw_q8(const esda_raw_desc *desc, const esda_raw_q8_args *args, void *stream) {
    return esda_decode_raw_q8_stages(desc, args, ESDA_STAGE_ATTEND | ESDA_STAGE_MERGE, stream);
}

int esda_rope_table(const float *inv_freq, int32_t rows, void *table, void *stream) {
    if (!inv_freq || !table) return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_rope_table: null pointer");
    if (rows < 0) return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_rope_table: rows must be >= 0");
    if (!aligned16(table) || (reinterpret_cast<uintptr_t>(inv_freq) & 3u))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_rope_table: table 16-byte, inv_freq 4-byte aligned");
    int rc = check_device();
    if (rc) return rc;
    const long long n = (long long) rows * kRopePairs;
    if (n == 0) return ESDA_OK;
    hipLaunchKernelGGL(rope_table_kernel, dim3((unsigned) ((n + 255) / 256)), dim3(256), 0,
                       reinterpret_cast<hipStream_t>(stream), inv_freq, n, static_cast<unsigned *>(table));
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? ESDA_OK : hip_fail(e, "rope_table_kernel launch");
}

int esda_quantize_raw_rows(const void *src, int32_t kv_heads, int32_t n_rows, void *q8, int64_t q_head_stride,
                           float *scale, float *bias, int64_t sb_head_stride, int32_t row0, void *stream) {
    if (!src || !q8 || !scale || !bias)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_quantize_raw_rows: null pointer");
    if (kv_heads <= 0 || n_rows < 0 || row0 < 0)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_quantize_raw_rows: bad sizes");
    if (!aligned16(src) || (reinterpret_cast<uintptr_t>(q8) & 7u) || (q_head_stride % 8))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_quantize_raw_rows: src 16-byte, q8 rows 8-byte aligned");
    if (q_head_stride < (int64_t) (row0 + n_rows) * kRawDim || sb_head_stride < row0 + n_rows)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_quantize_raw_rows: head strides smaller than the rows written");
    if (n_rows == 0) return ESDA_OK;
    int rc = check_device();
    if (rc) return rc;
    const long long rows = (long long) kv_heads * n_rows;
    const unsigned blocks = (unsigned) ((rows + 3) / 4);
    hipLaunchKernelGGL(quantize_rows_kernel, dim3(blocks), dim3(256), 0, reinterpret_cast<hipStream_t>(stream),
                       static_cast<const uint16_t *>(src), n_rows, rows, static_cast<unsigned char *>(q8),
                       q_head_stride, scale, bias, sb_head_stride, row0);
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? ESDA_OK : hip_fail(e, "quantize_rows_kernel launch");
}

int esda_decode_status(const esda_decode_desc *desc, void *workspace, int32_t *bad_sequences,
                       void *stream) {
    if (!workspace || !bad_sequences)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_decode_status: null pointer");
    (void) desc;
    hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    int32_t v = 0;
    hipError_t e = hipMemcpyAsync(&v, workspace, sizeof(v), hipMemcpyDeviceToHost, st);
    if (e == hipSuccess) e = hipStreamSynchronize(st);
    if (e != hipSuccess) return hip_fail(e, "esda_decode_status read");
    const int32_t zero = 0;
    e = hipMemcpyAsync(workspace, &zero, sizeof(zero), hipMemcpyHostToDevice, st);
    if (e == hipSuccess) e = hipStreamSynchronize(st);
    if (e != hipSuccess) return hip_fail(e, "esda_decode_status clear");
    *bad_sequences = v;
    return ESDA_OK;
}

int esda_kv_append(void *cache, int64_t seq_stride, int64_t head_stride, int32_t batch,
                   int32_t num_kv_heads, int32_t head_dim, int32_t cap, const void *src,
                   int32_t n_new, const int32_t *row0, void *stream) {
    if (!cache || !src || !row0)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_kv_append: null pointer");
    if (batch <= 0 || num_kv_heads <= 0 || n_new <= 0 || cap <= 0 || head_dim <= 0 || (head_dim % 8))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_kv_append: bad sizes");
    if (head_stride < (int64_t) cap * head_dim || seq_stride < (int64_t) num_kv_heads * head_stride ||
        (head_stride % 8) || (seq_stride % 8))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_kv_append: bad strides");
    if (!aligned16(cache) || !aligned16(src))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_kv_append: tensors must be 16-byte aligned");
    int rc = check_device();
    if (rc) return rc;
    const size_t total = (size_t) n_new * (head_dim / 8);
    int gx = (int) std::min<size_t>((total + 255) / 256, 1024);
    dim3 grid(gx, num_kv_heads, batch);
    hipLaunchKernelGGL(append_kernel, grid, dim3(256), 0, reinterpret_cast<hipStream_t>(stream),
                       static_cast<uint16_t *>(cache), (long long) seq_stride, (long long) head_stride,
                       num_kv_heads, head_dim, cap, static_cast<const uint16_t *>(src), n_new, row0,
                       nullptr);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return hip_fail(e, "append_kernel launch");
    return ESDA_OK;
}

int esda_stream_read(const void *src, size_t bytes, int32_t workgroups, uint32_t *sink, void *stream) {
    if (!src || !sink) return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_stream_read: null pointer");
    if (bytes == 0 || (bytes % 1024) || !aligned16(src))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_stream_read: bytes must be a positive multiple of 1024, src 16-byte aligned");
    if (workgroups < 1 || workgroups > 65535)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_stream_read: workgroups must be in 1 .. 65535");
    int rc = check_device();
    if (rc) return rc;
    hipLaunchKernelGGL(stream_read_kernel, dim3(workgroups), dim3(256), 0, reinterpret_cast<hipStream_t>(stream),
                       static_cast<const unsigned char *>(src), (long long) (bytes / 1024), sink);
    hipError_t e = hipGetLastError();
    return e == hipSuccess ? ESDA_OK : hip_fail(e, "stream_read_kernel launch");
}

int esda_fill_i32(int32_t *dst, int32_t value, int32_t n, void *stream) {
    if (!dst || n < 0) return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_fill_i32: null pointer or negative count");
    if (n == 0) return ESDA_OK;
    int rc = check_device();
    if (rc) return rc;
    hipLaunchKernelGGL(fill_i32_kernel, dim3((n + 255) / 256), dim3(256), 0,
                       reinterpret_cast<hipStream_t>(stream), dst, value, n);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return hip_fail(e, "fill_i32_kernel launch");
    return ESDA_OK;
}

}  // extern "C"
