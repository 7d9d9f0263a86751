// esda_stream.h -- decode attention over one run of cache rows by waves that do not wait for one
// another (gfx950): wave w takes the run's 16-row stages w, w + NW, .. over the whole head dim,
// from LDS slots of its own that it fills by DMA, and the waves' (m, l, O) meet once at the end.
// For workgroups whose stages are short (a 16-row stage of 128-dim rows is 8 KB: a barrier and a
// score exchange per stage, as in attend_kernel, take longer than its bytes: 571 MB 144 us, here 98),
// and for runs inside another kernel's workgroup.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "esda_device.h"

namespace esda_stream {

// What a run is given by: G query rows, rows [j0, j1) (in 16-row stages from j0 on), and
//   dense(jst, stage)    whether rows jst .. jst + 15 of the run lie one behind another: stage.k, stage.v;
//                        every wave calls it for its stages in order, before their loads
//   row(j, k, v)         where row j lies, for stages that are not dense
//   Stage::end           rows of the stage from it on have no weight
//   kUnseen, unseen(jst) whether, and which, rows jst .. jst + 15 have no weight for any query (bits)
//   begun()              called once by every wave after its first loads, before it asks for unseen rows
//   appended(wave, lane) called once by every wave after its last stage
// A run of linear or ring rows, the last one maybe new: rows [j0, j1) of a kv head's nvis visible ones.
template <int D, bool SH>
struct RunOf {
    static constexpr bool kUnseen = false;
    uint16_t *k, *v;               // the cache rows of the kv head
    const uint16_t *k_new, *v_new; // the new token's rows (the last visible row), or null
    int G, j0, j1, nvis, first, cap, newrow;

    struct Stage {
        const uint16_t *k, *v;
        int end;
    };
    __device__ __forceinline__ bool dense(int jst, Stage &st) const {
        st.end = j1;
        st.k = k + (size_t) (first + jst) * D;
        st.v = v + (size_t) (first + jst) * D;
        return jst + 16 < j1 && first + jst + 16 <= cap;  // sixteen consecutive cache rows, none clamped or new
    }
    __device__ __forceinline__ void row(int j, const uint16_t *&kr, const uint16_t *&vr) const {
        int r = first + j;
        if (r >= cap) r -= cap;
        const bool is_new = k_new != nullptr && j == nvis - 1;
        kr = is_new ? k_new : k + (size_t) r * D;
        if constexpr (!SH) vr = is_new ? v_new : v + (size_t) r * D;
    }
    __device__ __forceinline__ void begun() const {}
    // The new row into the cache (bit-exact) by the run that ends with it; no other run reads it.
    __device__ __forceinline__ void appended(int wave, int lane) const {
        if (k_new != nullptr && j1 == nvis && wave == 0)
            for (int c = lane; c < D / 8; c += 64) {
                *reinterpret_cast<u32x4 *>(k + (size_t) newrow * D + 8 * c) = *reinterpret_cast<const u32x4 *>(k_new + 8 * c);
                if constexpr (!SH)
                    *reinterpret_cast<u32x4 *>(v + (size_t) newrow * D + 8 * c) = *reinterpret_cast<const u32x4 *>(v_new + 8 * c);
            }
    }
};

// Rows of a stage that have a weight of 0 for every query: those from row `last` on repeat the run's last one
// or hold anything, and unseen ones do, too.  They are zeros in LDS, row r at rows + off(r): 0 x inf is NaN.
template <int D, class Layout, class Run>
__device__ __forceinline__ void clear_unseen(const Run &x, unsigned char *rows, int jst, int last, int lane) {
    for (unsigned todo = (x.unseen(jst) | 0xffffu << min(last, 16)) & 0xffffu; todo; todo &= todo - 1)
        if (lane < D / 8) *reinterpret_cast<u32x4 *>(rows + Layout::off(__builtin_ctz(todo)) + 16 * lane) = u32x4{0u, 0u, 0u, 0u};
}

// The log2-domain scores of a stage's raw products s (rows jst + 4 lg .. of query row 16 g + li), -inf for
// rows without weight: by score(x, j) one at a time, or by score(s, jst, end, g) together.
template <class Score>
__device__ __forceinline__ void stage_scores(const Score &score, f32x4 &s, int jst, int end, int lg, int g) {
    if constexpr (std::is_invocable<const Score &, f32x4 &, int, int, int>::value) {
        score(s, jst, end, g);
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r) s[r] = jst + 4 * lg + r < end ? score(s[r], jst + 4 * lg + r) : -INFINITY;
    }
}

// NW waves with SLOTS slots each; up to 16 NG query rows.
template <int D, bool SH, int NW, int SLOTS, int NG = 1>
struct Layout {
    static constexpr int BLK = 1056;                // LDS bytes per DMA block: 1 KB + 32 B pad
    static constexpr int NI = D / 32;               // DMA blocks of a tensor's 16-row stage
    static constexpr int HB = NI * BLK;
    static constexpr int SLOT = (SH ? 1 : 2) * HB;
    static constexpr int CPR = D / 8;               // 16-byte chunks per row
    static constexpr int ROWS = 16 * NG;
    static constexpr int CH = D < 32768 / (NW * ROWS) ? D : 32768 / (NW * ROWS);  // dims the waves' O are summed over at a time
    static constexpr int PITCH = CH + 4;            // floats between the rows of that sum (16 rows a multiple of 128
                                                    // bytes apart: each write 16; a 512-dim run of one stage 9.6 us, 12.6)
    static constexpr int SUM = NW * ROWS * PITCH * 4;
    static_assert(CH % 16 == 0 && D % CH == 0, "whole tiles of dims at a time");
    static constexpr int RING = NW * SLOTS * SLOT;
    static constexpr int TOTALS = RING > SUM ? RING : SUM;
    static constexpr int BYTES = TOTALS + (NW + 1) * ROWS * 8;
    // Row r of a stage: block r % NI, 2D bytes times r / NI into it (free of bank conflicts for both
    // the 128-bit row reads and the transpose reads).
    __device__ static constexpr int off(int r) { return (r % NI) * BLK + (r / NI) * 2 * D; }
};

// Attends the run; every thread of the workgroup calls it.  query(h): query row h; score: as
// stage_scores has it, of query row `lane & 15` (of each 16); put(h, d, o, M, T): called once for each
// query row h and four dims from d on, with O, its maximum and its sum.  Each K and V read from LDS serves
// NG products of 16 query rows.
template <int D, bool SH, int NW, int SLOTS, int NG, class Run, class Query, class Score, class Put>
__device__ __forceinline__ void attend_run(unsigned char *lds, Run &x, Query &&query, Score &&score, Put &&put) {
    using L = Layout<D, SH, NW, SLOTS, NG>;
    constexpr int KS = D / 32, DT = D / 16;
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int li = lane & 15, lg = lane >> 4;
    unsigned char *const ring = lds + wave * SLOTS * L::SLOT;
    const int nst = (x.j1 - x.j0 + 15) >> 4;

    const int drow = lane / L::CPR, chunk = lane % L::CPR;  // DMA: this lane's row among a block's, its chunk
    const unsigned voff = (unsigned) ((drow * L::NI * D + chunk * 8) * 2);
    auto dma = [&](int st, unsigned char *slot) -> int {  // the stage's end
        const int jst = x.j0 + 16 * st;
        const unsigned at = lds_addr(slot);
        typename Run::Stage rows;
        if (x.dense(jst, rows)) {
#pragma unroll
            for (int i = 0; i < L::NI; ++i) {
                lds_dma16_s(rows.k + i * D, voff, at + i * L::BLK);
                if constexpr (!SH) lds_dma16_s(rows.v + i * D, voff, at + L::HB + i * L::BLK);
            }
            return rows.end;
        }
#pragma unroll
        for (int i = 0; i < L::NI; ++i) {
            const int j = min(jst + i + L::NI * drow, x.j1 - 1);  // rows past the run repeat its last, masked
            const uint16_t *kr, *vr;
            x.row(j, kr, vr);
            lds_dma16(kr + chunk * 8, at + i * L::BLK);
            if constexpr (!SH) lds_dma16(vr + chunk * 8, at + L::HB + i * L::BLK);
        }
        return rows.end;
    };

    int end = 0, next_end = 0;  // of this stage and the next
    if (wave < nst) end = dma(wave, ring);
    x.begun();
    bf16x8 qv[NG][KS];  // B operands: query row 16 g + li, dims 32 ks + 8 lg ..
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        const bool there = 16 * g + li < x.G;
        const uint16_t *const qr = query(there ? 16 * g + li : 0) + 8 * lg;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const u32x4 w = *reinterpret_cast<const u32x4 *>(qr + 32 * ks);
            qv[g][ks] = __builtin_bit_cast(bf16x8, there ? w : u32x4{0u, 0u, 0u, 0u});
        }
    }
    const int qk_off = L::off(li) + lg * 16, tr_off = L::off(4 * lg + li / 4) + (li % 4) * 8;
    float m[NG], l[NG];
    f32x4 acc[NG][DT];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        m[g] = kNoScore;
        l[g] = 0.0f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) acc[g][dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    for (int st = wave, it = 0; st < nst; st += NW, ++it) {
        unsigned char *const slot = ring + (SLOTS > 1 ? (it & 1) * L::SLOT : 0);
        ESDA_WAIT_VM(0);  // this stage landed
        if (SLOTS > 1 && st + NW < nst) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the other slot's reads are done
            next_end = dma(st + NW, ring + ((it + 1) & 1) * L::SLOT);
        }
        asm volatile("" ::: "memory");
        // Rows past the run repeat its last one, with a weight of 0; but 0 x inf is NaN.
        if constexpr (Run::kUnseen) {
            clear_unseen<D, L>(x, slot + (SH ? 0 : L::HB), x.j0 + 16 * st, max(0, end - (x.j0 + 16 * st)), lane);
        } else {
            for (int r = max(0, end - (x.j0 + 16 * st)); r < 16; ++r)
                if (lane < D / 8) *reinterpret_cast<u32x4 *>(slot + (SH ? 0 : L::HB) + L::off(r) + 16 * lane) = u32x4{0u, 0u, 0u, 0u};
        }
        asm volatile("" ::: "memory");
        // Every K read of the stage, then the products, then every V read, which lands during the
        // softmax.  The scores of few rows go through several sums (a chain of D / 32 products waits for
        // each of them).
        constexpr int CHAINS = NG >= 4 ? 1 : 4 / NG;
        bf16x8 k8[KS];
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) k8[ks] = *reinterpret_cast<const bf16x8 *>(slot + qk_off + 64 * ks);
        __builtin_amdgcn_sched_barrier(0);
        f32x4 s[NG];  // rows 4 lg + r of query row 16 g + li
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            f32x4 part[CHAINS];
#pragma unroll
            for (int c = 0; c < CHAINS; ++c) part[c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
                part[ks % CHAINS] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k8[ks], qv[g][ks], part[ks % CHAINS], 0, 0, 0);
            s[g] = part[0];
#pragma unroll
            for (int c = 1; c < CHAINS; ++c) s[g] += part[c];
        }
        short4v va[DT];
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
            va[dt] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) short4v *) (slot + (SH ? 0 : L::HB) + tr_off + 32 * dt));
        __builtin_amdgcn_sched_barrier(0);
        float top[NG];
        bool raise = false;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            stage_scores(score, s[g], x.j0 + 16 * st, end, lg, g);
            top[g] = wave_max_across_groups(fmaxf(fmaxf(s[g][0], s[g][1]), fmaxf(s[g][2], s[g][3])));
            raise = raise || top[g] > m[g] + kRescaleSlack;
        }
        if (__any(raise)) {
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const float mn = top[g] > m[g] + kRescaleSlack ? top[g] : m[g];
                const float corr = mn == m[g] ? 1.0f : __builtin_amdgcn_exp2f(m[g] - mn);
                l[g] *= corr;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) acc[g][dt] *= corr;
                m[g] = mn;
            }
        }
        // The weights as they enter both sums: bf16, the product's operands.  (At most 2^-8 of a weight:
        // outputs are 0.0017 .. 0.0021 off in relative norm, 0.0017 of it by their own rounding to bf16.)
        short4v pb[NG];
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const __bf16 w = (__bf16) __builtin_amdgcn_exp2f(s[g][r] - m[g]);
                l[g] += (float) w;
                pb[g][r] = __builtin_bit_cast(short, w);
            }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int g = 0; g < NG; ++g) acc[g][dt] = __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(va[dt], pb[g], acc[g][dt], 0, 0, 0);
        if (SLOTS == 1 && st + NW < nst) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the slot's reads are done
            next_end = dma(st + NW, ring);
        }
        end = next_end;
    }
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        l[g] += __shfl_xor(l[g], 16);
        l[g] += __shfl_xor(l[g], 32);
    }

    x.appended(wave, lane);

    // The waves' totals, then their O over CH dims at a time.  A wave without a stage has m = kNoScore, l = 0.
    f32x2 *const ml = reinterpret_cast<f32x2 *>(lds + L::TOTALS), *const tot = ml + NW * L::ROWS;  // [NW][ROWS], [ROWS]
    float *const sum = reinterpret_cast<float *>(lds);                                           // [NW][G][PITCH]
    if (lg == 0)
#pragma unroll
        for (int g = 0; g < NG; ++g) ml[wave * L::ROWS + 16 * g + li] = f32x2{m[g], l[g]};
    lds_barrier();  // and every wave is done with its slots
    float c[NG];
#pragma unroll
    for (int g = 0; g < NG; ++g) {
        const f32x2 *const of = ml + 16 * g + li;
        float M = -INFINITY, T = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) M = fmaxf(M, of[w * L::ROWS][0]);
#pragma unroll
        for (int w = 0; w < NW; ++w) T = __builtin_fmaf(of[w * L::ROWS][1], __builtin_amdgcn_exp2f(of[w * L::ROWS][0] - M), T);
        if (wave == 0 && lg == 0) tot[16 * g + li] = f32x2{M, T};
        c[g] = __builtin_amdgcn_exp2f(m[g] - M);
    }
    const int live = nst < NW ? nst : NW;  // waves that had a stage
#pragma unroll
    for (int d0 = 0; d0 < D; d0 += L::CH) {
        if (wave < live)
#pragma unroll
            for (int g = 0; g < NG; ++g)
                if (16 * g + li < x.G) {
#pragma unroll
                    for (int dt = 0; dt < L::CH / 16; ++dt)
                        *reinterpret_cast<f32x4 *>(sum + (wave * x.G + 16 * g + li) * L::PITCH + 16 * dt + 4 * lg) = acc[g][d0 / 16 + dt] * c[g];
                }
        lds_barrier();
        for (int t = threadIdx.x; t < x.G * (L::CH / 4); t += 64 * NW) {
            const int h = t / (L::CH / 4), d = 4 * (t % (L::CH / 4));
            f32x4 o = *reinterpret_cast<const f32x4 *>(sum + h * L::PITCH + d);
            for (int w = 1; w < live; ++w) o += *reinterpret_cast<const f32x4 *>(sum + (w * x.G + h) * L::PITCH + d);
            put(h, d0 + d, o, tot[h][0], tot[h][1]);
        }
        lds_barrier();  // before the next dims, or the next run's DMAs
    }
}

// The same run by waves that work together, for up to 16 query rows whose O^T over the whole head dim
// takes long to sum (512 dims): groups of SUB 16-row stages in two slots; wave w < SUB scores stage w
// over the whole head dim, every wave reads all scores and holds O^T of D / NW dims.  Two barriers a
// group (64 rows of 1 KB in 1.9 us; attend_run's waves take them in 1.1), and nothing to sum at the end
// (3 us there).
template <int D, bool SH>
struct GroupLayout {
    static constexpr int BLK = 1056, NI = D / 32, HB = NI * BLK;  // (as in Layout)
    static constexpr int CPR = D / 8;
    static constexpr int SUB = (SH ? 1 : 2) * D > 512 ? 2 : 4;
    static constexpr int ROWS = 16 * SUB;
    static constexpr int SLOT = (SH ? 1 : 2) * SUB * HB;
    static constexpr int BYTES = 2 * SLOT + SUB * 1024;  // two slots, then the scores
    __device__ static constexpr int off(int r) { return (r % NI) * BLK + (r / NI) * 2 * D; }
};

// Arguments as attend_run's; put's four dims come from one lane, the rows of 16 side by side.
template <int D, bool SH, int NW, class Run, class Query, class Score, class Put>
__device__ __forceinline__ void attend_groups(unsigned char *lds, Run &x, Query &&query, Score &&score, Put &&put) {
    using L = GroupLayout<D, SH>;
    constexpr int KS = D / 32, DT = D / 16 / NW, SUB = L::SUB;  // k-steps; O^T dim tiles a wave
    constexpr int LOADS = (SH ? 1 : 2) * L::NI;                 // DMAs of a stage
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int li = lane & 15, lg = lane >> 4;
    const bool scores = wave < SUB;
    const int groups = (x.j1 - x.j0 + L::ROWS - 1) / L::ROWS;
    f32x4 *const xch = reinterpret_cast<f32x4 *>(lds + 2 * L::SLOT);  // [SUB][64 lanes]

    const int drow = lane / L::CPR, chunk = lane % L::CPR;
    const unsigned voff = (unsigned) ((drow * L::NI * D + chunk * 8) * 2);
    // This wave's stage of group i; false where it has none or holds no row.
    int end = x.j1, next_end = x.j1;  // of this wave's stage in this group and the next
    auto dma = [&](int i) {
        const int jst = x.j0 + L::ROWS * i + 16 * wave;
        if (!scores || jst >= x.j1) return false;
        const unsigned at = lds_addr(lds) + (i & 1) * L::SLOT + wave * L::HB;
        typename Run::Stage rows;
        const bool dense = x.dense(jst, rows);
        next_end = rows.end;
        if (dense) {
#pragma unroll
            for (int t = 0; t < L::NI; ++t) {
                lds_dma16_s(rows.k + t * D, voff, at + t * L::BLK);
                if constexpr (!SH) lds_dma16_s(rows.v + t * D, voff, at + SUB * L::HB + t * L::BLK);
            }
            return true;
        }
#pragma unroll
        for (int t = 0; t < L::NI; ++t) {
            const int j = min(jst + t + L::NI * drow, x.j1 - 1);  // rows past the run repeat its last, masked
            const uint16_t *kr, *vr;
            x.row(j, kr, vr);
            lds_dma16(kr + chunk * 8, at + t * L::BLK);
            if constexpr (!SH) lds_dma16(vr + chunk * 8, at + SUB * L::HB + t * L::BLK);
        }
        return true;
    };

    dma(0);
    end = next_end;
    x.begun();
    u32x4 qv[KS];  // B operands: query row li, dims 32 ks + 8 lg ..
    const bool there = scores && li < x.G;
    const uint16_t *const qr = query(there ? li : 0) + 8 * lg;
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) {
        const u32x4 w = *reinterpret_cast<const u32x4 *>(qr + 32 * ks);
        qv[ks] = there ? w : u32x4{0u, 0u, 0u, 0u};
    }
    // q in registers before the second group's DMAs (its loads would be waited for with them)
#pragma unroll
    for (int ks = 0; ks < KS; ++ks) asm volatile("" : "+v"(qv[ks]));
    ESDA_WAIT_VM(0);
    bool ahead = groups > 1 && dma(1);  // the next group's stage is under way
    const int qk_off = L::off(li) + lg * 16, tr_off = L::off(4 * lg + li / 4) + (li % 4) * 8;
    float m = kNoScore, l = 0.0f;
    f32x4 acc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) acc[dt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    for (int i = 0; i < groups; ++i) {
        unsigned char *const slot = lds + (i & 1) * L::SLOT;
        if (ahead) ESDA_WAIT_VM(LOADS);
        else ESDA_WAIT_VM(0);
        if (scores) {
            unsigned char *const kb = slot + wave * L::HB, *const vb = SH ? kb : kb + SUB * L::HB;
            const int jst = x.j0 + L::ROWS * i + 16 * wave;
            // Rows past the run repeat its last one or hold anything, with a weight of 0; but 0 x inf is NaN.
            if constexpr (Run::kUnseen) {
                clear_unseen<D, L>(x, vb, jst, max(0, end - jst), lane);
            } else {
                for (int r = max(0, end - jst); r < 16; ++r)
                    if (lane < D / 8) *reinterpret_cast<u32x4 *>(vb + L::off(r) + 16 * lane) = u32x4{0u, 0u, 0u, 0u};
            }
            asm volatile("" ::: "memory");
            f32x4 s = {0.0f, 0.0f, 0.0f, 0.0f};  // (in four sums, as attend_run's, the step took as long)
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const bf16x8 k8 = *reinterpret_cast<const bf16x8 *>(kb + qk_off + 64 * ks);
                s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(k8, __builtin_bit_cast(bf16x8, qv[ks]), s, 0, 0, 0);
            }
            stage_scores(score, s, jst, end, lg, 0);
            xch[wave * 64 + lane] = s;
        }
        lds_barrier();  // every score written, every stage landed
        const unsigned char *const vt = slot + (SH ? 0 : SUB * L::HB) + tr_off + 32 * DT * wave;
        short4v va[DT][SUB];  // V^T, in flight during the softmax
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int u = 0; u < SUB; ++u)
                va[dt][u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) short4v *) (vt + u * L::HB + 32 * dt));
        f32x4 s[SUB];
        float top = -INFINITY;
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
            s[u] = xch[u * 64 + lane];
            top = fmaxf(top, fmaxf(fmaxf(s[u][0], s[u][1]), fmaxf(s[u][2], s[u][3])));
        }
        top = wave_max_across_groups(top);
        if (__any(top > m + kRescaleSlack)) {
            const float mn = top > m + kRescaleSlack ? top : m;
            const float corr = mn == m ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            l *= corr;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) acc[dt] *= corr;
            m = mn;
        }
        bf16x8 pb[SUB / 2];  // the weights as they enter both sums: bf16, the product's operands
#pragma unroll
        for (int u = 0; u < SUB; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const __bf16 w = (__bf16) __builtin_amdgcn_exp2f(s[u][r] - m);
                l += (float) w;
                pb[u / 2][4 * (u % 2) + r] = w;
            }
#pragma unroll
        for (int u = 0; u < SUB; u += 2)
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const short4v a0 = va[dt][u], a1 = va[dt][u + 1];
                const short8v a8 = {a0[0], a0[1], a0[2], a0[3], a1[0], a1[1], a1[2], a1[3]};
                acc[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a8), pb[u / 2], acc[dt], 0, 0, 0);
            }
        lds_barrier();  // every wave is done with the slot and the scores
        end = next_end;
        ahead = i + 2 < groups && dma(i + 2);
    }

    x.appended(wave, lane);
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (li < x.G)
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) put(li, 16 * (DT * wave + dt) + 4 * lg, acc[dt], m, l);
}

}  // namespace esda_stream
