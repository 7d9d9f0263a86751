// esda_prefill.hip -- Gemma-4 prefill attention for MI355X (gfx950, CDNA4).
//
// Reference behaviour (Apertura tree): a chunk of seq > 1 new tokens attends the cache
// through mx::fast::scaled_dot_product_attention (ESAttention.mm:188; raw-K layers
// :328 after the op-level reconstruction :306-326) with the additive mask of
// ESGemma4TextModel.mm:68-83 aligned by ESAttention.mm:17-22; the op-level tiled core
// (ESAttention.mm:195-251) computes the same quantity by online softmax.
//
// Kernels
//   prefill_kernel<D, QB>  one workgroup per (query tile, kv head, key split), 8 waves
//                       (two per SIMD), one workgroup per CU; QB 16-query blocks per wave
//                       (one at D = 512, one or two at D = 256, two at D = 128).  A
//                       query tile is 128 QB query rows of one kv head's GQA group,
//                       ordered position-major (row r: position r / G, group head r % G);
//                       wave w owns rows 16 QB w .. as QB blocks of 16 -- the MFMA N
//                       dimension.  The tile's visible keys (or one split of them)
//                       stream through an LDS ring of 32-key stages filled by LDS DMA,
//                       the next stage landing during this one.  Per stage each
//                       wave forms S^T[32 keys x its queries] over the whole head dim
//                       with v_mfma_f32_16x16x32_bf16 (K rows from LDS, Q^T held in
//                       registers), masks boundary stages by position, runs an fp32
//                       online softmax per query column, and accumulates O^T[D x its
//                       queries] += V^T . P^T, V^T by transpose reads from LDS and P^T
//                       straight from the score registers (the 32 keys are ordered so
//                       that the score layout is the B-operand layout).  O^T stays in
//                       registers (D/16 x QB tiles: QB * D / 16 accumulators per lane).
//                       Four waves and 64-row tiles at D = 512 where the plan
//                       (esda_prefill_plan.h) finds them faster: mostly chunks whose 128-row
//                       tiles would leave CUs idle.
//   prefill_kernel<256, 1, true>  the same with 64-row tiles whose even and odd stages go
//                       to the two wave groups (waves 0-3 and 4-7 on the same query
//                       blocks), folded together through LDS at the end: chunks whose
//                       128-row tiles would leave CUs idle at D = 256.
//   prefill_merge_kernel  reduces split partials (m, l, acc) per (query row, head).
//   raw_prefill_kv_kernel rebuilds K and V of a raw-K (or q8 raw-K) stream by the
//                       reference's op-level rounding points.
// prefill_kernel, its merge and their launch are in esda_prefill_kernel.h, which other entry points
// use too.  The C ABI (include/esda_prefill.h) is at the end of the file.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdint>
#include <cstring>
#include <string>

#include "esda.h"
#include "esda_device.h"
#include "esda_internal.h"
#include "esda_prefill.h"
#include "esda_prefill_kernel.h"
#include "esda_prefill_plan.h"

namespace {

using namespace esda_prefill_plan;

// ------------------------------------------------------------ raw-K reconstruction
//
// Memory-bound: a raw row read, a K and a V row written.  LPR = D / 2E lanes hold a row, each
// E dims of either half (E = 8: 16-byte loads and stores; every rotary pair (d, d + D/2) in one
// lane), so a wave holds 64/LPR consecutive rows, and it does HG kv heads of them: their
// loads are in flight together and share one set of cos / sin and k-norm weights.  Few rows
// take fewer dims a lane (launch_raw_kv).  4 heads
// x 8256 rows 20.0 us (5.1 TB/s), x 16384 rows 33.5 (6.0); one wave per row with 8-byte
// accesses, its own cos / sin and its own weight loads took 33.1 and 58.1.  The sum of squares is an
// fp32 sum by pairs, within the lane and then over the row's lanes (a lane's 16 one after the
// other leave it 3% further from the 64-bit sum); rinv = 1 / sqrt(mean + eps) with
// IEEE division and square root.
struct RawKvParams {
    const uint16_t *raw;        // bf16 rows, or NULL with q8 / scale / bias
    const unsigned char *q8;
    const float *sc, *bs;
    long long raw_hs, sb_hs, out_hs;
    const uint16_t *kw;
    const float *inv_freq;
    float eps;
    int Hkv, rows, pos0;
    uint16_t *k, *v;
};

__device__ __forceinline__ float bf16r(float x) { return (float) (__bf16) x; }

template <int D, bool Q8, int HG, int E>
__global__ __launch_bounds__(256) void raw_prefill_kv_kernel(RawKvParams p) {
#pragma clang fp contract(off)  // every rounding point as written (no fused multiply-add)
    constexpr int HALF = D / 2, LPR = HALF / E, RPW = 64 / LPR;
    typedef uint16_t row_piece __attribute__((ext_vector_type(E), aligned(2)));
    typedef unsigned char code_piece __attribute__((ext_vector_type(E), aligned(1)));
    typedef __bf16 out_piece __attribute__((ext_vector_type(E)));
    const int lane = threadIdx.x & 63, l = lane % LPR;
    const long long wv = (long long) blockIdx.x * 4 + uniform(threadIdx.x >> 6);
    const int row_groups = (p.rows + RPW - 1) / RPW;
    const int h0 = (int) (wv / row_groups) * HG;
    if (h0 >= p.Hkv) return;
    const int tt = (int) (wv % row_groups) * RPW + lane / LPR;
    const int t = min(tt, p.rows - 1);  // rows past the end repeat the last one, unwritten

    row_piece raw[HG][2];
    code_piece code[Q8 ? HG : 1][2];
    float sc[HG], bs[HG];
#pragma unroll
    for (int g = 0; g < HG; ++g) {
        const int h = min(h0 + g, p.Hkv - 1);
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const size_t at = (size_t) h * p.raw_hs + (size_t) t * D + half * HALF + E * l;
            if constexpr (Q8) code[g][half] = *reinterpret_cast<const code_piece *>(p.q8 + at);
            else raw[g][half] = *reinterpret_cast<const row_piece *>(p.raw + at);
        }
        if constexpr (Q8) {
            sc[g] = p.sc[(size_t) h * p.sb_hs + t];
            bs[g] = p.bs[(size_t) h * p.sb_hs + t];
        }
    }
    const row_piece kwa = *reinterpret_cast<const row_piece *>(p.kw + E * l);
    const row_piece kwb = *reinterpret_cast<const row_piece *>(p.kw + HALF + E * l);
    auto bf = [](uint16_t w) { return __builtin_bit_cast(float, (unsigned) w << 16); };
    float c[E], s[E];
    const float pos = (float) (p.pos0 + t);
#pragma unroll
    for (int e = 0; e < E; ++e) {
        float sn, cs;
        sincos_f32(pos * p.inv_freq[E * l + e], sn, cs);
        c[e] = bf16r(cs);
        s[e] = bf16r(sn);
    }
#pragma unroll
    for (int g = 0; g < HG; ++g) {
        if (h0 + g >= p.Hkv) break;
        float x[2][E];
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int e = 0; e < E; ++e) {
                if constexpr (Q8) {
                    const float prod = (float) code[g][half][e] * sc[g];
                    x[half][e] = bf16r(prod + bs[g]);  // the bf16 raw view of the q8 row
                } else {
                    x[half][e] = bf(raw[g][half][e]);
                }
            }
        float sq[E];
#pragma unroll
        for (int e = 0; e < E; ++e) sq[e] = x[0][e] * x[0][e] + x[1][e] * x[1][e];
#pragma unroll
        for (int o = E / 2; o >= 1; o >>= 1)
#pragma unroll
            for (int e = 0; e < o; ++e) sq[e] += sq[e + o];
        float ss = sq[0];
#pragma unroll
        for (int o = LPR / 2; o >= 1; o >>= 1) ss += __shfl_xor(ss, o);
        const float rinv = 1.0f / sqrtf(ss / (float) D + p.eps);
        out_piece ka, kb, va, vb;
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float k0a = bf16r(x[0][e] * rinv * bf(kwa[e]));
            const float k0b = bf16r(x[1][e] * rinv * bf(kwb[e]));
            ka[e] = (__bf16) (bf16r(k0a * c[e]) + bf16r(-k0b * s[e]));
            kb[e] = (__bf16) (bf16r(k0b * c[e]) + bf16r(k0a * s[e]));
            va[e] = (__bf16) (x[0][e] * rinv);
            vb[e] = (__bf16) (x[1][e] * rinv);
        }
        if (tt < p.rows) {
            const size_t at = (size_t) (h0 + g) * p.out_hs + (size_t) t * D + E * l;
            *reinterpret_cast<row_piece *>(p.k + at) = __builtin_bit_cast(row_piece, ka);
            *reinterpret_cast<row_piece *>(p.k + at + HALF) = __builtin_bit_cast(row_piece, kb);
            *reinterpret_cast<row_piece *>(p.v + at) = __builtin_bit_cast(row_piece, va);
            *reinterpret_cast<row_piece *>(p.v + at + HALF) = __builtin_bit_cast(row_piece, vb);
        }
    }
}

// ------------------------------------------------------------ LDS read ceiling
//
// The read rate of the LDS on the prefill kernel's two read forms, for its roofline: each
// wave of W reads its 4 KB share of a 64 KB array, 8 reads in flight per round, with the
// QK operand's 128-bit row reads (TR = false) or the PV operand's 64-bit transpose reads
// ds_read_b64_tr_b16 (TR = true), every lane group of a read on consecutive addresses
// (bank-conflict-free).  Every address is masked into the array.
template <int W, bool TR>
__global__ __launch_bounds__(64 * W, 1) void lds_read_kernel(int iters, unsigned *sink) {
    __shared__ __attribute__((aligned(16))) unsigned char buf[65536];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    for (int i = tid; i < 65536 / 4; i += 64 * W) reinterpret_cast<unsigned *>(buf)[i] = (unsigned) i * 2654435761u;
    __syncthreads();
    const unsigned base = lds_addr(buf);
    constexpr unsigned kStep = TR ? 512u : 1024u, kLane = TR ? 8u : 16u;
    unsigned acc = 0u;
    // The wait names the read registers as operands, so that no use of them is scheduled
    // above it (the compiler does not count the assembly reads).
    for (int it = 0; it < iters; ++it) {
        unsigned a[8];
#pragma unroll
        for (int u = 0; u < 8; ++u)
            a[u] = base + (((unsigned) (it * 8 + u) * kStep + (unsigned) wave * 4096u + (unsigned) lane * kLane) & 65535u);
        if constexpr (TR) {
            u32x2 y[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) asm volatile("ds_read_b64_tr_b16 %0, %1" : "=v"(y[u]) : "v"(a[u]));
            asm volatile("s_waitcnt lgkmcnt(0)"
                         : "+v"(y[0]), "+v"(y[1]), "+v"(y[2]), "+v"(y[3]), "+v"(y[4]), "+v"(y[5]), "+v"(y[6]), "+v"(y[7])
                         :: "memory");
#pragma unroll
            for (int u = 0; u < 8; ++u) acc ^= y[u][0] ^ y[u][1];
        } else {
            u32x4 x[8];
#pragma unroll
            for (int u = 0; u < 8; ++u) asm volatile("ds_read_b128 %0, %1" : "=v"(x[u]) : "v"(a[u]));
            asm volatile("s_waitcnt lgkmcnt(0)"
                         : "+v"(x[0]), "+v"(x[1]), "+v"(x[2]), "+v"(x[3]), "+v"(x[4]), "+v"(x[5]), "+v"(x[6]), "+v"(x[7])
                         :: "memory");
#pragma unroll
            for (int u = 0; u < 8; ++u) acc ^= x[u][0] ^ x[u][1] ^ x[u][2] ^ x[u][3];
        }
    }
    sink[(size_t) blockIdx.x * 64 * W + tid] = acc;
}

// ------------------------------------------------------------ host side

int fail(int code, const std::string &msg) {
    esda_detail::set_error(msg);
    return code;
}

bool aligned16(const void *ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15u) == 0; }

constexpr long long kRawKvWaves = 4 * kTargetGroups;

template <int D, bool Q8>
void launch_raw_kv(const RawKvParams &p, hipStream_t st) {
    auto waves = [&](int E, int HG) {  // HG heads of 128 E / D rows each
        const long long groups = (p.rows + (128 * E / D) - 1) / (128 * E / D);
        return groups * ((p.Hkv + HG - 1) / HG);
    };
    auto grid = [&](int E, int HG) { return dim3((unsigned) ((waves(E, HG) + 3) / 4)); };
    const dim3 block(256);
    // Fewer waves than SIMDs: a call is one wave's latency, and its E cos / sin most of that (us,
    // 8 dims a half / fewer): D = 128 one head x 500 rows 3.4 / 2.7 with one row per wave, x 4000
    // 3.7 / 3.3 (four dims 3.3), x 8000 4.1 / 4.5 (3.8), x 16000 5.0 / 6.8 (5.1); D = 256 x 1000
    // 3.5 / 2.9, x 4000 4.0 / 3.9 (3.8); D = 512, where a row per wave is four dims, x 500 3.6 /
    // 3.2, x 4000 5.1 / 5.0, x 8000 7.5 / 8.1.
    if (waves(8, 1) <= kRawKvWaves / 2)
        hipLaunchKernelGGL((raw_prefill_kv_kernel<D, Q8, 1, D / 128>), grid(D / 128, 1), block, 0, st, p);
    else if (waves(8, 1) <= kRawKvWaves)
        hipLaunchKernelGGL((raw_prefill_kv_kernel<D, Q8, 1, 4>), grid(4, 1), block, 0, st, p);
    // Two heads per wave once that leaves a wave for every SIMD (4 heads x 3000 rows 9.4 us with
    // two, 10.3 with four).
    else if (waves(8, 2) < kRawKvWaves)
        hipLaunchKernelGGL((raw_prefill_kv_kernel<D, Q8, 1, 8>), grid(8, 1), block, 0, st, p);
    else
        hipLaunchKernelGGL((raw_prefill_kv_kernel<D, Q8, 2, 8>), grid(8, 2), block, 0, st, p);
}

int run_raw_kv(const RawKvParams &p, int D, bool q8, hipStream_t st) {
    int rc = esda_detail::check_device();
    if (rc != ESDA_OK) return rc;
    if (p.rows == 0) return ESDA_OK;
    if (q8) launch_raw_kv<512, true>(p, st);
    else if (D == 512) launch_raw_kv<512, false>(p, st);
    else if (D == 256) launch_raw_kv<256, false>(p, st);
    else launch_raw_kv<128, false>(p, st);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(ESDA_ERR_HIP, std::string("raw_prefill_kv launch: ") + hipGetErrorString(e));
    return ESDA_OK;
}

}  // namespace

extern "C" {

int esda_prefill_workspace_size(const esda_prefill_desc *desc, size_t *bytes) {
    if (!bytes) return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_prefill_workspace_size: null output");
    PrefillParams p;
    if (const char *why = last_plan(desc, 0, &p)) return fail(ESDA_ERR_INVALID_ARGUMENT, why);
    *bytes = workspace_of(p, desc->head_dim);
    return ESDA_OK;
}

int esda_prefill_stages(const esda_prefill_desc *desc, const esda_prefill_args *a, int stages, void *stream) {
    PrefillParams p;
    if (const char *why = last_plan(desc, 0, &p)) return fail(ESDA_ERR_INVALID_ARGUMENT, why);
    if (!a || !a->q || !a->k || !a->v || !a->out) return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_prefill: null pointer");
    if (!aligned16(a->q) || !aligned16(a->k) || !aligned16(a->v) || !aligned16(a->out))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_prefill: tensors must be 16-byte aligned");
    const int D = desc->head_dim;
    const size_t need = workspace_of(p, D);
    if (need) {
        if (!a->workspace || a->workspace_bytes < need || !aligned16(a->workspace))
            return fail(ESDA_ERR_WORKSPACE, "esda_prefill: workspace missing or smaller than "
                                            "esda_prefill_workspace_size");
        const size_t rows = (size_t) p.Sq * p.Hq;
        p.part_acc = static_cast<float *>(a->workspace);
        p.part_ml = reinterpret_cast<float *>(static_cast<char *>(a->workspace) + (size_t) p.splits * rows * D * 4);
    }
    const int rc = esda_detail::check_device();
    if (rc != ESDA_OK) return rc;
    p.q = static_cast<const uint16_t *>(a->q);
    p.k = static_cast<const uint16_t *>(a->k);
    p.v = static_cast<const uint16_t *>(a->v);
    p.out = static_cast<uint16_t *>(a->out);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (D == 512) launch_prefill<512>(p, stages, st);
    else if (D == 256) launch_prefill<256>(p, stages, st);
    else launch_prefill<128>(p, stages, st);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(ESDA_ERR_HIP, std::string("esda_prefill launch: ") + hipGetErrorString(e));
    return ESDA_OK;
}

int esda_prefill(const esda_prefill_desc *desc, const esda_prefill_args *a, void *stream) {
    return esda_prefill_stages(desc, a, 3, stream);
}

int esda_raw_prefill_kv(const void *raw, int64_t raw_head_stride, int32_t kv_heads, int32_t rows, int32_t head_dim,
                        const void *kw, float eps, const float *inv_freq, int32_t pos0, void *k_out, void *v_out,
                        int64_t out_head_stride, void *stream) {
    if (head_dim != 128 && head_dim != 256 && head_dim != 512)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_raw_prefill_kv: head_dim must be 128, 256 or 512");
    if (!raw || !kw || !inv_freq || !k_out || !v_out)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_raw_prefill_kv: null pointer");
    if (kv_heads <= 0 || rows < 0 || pos0 < 0 || !(eps >= 0.0f) ||
        (kv_heads > 1 && (raw_head_stride < (int64_t) rows * head_dim || out_head_stride < (int64_t) rows * head_dim)))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_raw_prefill_kv: invalid sizes or strides");
    RawKvParams p{};
    p.raw = static_cast<const uint16_t *>(raw);
    p.raw_hs = raw_head_stride;
    p.out_hs = out_head_stride;
    p.kw = static_cast<const uint16_t *>(kw);
    p.inv_freq = inv_freq;
    p.eps = eps;
    p.Hkv = kv_heads;
    p.rows = rows;
    p.pos0 = pos0;
    p.k = static_cast<uint16_t *>(k_out);
    p.v = static_cast<uint16_t *>(v_out);
    return run_raw_kv(p, head_dim, false, static_cast<hipStream_t>(stream));
}

int esda_raw_q8_prefill_kv(const void *q8, int64_t q_head_stride, const float *scale, const float *bias,
                           int64_t sb_head_stride, int32_t kv_heads, int32_t rows, const void *kw, float eps,
                           const float *inv_freq, int32_t pos0, void *k_out, void *v_out, int64_t out_head_stride,
                           void *stream) {
    if (!q8 || !scale || !bias || !kw || !inv_freq || !k_out || !v_out)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_raw_q8_prefill_kv: null pointer");
    if (kv_heads <= 0 || rows < 0 || pos0 < 0 || !(eps >= 0.0f) ||
        (kv_heads > 1 && (q_head_stride < (int64_t) rows * 512 || sb_head_stride < rows ||
                          out_head_stride < (int64_t) rows * 512)))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_raw_q8_prefill_kv: invalid sizes or strides");
    RawKvParams p{};
    p.q8 = static_cast<const unsigned char *>(q8);
    p.sc = scale;
    p.bs = bias;
    p.raw_hs = q_head_stride;
    p.sb_hs = sb_head_stride;
    p.out_hs = out_head_stride;
    p.kw = static_cast<const uint16_t *>(kw);
    p.inv_freq = inv_freq;
    p.eps = eps;
    p.Hkv = kv_heads;
    p.rows = rows;
    p.pos0 = pos0;
    p.k = static_cast<uint16_t *>(k_out);
    p.v = static_cast<uint16_t *>(v_out);
    return run_raw_kv(p, 512, true, static_cast<hipStream_t>(stream));
}

int esda_lds_read(int32_t waves, int32_t transpose, int32_t iters, int32_t workgroups, uint32_t *sink,
                  void *stream) {
    if (!sink) return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_lds_read: null sink");
    if (iters <= 0 || workgroups <= 0 || workgroups > 65535)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_lds_read: iters must be positive, workgroups in 1 .. 65535");
    const hipStream_t st = reinterpret_cast<hipStream_t>(stream);
    const dim3 grid(workgroups);
    const bool tr = transpose != 0;
    if (waves != 4 && waves != 8 && waves != 16)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_lds_read: waves must be 4, 8 or 16");
    if (waves == 4 && tr) hipLaunchKernelGGL((lds_read_kernel<4, true>), grid, dim3(256), 0, st, iters, sink);
    if (waves == 4 && !tr) hipLaunchKernelGGL((lds_read_kernel<4, false>), grid, dim3(256), 0, st, iters, sink);
    if (waves == 8 && tr) hipLaunchKernelGGL((lds_read_kernel<8, true>), grid, dim3(512), 0, st, iters, sink);
    if (waves == 8 && !tr) hipLaunchKernelGGL((lds_read_kernel<8, false>), grid, dim3(512), 0, st, iters, sink);
    if (waves == 16 && tr) hipLaunchKernelGGL((lds_read_kernel<16, true>), grid, dim3(1024), 0, st, iters, sink);
    if (waves == 16 && !tr) hipLaunchKernelGGL((lds_read_kernel<16, false>), grid, dim3(1024), 0, st, iters, sink);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? ESDA_OK : fail(ESDA_ERR_HIP, std::string("lds_read_kernel launch: ") + hipGetErrorString(e));
}

}  // extern "C"
