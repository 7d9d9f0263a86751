// esda_rope.hip -- rotary positions of q and k rows for MI355X (gfx950).
//
// Replaces the reference's rotation by ops (ESRotaryEmbedding.mm:8-46, ESOps.h:58-62) in front
// of the attention entry points.  The C ABI (include/esda_rope.h) is at the end of the file.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <string>

#include "esda.h"
#include "esda_device.h"
#include "esda_internal.h"
#include "esda_rope.h"
#include "esda_views.h"

namespace {

struct RopeParams {
    const uint16_t *q, *k;
    uint16_t *qo, *ko;
    const int *pos;
    const float *inv_freq;
    long long q_rs, q_hs, k_rs, k_hs, qo_rs, qo_hs, ko_rs, ko_hs;
    int T, Hq, H;        // H: q and k heads together
    int rot, interleaved;
    int np, pieces;      // rotated pieces of a row, and all of them
    int groups;          // threads of one piece over a token's heads
    float c_factor, s_factor;  // attn_factor; the same, negated for the inverse rotation
};

// cos and sin of pos * inv_freq.  The product of an int32 and an fp32 is exact in 64 bits for
// |pos| < 2^29 (within 2^-22 rad up to 2^31), and so is its reduction to |r| <= pi/4 to far
// below fp32: an fp32 product alone is off by 0.06 rad at position 10^6.
__device__ __forceinline__ void sincos_far(int pos, float inv_freq, float &s, float &c) {
    const double a = (double) pos * (double) inv_freq;
    const double n = __builtin_rint(a * 0.63661977236758134308);
    double r = __builtin_fma(-n, 1.57079632679489655800, a);
    r = __builtin_fma(-n, 6.12323399573676603587e-17, r);
    sincos_quadrant((float) r, (int) (n - 4.0 * __builtin_floor(n * 0.25)), s, c);
}

// One thread owns a piece of VEC pairs of one token and walks the token's heads with their cos
// and sin in registers: threads of consecutive pieces are consecutive, then the `groups` threads
// that share the heads of a piece, then tokens.  A piece is two runs of VEC elements: dims VEC i
// on and their partners rot/2 on; interleaved, the two halves of the 2 VEC consecutive elements;
// past the rotated dims, 2 VEC elements to copy.
// y0 = x0 c - x1 s, y1 = x1 c + x0 s, c and s from 64-bit angles, rounded once.  Bound by memory: 8192
// tokens of 40 heads x 128, 168 MB read and written in 35 us (4.75 TB/s; a copy of 1 GB 5.1), the cos
// and sin of a piece formed once for its heads; 64 of 256 dims of 48 heads turned in interleaved pairs
// into other tensors, 2049 tokens, 22.6 us (101 MB, 4.4 TB/s), in place, where the rest is not touched,
// 7.7 (25 MB in pieces of 128 bytes, 3.2 TB/s).  One token is a launch: 4.3 us.
template <int VEC>
__global__ __launch_bounds__(256) void rope_kernel(RopeParams p) {
    typedef uint16_t run __attribute__((ext_vector_type(VEC), aligned(VEC * 2)));
    typedef __bf16 brun __attribute__((ext_vector_type(VEC)));
    constexpr int U = 4;  // heads in flight
    const int per_token = p.groups * p.pieces;
    const int tpb = per_token <= 256 ? 256 / per_token : 1;    // tokens per block
    const int bpt = (per_token + 255) / 256;                   // blocks per token
    const int tid = threadIdx.x;
    const int in_block = tid / per_token;                      // 0 where a token takes whole blocks
    if (in_block >= tpb) return;
    const long long nblk = tpb > 1 ? ((long long) p.T + tpb - 1) / tpb : (long long) p.T * bpt;
    for (long long blk = blockIdx.x; blk < nblk; blk += gridDim.x) {
        const int t = bpt == 1 ? (int) blk * tpb + in_block : (int) (blk / bpt);
        const int x = bpt == 1 ? tid - in_block * per_token : (int) (blk % bpt) * 256 + tid;
        if (t >= p.T || x >= per_token) continue;
        const int hs = x / p.pieces, i = x - hs * p.pieces;
        const bool turns = i < p.np;
        int oa, ob;
        if (!turns) {
            oa = p.rot + 2 * VEC * (i - p.np);
            ob = oa + VEC;
        } else if (p.interleaved) {
            oa = 2 * VEC * i;
            ob = oa + VEC;
        } else {
            oa = VEC * i;
            ob = oa + p.rot / 2;
        }
        float c[VEC], s[VEC];
        if (turns) {
            const int pos = p.pos[t];
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                sincos_far(pos, p.inv_freq[VEC * i + e], s[e], c[e]);
                c[e] *= p.c_factor;
                s[e] *= p.s_factor;
            }
        }
        auto bf = [](uint16_t w) { return __builtin_bit_cast(float, (unsigned) w << 16); };
        for (int h0 = hs; h0 < p.H; h0 += U * p.groups) {
            run a[U], b[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int h = h0 + u * p.groups;
                if (h < p.H) {
                    const uint16_t *src = h < p.Hq ? p.q + t * p.q_rs + h * p.q_hs
                                                   : p.k + t * p.k_rs + (h - p.Hq) * p.k_hs;
                    a[u] = *reinterpret_cast<const run *>(src + oa);
                    b[u] = *reinterpret_cast<const run *>(src + ob);
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int h = h0 + u * p.groups;
                if (h >= p.H) break;
                if (turns) {
                    brun ya, yb;
                    if (VEC > 1 && p.interleaved) {
                        // pair e: elements 2e, 2e + 1 of the piece
#pragma unroll
                        for (int e = 0; e < VEC; ++e) {
                            const float x0 = bf(e < VEC / 2 ? a[u][(2 * e) % VEC] : b[u][(2 * e) % VEC]);
                            const float x1 = bf(e < VEC / 2 ? a[u][(2 * e + 1) % VEC] : b[u][(2 * e + 1) % VEC]);
                            const __bf16 y0 = (__bf16) (x0 * c[e] - x1 * s[e]), y1 = (__bf16) (x1 * c[e] + x0 * s[e]);
                            if (e < VEC / 2) {
                                ya[(2 * e) % VEC] = y0;
                                ya[(2 * e + 1) % VEC] = y1;
                            } else {
                                yb[(2 * e) % VEC] = y0;
                                yb[(2 * e + 1) % VEC] = y1;
                            }
                        }
                    } else {
#pragma unroll
                        for (int e = 0; e < VEC; ++e) {
                            const float x0 = bf(a[u][e]), x1 = bf(b[u][e]);
                            ya[e] = (__bf16) (x0 * c[e] - x1 * s[e]);
                            yb[e] = (__bf16) (x1 * c[e] + x0 * s[e]);
                        }
                    }
                    a[u] = __builtin_bit_cast(run, ya);
                    b[u] = __builtin_bit_cast(run, yb);
                }
                uint16_t *dst = h < p.Hq ? p.qo + t * p.qo_rs + h * p.qo_hs : p.ko + t * p.ko_rs + (h - p.Hq) * p.ko_hs;
                *reinterpret_cast<run *>(dst + oa) = a[u];
                *reinterpret_cast<run *>(dst + ob) = b[u];
            }
        }
    }
}

// ------------------------------------------------------------------------ host side

int fail(int code, const std::string &msg) {
    esda_detail::set_error(msg);
    return code;
}

constexpr long long kThreads = 256 * 512;  // aimed at: 8 waves a CU
constexpr unsigned kMaxBlocks = 1u << 20;

}  // namespace

extern "C" {

int esda_rope(const esda_rope_desc *d, const esda_rope_args *a, void *stream) {
    if (!d || !a) return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_rope: null description or arguments");
    const int D = d->head_dim, T = d->tokens, Hq = d->num_q_heads, Hk = d->num_k_heads;
    if (D != 128 && D != 256 && D != 512)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_rope: head_dim must be 128, 256 or 512");
    if (d->rot_dim < 2 || d->rot_dim > D || d->rot_dim % 2)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_rope: rot_dim must be even, 2 .. head_dim");
    if (T < 0 || T > 1 << 30 || Hq < 0 || Hk < 0 || Hq > 65536 || Hk > 65536 || Hq + Hk == 0)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_rope: 0 .. 2^30 tokens, 0 .. 65536 heads of each kind, and some head given");
    if ((d->interleaved & ~1) || (d->inverse & ~1))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_rope: interleaved and inverse are 0 or 1");
    if (!std::isfinite(d->attn_factor))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_rope: attn_factor must be finite");
    if (T == 0) return ESDA_OK;
    if (!a->pos || !a->inv_freq || (Hq && (!a->q || !a->q_out)) || (Hk && (!a->k || !a->k_out)))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_rope: null device pointer");
    if ((reinterpret_cast<uintptr_t>(a->pos) & 3u) || (reinterpret_cast<uintptr_t>(a->inv_freq) & 3u))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_rope: pos and inv_freq must be 4-byte aligned");
    const char *const names[4] = {"q", "q_out", "k", "k_out"};
    auto view = [&](const void *ptr, int heads, long long rs, long long hs) {
        return esda_views::View{reinterpret_cast<uintptr_t>(ptr), {T, heads}, {rs, hs}, D};
    };
    const esda_views::View v[4] = {view(a->q, Hq, d->q_row_stride, d->q_head_stride),
                                   view(a->q_out, Hq, d->q_out_row_stride, d->q_out_head_stride),
                                   view(a->k, Hk, d->k_row_stride, d->k_head_stride),
                                   view(a->k_out, Hk, d->k_out_row_stride, d->k_out_head_stride)};
    int vec = 8;
    bool copy = false;
    for (int i = 0; i < 4; ++i) {
        const long long heads = v[i].n[1], rs = v[i].st[0], hs = v[i].st[1];
        if (!heads) continue;
        const std::string name = std::string("esda_rope: ") + names[i];
        if (rs < 0 || hs < 0) return fail(ESDA_ERR_INVALID_ARGUMENT, name + " strides must not be negative");
        if (v[i].extent() > (__int128) 1 << 60) return fail(ESDA_ERR_INVALID_ARGUMENT, name + " strides are too large");
        const uintptr_t at = v[i].ptr;
        if (at & 1u) return fail(ESDA_ERR_INVALID_ARGUMENT, name + " must be 2-byte aligned");
        // runs of VEC elements need every row to start on one
        while (vec > 1 && (at % (2 * vec) || (T > 1 && rs % vec) || (heads > 1 && hs % vec))) vec /= 2;
        if (i & 1) {
            if (esda_views::overlaps_itself(v[i]))
                return fail(ESDA_ERR_INVALID_ARGUMENT, name + " strides make rows overlap");
            if (v[i - 1].ptr != v[i].ptr) copy = true;
        }
    }
    // An output may be its own input; otherwise no output shares an element with another tensor.
    for (int o = 1; o < 4; o += 2)
        for (int i = 0; i < 4; ++i) {
            if (i == o || !v[o].n[1] || !v[i].n[1]) continue;
            const bool same = i == o - 1 && v[i].ptr == v[o].ptr && (T == 1 || v[i].st[0] == v[o].st[0]) &&
                              (v[i].n[1] == 1 || v[i].st[1] == v[o].st[1]);
            if (!same && !esda_views::disjoint(v[i], v[o]))
                return fail(ESDA_ERR_INVALID_ARGUMENT, std::string("esda_rope: ") + names[o] + " overlaps " + names[i] +
                                                           (i == o - 1 ? " without being the same view" : ""));
        }
    while (vec > 1 && (d->rot_dim / 2 % vec || (D - d->rot_dim) % (2 * vec))) vec /= 2;
    RopeParams p{};
    p.q = static_cast<const uint16_t *>(a->q);
    p.k = static_cast<const uint16_t *>(a->k);
    p.qo = static_cast<uint16_t *>(a->q_out);
    p.ko = static_cast<uint16_t *>(a->k_out);
    p.pos = a->pos;
    p.inv_freq = a->inv_freq;
    p.q_rs = d->q_row_stride;
    p.q_hs = d->q_head_stride;
    p.k_rs = d->k_row_stride;
    p.k_hs = d->k_head_stride;
    p.qo_rs = d->q_out_row_stride;
    p.qo_hs = d->q_out_head_stride;
    p.ko_rs = d->k_out_row_stride;
    p.ko_hs = d->k_out_head_stride;
    p.T = T;
    p.Hq = Hq;
    p.H = Hq + Hk;
    p.rot = d->rot_dim;
    p.interleaved = d->interleaved;
    p.np = d->rot_dim / 2 / vec;
    p.pieces = p.np + (copy ? (D - d->rot_dim) / (2 * vec) : 0);
    p.c_factor = d->attn_factor;
    p.s_factor = d->inverse ? -d->attn_factor : d->attn_factor;
    // Threads of a piece share its heads: enough of them to fill the GPU, and a wave's worth of
    // consecutive memory per head run.
    const long long fill = (kThreads + (long long) T * p.pieces - 1) / ((long long) T * p.pieces);
    p.groups = (int) std::min<long long>(p.H, std::max<long long>(fill, (64 + p.pieces - 1) / p.pieces));
    const int rc = esda_detail::check_device();
    if (rc != ESDA_OK) return rc;
    const long long per_token = (long long) p.groups * p.pieces;
    const long long tpb = per_token <= 256 ? 256 / per_token : 1, bpt = (per_token + 255) / 256;
    const long long blocks = tpb > 1 ? (T + tpb - 1) / tpb : T * bpt;
    const dim3 grid((unsigned) std::min<long long>(blocks, kMaxBlocks)), block(256);
    hipStream_t st = static_cast<hipStream_t>(stream);
    if (vec == 8) hipLaunchKernelGGL(rope_kernel<8>, grid, block, 0, st, p);
    else if (vec == 4) hipLaunchKernelGGL(rope_kernel<4>, grid, block, 0, st, p);
    else if (vec == 2) hipLaunchKernelGGL(rope_kernel<2>, grid, block, 0, st, p);
    else hipLaunchKernelGGL(rope_kernel<1>, grid, block, 0, st, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return fail(ESDA_ERR_HIP, std::string("rope_kernel launch: ") + hipGetErrorString(e));
    return ESDA_OK;
}

int esda_rope_frequencies(const esda_rope_scaling *s, int32_t rot_dim, float *inv_freq, float *attn_factor) {
    if (!s || !inv_freq || !attn_factor)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_rope_frequencies: null argument");
    if (s->kind < ESDA_ROPE_NONE || s->kind > ESDA_ROPE_YARN)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_rope_frequencies: unknown kind");
    if (rot_dim < 2 || rot_dim % 2 || rot_dim > 512)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_rope_frequencies: rot_dim must be even, 2 .. 512");
    if (!(s->base > 1.0) || !std::isfinite(s->base))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_rope_frequencies: base must be finite and above 1");
    if (s->kind != ESDA_ROPE_NONE && (!(s->factor >= 1.0) || !std::isfinite(s->factor)))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_rope_frequencies: factor must be finite and at least 1");
    if (s->kind == ESDA_ROPE_NTK && rot_dim < 4)
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_rope_frequencies: NTK needs rot_dim of 4 or more");
    const bool ramp = s->kind == ESDA_ROPE_BANDS || s->kind == ESDA_ROPE_YARN;
    if (ramp && (s->trained_len <= 0 || !(s->low > 0.0) || !(s->high > s->low) || !std::isfinite(s->high)))
        return fail(ESDA_ERR_INVALID_ARGUMENT, "esda_rope_frequencies: this kind needs trained_len > 0 and 0 < low < high");
    const double r = rot_dim, two_pi = 6.283185307179586476925;
    const double base = s->kind == ESDA_ROPE_NTK ? s->base * std::pow(s->factor, r / (r - 2.0)) : s->base;
    // the pair that makes `turns` turns over the trained length
    auto pair_of = [&](double turns) { return r * std::log(s->trained_len / (turns * two_pi)) / (2.0 * std::log(s->base)); };
    double lo = 0.0, hi = 0.0;
    if (s->kind == ESDA_ROPE_YARN) {
        lo = std::min(std::max(std::floor(pair_of(s->high)), 0.0), r - 1.0);
        hi = std::min(std::max(std::ceil(pair_of(s->low)), 0.0), r - 1.0);
        if (hi <= lo) hi = lo + 0.001;  // one pair: a step
    }
    for (int i = 0; i < rot_dim / 2; ++i) {
        double f = std::pow(base, -2.0 * i / r);
        if (s->kind == ESDA_ROPE_LINEAR) f /= s->factor;
        if (ramp) {
            const double w = s->kind == ESDA_ROPE_BANDS ? (s->trained_len * f / two_pi - s->low) / (s->high - s->low)
                                                        : 1.0 - (i - lo) / (hi - lo);
            const double keep = std::min(std::max(w, 0.0), 1.0);
            f = keep * f + (1.0 - keep) * f / s->factor;
        }
        inv_freq[i] = (float) f;
    }
    *attn_factor = s->kind == ESDA_ROPE_YARN ? (float) (0.1 * std::log(s->factor) + 1.0) : 1.0f;
    return ESDA_OK;
}

}  // extern "C"
