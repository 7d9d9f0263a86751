/*
 * esda_rope.h -- C ABI of libesda.so's rotary positions (MI355X, gfx950): the rows that the
 * attention entry points take after their rotation.  Conventions as in esda.h (plain pointers,
 * caller-owned device memory, explicit HIP stream, ESDA_OK or an error code with
 * esda_last_error()).
 *
 * The reference rotates q and k by ops on bf16 tables (ESRotaryEmbedding.mm:8-46, rotateHalf
 * ESOps.h:58-62); here the angle is reduced in 64 bits, cos and sin are fp32, and a row is
 * rounded once.  (The raw-K entry points keep the reference's bf16 cos / sin.)
 */
#ifndef APERTURA_ESDA_ROPE_H
#define APERTURA_ESDA_ROPE_H

#include <stdint.h>

#include "esda.h"

#ifdef __cplusplus
extern "C" {
#endif

/* One call: the q and the k rows of `tokens` tokens.
 *
 * Element (t, h, d) of q at q[t*q_row_stride + h*q_head_stride + d], of k and the outputs
 * likewise (bf16).  Pair i < rot_dim / 2 of a row is (x0, x1) = dims (i, i + rot_dim/2), or
 * (2i, 2i + 1) when interleaved; with a = pos[t] * inv_freq[i]:
 *   y0 = f (x0 cos a - x1 sin a),  y1 = f (x1 cos a + x0 sin a),  f = attn_factor
 * and with -a for a when inverse (the rotation's gradient; un-rotating cached rows, with 1 / f where they
 * were turned with f).  Dims rot_dim .. head_dim - 1 are copied.  An inverse frequency of 0 leaves its pair unturned, so a
 * rotation of pairs (d, d + head_dim/2), d < n, alone is rot_dim = head_dim with zeros behind
 * the first n frequencies (the reference's global layers).
 * An output may be its input with the same strides; otherwise they must not overlap. */
typedef struct esda_rope_desc {
    int32_t tokens;       /* 0 .. 2^30                                        */
    int32_t num_q_heads;  /* 0 .. 65536; 0: no q                              */
    int32_t num_k_heads;  /* 0 .. 65536; 0: no k                              */
    int32_t head_dim;     /* 128, 256 or 512                                  */
    int32_t rot_dim;      /* even, 2 .. head_dim                              */
    int32_t interleaved;  /* 0: pairs (i, i + rot_dim/2); 1: pairs (2i, 2i+1) */
    int32_t inverse;      /* 1: by the negative angle                         */
    float attn_factor;    /* multiplies cos and sin (1: a rotation)           */
    int64_t q_row_stride, q_head_stride; /* elements, >= 0                    */
    int64_t k_row_stride, k_head_stride;
    int64_t q_out_row_stride, q_out_head_stride;
    int64_t k_out_row_stride, k_out_head_stride;
} esda_rope_desc;

typedef struct esda_rope_args {
    const void *q, *k;     /* bf16, 2-byte aligned (16-byte aligned rows run fastest) */
    void *q_out, *k_out;
    const int32_t *pos;    /* [tokens] int32, device memory; any value                */
    const float *inv_freq; /* [rot_dim / 2] f32, device memory                        */
} esda_rope_args;

int esda_rope(const esda_rope_desc *desc, const esda_rope_args *args, void *stream);

/* Inverse frequencies of a rotary base, scaled for contexts beyond the trained one.  With
 * f_i = base^(-2i / rot_dim), s = factor, L = trained_len and turns_i = L f_i / (2 pi):
 *   NONE    f_i
 *   LINEAR  f_i / s
 *   NTK     (base s^(rot_dim / (rot_dim - 2)))^(-2i / rot_dim)          (rot_dim > 2)
 *   BANDS   w f_i + (1 - w) f_i / s, w = clamp((turns_i - low) / (high - low), 0, 1)
 *   YARN    w f_i + (1 - w) f_i / s, w = 1 - clamp((i - a) / (b - a), 0, 1), where a and b are
 *           the (fractional) pairs of `high` and `low` turns, rounded down and up, within
 *           0 .. rot_dim - 1; attn_factor = 0.1 ln s + 1 (s > 1)
 * attn_factor is 1 except for YARN. */
#define ESDA_ROPE_NONE 0
#define ESDA_ROPE_LINEAR 1
#define ESDA_ROPE_NTK 2
#define ESDA_ROPE_BANDS 3
#define ESDA_ROPE_YARN 4

typedef struct esda_rope_scaling {
    int32_t kind;        /* ESDA_ROPE_*                                     */
    int32_t trained_len; /* BANDS, YARN: > 0                                */
    double base;         /* > 1                                             */
    double factor;       /* >= 1 (ignored by NONE)                          */
    double low, high;    /* BANDS, YARN: turns, 0 < low < high              */
} esda_rope_scaling;

/* Writes rot_dim / 2 floats to inv_freq and one to attn_factor, both HOST memory. */
int esda_rope_frequencies(const esda_rope_scaling *scaling, int32_t rot_dim, float *inv_freq, float *attn_factor);

#ifdef __cplusplus
}
#endif
#endif
