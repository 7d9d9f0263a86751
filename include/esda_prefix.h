/*
 * esda_prefix.h -- C ABI of libesda.so's decode step over a shared prefix (MI355X, gfx950): a
 * batch whose sequences all begin with the same tokens (one system prompt, several samples of
 * one document) keeps those tokens' K / V rows once, and a step reads them once for the whole
 * batch.  Conventions as in esda.h (plain pointers, caller-owned device memory, explicit HIP
 * stream, ESDA_OK or an error code with esda_last_error()).
 *
 * The reference is batch 1; its counterpart is the prefix kept in one cache under a marker
 * (ESKVCache::markPrefix, ESKVCache.mm:123-143) and attended by the step of ESAttention.mm:188.
 *
 * Sequence b's keys are the prefix rows, positions 0 .. prefix_len - 1, then the rows of its own
 * cache, positions prefix_len .. pos[b] (the row of position p is p - prefix_len):
 *   out = softmax(scale q.k over both) v
 * the values of esda_decode over one cache that holds prefix and own rows, to its rounding.  A value
 * that is not finite reaches only the queries that see its row. */
#ifndef APERTURA_ESDA_PREFIX_H
#define APERTURA_ESDA_PREFIX_H

#include <stddef.h>
#include <stdint.h>

#include "esda.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct esda_prefix_desc {
    esda_decode_desc own;       /* batch, heads, head_dim, scale, and the sequences' own caches: linear
                                   rows (ring 0), no window; cap, max_visible and split_rows count own
                                   rows.  kv_shared: V aliases K in the prefix and in the own caches */
    int32_t prefix_len;         /* 1 .. 2^30; prefix_len + own.cap below 2^31                */
    int32_t split_keys;         /* prefix keys per split (0 = automatic; multiple of 32)     */
    int64_t prefix_head_stride; /* elements; >= prefix_len * head_dim, multiple of 8: element
                                   (kvh, j, d) at prefix[kvh*prefix_head_stride + j*head_dim + d] */
} esda_prefix_desc;

typedef struct esda_prefix_args {
    esda_decode_args own;  /* q, k_new, v_new, own caches, pos (absolute: >= prefix_len; others are
                              skipped and counted, esda_decode_status), out, workspace; row_base
                              must be NULL                                                    */
    const void *prefix_k;  /* bf16 [Hkv, prefix_len, D], 16-byte aligned                      */
    const void *prefix_v;  /* the same; must equal prefix_k when own.kv_shared                */
} esda_prefix_args;

int esda_prefix_decode_workspace_size(const esda_prefix_desc *desc, size_t *bytes);

/* Append the new rows to the own caches and attend prefix and own rows. */
int esda_prefix_decode(const esda_prefix_desc *desc, const esda_prefix_args *args, void *stream);

#ifdef __cplusplus
}
#endif
#endif
