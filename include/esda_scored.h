/*
 * esda_scored.h -- C ABI of libesda.so's attention with modified scores and masks (MI355X,
 * gfx950): the decode step and the prefill chunk of esda.h and esda_prefill.h for layers whose
 * scores are capped by a tanh or biased by distance, and for chunks with a document or a prefix
 * mask.  Conventions as in esda.h (plain pointers, caller-owned device memory, explicit HIP
 * stream, ESDA_OK or an error code with esda_last_error()).
 *
 * The reference has the plain scores only (ESAttention.mm:136-193; its one tanh cap is on the
 * logits, ESGemma4TextForCausalLM.mm:58-67) and adds causal and sliding masks
 * (ESGemma4TextModel.mm:68-83).
 *
 * With x = scale q.k of query position qAbs (query head h) and key position kAbs:
 *   s = softcap tanh(x / softcap)      (softcap 0: s = x; within 2^-21 softcap of it up to a softcap
 *                                       of 256, within 2^-21 of itself past that)
 *   s = s - slopes[h] |qAbs - kAbs|    (slopes NULL: no bias)
 * and key j visible to query i iff
 *   (kAbs <= qAbs or kAbs < prefix) and (window == 0 or kAbs > qAbs - window)
 *   and (q_doc NULL or q_doc[i] == k_doc[j] >= 0)
 * out = softmax(s over the visible keys) v; a query that sees no key gives 0.
 */
#ifndef APERTURA_ESDA_SCORED_H
#define APERTURA_ESDA_SCORED_H

#include <stddef.h>
#include <stdint.h>

#include "esda.h"
#include "esda_prefill.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef struct esda_score {
    float softcap;       /* > 0: the cap; 0: none.  One whose quotient with the scale fp32
                            cannot hold, or near fp32's largest number, is refused         */
    int32_t prefix;      /* prefill: keys at positions below it are visible to earlier queries,
                            too (>= 0).  In a decode step every visible key is at or before the
                            token, so it changes nothing                                   */
    const float *slopes; /* [num_q_heads] f32, device memory, or NULL                      */
} esda_score;

/* ------------------------------------------------------------------------- prefill
 * esda_prefill with these scores and masks.  The keys need not hold the queries' own positions
 * (key positions stay below 2^31 - 64).  A value of k or v that is not finite reaches only the
 * queries that see its key.  out must not overlap q, k or v (unlike the plain call's, q's rows may
 * be read after rows of out are written). */
typedef struct esda_scored_prefill_args {
    const void *q, *k, *v; /* as esda_prefill_args; k == v allowed            */
    void *out;
    void *workspace;       /* esda_scored_prefill_workspace_size bytes (may be 0) */
    size_t workspace_bytes;
    const int32_t *q_doc;  /* [seq_q] document ids, device memory, or NULL    */
    const int32_t *k_doc;  /* [seq_k]; given with q_doc only                  */
} esda_scored_prefill_args;

int esda_scored_prefill_workspace_size(const esda_prefill_desc *desc, const esda_score *score, size_t *bytes);
int esda_scored_prefill(const esda_prefill_desc *desc, const esda_score *score, const esda_scored_prefill_args *args,
                        void *stream);

/* ------------------------------------------------------------------------- decode
 * esda_decode with these scores: append, attend, merge (esda_decode_args; every cache mode of
 * esda_decode_desc).  Workspace: esda_decode_workspace_size; skipped sequences:
 * esda_decode_status.  A value of k or v that is not finite reaches only the queries of its
 * sequence and kv head. */
int esda_scored_decode(const esda_decode_desc *desc, const esda_score *score, const esda_decode_args *args,
                       void *stream);

#ifdef __cplusplus
}
#endif
#endif
