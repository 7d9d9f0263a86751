/*
 * esda_tree.h -- C ABI of libesda.so's step of drafted tokens (MI355X, gfx950): up to 64 new tokens
 * of each sequence, one behind another or as a tree of alternatives, attend a cache in pages
 * (esda_pages.h) or a linear one in one call, and the rows of those that are accepted are moved
 * behind the committed ones.  One token a sequence is the decode step over pages.  Conventions as
 * in esda.h (plain pointers, caller-owned device memory, explicit HIP stream, ESDA_OK or an error code
 * with esda_last_error()).
 *
 * The reference decodes one token of one sequence a step (ESAttention.mm:110-135), and attends a
 * chunk of several causally (ESAttention.mm:195-251).
 *
 * Node i < nodes of sequence b hangs on node parent[b][i] < i, or, where that is -1, on the committed
 * rows; any other value is no node, nor is a node on no node.  parent NULL: a chain, node i on node
 * i - 1.  Node i stands at position length[b] + depth_i (depth 0: on the committed rows) and sees
 *   the committed rows r < length[b] with window == 0 or r > length[b] + depth_i - window,
 *   the nodes above it, and itself:
 *   out[b][i] = softmax(scale q.k over them) v;  0 where i is no node.
 * Node i's K / V row is written to row length[b] + i of its sequence.  length stays: every layer of a
 * step is given the same; esda_tree_commit moves it on.
 * A committed row whose table entry is no page is left out.  A sequence with a negative length, or one
 * whose nodes' rows do not all lie in its pages, is skipped: nothing is written for it, and it is
 * counted (esda_pages_status); one of length 0 whose nodes are all none is a batch's padding: it needs no
 * pages and gives 0.  Pages of the nodes' rows belong to one sequence.  Calls that overlap need
 * workspaces of their own.  A value of k or v that is not finite reaches only the queries that see
 * its row, and what q holds where there is no node none.
 * Scores, maxima and sums are fp32; a weight enters the sum of the weights and that of the values rounded to
 * bf16. */
#ifndef APERTURA_ESDA_TREE_H
#define APERTURA_ESDA_TREE_H

#include <stddef.h>
#include <stdint.h>

#include "esda.h"
#include "esda_pages.h"

#ifdef __cplusplus
extern "C" {
#endif

/* batch * nodes * num_q_heads * head_dim must be below 2^30. */
typedef struct esda_tree_desc {
    int32_t batch;        /* 1 .. 256                                               */
    int32_t nodes;        /* 1 .. 64                                                */
    int32_t num_q_heads;  /* Hq                                                     */
    int32_t num_kv_heads; /* Hkv; Hq / Hkv <= 16; query head h reads kv head h / (Hq / Hkv) */
    int32_t head_dim;     /* 128, 256 or 512                                        */
    int32_t kv_shared;    /* 1: V aliases K (one buffer)                            */
    int32_t window;       /* 0: none; else >= nodes                                 */
    int32_t num_pages;    /* pages of the pool, 1 .. 2^22 (linear: batch)           */
    int32_t page_rows;    /* a power of two, 16 .. 4096 (linear: rows of a sequence, 1 .. 2^30) */
    int32_t max_pages;    /* entries of a sequence's table; 0: linear caches, sequence b in page b */
    int64_t table_stride; /* ints; >= max_pages                                     */
    int64_t page_stride;  /* elements: (page, kvh, row, d) at page*page_stride + kvh*head_stride + row*head_dim + d */
    int64_t head_stride;  /* both multiples of 8; blocks of page_rows * head_dim elements must not overlap */
    int32_t split_rows;   /* rows per split (0: from the lengths, on the device; multiple of 32, of
                             which a sequence's room holds at most 4096)            */
    float scale;          /* softmax scale, positive                                */
} esda_tree_desc;

typedef struct esda_tree_args {
    const void *q;         /* [B, nodes, Hq, D] bf16, 16-byte aligned                */
    const void *k_new;     /* [B, nodes, Hkv, D] bf16                                */
    const void *v_new;     /* the same; ignored when kv_shared                       */
    void *k_pages;         /* a plane of a pool, or a linear cache                   */
    void *v_pages;         /* another, that does not overlap it; must equal k_pages when kv_shared */
    const int32_t *table;  /* [B][max_pages] int32, device memory (linear: NULL)     */
    const int32_t *length; /* [B] int32, device memory: committed rows               */
    const int32_t *parent; /* [B, nodes] int32, device memory, or NULL: a chain      */
    void *out;             /* [B, nodes, Hq, D] bf16; must not overlap q, the new rows or the pages, nor
                              the new rows the pages                                 */
    void *workspace;       /* esda_tree_workspace_size bytes, 16-byte aligned; first 256 zeroed once;
                              must not overlap the other tensors                     */
    size_t workspace_bytes;
} esda_tree_args;

int esda_tree_workspace_size(const esda_tree_desc *desc, size_t *bytes);
int esda_tree_decode(const esda_tree_desc *desc, const esda_tree_args *args, void *stream);

/* The accepted rows behind the committed ones, in every plane of the cache's pools: row length[s] + i
 * becomes row length[s] + accept[s][i] for i < count[s], and length[s] grows by count[s].
 * accept: [slots][max_accept], accept_stride ints apart, and count: [slots], device memory; a slot's
 * entries rise and lie in 0 .. 63.  A slot with another list, a count outside 0 .. max_accept or rows
 * that lie in no page is left as it was and counted.  max_accept: 1 .. 64.  Workgroups of 4096 elements
 * of a row of every plane and head: slots * (planes * num_kv_heads * head_dim / 4096, up, over the pools)
 * at most 2^23.
 * cache->table NULL: linear caches, slot s in page s (num_pages == slots, max_pages 1, page_rows any
 * 1 .. 2^30); refs is not used.  The workspace is esda_pages.h's, zeroed once. */
int esda_tree_commit(const esda_pages *cache, const int32_t *accept, int64_t accept_stride, int32_t max_accept,
                     const int32_t *count, void *stream);

#ifdef __cplusplus
}
#endif
#endif
