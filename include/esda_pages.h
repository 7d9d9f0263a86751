/*
 * esda_pages.h -- C ABI of libesda.so's caches in pages (MI355X, gfx950): K / V rows of many
 * sequences in one pool of fixed-size pages, found through a table, shared between sequences by
 * reference counts, and kept in order on the device.  Conventions as in esda.h (plain pointers,
 * caller-owned device memory, explicit HIP stream, ESDA_OK or an error code with
 * esda_last_error()).  esda_tree.h attends such caches.
 *
 * The reference keeps one growing buffer per layer (ESKVCache.mm:64-109), marks and rewinds it
 * (ESKVCache.mm:123-213) and has one sequence; a page pool is what its capacity, its prefix
 * marker and its rewind become for many.
 *
 * Row r of slot s lies in page table[s][r / page_rows], at row r % page_rows of it, in every plane
 * of every pool (a plane is the K or the V of one layer).  length[s] rows are committed; pages
 * behind them may be mapped for rows to come.  A table entry outside 0 .. num_pages - 1 is no page
 * (the calls write -1).  refs[p] is the number of table entries that hold page p; a page of 0 is free.
 * Pages of committed rows may be shared as long as they are full: the page of row length[s] and those
 * behind it belong to s alone (what these calls keep up).
 *
 * Each call takes effect as one step: a fork reads every source as it was before the call.  Pages are
 * taken lowest number first, so the outcome depends on the table, refs and the lists alone.  Nothing
 * is read back: what cannot be done is left out and counted in the workspace's status word
 * (esda_pages_status).  Calls may be captured in a graph; calls on one cache are ordered on one
 * stream, and calls that overlap need workspaces of their own.  What a workspace holds between calls
 * lies where num_pages, slots and max_pages put it: another cache's sizes need another workspace. */
#ifndef APERTURA_ESDA_PAGES_H
#define APERTURA_ESDA_PAGES_H

#include <stddef.h>
#include <stdint.h>

#include "esda.h"

#ifdef __cplusplus
extern "C" {
#endif

#define ESDA_MAX_POOLS 8
#define ESDA_MAX_ENTRIES 1024 /* slots a call names */

/* Element (plane, page, kvh, row, d) at data[plane*plane_stride + page*page_stride +
 * kvh*head_stride + row*head_dim + d] (bf16).  The strides may come in any order; the blocks of
 * page_rows * head_dim elements must not overlap. */
typedef struct esda_pool {
    void *data;           /* device memory, 16-byte aligned             */
    int32_t planes;       /* 1 .. 4096                                  */
    int32_t num_kv_heads; /* 1 .. 4096                                  */
    int32_t head_dim;     /* 128, 256 or 512                            */
    int32_t pad;          /* 0                                          */
    int64_t plane_stride, page_stride, head_stride; /* elements; multiples of 8 */
} esda_pool;

typedef struct esda_pages {
    int32_t num_pages;    /* 1 .. 2^22                                  */
    int32_t page_rows;    /* a power of two, 16 .. 4096                 */
    int32_t slots;        /* 1 .. 2^20                                  */
    int32_t max_pages;    /* 1 .. 2^20; max_pages * page_rows below 2^31 */
    int64_t table_stride; /* ints; >= max_pages                         */
    int32_t *table;       /* [slots][max_pages], device memory          */
    int32_t *refs;        /* [num_pages], device memory                 */
    int32_t *length;      /* [slots], device memory                     */
    int32_t num_pools;    /* 0 .. ESDA_MAX_POOLS                        */
    int32_t pad;          /* 0                                          */
    esda_pool pools[ESDA_MAX_POOLS]; /* one table for all of them; they must not overlap, but may lie
                                        between one another where strides that both have show it */
    void *workspace;      /* esda_pages_workspace_size bytes, 16-byte aligned; zeroed once; must not
                             overlap the pools, table, refs or length */
    size_t workspace_bytes;
} esda_pages;

/* Goes by num_pages, slots and max_pages. */
int esda_pages_workspace_size(const esda_pages *cache, size_t *bytes);

/* Pages for rows up to rows[i] (exclusive) of slot slots[i], from its committed rows on; entries that
 * are mapped stay.  slots, rows: [n], device memory, n <= ESDA_MAX_ENTRIES.  In the order of the list:
 * from the first entry on that the free pages do not suffice for, entries in need of pages are left
 * out and counted; so are entries outside the cache and slots named before in the list. */
int esda_pages_reserve(const esda_pages *cache, const int32_t *slots, const int32_t *rows, int32_t n, void *stream);

/* Slots give up their pages: their entries become -1, their lengths 0.  Entries outside the cache and
 * slots named before in the list are left out and counted. */
int esda_pages_free(const esda_pages *cache, const int32_t *slots, int32_t n, void *stream);

/* Slot dst[i] becomes the first rows[i] rows of slot src[i] (rows NULL, or more than it holds: all of
 * them).  What dst[i] held is given up; full pages are shared; the rows of a last page that is not full
 * are copied to a page of dst[i]'s own in every pool.  dst[i] == src[i] cuts a sequence, which keeps a
 * last page that nobody else holds.  Entries outside the cache, with rows below 0, with rows that lie in
 * no page, and slots named before in dst are left out and counted; an entry that finds no free page
 * leaves its dst empty and is counted.  n <= slots. */
int esda_pages_fork(const esda_pages *cache, const int32_t *src, const int32_t *dst, const int32_t *rows, int32_t n,
                    void *stream);

/* The pages in use move to the front of the pools: with m of them, those numbered m and above, in
 * order, to the free ones below m, in order.  table and refs follow. */
int esda_pages_compact(const esda_pages *cache, void *stream);

/* Reads (synchronously) and clears the status word of a workspace: what the calls on it left out
 * since the last time.  Not for a stream that is being captured. */
int esda_pages_status(void *workspace, int32_t *left_out, void *stream);

/* ------------------------------------------------------------ rows in and out
 * Rows row0[b] .. row0[b] + rows - 1 of sequence b < batch between its pages and a linear buffer, in
 * every plane: element (plane, b, kvh, i, d) at linear[plane*linear_plane_stride + b*linear_seq_stride +
 * kvh*linear_head_stride + i*head_dim + d].  Rows that lie in no page are not written, and read as 0.
 * The linear rows must not overlap the pool. */
typedef struct esda_page_rows_desc {
    esda_pool pool;
    int32_t num_pages, page_rows; /* as in esda_pages                         */
    int32_t batch, max_pages;     /* rows of the table: [batch][max_pages]    */
    int64_t table_stride;
    int32_t rows;                 /* 0 .. 2^30                                */
    int32_t pad;                  /* 0                                        */
    int64_t linear_plane_stride, linear_seq_stride, linear_head_stride; /* elements; multiples of 8 */
} esda_page_rows_desc;

/* linear -> pages.  (Pages of the rows belong to one sequence.) */
int esda_pages_write(const esda_page_rows_desc *desc, const int32_t *table, const int32_t *row0, const void *linear,
                     void *stream);
/* pages -> linear, whose rows must not overlap. */
int esda_pages_read(const esda_page_rows_desc *desc, const int32_t *table, const int32_t *row0, void *linear,
                    void *stream);

#ifdef __cplusplus
}
#endif
#endif
