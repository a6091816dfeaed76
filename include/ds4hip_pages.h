/* ds4hip_pages.h — a paged FP8 KV cache: its pages, and the attention that
 * reads them.
 *
 * Same status convention as ds4hip.h. Every call is asynchronous on `stream`,
 * allocates nothing and may be captured into a graph; calls on one pool are ordered
 * on one stream by the caller. No counterpart in the reference, whose cache is
 * one ring and one compressed list per layer (include/ds4cuda.h:310-425).
 */
#ifndef DS4HIP_PAGES_H
#define DS4HIP_PAGES_H

#include <stddef.h>
#include <stdint.h>

#include "ds4hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- the pool ------------------------------------------------------------------ */

#define DS4HIP_PAGES_MAX_JOBS 1024   /* sequences of one call */
#define DS4HIP_PAGES_MAX_SEQS 65536  /* sequences of one pool */

/* n_pages pages of page_rows rows (a power of two) in the row layout of
 * ds4hip.h, for n_layers layers: row r of page g is row g * page_rows + r, of layer l
 * at l * layer_rows more. All arrays are caller-owned device memory; codes and
 * tail are 16-byte aligned, sexp 8-byte.
 *   refs   [n_pages] how many sequences hold the page; 0: free
 *   table  [n_seqs][table_stride] the pages of each sequence, in order; entries
 *          past those its rows take have no meaning and may be overwritten
 *   rows   [n_seqs] rows each sequence holds (0: it holds no page)
 *   status [1] what a call finds out on the device: -22 (a sequence, page or
 *          count outside the pool, or a case that the call names), -28 (too few
 *          free pages, or a table row is full). Written by a refused call
 *          only, never reset by the library. A refused call changes nothing else
 *          that has a meaning.
 * A page that has room left is held by one sequence only: fork copies a partly
 * filled last page. Sequences are numbered by their table row. */
typedef struct ds4hip_kv_pages {
    uint8_t *codes;
    int8_t *sexp;
    uint16_t *tail;
    long long layer_rows;
    int n_layers, n_pages, page_rows;
    int table_stride, n_seqs;
    int32_t *refs, *table, *rows, *status;
} ds4hip_kv_pages;

/* An empty pool: refs, rows and status 0, table -1. */
int ds4hip_kv_pages_init(const ds4hip_kv_pages *p, void *stream);

/* Bytes of workspace for fork, compact, keep and accept on this pool (8-byte aligned; calls
 * that share one are ordered on one stream). */
size_t ds4hip_kv_pages_workspace_bytes(const ds4hip_kv_pages *p);

/* Gives sequence seqs[j] n_new[j] >= 0 more rows (device int32 arrays, n_jobs
 * <= DS4HIP_PAGES_MAX_JOBS, no sequence twice): the lowest free pages are taken, in
 * the order of the jobs, and dst_rows (device int64 [n_dst]) receives the rows'
 * places, job after job, the dst_rows argument of ds4hip_kv_pages_append. Entries
 * past the last job's are -1, and all are -1 where the call is refused. -22:
 * also more rows than n_dst, or a last page with room that another sequence
 * holds too. */
int ds4hip_kv_pages_extend(const ds4hip_kv_pages *p, const int32_t *seqs, const int32_t *n_new, int n_jobs,
                           long long *dst_rows, int n_dst, void *stream);

/* ds4hip_fp8_kv_quantize_append of n_rows fp32 rows [n_rows][512] into layer
 * `layer` at dst_rows; a row whose place is outside the pool (-1) is skipped. */
int ds4hip_kv_pages_append(const ds4hip_kv_pages *p, int layer, const float *kv, int n_rows,
                           const long long *dst_rows, void *stream);

/* Makes children[j], which must hold nothing, a copy of the first n_rows[j] rows of
 * parents[j] (all of them where n_rows is NULL or n_rows[j] < 0). deep 0: full
 * pages are shared and a partly filled last one is copied to a free page; 1: every
 * page is copied. A parent may be named many times, a child once; what is
 * read is the pool before the call. */
int ds4hip_kv_pages_fork(const ds4hip_kv_pages *p, const int32_t *parents, const int32_t *children,
                         const int32_t *n_rows, int n_jobs, int deep, void *workspace, size_t workspace_bytes,
                         void *stream);

/* Cuts sequence seqs[j] down to its first keep[j] rows (none where keep is NULL)
 * and releases the pages past them; a page that no sequence holds any more is free.
 * No sequence twice; 0 <= keep[j] <= its rows. -22: also a cut inside a page
 * that another sequence holds too (fork the first keep[j] rows instead). */
int ds4hip_kv_pages_free(const ds4hip_kv_pages *p, const int32_t *seqs, const int32_t *keep, int n_jobs,
                         void *stream);

/* Moves the held pages to the front of the pool: with n held pages, those at n and
 * above go, in order, to the free ones below n, in all layers, and the tables
 * name them there. *n_live (device) receives n. */
int ds4hip_kv_pages_compact(const ds4hip_kv_pages *p, int32_t *n_live, void *workspace, size_t workspace_bytes,
                            void *stream);

/* ---- drafted trees ------------------------------------------------------------------ */

#define DS4HIP_TREE_MAX_NODES 1024   /* drafted nodes of one sequence */

/* After a step over drafted tokens: of job j's tree, whose q_start[j + 1] - q_start[j] nodes (device int32
 * [n_jobs + 1], ascending, 0 <= .. <= n_nodes) are the last rows of sequence seqs[j], the n_path[j] nodes path[q_start[j]], ..
 * stay (ascending, each a node of its own tree): the row of the i-th becomes the i-th row behind
 * those before the tree's, in all layers, and the sequence ends there; pages past it are
 * released. No sequence twice. -22: also a path that is not such nodes, more nodes than the
 * sequence has rows, or a page with rows of the tree's in it that another sequence holds too. */
int ds4hip_kv_pages_keep(const ds4hip_kv_pages *p, const int32_t *seqs, const int32_t *q_start, int n_jobs,
                         const int32_t *path, int n_nodes, const int32_t *n_path, void *workspace, size_t workspace_bytes,
                         void *stream);

/* The same with the paths found here, by what the model says after each node. parents, tokens and targets (device int32
 * [n_nodes], as ds4hip_flash_attn_tree_fp8 takes the nodes): each node's parent, its drafted token, and
 * the token that follows it (sampled; < 0 agrees with no draft). A path begins with node 0 and goes on with the first
 * node that has its last one as parent and that one's target as token, until there is none. path receives the
 * nodes (-1 behind them and where no job has nodes, also where there are no jobs), n_path their numbers and next [n_jobs] the
 * target of each last one: the token that the step adds behind the drafts (no nodes: 0 and -1). Where the call is
 * refused, path and next are -1 and n_path 0. -22: also more than DS4HIP_TREE_MAX_NODES nodes. */
int ds4hip_kv_pages_accept(const ds4hip_kv_pages *p, const int32_t *seqs, const int32_t *q_start, int n_jobs,
                           const int32_t *parents, const int32_t *tokens, const int32_t *targets, int n_nodes,
                           int32_t *path, int32_t *n_path, int32_t *next, void *workspace, size_t workspace_bytes,
                           void *stream);

/* ---- attention over pages --------------------------------------------------------- */

/* Attention of n_q packed queries [n_q][n_head][512] over the rows of their
 * sequences, of one layer. Entry s < n_seqs (at most 4096) is the sequence in table
 * row seq_ids[s] (or s), with rows[] rows in all; its queries are q_start[s] ..
 * q_start[s + 1] - 1, its last tokens in order (their own rows are in the
 * cache): query i of n sits at position rows - n + i. q_start NULL: one query
 * each, at its last row. A query at position p sees row k where
 *   k <= p and (window == 0 or k > p - window or k < n_first),
 * and its softmax runs over those rows and, where sinks is not NULL, the
 * head's sink logit (a term of the denominator with no row). It is 0 where it sees
 * nothing; outputs of queries that no entry names are left as they were.
 * n_head: 8, 16, 32, 64 or 128. io_f32 0: q and out are bf16, and weights are rounded to
 * one f16; 1: both are fp32, with q and weights as f16 hi + lo halves. Beside its own rounding and
 * that of fp32 sums, an output is off by up to 2^-10 (io_f32 1: 2^-21) of the same average of
 * |V| and by 2^-15 (2^-21) of the largest weight times the largest |V|, over however many rows (up to
 * 2^23 in bf16, 2^17 in fp32; over more, by as many times more).
 * All arrays are device memory (q, out, codes, tail and workspace 16-byte aligned, sexp
 * 8-byte). The lengths are read on the device, so a captured call follows them. No
 * entry outside the table and no row outside [0, n_cache_rows) is read: queries are NaN
 * where their sequence is outside the table, has more rows than its table row holds (or
 * than 2^31 - 256), or where a group of 32 rows from a multiple of 32 on in which they
 * see one names such a row (with them, up to 64 / n_head - 1 queries next to them in their
 * sequence: 7 of 8 heads, none of 64 or more).
 * A row that is not finite reaches only the queries that see it. */
typedef struct ds4hip_window_attn {
    const void *q;
    void *out;
    int io_f32;
    const float *sinks; /* [n_head] or NULL */
    const uint8_t *codes;
    const int8_t *sexp;
    const uint16_t *tail;
    long long n_cache_rows;
    const int32_t *table; /* [n_slots][table_stride] */
    const int32_t *rows;  /* [n_slots] */
    int n_slots, table_stride, page_rows;
    const int32_t *q_start; /* [n_seqs + 1] or NULL */
    const int32_t *seq_ids; /* [n_seqs] or NULL */
    int n_seqs, n_q, n_head, window, n_first;
} ds4hip_window_attn;
/* Bytes of workspace; enough also for fewer sequences and fewer queries. Two calls that can
 * run at the same time need one each. */
size_t ds4hip_flash_attn_window_fp8_workspace_bytes(int n_seqs, int n_q, int n_head);
int ds4hip_flash_attn_window_fp8(const ds4hip_window_attn *a, void *workspace, size_t workspace_bytes, void *stream);

/* The same attention of trees of drafted tokens. A sequence's queries are the nodes of its tree
 * (n of them, DS4HIP_TREE_MAX_NODES at most), in the order of their rows, its last n: node i is row
 * rows - n + i. parents (device int32 [n_q]) has each node's parent as a node of its own tree, -1 <= parent < i;
 * -1: the node follows the rows before the tree's (at least one such node, the first one). A node's
 * position is rows - n plus the number of its ancestors. It sees the rows before the tree's as a query at its
 * position does, and of the tree its own row and its ancestors', by their positions (p - window < position, or
 * position < n_first); no others. (Chains of parents i - 1 give what ds4hip_flash_attn_window_fp8 gives.) Queries are also
 * NaN where their sequence has more nodes than that or than rows, or where a parent of
 * theirs or of an ancestor's is outside [-1, i) (with the queries next to them, as above).
 * The workspace is ds4hip_flash_attn_window_fp8_workspace_bytes(). */
int ds4hip_flash_attn_tree_fp8(const ds4hip_window_attn *a, const int32_t *parents, void *workspace,
                               size_t workspace_bytes, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* DS4HIP_PAGES_H */
