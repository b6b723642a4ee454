/* exl3_paged.h -- a paged KV cache and the operators that serve drafted tokens
 * from it, exported by libexl3_mi355x.so next to the decode step's operations
 * (exl3_decoder.h), which keep one contiguous cache and one new row a sequence.
 *
 * The cache of a model is two arrays, keys and values, of
 * [layers][pages][kv_heads][page][dim]: `page` keys of every head of one layer
 * lie together.  A table of pages gives key number x of sequence s its place:
 * page table[s][x / page], row x % page ("slot" table[s][x / page] * page +
 * x % page).  A step brings new rows: a token, the rows of a prompt, or a tree
 * of drafted tokens, for any number of sequences side by side.  Row i of
 * sequence s is its key number len[s] + i, whatever its place in the tree.
 *
 *   exl3p_tree_plan   positions, slots and ancestor masks of the rows (a step)
 *   exl3p_qkv_append  head norms, rotation, keys and values into pages (a layer)
 *   exl3p_attend      attention over the cache and the rows      (a layer)
 *   exl3p_commit      which rows the model's own tokens accept, and their keys
 *                     and values moved behind the context, all layers (a step)
 *   exl3p_copy_pages  pages copied in all layers (forks, compaction)
 *   exl3p_book_*      which pages are whose: host bookkeeping, no device work
 *
 * Device pointers unless said otherwise; every entry records its work on the
 * stream (of the current device), allocates nothing, synchronizes nothing and may
 * be captured into a graph: what is on the device -- lengths, table, tokens -- is
 * read when the work runs.  Refusals are named (exl3_verdict) and launch nothing.
 * What only the device can see is checked by the kernels, which never leave the
 * arrays:
 *  - a sequence whose len is negative, or whose len + rows pass max_pages *
 *    page, has slots of -1 and attends to NaN; exl3p_commit gives it count 0;
 *  - a page number outside [0, pages) among a sequence's keys likewise: slot -1, a
 *    row not moved, and NaN for every row that sees a key of it (and for others of
 *    the sequence that are worked on with such a row);
 *  - cu must ascend from 0 to at most `rows`; rows behind cu[seqs], and a
 *    sequence's rows behind max_rows, get slot -1 and are left as they were by
 *    every other entry.  Where cu goes back, exl3p_attend writes no row.
 */
#ifndef EXL3_PAGED_H
#define EXL3_PAGED_H

#include <stddef.h>
#include <stdint.h>

#include "exl3_mi355x.h"

#ifdef __cplusplus
extern "C" {
#endif

/* A cache.  k, v on a 16-byte boundary; dtype EXL3_DT_F16 or EXL3_DT_BF16 (of
 * q, k, v, the norm weights and the output too); page a power of two from 16
 * to 256; dim 64 or 128; pages * page below 2^31, max_pages * page up to 2^30. */
typedef struct exl3p_cache {
  uint32_t size; /* sizeof(exl3p_cache) */
  int32_t dtype;
  void *k, *v;
  int32_t layers, pages, kv_heads, page, dim;
  int32_t seqs, max_pages;
  const int32_t *table; /* [seqs][max_pages] */
} exl3p_cache;

/* A step's new rows: sequence s has rows cu[s] .. cu[s + 1] - 1 of the step's
 * tensors (none where they are equal) behind len[s] cached keys. */
typedef struct exl3p_rows {
  uint32_t size; /* sizeof(exl3p_rows) */
  int32_t seqs;     /* at most the cache's */
  int32_t rows;     /* rows of the step's tensors, at most 2^30 */
  int32_t max_rows; /* no sequence has more */
  const int32_t *cu;  /* [seqs + 1] */
  const int32_t *len; /* [seqs]; may be NULL where seqs is 0 */
} exl3p_rows;

/* The most rows a sequence may have where a tree is given. */
#define EXL3P_TREE_MAX 1024

/* pos[t] = len + depth of row t (its rotation's position), slot[t] its cache
 * slot, and, with mask [rows][words]: bit j of row i's words is set where j is
 * i or an ancestor of i.  parent[t] is the index of a row's parent among its
 * sequence's rows, -1 for a root; one that does not lie before its row counts
 * as -1.  parent NULL: each row follows the one before it (a prompt).  mask may
 * be NULL (words then 0); words * 64 >= max_rows otherwise.  No output lies over
 * another, or over parent, cu, len or the table. */
exl3_verdict exl3p_tree_plan(const exl3p_cache *c, const exl3p_rows *r, const int32_t *parent,
                             int32_t *pos, int32_t *slot, uint64_t *mask, int32_t words,
                             exl3_stream s);

/* For each of `rows` rows with slot[t] >= 0: q's heads normalized (RMS over the
 * head and finite eps >= 0, times q_norm[dim]; q_norm NULL: as they are), rotated
 * at pos[t] (halves i and i + dim / 2 by pos * theta^(-2 i / dim), the angle in 64
 * bits) to q_out;
 * k's heads the same with k_norm into the cache's keys at slot[t]; v's copied
 * into its values.  One rounding, at the end.  q, k, v and q_out have row
 * strides (in elements, multiples of 8) and 16-byte bases.  q_out may be q, rows
 * of the same stride; apart from that what is written (q_out, the layer's pages)
 * lies over nothing else that is read or written (slices of one matrix are fine).
 * Two rows of one slot: its keys and values are pieces of either's.  Fewer than
 * 2^24 rows a call. */
exl3_verdict exl3p_qkv_append(const exl3p_cache *c, int32_t layer, int32_t rows, int32_t heads,
                              const void *q, int64_t q_stride, const void *k, int64_t k_stride,
                              const void *v, int64_t v_stride, const void *q_norm,
                              const void *k_norm, const int32_t *pos, const int32_t *slot,
                              void *q_out, int64_t out_stride, float eps, double theta,
                              exl3_stream s);

/* out[t] = softmax(q[t] k^T * scale) v over what row t sees: the sequence's
 * first len keys and, of its rows, those in its mask (mask NULL: rows 0 .. i).
 * heads is a multiple of the cache's kv_heads, query head h reads kv head
 * h / (heads / kv_heads).  scale, and scale times log2(e), are finite.  A row that
 * sees nothing is zeros; what a row does not see cannot touch it, NaN or not.
 * scratch: exl3p_attend_scratch_bytes() of the same device, written and read within
 * the call (calls that may overlap need their own); its size goes by the device and
 * the heads, a little by the sequences, and not by the rows once they are many.
 * out may be q, rows of the same stride; apart from that out and the scratch lie
 * over nothing that is read, nor over each other.
 * The sums' order goes by the sizes and lengths alone: results repeat. */
size_t exl3p_attend_scratch_bytes(const exl3p_cache *c, const exl3p_rows *r, int32_t heads);
exl3_verdict exl3p_attend(const exl3p_cache *c, int32_t layer, const exl3p_rows *r, int32_t heads,
                          const void *q, int64_t q_stride, const uint64_t *mask, int32_t words,
                          float scale, void *out, int64_t out_stride, void *scratch,
                          size_t scratch_bytes, exl3_stream s);

/* The walk of each sequence's tree: row 0 is accepted, then from a row the
 * lowest of its children whose ids[] is the row's target[] (the token that the
 * model gives after it), until there is none or max_path rows are accepted.
 * path [seqs][max_path] (indices among the sequence's rows, -1 behind them),
 * count [seqs], next [seqs] = target of the last accepted row (-1 for a
 * sequence without rows), new_len = len + count.  The accepted rows' keys and
 * values move to key numbers len, len + 1, ... in every layer.  No output lies over
 * an input (several workgroups read them: new_len is not r->len, next not ids, and
 * none is in the table), over another output or over the cache.
 * parent NULL: a chain.  At most EXL3P_TREE_MAX rows of a sequence. */
exl3_verdict exl3p_commit(const exl3p_cache *c, const exl3p_rows *r, const int32_t *parent,
                          const int32_t *ids, const int32_t *target, int32_t *path,
                          int32_t max_path, int32_t *count, int32_t *next, int32_t *new_len,
                          exl3_stream s);

/* Page dst[i] = page src[i] in every layer, keys and values.  src and dst are
 * HOST arrays, read before the call returns.  Refused: a page outside the
 * cache, a page written twice, a page both read and written. */
exl3_verdict exl3p_copy_pages(const exl3p_cache *c, const int32_t *src, const int32_t *dst,
                              int32_t count, exl3_stream s);

/* The book of a cache's pages: HOST memory, one user at a time.  Pages have
 * reference counts; free ones are taken lowest first.  Keys of a sequence are
 * numbered from 0; a sequence holds the pages of its first keys. */
typedef struct exl3p_book exl3p_book;
exl3p_book *exl3p_book_open(int32_t pages, int32_t page, int32_t seqs, int32_t max_pages,
                            exl3_verdict *why); /* NULL: *why says why */
void exl3p_book_close(exl3p_book *b);
/* Pages for keys up to `to` of a sequence, and keys from .. to - 1 writable:
 * those of their pages that others hold too are replaced by pages of its own,
 * and *pairs (0 or 1, at most `room`) pairs src[], dst[] say what
 * exl3p_copy_pages has to copy before the keys are written: the page that holds
 * earlier keys too.  A page replaced without a copy has lost what it held of the
 * sequence, keys behind `to` in it among them.  Pages behind that of key to - 1
 * stay the sequence's as they are, those that others hold too still shared: not
 * writable, until a reserve that covers them, or exl3p_book_trim, which gives
 * them back (after a fork, trim to `from` before rows are written again from
 * there on).  All or nothing: too_large where pages, table or room do not
 * suffice. */
exl3_verdict exl3p_book_reserve(exl3p_book *b, int32_t seq, int32_t from, int32_t to, int32_t *src,
                                int32_t *dst, int32_t room, int32_t *pairs);
/* Sequence dst, which holds no page, shares src's pages of its first `keys` keys. */
exl3_verdict exl3p_book_fork(exl3p_book *b, int32_t src, int32_t dst, int32_t keys);
/* The pages behind the sequence's first `keys` keys are given back (0: all). */
exl3_verdict exl3p_book_trim(exl3p_book *b, int32_t seq, int32_t keys);
/* The pages in use become the lowest ones: pairs to copy, at most `room` of
 * them (fewer moves than needed are made where room is short). */
exl3_verdict exl3p_book_compact(exl3p_book *b, int32_t *src, int32_t *dst, int32_t room,
                                int32_t *pairs);
/* The table [seqs][max_pages] (-1: no page), valid until the book closes. */
const int32_t *exl3p_book_table(const exl3p_book *b);
int32_t exl3p_book_free_pages(const exl3p_book *b);
int32_t exl3p_book_held(const exl3p_book *b, int32_t seq);  /* pages of a sequence, -1 refused */
int32_t exl3p_book_shared(const exl3p_book *b, int32_t page); /* a page's holders, -1 refused */

#ifdef __cplusplus
}
#endif

#endif /* EXL3_PAGED_H */
