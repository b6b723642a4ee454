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
 *   exl3p_verify      the tokens that sampling accepts or gives, from the
 *                     target's logits and given random numbers    (a step)
 *   exl3p_weigh       the attention weight of every cached key    (a layer)
 *   exl3p_evict       the keys of most weight stay, up to a budget (as needed)
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

/* Sampled verification: target[t] is the token that follows row t on each
 * sequence's walk, -1 for rows that are not on it, so that exl3p_commit with these
 * targets walks the same way.  Row t's logits are the model's after row t; its
 * probabilities p are their softmax at the sequence's temperature.  The walk
 * begins at row 0.  A row's children, in their order, are drafted tokens that
 * were drawn from draft[t], the probabilities q that the draft had after row t:
 * one is accepted with probability min(1, p~ / q~) of its token (u[child] * q~ <
 * p~), and after a refusal p~ is max(p~ - q~, 0), normalized.  q~ is q, or, with
 * `distinct` not 0 (siblings drawn without replacement), q without the refused
 * ones, normalized.  draft NULL: drafted tokens are certain (q~ is 1 at each), as
 * where a draft's most likely ones were taken.  A refusal that would leave nothing of
 * p~ -- the draft's numbers are rounded, and may add up to more than 1 -- is none: its
 * child is accepted, or p~ stays as it was where it had nothing of the child's token, so
 * that a token that may follow is always accepted or left.  Where no child is accepted the
 * token is sampled from what p~ is then: the first of positive probability whose
 * cumulative sum, in 64 bits and in the vocabulary's order, passes u[row 0]
 * times the whole.  So the tokens have the distribution that sampling without
 * drafts has; a step of single rows is the sampler itself.
 *   temperature [seqs], NULL: 1.  0: the largest logit, the first of equals.
 *   u [rows], in [0, 1).  A number that is none (NaN) accepts nothing and samples
 *   the last token of positive probability (a refused child's, where there are no others:
 *   the walk of exl3p_commit then ends in a row of target -1).
 * logits [rows][vocab] and draft (logits_dtype, draft_dtype: EXL3_DT_F32, F16 or
 * BF16; strides in elements, rows apart), -inf: never.  Of the draft, rows without
 * children are not read, nor what a walk does not need.  A token outside the
 * vocabulary is refused as any other.  Where a row's logits have a NaN, no finite
 * one, or +inf (temperature 0 takes it), or the temperature is negative or not
 * finite, the walk ends there with target -1.  parent as in exl3p_tree_plan; at
 * most EXL3P_TREE_MAX rows of a sequence; vocab up to 2^24.  r->len is not read.
 * scratch: exl3p_verify_scratch_bytes(), written and read within the call.  target
 * and the scratch lie over nothing that is read, nor over each other. */
size_t exl3p_verify_scratch_bytes(const exl3p_rows *r, int32_t vocab);
exl3_verdict exl3p_verify(const exl3p_rows *r, const int32_t *parent, const int32_t *ids,
                          int32_t vocab, const void *logits, int32_t logits_dtype,
                          int64_t logits_stride, const void *draft, int32_t draft_dtype,
                          int64_t draft_stride, int32_t distinct, const float *temperature,
                          const double *u, int32_t *target, void *scratch, size_t scratch_bytes,
                          exl3_stream s);

/* score[s][h][x] = had + the sum, over the rows of sequence s that count and the
 * query heads of kv head h, of the softmax weight that each gives key number x:
 * exl3p_attend's weights, of the same q, mask and scale.  had is decay * score[s][h][x]
 * for x < base[s] (base NULL: r->len, the keys cached before the step) and 0 for
 * the others, whose scores begin here.  The last `window` rows of a sequence count,
 * 0: all.  score [seqs][kv_heads][room] of 32-bit floats, one layer's; keys behind
 * the sequence's, and sequences without rows, stay as they are, and so does one
 * whose keys are more than `room`, or do not fit its table.  A sequence with a
 * page number outside the cache among its keys has scores of NaN at every key that
 * a row that counts sees.  decay is finite.  Sums are of 32 bits, in an order that
 * goes by the sizes and lengths alone: results repeat.  q as in exl3p_attend; values
 * are not read.
 * scratch: exl3p_weigh_scratch_bytes(), as in exl3p_attend, but by `room` too: up to
 * 32 pairs of a row and a query head keep a number each for every key that there is
 * room for, where that is up to 2^30 bytes in all; more pairs two numbers each, and
 * for every such key sums, up to 2^28 bytes of them or two a key and kv head.  score
 * and the scratch lie over nothing else that is read, nor over each other. */
size_t exl3p_weigh_scratch_bytes(const exl3p_cache *c, const exl3p_rows *r, int32_t heads,
                                 int32_t window, int32_t room);
exl3_verdict exl3p_weigh(const exl3p_cache *c, int32_t layer, const exl3p_rows *r, int32_t heads,
                         const void *q, int64_t q_stride, const uint64_t *mask, int32_t words,
                         float scale, int32_t window, float decay, const int32_t *base,
                         float *score, int32_t room, void *scratch, size_t scratch_bytes,
                         exl3_stream s);

/* Eviction: a sequence of more keys than its budget, min(keep[s], most) (keep
 * NULL: most), keeps that many in every layer and kv head: its first `first` keys,
 * its last `last` ones (as far as the budget goes, the first before the last), and
 * the others of the highest score, of equals the earlier; a NaN is below all
 * numbers.  The kept keys and values move together, in their order, to key numbers
 * 0, 1, ..., in the sequence's own pages.  len [seqs]: keys cached; new_len the
 * same after it.  score [layers][seqs][kv_heads][room]; kept [layers][seqs]
 * [kv_heads][most]: the numbers that the kept keys had, -1 behind them; new_score,
 * laid out as score, gets the kept keys' scores (behind them it stays as it is).
 * new_score may be score itself.  A sequence within its budget, with keep[s]
 * below 0, more keys than `room` or its table, or a page number outside the cache
 * among them, stays as it is: kept is -1 throughout, new_len its len.
 * A sequence that loses keys has its key numbers below new_len written: their pages
 * are its alone (exl3p_book_shared); those behind them are only read.  No output lies over an input (but
 * new_score), another output or the cache. */
exl3_verdict exl3p_evict(const exl3p_cache *c, int32_t seqs, const int32_t *len,
                         const float *score, int32_t room, const int32_t *keep, int32_t most,
                         int32_t first, int32_t last, int32_t *kept, float *new_score,
                         int32_t *new_len, exl3_stream s);

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
